"""The operators of a paged KV cache held in 8 bits, as they are measured: the cache
writes of a decode step and of prompts (rotary embedding, quantisation, append, fork
copies), decode attention and causal prefill attention over such a cache.

The cache holds e4m3 codes ``[pages, 2, page, kv heads, head_dim]`` and, for each
block (the tokens of one page, K or V, one head), a power-of-two scale as an e8m0
byte ``[pages, 2, kv heads]``: a code c stands for c * 2**(byte - 127).  A block's
scale is the least power of two with ``amax <= 448 * scale``.

``own`` false: plain torch operations in 32 bits.  ``own`` true: the calls a decoding
program makes of ``beam_engine_amd``.
"""

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
# the largest e4m3 value times a power of two that the type holds: stored values saturate there
LARGEST = {torch.float16: 61440.0, torch.bfloat16: 1.875 * 2.0 ** 127}
LEAST_EXPONENT = -100
WORKSPACE = 256 << 20       # the engine's attention workspace
POSITIONS = 8192            # rows of the rotary tables


def _decode(name, requests, beams, prefix, suffix, ragged, strategy, hq, hkv, d, page, dtype, layers):
    return dict(name=name, kind="decode", requests=requests, beams=beams, prefix=prefix, suffix=suffix, ragged=ragged,
                strategy=strategy, hq=hq, hkv=hkv, d=d, page=page, dtype=dtype, layers=layers)


def _prefill(name, requests, longest, cached, ragged, hq, hkv, d, page, dtype, layers):
    return dict(name=name, kind="prefill", requests=requests, longest=longest, cached=cached, ragged=ragged, hq=hq,
                hkv=hkv, d=d, page=page, dtype=dtype, layers=layers)


def listed():
    return [
        # one request, four beams, a small model's head_dim: the smallest call, bound by launches and latency
        _decode("decode-small", 1, 4, 512, 32, False, "cascade", 8, 8, 64, 16, "bfloat16", 1),
        # an interactive prompt on PageTable's default page size and type, eight beams some tokens into the answer
        _decode("decode-page8", 1, 8, 350, 24, True, "cascade", 32, 8, 128, 8, "float16", 8),
        # the serving step: 8 requests x 16 beams, short private tails (eight of the model's layers)
        _decode("decode-step", 8, 16, 1136, 24, True, "cascade", 32, 8, 128, 16, "bfloat16", 8),
        # the same batch on a 4k prompt with longer answers: the HBM-bound shape
        _decode("decode-prefix4k", 8, 16, 4096, 128, False, "cascade", 32, 8, 128, 16, "bfloat16", 4),
        # sequences that share nothing, of all lengths: every one reads its own pages
        _decode("decode-flat", 16, 1, 64, 6000, True, "flat", 32, 8, 128, 16, "bfloat16", 2),
        # long context, wide beams, a large model's layer: the largest decode call
        _decode("decode-long", 2, 64, 32768, 512, True, "cascade", 64, 8, 128, 16, "bfloat16", 1),
        # the batch's prompts, fresh, one layer after another
        _prefill("prefill-prompts", 8, 1024, 0, False, 32, 8, 128, 16, "bfloat16", 2),
        # prompts of different lengths that continue a cached conversation, default page size and type
        _prefill("prefill-page8", 3, 1500, 400, True, 32, 8, 128, 8, "float16", 2),
        # a short question after a long cached one, a small model's heads
        _prefill("prefill-short", 1, 40, 3000, False, 16, 4, 64, 16, "bfloat16", 4),
        # the cache writes of a serving step: forked pages copied on every layer, then rotation and append per layer
        dict(name="append-step", kind="append", requests=8, beams=16, forks=40, hq=32, hkv=8, d=128, page=16,
             dtype="bfloat16", layers=8),
        # the prompts of a batch written to their pages
        dict(name="append-prompts", kind="prompts", requests=8, longest=1024, cached=0, ragged=False, hq=32, hkv=8, d=128,
             page=16, dtype="bfloat16", layers=2),
        # prompts that go on in the middle of a page, default page size and type, a small model's heads
        dict(name="append-page8", kind="prompts", requests=5, longest=700, cached=300, ragged=True, hq=16, hkv=4, d=64, page=8,
             dtype="float16", layers=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["decode", "prefill", "append", "prompts"], [5, 3, 2, 2])[0]
    hq, hkv = rng.choice([(32, 8), (32, 8), (64, 8), (8, 8), (16, 4), (12, 2)])
    heads = dict(hq=hq, hkv=hkv, d=rng.choice([128, 128, 128, 64, 256]), page=rng.choice([16, 16, 16, 8, 8, 4, 32, 5]),
                 dtype=rng.choice(["bfloat16", "bfloat16", "float16"]))
    if kind == "decode":
        requests, beams, suffix = _log(rng, 1, 12), _log(rng, 1, 40), _log(rng, 1, 400)
        prefix = max(heads["page"], min(20000, _log(rng, 2000, 100000) // requests))
        tokens = requests * (prefix + beams * suffix)
        flat = requests * beams * (prefix + suffix) < 100000 and rng.random() < 0.3
        if flat:
            tokens = requests * beams * (prefix + suffix)
        while prefix > 64 and 4.0 * heads["d"] * hq * requests * beams * (prefix + suffix) > 1.2e11:
            prefix = prefix * 4 // 5 + rng.randrange(3)
        most = min(100000 // tokens, int(1.2e11 / (4.0 * heads["d"] * hq * requests * beams * (prefix + suffix))))
        return dict(kind=kind, requests=requests, beams=beams, prefix=prefix, suffix=suffix, ragged=rng.random() < 0.8,
                    strategy="flat" if flat else "cascade", **heads, layers=max(1, min(rng.choice([1, 2, 4]), most)))
    if kind == "append":
        requests, beams = _log(rng, 1, 12), _log(rng, 1, 32)
        return dict(kind=kind, requests=requests, beams=beams, forks=rng.randint(0, requests * beams // 2), **heads,
                    layers=rng.choice([1, 2, 4, 8]))
    requests, longest = _log(rng, 1, 10), _log(rng, 1, 2500)
    cached = rng.choice([0, 0, _log(rng, 10, 1500)])
    while longest > 24 and 4.0 * heads["d"] * hq * requests * longest * (longest / 2 + cached) > 1.2e11:
        longest = longest * 4 // 5 + rng.randrange(3)
    return dict(kind=kind, requests=requests, longest=longest, cached=cached, ragged=rng.random() < 0.7, **heads, layers=1)


# ------------------------------------------------------------------ shapes of a case
def _fixed(case, salt):
    """Lengths and pages belong to the case, not to the seed of its values."""
    return random.Random(salt + "/".join(f"{k}={case[k]}" for k in sorted(case) if k != "name"))


def _suffixes(case):
    r, n = _fixed(case, "suffix"), case["requests"] * case["beams"]
    return [r.randint(1, case["suffix"]) if case["ragged"] else case["suffix"] for _ in range(n)]


def _prompts(case):
    """(new tokens, cached tokens) of each request."""
    r, out = _fixed(case, "prompt"), []
    for _ in range(case["requests"]):
        n = r.randint(max(1, case["longest"] // 4), case["longest"]) if case["ragged"] else case["longest"]
        c = r.randint(0, case["cached"]) if case["ragged"] else case["cached"]
        out.append((n, c))
    return out


class _Pages:
    """Pages in the shuffled order a pool in use hands them out."""

    def __init__(self, case, total):
        self.order = list(range(total))
        _fixed(case, "pages").shuffle(self.order)

    def take(self, tokens, page):
        n = -(-tokens // page)
        got, self.order = self.order[:n], self.order[n:]
        return got, tokens - (n - 1) * page


def _decode_layout(case):
    """Per request (prefix pages, last), per beam (suffix pages, last); pages in the pool.  Beams share the
    prompt's whole pages (a partial page is copied to each beam at the fork)."""
    page, suf = case["page"], _suffixes(case)
    whole = max(1, case["prefix"] // page) * page
    total = case["requests"] * (whole // page) + sum(-(-s // page) for s in suf)
    pool = _Pages(case, total)
    pre, tails = [], []
    for r in range(case["requests"]):
        pre.append(pool.take(whole, page))
        tails.append([pool.take(s, page) for s in suf[r * case["beams"]:(r + 1) * case["beams"]]])
    return pre, tails, total


def _prompt_layout(case):
    """(new, cached, pages, last) of each request; pages in the pool."""
    page, lens = case["page"], _prompts(case)
    total = sum(-(-(n + c) // page) for n, c in lens)
    pool = _Pages(case, total)
    return [(n, c, *pool.take(n + c, page)) for n, c in lens], total


def _append_layout(case):
    """Every beam's page and its next slot; the fork copies [source, new page, tokens] that come first.  A forked
    beam writes behind the tokens copied for it."""
    r, n = _fixed(case, "append"), case["requests"] * case["beams"]
    order = list(range(n + case["forks"]))
    r.shuffle(order)
    pages, slots = order[:n], [r.randrange(case["page"]) for _ in range(n)]
    copies, own_page, own_slot = [], list(pages), list(slots)
    for new, beam in zip(order[n:], r.sample(range(n), case["forks"])):
        source = r.randrange(n)
        tokens = r.randint(0, own_slot[source])
        copies.append([own_page[source], new, tokens])
        pages[beam], slots[beam] = new, tokens
    return pages, slots, copies, n + case["forks"]


# ------------------------------------------------------------------ the format
def _exponent(amax):
    """The least E >= LEAST_EXPONENT with amax <= 448 * 2**E, for float32 amax >= 0: 448 is 1.75 * 2**8."""
    return (((amax.view(torch.int32) + 0x1FFFFF) >> 23) - 127 - 8).clamp(min=LEAST_EXPONENT)


def _power(e):
    """2.0**e of int32 exponents in [-126, 127]."""
    return ((e + 127) << 23).view(torch.float32)


def _quantise(x):
    """Codes and e8m0 scale bytes of float32 blocks x [pages, 2, page, heads, d]."""
    e = _exponent(x.abs().amax(dim=(2, 4)))
    codes = (x * _power(-e)[:, :, None, :, None]).to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8)


def _values(codes, scale):
    """float32 values of codes [..., 2, page, heads, d] under scale bytes [..., 2, heads]."""
    return codes.float() * _power(scale.int() - 127)[..., None, :, None]


# ------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _heads_like(shape, g, channels):
    """Values as projections give them: normal, some channels several times wider than the others."""
    return torch.randn(shape, generator=g, device="cuda") * channels


def _channels(case, g):
    """Gains [2, kv heads, d] of the K and V channels: a few K channels of each head stand out."""
    c = torch.exp(0.3 * torch.randn((2, case["hkv"], case["d"]), generator=g, device="cuda"))
    c[0] *= 1.0 + 3.0 * (torch.rand((case["hkv"], case["d"]), generator=g, device="cuda") < 0.04)
    return c


def _attention_inputs(case, seed, queries, pages):
    """q, codes and scale bytes of every layer; scores of about unit variance."""
    g, dt = _generator(seed), DTYPES[case["dtype"]]
    q, kv, scale = [], [], []
    for _ in range(case["layers"]):
        c = _channels(case, g)
        wide = c[0].square().mean(-1).sqrt().repeat_interleave(case["hq"] // case["hkv"], 0)
        q.append((torch.randn((queries, case["hq"], case["d"]), generator=g, device="cuda") / wide[None, :, None]).to(dt))
        codes, s = _quantise(_heads_like((pages, 2, case["page"], case["hkv"], case["d"]), g, c[None, :, None]))
        kv.append(codes)
        scale.append(s)
    return q, kv, scale


def _write_inputs(case, seed, n, pages):
    """The projections of n tokens and a pool that holds earlier tokens, for every layer; rotary tables."""
    g, dt = _generator(seed), DTYPES[case["dtype"]]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    qkv, codes, scale = [], [], []
    for _ in range(case["layers"]):
        c = _channels(case, g)
        wide = torch.cat([torch.ones((hq, d), device="cuda"), c[0], c[1]]).reshape(-1)
        qkv.append(_heads_like((n, (hq + 2 * hkv) * d), g, wide).to(dt))
        a, b = _quantise(_heads_like((pages, 2, case["page"], hkv, d), g, c[None, :, None]))
        codes.append(a)
        scale.append(b)
    freq = torch.outer(torch.arange(POSITIONS, dtype=torch.float64, device="cuda"),
                       500000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d))
    emb = torch.cat([freq, freq], dim=-1)
    return qkv, torch.stack(codes), torch.stack(scale), emb.cos().to(dt), emb.sin().to(dt)


def _on_gpu(x, dtype=torch.int64):
    return torch.tensor(x, dtype=dtype, device="cuda")


# ------------------------------------------------------------------ prepare
def prepare(case, seed):
    return {"decode": _prepare_decode, "prefill": _prepare_prefill, "append": _prepare_append,
            "prompts": _prepare_prompts}[case["kind"]](case, seed)


def _padded(groups, page):
    """Token slots [groups, longest] of (pages, last) groups as page * size + slot, and which of them are tokens."""
    lens = [(len(p) - 1) * page + last for p, last in groups]
    at = np.zeros((len(groups), max(lens)), np.int64)
    for i, (p, _) in enumerate(groups):
        at[i, :lens[i]] = (np.repeat(np.asarray(p, np.int64) * page, page) + np.tile(np.arange(page), len(p)))[:lens[i]]
    return _on_gpu(at), torch.arange(at.shape[1], device="cuda")[None, :] < _on_gpu(lens)[:, None]


def _prepare_decode(case, seed):
    pre, tails, total = _decode_layout(case)
    beams, page = case["beams"], case["page"]
    q, kv, scale = _attention_inputs(case, seed, case["requests"] * beams, total)
    tail = [t for ts in tails for t in ts]
    paths = [(pre[i // beams][0] + p, last) for i, (p, last) in enumerate(tail)]
    levels = [(paths, 1)] if case["strategy"] == "flat" else [(pre, beams), (tail, 1)]
    if not own:
        return _plain_decode, q, kv, scale, [(*_padded(groups, page), per) for groups, per in levels]
    from beam_engine_amd import BatchDecodeWithPagedKVCacheWrapper, MultiLevelCascadeAttentionWrapper
    ws = torch.empty(WORKSPACE, dtype=torch.uint8, device="cuda")
    heads, types = (case["hq"], case["hkv"], case["d"], page), dict(q_data_type=DTYPES[case["dtype"]],
                                                                    kv_data_type=torch.float8_e4m3fn)
    lists = [[], [], [], []]
    for groups, per in levels:
        ptr, ind = [0], []
        for p, _ in groups:
            ind += p
            ptr.append(len(ind))
        for of, x in zip(lists, ([i * per for i in range(len(groups) + 1)], ptr, ind, [last for _, last in groups])):
            of.append(x)
    if case["strategy"] == "flat":
        w = BatchDecodeWithPagedKVCacheWrapper(ws)
        w.plan(lists[1][0], lists[2][0], lists[3][0], *heads, **types)
    else:
        w = MultiLevelCascadeAttentionWrapper(2, ws)
        w.plan(*lists, *heads, causal=True, **types)
    return _own_attention, w, q, kv, [s.view(torch.float8_e8m0fnu) for s in scale]


def _prepare_prefill(case, seed):
    lens, total = _prompt_layout(case)
    page, new = case["page"], [n for n, _, _, _ in lens]
    q, kv, scale = _attention_inputs(case, seed, sum(new), total)
    if not own:
        at, is_key = _padded([(p, last) for _, _, p, last in lens], page)
        first = [sum(new[:i]) for i in range(len(new))]
        row = np.zeros((len(new), max(new)), np.int64)          # the query of each request's i-th new token
        for i, n in enumerate(new):
            row[i, :n] = first[i] + np.arange(n)
        is_row = torch.arange(max(new), device="cuda")[None, :] < _on_gpu(new)[:, None]
        sees = _on_gpu([c for _, c, _, _ in lens])[:, None] + torch.arange(max(new), device="cuda")[None, :] + 1
        return _plain_prefill, q, kv, scale, at, is_key, _on_gpu(row), is_row, sees
    from beam_engine_amd import BatchPrefillWithPagedKVCacheWrapper
    qo, ptr, ind = [0], [0], []
    for n, _, p, _ in lens:
        ind += p
        ptr.append(len(ind))
        qo.append(qo[-1] + n)
    w = BatchPrefillWithPagedKVCacheWrapper(torch.empty(WORKSPACE, dtype=torch.uint8, device="cuda"))
    w.plan(qo, ptr, ind, [last for _, _, _, last in lens], case["hq"], case["hkv"], case["d"], page, causal=True,
           q_data_type=DTYPES[case["dtype"]], kv_data_type=torch.float8_e4m3fn)
    return _own_attention, w, q, kv, [s.view(torch.float8_e8m0fnu) for s in scale]


def _table(case, codes, scale):
    from beam_engine_amd import PageTable
    table = PageTable(case["layers"], page_size=case["page"], max_num_pages=codes.shape[1], head_num=case["hkv"],
                      head_dim=case["d"], store_dtype=torch.float8_e4m3fn, compute_dtype=DTYPES[case["dtype"]])
    table.kv_pool.view(torch.uint8).copy_(codes.view(torch.uint8))
    table.kv_scale.view(torch.uint8).copy_(scale)
    return table


def _prepare_append(case, seed):
    pages, slots, copies, total = _append_layout(case)
    qkv, codes, scale, cos, sin = _write_inputs(case, seed, len(pages), total)
    r = _fixed(case, "positions")
    positions = _on_gpu([r.randrange(POSITIONS) for _ in pages])
    if not own:
        src, dst, tokens = _on_gpu(copies).reshape(-1, 3).unbind(1)
        return (_plain_append, codes, scale, (src, dst, tokens), qkv, case["hq"], positions, cos, sin, _on_gpu(pages),
                _on_gpu(slots))
    return (_own_append, _table(case, codes, scale), np.array(copies, np.int32).reshape(-1, 3), qkv, case["hq"], positions,
            cos, sin, _on_gpu(pages, torch.int32), _on_gpu(slots, torch.int32))


def _prepare_prompts(case, seed):
    lens, total = _prompt_layout(case)
    page = case["page"]
    pages = [p[t // page] for n, c, p, _ in lens for t in range(c, c + n)]
    where = [t for n, c, _, _ in lens for t in range(c, c + n)]
    qkv, codes, scale, cos, sin = _write_inputs(case, seed, len(pages), total)
    slots = [t % page for t in where]
    if not own:
        return (_plain_append, codes, scale, None, qkv, case["hq"], _on_gpu(where), cos, sin, _on_gpu(pages),
                _on_gpu(slots))
    return (_own_append, _table(case, codes, scale), None, qkv, case["hq"], _on_gpu(where), cos, sin,
            _on_gpu(pages, torch.int32), _on_gpu(slots, torch.int32))


# ------------------------------------------------------------------ run
def run(state):
    return state[0](*state[1:])


def _own_attention(wrapper, q, kv, scale):
    return [wrapper.run(a, b, kv_scale=s) for a, b, s in zip(q, kv, scale)]


def _own_append(table, copies, qkv, hq, positions, cos, sin, pages, slots):
    if copies is not None:
        table.copy_pages(copies)
    q = [table.write_rope_qkv(layer, x, hq, positions, cos, sin, pages, slots) for layer, x in enumerate(qkv)]
    return q, table.dequantized()


def _level(q, kv, scale, at, is_key, per, sm_scale):
    """Scores [groups, kv heads, per * g, longest] of q [groups * per, heads, d], masked, and the values."""
    page, hkv, d = kv.shape[2:]
    x = _values(kv, scale)
    k, v = (x[:, i].reshape(-1, hkv, d)[at].transpose(1, 2) for i in (0, 1))      # [groups, kv heads, longest, d]
    rows = q.float().reshape(at.shape[0], per, hkv, -1, d).permute(0, 2, 1, 3, 4).reshape(at.shape[0], hkv, -1, d)
    s = torch.matmul(rows, k.transpose(2, 3)) * sm_scale
    return s.masked_fill_(~is_key[:, None, None, :], -math.inf), v


def _plain_decode(q, kv, scale, levels):
    out = []
    for a, c, e in zip(q, kv, scale):
        n, hq, d = a.shape
        hkv = c.shape[3]
        parts = []
        for at, is_key, per in levels:
            s, v = _level(a, c, e, at, is_key, per, d ** -0.5)
            m = s.amax(-1, keepdim=True)
            p = s.sub_(m).exp_()
            parts.append((m, p.sum(-1, keepdim=True), torch.matmul(p, v), at.shape[0], per))
        rows = []
        for m, z, o, groups, per in parts:       # back to one row for each query and head
            rows.append([t.reshape(groups, hkv, per, hq // hkv, -1).transpose(1, 2).reshape(n, hq, -1) for t in (m, z, o)])
        top = torch.stack([m for m, _, _ in rows]).amax(0)
        z = sum(x * torch.exp(m - top) for m, x, _ in rows)
        o = sum(x * torch.exp(m - top) for m, _, x in rows)
        out.append((o / z).to(a.dtype))
    return out


def _plain_prefill(q, kv, scale, at, is_key, row, is_row, sees):
    out = []
    for a, c, e in zip(q, kv, scale):
        n, hq, d = a.shape
        r, t = row.shape
        hkv = c.shape[3]
        s, v = _level(a[row].reshape(r * t, hq, d), c, e, at, is_key, t, d ** -0.5)
        s = s.reshape(r, hkv, t, hq // hkv, -1)
        s.masked_fill_((torch.arange(s.shape[-1], device=s.device) >= sees[..., None])[:, None, :, None, :], -math.inf)
        p = s.sub_(s.amax(-1, keepdim=True)).exp_()
        p /= p.sum(-1, keepdim=True)
        o = torch.matmul(p.reshape(r, hkv, -1, p.shape[-1]), v).reshape(r, hkv, t, hq // hkv, d)
        out.append(o.transpose(1, 2).reshape(r, t, hq, d)[is_row].to(a.dtype))
    return out


def _plain_append(codes, scale, copies, qkv, hq, positions, cos, sin, pages, slots):
    layers, total, _, page, hkv, d = codes.shape
    slot_of = torch.arange(page, device=codes.device)
    if copies is not None:
        src, dst, tokens = copies
        head = (slot_of[None, :] < tokens[:, None])[None, :, None, :, None, None]
        raw = codes.view(torch.uint8)
        raw[:, dst] = torch.where(head, raw[:, src], raw[:, dst])
        some = (tokens > 0)[None, :, None, None]
        scale[:, dst] = torch.where(some, scale[:, src], scale[:, dst])
    c, s = cos[positions].float()[:, None], sin[positions].float()[:, None]
    first = torch.full((total,), page, device=codes.device).scatter_reduce(0, pages, slots, "amin")   # page: not written
    out = []
    for x, code, e in zip(qkv, codes, scale):
        largest = LARGEST[x.dtype]
        x = x.float().reshape(x.shape[0], hq + 2 * hkv, d)
        r = x[:, :hq + hkv]
        r = r * c + torch.cat([-r[..., d // 2:], r[..., :d // 2]], dim=-1) * s
        out.append(r[:, :hq].to(qkv[0].dtype))
        new = torch.stack([r[:, hq:], x[:, hq + hkv:]], dim=1).clamp_(-largest, largest)          # [n, 2, hkv, d]
        amax = torch.zeros((total, 2, hkv), device=x.device)
        amax.scatter_reduce_(0, pages[:, None, None].expand(-1, 2, hkv), new.abs().amax(-1), "amax")
        old = e.int() - 127
        need = _exponent(amax)
        starts, grows = (first == 0)[:, None, None], ((first > 0) & (first < page))[:, None, None]
        now = torch.where(starts, need, torch.where(grows, torch.maximum(old, need), old))
        kept = (slot_of[None, :] < first[:, None]) & (first < page)[:, None]
        again = (code.float() * _power((old - now).clamp(-126, 0))[:, :, None, :, None]).to(torch.float8_e4m3fn)
        raw = code.view(torch.uint8)
        raw.copy_(torch.where(kept[:, None, :, None, None], again.view(torch.uint8), raw))
        raw[pages, :, slots] = (new * _power(-now)[pages][..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
        e.copy_((now + 127).to(torch.uint8))
    return out, _values(codes, scale).to(qkv[0].dtype)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    hq, hkv, d, page, layers = (case[k] for k in ("hq", "hkv", "d", "page", "layers"))
    if case["kind"] in ("decode", "prefill"):
        if case["kind"] == "decode":
            suf, n = _suffixes(case), case["requests"] * case["beams"]
            pre = max(1, case["prefix"] // page) * page
            tokens = case["requests"] * pre + sum(suf)
            seen = n * pre + sum(suf)
        else:
            lens = _prompts(case)
            n, tokens = sum(a for a, _ in lens), sum(a + c for a, c in lens)
            seen = sum(a * c + a * (a + 1) // 2 for a, c in lens)
        cache = 2 * tokens * hkv * d + 2 * hkv * (tokens / page)
        return {"bytes": layers * (cache + 4 * n * hq * d), "flops": layers * 4.0 * d * hq * seen}
    if case["kind"] == "append":
        pages, slots, copies, total = _append_layout(case)
        n, copied = len(pages), sum(c[2] for c in copies)
    else:
        lens, total = _prompt_layout(case)
        n, copied = sum(x[0] for x in lens), 0
    rows = 2 * n * (hq + 2 * hkv) * d + 2 * n * hq * d + 2 * n * hkv * d          # read, q and codes written
    values = total * page * hkv * d * 2 * 3                                       # codes read, values written
    return {"bytes": layers * (rows + 2 * 2 * copied * hkv * d + values), "flops": layers * 6.0 * n * (hq + hkv) * d}


# ------------------------------------------------------------------ results in 64 bits
def exact(case, seed):
    return {"decode": _exact_decode, "prefill": _exact_prefill, "append": _exact_append,
            "prompts": _exact_append}[case["kind"]](case, seed)


def _stored(kv, scale, pages, tokens):
    """K and V [tokens, heads, d] in float64 of a token range's pages."""
    at = torch.tensor(pages, device=kv.device)
    x = kv[at].to(torch.float64) * torch.exp2(scale[at].to(torch.float64) - 127.0)[:, :, None, :, None]
    return x[:, 0].reshape(-1, *kv.shape[3:])[:tokens], x[:, 1].reshape(-1, *kv.shape[3:])[:tokens]


def _softmax_rows(q, k, v, sees=None):
    """softmax(q k^T / sqrt(d)) v of q [n, hq, d]; row i sees the first sees[i] keys."""
    n, hq, d = q.shape
    hkv = k.shape[1]
    out = torch.empty((n, hq, d), dtype=torch.float64, device=q.device)
    for h in range(hkv):
        mine = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
        s = q[:, mine].double().reshape(-1, d) @ k[:, h].t().contiguous() / math.sqrt(d)
        if sees is not None:
            hide = torch.arange(k.shape[0], device=q.device)[None, :] >= sees[:, None]
            s = s.masked_fill(hide.repeat_interleave(hq // hkv, 0), -math.inf)
        out[:, mine] = (torch.softmax(s, -1) @ v[:, h].contiguous()).reshape(n, -1, d)
    return out


def _joined(q, parts):
    """One row [hq, d] over the keys of several (k, v) in turn."""
    return _softmax_rows(q, torch.cat([k for k, _ in parts]), torch.cat([v for _, v in parts]))


def _exact_decode(case, seed):
    pre, tails, total = _decode_layout(case)
    beams, page, hq, hkv, d = (case[k] for k in ("beams", "page", "hq", "hkv", "d"))
    if case["requests"] * beams * (case["prefix"] + case["suffix"]) * hq * case["layers"] > 4e9:
        return None
    q, kv, scale = _attention_inputs(case, seed, case["requests"] * beams, total)
    out = []
    for a, c, e in zip(q, kv, scale):
        o = torch.empty(a.shape, dtype=torch.float64, device=a.device)
        for r, (pp, plast) in enumerate(pre):
            shared = _stored(c, e, pp, (len(pp) - 1) * page + plast)
            mine = [_stored(c, e, tp, (len(tp) - 1) * page + last) for tp, last in tails[r]]
            rows = a[r * beams:(r + 1) * beams].double()
            for h in range(hkv):
                heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
                x = rows[:, heads].reshape(-1, d)
                s = (x @ shared[0][:, h].t().contiguous() / math.sqrt(d)).reshape(beams, -1, shared[0].shape[0])
                m = s.amax(-1)
                p = torch.exp(s - m[..., None])
                z, w = p.sum(-1), (p.reshape(-1, p.shape[-1]) @ shared[1][:, h].contiguous()).reshape(beams, -1, d)
                for b, (k, v) in enumerate(mine):
                    t = rows[b, heads] @ k[:, h].t().contiguous() / math.sqrt(d)
                    top = torch.maximum(m[b], t.amax(-1))
                    u, f = torch.exp(t - top[:, None]), torch.exp(m[b] - top)
                    o[r * beams + b, heads] = ((w[b] * f[:, None] + u @ v[:, h].contiguous())
                                               / (z[b] * f + u.sum(-1))[:, None])
        out.append(o)
    return out


def _exact_prefill(case, seed):
    lens, total = _prompt_layout(case)
    q, kv, scale = _attention_inputs(case, seed, sum(x[0] for x in lens), total)
    out = []
    for a, c, e in zip(q, kv, scale):
        parts, at = [], 0
        for n, cached, pages, _ in lens:
            k, v = _stored(c, e, pages, n + cached)
            parts.append(_softmax_rows(a[at:at + n], k, v, cached + 1 + torch.arange(n, device=a.device)))
            at += n
        out.append(torch.cat(parts))
    return out


def _nearest_code(x):
    """The e4m3 value nearest to x (ties to the even code) for |x| <= 448, in float64."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3.0)
    return torch.round(x / step) * step


def _exact_append(case, seed):
    if case["kind"] == "append":
        pages, slots, copies, total = _append_layout(case)
        r = _fixed(case, "positions")
        positions = [r.randrange(POSITIONS) for _ in pages]
    else:
        lens, total = _prompt_layout(case)
        positions = [t for n, c, _, _ in lens for t in range(c, c + n)]
        pages = [p[t // case["page"]] for n, c, p, _ in lens for t in range(c, c + n)]
        slots, copies = [t % case["page"] for t in positions], []
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    qkv, codes, scale, cos, sin = _write_inputs(case, seed, len(pages), total)
    positions, largest = torch.tensor(positions, device="cuda"), LARGEST[qkv[0].dtype]
    c, s = cos[positions].double()[:, None], sin[positions].double()[:, None]
    least = {}
    for p, t in zip(pages, slots):
        least[p] = min(t, least.get(p, page))
    at = torch.tensor(list(least), device="cuda")
    low = torch.tensor(list(least.values()), device="cuda")
    where = {p: i for i, p in enumerate(least)}
    group = torch.tensor([where[p] for p in pages], device="cuda")
    slots = torch.tensor(slots, device="cuda")
    out, values = [], []
    for x, code, e in zip(qkv, codes, scale):
        code, exponent = code.double(), e.double() - 127.0
        for src, dst, n in copies:
            code[dst, :, :n] = code[src, :, :n]
            if n:
                exponent[dst] = exponent[src]
        x = x.double().reshape(x.shape[0], hq + 2 * hkv, d)
        rotated = torch.empty_like(x[:, :hq + hkv])
        a, b = x[:, :hq + hkv, :d // 2], x[:, :hq + hkv, d // 2:]
        rotated[..., :d // 2] = a * c[..., :d // 2] - b * s[..., :d // 2]
        rotated[..., d // 2:] = b * c[..., d // 2:] + a * s[..., d // 2:]
        out.append(rotated[:, :hq])
        new = torch.stack([rotated[:, hq:], x[:, hq + hkv:]], dim=1).clamp(-largest, largest)
        amax = torch.zeros((len(least), 2, hkv), dtype=torch.float64, device="cuda")
        amax.scatter_reduce_(0, group[:, None, None].expand(-1, 2, hkv), new.abs().amax(-1), "amax")
        need = torch.ceil(torch.log2(amax / 448.0)).clamp(min=LEAST_EXPONENT)
        old = exponent[at]
        now = torch.where((low == 0)[:, None, None], need, torch.maximum(old, need))
        again = _nearest_code(code[at] * torch.exp2(old - now)[:, :, None, :, None])
        kept = torch.arange(page, device="cuda")[None, :] < low[:, None]
        block = torch.where(kept[:, None, :, None, None], again, code[at])
        block[group, :, slots] = _nearest_code(new * torch.exp2(-now)[group][..., None])
        code[at], exponent[at] = block, now
        values.append(code * torch.exp2(exponent)[:, :, None, :, None])
    return out, torch.stack(values)
