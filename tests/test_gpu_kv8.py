"""The 8-bit paged KV cache on the GPU: writes (bit-exact against the numpy
restatement), fork copies, reading back, decode and prefill attention over it against
64-bit results, and the decoder running on it.

Attention tolerance, element by element: with u half a step of the 16-bit type
(eps / 2), A the reference's sum of weights times |v| and P the rounded weights,
|o - o64| <= u A (the output's rounding, |o| <= A) + u A (each weight's rounding) +
2 S A, S = head_dim 2^-24 sm_scale max sum |q||k| (the fp32 sums of the scores, which
move a weight by at most a factor e^(2S)) + 2^-18 A (fp32 sums, exp2, merge); fp16
weights, values and outputs below 2^-14 keep a step of 2^-24: + 2^-25 times the sum of
|v|, and 2^-25 for the values and for the output.
"""

import math
import random
import sys

import numpy as np
import pytest
import torch

from oracle import kv8

pytestmark = pytest.mark.gpu
F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def say(msg):
    print(f"[case] {msg}", flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module", autouse=True)
def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def table(pages, page, hkv, d, dtype, layers=1, seed=None):
    """A page table; with a seed its pool holds earlier tokens."""
    from beam_engine_amd import PageTable
    t = PageTable(layers, page_size=page, max_num_pages=pages, head_num=hkv, head_dim=d, store_dtype=F8, compute_dtype=dtype)
    if seed is not None:
        g = np.random.default_rng(seed)
        c = g.integers(0, 256, t.kv_pool.shape, dtype=np.uint8)
        c[(c & 127) == 127] = 5
        s = g.integers(110, 130, t.kv_scale.shape, dtype=np.uint8)
        t.kv_pool.view(torch.uint8).copy_(torch.from_numpy(c))
        t.kv_scale.view(torch.uint8).copy_(torch.from_numpy(s))
    return t


def state(t, layer=0):
    return (t.kv_pool.view(torch.uint8)[layer].cpu().numpy().copy(), t.kv_scale.view(torch.uint8)[layer].cpu().numpy().copy())


def same_codes(got, want):
    nan = (want & 127) == 127
    assert np.array_equal((got & 127) == 127, nan)
    bad = np.argwhere((got != want) & ~nan)
    assert bad.size == 0, f"{len(bad)} codes differ, first at {bad[0]}"


# ------------------------------------------------------------------ writes
def orders(kind, n, page, r):
    """(pages in the pool, page and slot of each entry)."""
    if kind == "prompt":                       # one prompt from a page's start
        ids = r.sample(range(n // page + 3), -(-n // page))
        at = [(ids[t // page], t % page) for t in range(n)]
        return n // page + 3, at
    if kind == "ragged":                       # prompts that go on inside a page, back to back
        at, used = [], 0
        while len(at) < n:
            c, m = r.randrange(2 * page), min(r.randint(1, 3 * page), n - len(at))
            at += [(used + t // page, t % page) for t in range(c, c + m)]
            used += -(-(c + m) // page)
        return used, at
    if kind == "step":                         # a decode step: a page and a slot of its own each
        return n + 2, [(p, r.randrange(page)) for p in r.sample(range(n + 2), n)]
    if kind == "token-major":                  # several prompts, token by token
        m = max(1, min(9, n // 3))
        per = -(-(-(-n // m)) // page) + 1
        return m * per, [((i % m) * per + (i // m) // page, (i // m) % page) for i in range(n)]
    if kind == "shuffled":                     # any order, some (page, slot) several times
        few = max(2, n // (2 * page))
        return few + 1, [(r.randrange(few), r.randrange(page)) for _ in range(n)]
    assert kind == "one"                       # every entry the same slot
    return 2, [(1, 0)] * n


@pytest.mark.parametrize("kind", ["prompt", "ragged", "step", "token-major", "shuffled", "one"])
@pytest.mark.parametrize("n,page,hkv,d,dtype", [
    (1, 16, 2, 64, torch.bfloat16), (7, 1, 1, 128, torch.float16), (17, 4, 3, 64, torch.float16), (37, 16, 8, 128, torch.bfloat16),
    (64, 5, 2, 256, torch.bfloat16), (129, 8, 8, 64, torch.float16), (300, 64, 2, 128, torch.float16), (1100, 16, 2, 64, torch.bfloat16),
    (1500, 96, 1, 128, torch.bfloat16)])
def test_append_is_the_definition(kind, n, page, hkv, d, dtype):
    say(f"append {kind} n {n} page {page} heads {hkv} d {d} {dtype}")
    r = random.Random(n * page + d)
    pool, at = orders(kind, n, page, r)
    t = table(pool, page, hkv, d, dtype, layers=2, seed=n)
    before, other = state(t), state(t, 1)
    g = torch.Generator().manual_seed(n)
    x = torch.randn((n, 2, hkv, d), generator=g) * torch.exp2(torch.randint(-9, 9, (n, 2, hkv, 1), generator=g).float())
    x[torch.rand((n, 2, hkv), generator=g) < 0.1] = 0.0
    x = x.to(dtype)
    pages, slots = [p for p, _ in at], [s for _, s in at]
    k, v = x[:, 0].cuda(), x[:, 1].cuda()
    t.write_blocks_vectorized(0, i32(pages), k, v, i32(slots))
    t.check_errors()
    codes, scale = before
    kv8.append(codes, scale, pages, slots, x[:, 0].float().numpy(), x[:, 1].float().numpy(), str(dtype)[6:])
    got = state(t)
    assert np.array_equal(got[1], scale)
    same_codes(got[0], codes)
    assert all(np.array_equal(a, b) for a, b in zip(state(t, 1), other))       # the other layer stays as it was
    t.write_blocks_vectorized(0, i32(pages), k, v, i32(slots))                 # the same again: the same bytes
    again = state(t)
    kv8.append(codes, scale, pages, slots, x[:, 0].float().numpy(), x[:, 1].float().numpy(), str(dtype)[6:])
    assert np.array_equal(again[1], scale)
    same_codes(again[0], codes)


@pytest.mark.parametrize("n,page,hq,hkv,d,dtype", [
    (1, 16, 32, 8, 128, torch.bfloat16), (5, 8, 3, 1, 64, torch.float16), (40, 4, 12, 2, 256, torch.float16),
    (128, 16, 32, 8, 128, torch.bfloat16), (1300, 16, 8, 4, 64, torch.bfloat16), (260, 3, 5, 2, 128, torch.float16)])
@pytest.mark.parametrize("kind", ["prompt", "step", "ragged", "shuffled"])
def test_rope_append_is_the_definition(n, page, hq, hkv, d, dtype, kind):
    say(f"rope append {kind} n {n} page {page} heads {hq}/{hkv} d {d} {dtype}")
    r = random.Random(n + d)
    pool, at = orders(kind, n, page, r)
    t = table(pool, page, hkv, d, dtype, seed=n + 1)
    codes, scale = state(t)
    g = torch.Generator().manual_seed(n)
    wide = (torch.randn((n, (hq + 2 * hkv) * d + 8), generator=g) * 3).to(dtype)
    qkv = wide.cuda()[:, :-8]                                                  # rows with a stride of their own
    pos = torch.randint(0, 700, (n,), generator=g)
    angle = torch.outer(torch.arange(700).double(), 10000.0 ** (-torch.arange(0, d, 2).double() / d))
    cos, sin = (f(torch.cat([angle, angle], -1)).to(dtype) for f in (torch.cos, torch.sin))
    pages, slots = [p for p, _ in at], [s for _, s in at]
    q = t.write_rope_qkv(0, qkv, hq, pos.cuda(), cos.cuda(), sin.cuda(), i32(pages), i32(slots))
    t.check_errors()
    x = wide[:, :-8].float().numpy().reshape(n, hq + 2 * hkv, d)
    turned = kv8.rotate(x[:, :hq + hkv], cos[pos].float().numpy(), sin[pos].float().numpy())
    assert torch.equal(q.cpu(), torch.from_numpy(turned[:, :hq].copy()).to(dtype))
    kv8.append(codes, scale, pages, slots, turned[:, hq:], x[:, hq + hkv:], str(dtype)[6:])
    got = state(t)
    assert np.array_equal(got[1], scale)
    same_codes(got[0], codes)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_keeps_the_ends_of_the_range(dtype):
    """The type's largest and smallest values, infinities and NaN beside others, a
    block of zeros, of NaN alone, and a growth of many binades."""
    say(f"append ends of the range {dtype}")
    t = table(4, 8, 2, 64, dtype)
    f = torch.finfo(dtype)
    rows = torch.zeros((9, 2, 64), dtype=dtype)
    rows[0, 0, :6] = torch.tensor([f.max, -f.max, f.tiny, f.smallest_normal / 8, 1.0, -0.0]).to(dtype)
    rows[1, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 3.0])
    rows[2, 0] = math.nan
    rows[3, 1] = f.tiny * 4
    rows[4] = 2.0 ** -14
    rows[5] = 1.0
    rows[6] = f.max
    rows[7, :, 3] = 448.0
    rows[8, :, 3] = 450.0
    pages, slots = [0, 1, 2, 2, 3, 3, 3, 0, 1], [0, 0, 0, 1, 0, 1, 2, 5, 6]
    codes, scale = state(t)
    for lo, hi in ((0, 5), (5, 6), (6, 9)):
        t.write_blocks_vectorized(0, i32(pages[lo:hi]), rows[lo:hi].cuda(), rows[lo:hi].neg().cuda(), i32(slots[lo:hi]))
        kv8.append(codes, scale, pages[lo:hi], slots[lo:hi], rows[lo:hi].float().numpy(), -rows[lo:hi].float().numpy(),
                   str(dtype)[6:])
        got = state(t)
        assert np.array_equal(got[1], scale)
        same_codes(got[0], codes)
    v = t.dequantized(0)
    assert torch.isfinite(v[3]).all() and not torch.isfinite(v[1]).all()


def test_append_skips_what_is_out_of_range():
    say("append out of range")
    t = table(6, 8, 2, 128, torch.bfloat16, seed=2)
    codes, scale = state(t)
    n, hq = 7, 4
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn((n, (hq + 4) * 128), generator=g).to(torch.bfloat16)
    pages, slots, pos = [0, 6, 1, -1, 2, 3, 0], [0, 0, 8, 0, -1, 1, 1], [0, 1, 2, 3, 4, 50, 49]
    cos, sin = torch.ones((50, 128), dtype=torch.bfloat16), torch.zeros((50, 128), dtype=torch.bfloat16)
    q = torch.full((n, hq, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    t.write_rope_qkv(0, qkv.cuda(), hq, torch.tensor(pos).cuda(), cos.cuda(), sin.cuda(), i32(pages), i32(slots), q_out=q)
    with pytest.raises(ValueError, match="5 KV append"):
        t.check_errors()
    x = qkv.float().numpy().reshape(n, hq + 4, 128)
    good = [0, 6]
    kv8.append(codes, scale, [pages[i] for i in good], [slots[i] for i in good], x[good, hq:hq + 2], x[good, hq + 2:], "bfloat16")
    got = state(t)
    assert np.array_equal(got[1], scale)
    same_codes(got[0], codes)
    assert torch.equal(q[5].cpu(), torch.full((hq, 128), 7.0, dtype=torch.bfloat16))     # no position, no q
    assert torch.equal(q[1].cpu(), qkv[1, :hq * 128].reshape(hq, 128))


@pytest.mark.parametrize("n", [90, 700])
@pytest.mark.parametrize("bad", [-1, -2, 12])
def test_append_skips_whole_runs(n, bad):
    """Workgroups all of whose entries are out of range, with entries of the same page
    number before and behind them: nothing is written for any."""
    say(f"append runs of page {bad}, {n} entries")
    t = table(14, 8, 2, 64, torch.bfloat16, seed=4)
    t.max_num_pages = 12                                    # two pages behind the pool that is named
    codes, scale = state(t)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn((n, 2, 64), generator=g).to(torch.bfloat16) for _ in range(2))
    pages = [1 + i // 8 if i < 32 else 5 + i % 3 if i % 40 == 39 else bad for i in range(n)]
    slots = [i % 8 for i in range(n)]
    t.write_blocks_vectorized(0, i32(pages), k.cuda(), v.cuda(), i32(slots))
    with pytest.raises(ValueError, match=f"{sum(p == bad for p in pages)} KV append"):
        t.check_errors()
    good = [i for i in range(n) if pages[i] != bad]
    kv8.append(codes, scale, [pages[i] for i in good], [slots[i] for i in good], k.float().numpy()[good], v.float().numpy()[good], "bfloat16")
    got = state(t)
    assert np.array_equal(got[1], scale)
    same_codes(got[0], codes)


def test_append_takes_any_layout_and_stream():
    """Strided and unaligned keys, int64 indices, nothing to write, another stream."""
    say("append layouts and streams")
    t = table(40, 16, 2, 64, torch.float16)
    codes, scale = state(t)
    g = torch.Generator().manual_seed(5)
    wide = torch.randn((20, 2, 131), generator=g).to(torch.float16)
    k, v = wide.cuda()[:, :, 1:65], wide.cuda()[:, :, 66:130]
    pages, slots = list(range(10, 30)), [i % 16 for i in range(20)]
    t.write_blocks_vectorized(0, i32([]), k[:0], v[:0], i32([]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        t.write_blocks_vectorized(0, torch.tensor(pages).cuda(), k, v, torch.tensor(slots).cuda())
    torch.cuda.current_stream().wait_stream(side)
    kv8.append(codes, scale, pages, slots, wide[:, :, 1:65].float().numpy(), wide[:, :, 66:130].float().numpy(), "float16")
    got = state(t)
    assert np.array_equal(got[1], scale)
    same_codes(got[0], codes)
    # the reference's prefill write, page by page
    p = t.allocate_block()
    t.write_block(0, p, k[:5], v[:5], 3)
    kv8.append(codes, scale, [p] * 5, range(3, 8), wide[:5, :, 1:65].float().numpy(), wide[:5, :, 66:130].float().numpy(),
               "float16")
    got = state(t)
    assert np.array_equal(got[1], scale)
    same_codes(got[0], codes)


def test_copies_take_codes_and_scales():
    say("fork copies")
    for page, hkv, d in ((16, 8, 128), (5, 3, 64), (1, 1, 256)):
        t = table(30, page, hkv, d, torch.bfloat16, layers=3, seed=9)
        r = random.Random(page)
        copies = np.array([[r.randrange(15), 15 + i, r.randint(0, page)] for i in range(12)] + [[3, 30, 1]], np.int32)
        want = [state(t, l) for l in range(3)]
        for s, e, n in copies[:-1]:
            for codes, scale in want:
                codes[e, :, :n] = codes[s, :, :n]
                if n:
                    scale[e] = scale[s]
        t.copy_pages(copies)
        with pytest.raises(ValueError, match="1 KV append"):
            t.check_errors()
        for l in range(3):
            assert all(np.array_equal(a, b) for a, b in zip(state(t, l), want[l]))
        # the staged list, as a step graph runs it
        t.enable_staged_copies(8)
        t.stage_copies(np.array([[20, 1, page], [21, 2, 1]], np.int32))
        t.run_staged_copies()
        for codes, scale in want:
            for s, e, n in ((20, 1, page), (21, 2, 1)):
                codes[e, :, :n] = codes[s, :, :n]
                scale[e] = scale[s]
        for l in range(3):
            assert all(np.array_equal(a, b) for a, b in zip(state(t, l), want[l]))


def test_copies_in_a_row():
    """Many lists of copies in a row, each reading what the last one wrote, from two streams
    that wait for each other: none sees another's list."""
    say("copies in a row")
    t = table(40, 4, 2, 64, torch.bfloat16, seed=8)
    want = state(t)
    side, main = torch.cuda.Stream(), torch.cuda.current_stream()
    for i in range(14):
        a = [(7 * i + 3 * j) % 20 for j in range(1 + 5 * i % 11)]
        todo = np.array([(s, 20 + (s + i) % 20 if i % 2 else (s + 1) % 20, 1 + (s + i) % 4) for s in dict.fromkeys(a)], np.int32)
        todo = todo[[k for k in range(len(todo)) if todo[k, 1] not in todo[:, 0] and todo[k, 1] not in todo[:k, 1]]]
        for s, d, n in todo:
            want[0][d, :, :n] = want[0][s, :, :n]
            want[1][d] = want[1][s]
        with torch.cuda.stream(side if i % 3 == 0 else main):
            t.copy_pages(todo)
        (main if i % 3 == 0 else side).wait_stream(side if i % 3 == 0 else main)
    torch.cuda.synchronize()
    got = state(t)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_values_are_exact(dtype):
    """The values, in the type (fp16 rounds what lies below its subnormal step)."""
    say(f"values {dtype}")
    t = table(37, 5, 3, 64, dtype, layers=2, seed=4)
    for layer in range(2):
        want = torch.from_numpy(kv8.values(*state(t, layer))).to(dtype)
        got = t.dequantized(layer)
        assert got.dtype == dtype and torch.equal(got.cpu(), want)
        assert torch.equal(t.dequantized()[layer], got)
        assert torch.equal(t.get_k_buffer(layer).cpu(), want[:, 0].reshape(37 * 5, 3, 64))
        assert torch.equal(t.get_v_buffer(layer).cpu(), want[:, 1].reshape(37 * 5, 3, 64))


# ------------------------------------------------------------------ attention
def cache(pages, page, hkv, d, seed, spread=0):
    """Codes and scales of random tokens (scales within 2^spread of each other)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((pages, 2, page, hkv, d), generator=g, device="cuda")
    codes = (x * 100).to(F8)
    s = torch.randint(119 - spread, 121, (pages, 2, hkv), generator=g, device="cuda").to(torch.uint8)
    return codes, s.view(E8)


def attend(q, codes, scale, slots, sees=None, sm_scale=None):
    """(o, lse, tolerance per element) in float64 of q [n, hq, d] over the token slots
    [t] of a group; row i sees its first sees[i]."""
    n, hq, d = q.shape
    hkv, page = codes.shape[3], codes.shape[2]
    sm = d ** -0.5 if sm_scale is None else sm_scale
    at = torch.tensor(slots, dtype=torch.long, device=q.device)
    val = codes[at // page].double() * torch.exp2(scale.view(torch.uint8)[at // page].double() - 127.0)[:, :, None, :, None]
    kv = torch.gather(val, 2, (at % page)[:, None, None, None, None].expand(-1, 2, 1, hkv, d))[:, :, 0]
    o = torch.zeros((n, hq, d), dtype=torch.float64, device=q.device)
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o)
    if not len(slots):
        return o, lse, tol
    u = torch.finfo(q.dtype).eps / 2
    for h in range(hq):
        k, v = kv[:, 0, h // (hq // hkv)].contiguous(), kv[:, 1, h // (hq // hkv)].contiguous()
        x = q[:, h].double()
        s = (x @ k.t().contiguous()) * sm
        if sees is not None:
            s = s.masked_fill(torch.arange(len(slots), device=q.device)[None] >= sees[:, None], -math.inf)
        m = s.amax(-1, keepdim=True)
        m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
        p = torch.exp(s - m)
        z = p.sum(-1, keepdim=True)
        w = torch.where(z == 0, torch.zeros_like(p), p / z)
        # (a NaN value reaches the rows that see it, by any weight)
        bad = torch.isnan(v)
        v = torch.where(bad, torch.zeros_like(v), v)
        o[:, h] = torch.where((w > 0).double() @ bad.double() > 0, math.nan, w @ v)
        lse[:, h] = torch.where(z == 0, torch.full_like(z, -math.inf), m + torch.log(z))[:, 0]
        A = w @ v.abs()
        S = d * 2.0 ** -24 * abs(sm) * float((x.abs() @ torch.nan_to_num(k).abs().t().contiguous()).max())
        tol[:, h] = A * (2 * u + 2 * S + 2.0 ** -18)
        if q.dtype == torch.float16:
                tol[:, h] += 2.0 ** -25 * v.abs().sum(0) + 2.0 ** -24
    return o, lse, tol


def close(got, o, tol, what):
    d = (got.double() - o).abs()
    bad = ~(d <= tol) & ~(torch.isnan(o) & torch.isnan(got))
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst {float((d - tol).max()):.3g} beyond, at {bad.nonzero()[0].tolist()}"


def lse_close(lse, want, d, what):
    """fp32 scores and sums: 2^-12 is far above S + 2^-18 at these sizes.  (A row of NaN
    scores has lse NaN or -inf, as everywhere in this package.)"""
    fine = torch.isfinite(want)
    assert torch.equal(torch.isinf(lse) | torch.isnan(lse), ~fine), what
    if fine.any():
        assert float((lse.double() - want)[fine].abs().max()) < 2.0 ** -12, what


def lists(lens, page, r, spare=3):
    """Page lists (shuffled ids), last lengths and token slots of groups of these lengths."""
    total = sum(-(-n // page) for n in lens) + spare
    ids = list(range(total))
    r.shuffle(ids)
    ptr, ind, last, slots = [0], [], [], []
    for n in lens:
        m = -(-n // page)
        mine, ids = ids[:m], ids[m:]
        ind += mine
        ptr.append(len(ind))
        last.append(n - (m - 1) * page if m else 0)
        slots.append([mine[t // page] * page + t % page for t in range(n)])
    return total, ptr, ind, last, slots


def workspace(mb=64):
    return torch.empty(mb << 20, dtype=torch.uint8, device="cuda")


HEADS = [(32, 8, 128, torch.bfloat16), (8, 8, 64, torch.float16), (12, 2, 256, torch.bfloat16), (64, 1, 128, torch.float16),
         (20, 4, 64, torch.bfloat16), (16, 1, 256, torch.float16)]


@pytest.mark.parametrize("page", [1, 3, 4, 8, 16, 48])
@pytest.mark.parametrize("hq,hkv,d,dtype", HEADS)
def test_flat_decode(hq, hkv, d, dtype, page):
    from beam_engine_amd import BatchDecodeWithPagedKVCacheWrapper
    say(f"flat decode {hq}/{hkv} d {d} {dtype} page {page}")
    lens = [1, 2, 0, 15, 16, 17, 63, 64, 65, 127, 129, 300, 1025]
    r = random.Random(page)
    total, ptr, ind, last, slots = lists(lens, page, r)
    codes, scale = cache(total, page, hkv, d, page, spread=3)
    g = torch.Generator(device="cuda").manual_seed(d)
    q = torch.randn((len(lens), hq, d), generator=g, device="cuda").to(dtype)
    for cus in (None, 3):
        w = BatchDecodeWithPagedKVCacheWrapper(workspace())
        w._num_cus = cus
        w.plan(ptr, ind, last, hq, hkv, d, page, q_data_type=dtype, kv_data_type=F8)
        assert w.stats.kernel == "kv8"
        o, lse = w.run(q, codes, kv_scale=scale, return_lse=True)
        for i in range(len(lens)):
            want, wl, tol = attend(q[i:i + 1], codes, scale, slots[i])
            close(o[i:i + 1], want, tol, f"len {lens[i]} cus {cus}")
            lse_close(lse[i:i + 1], wl, d, f"len {lens[i]}")


@pytest.mark.parametrize("page,beams,prefix,hq,hkv,d,dtype", [
    (16, 16, 200, 32, 8, 128, torch.bfloat16), (8, 40, 333, 16, 4, 64, torch.float16), (16, 64, 700, 64, 8, 128, torch.bfloat16),
    (5, 7, 95, 12, 2, 256, torch.float16), (16, 3, 1, 8, 8, 128, torch.bfloat16), (32, 130, 96, 8, 8, 128, torch.float16)])
def test_cascade(page, beams, prefix, hq, hkv, d, dtype):
    """Two requests whose beams share a prefix, some beams without a tail."""
    from beam_engine_amd import MultiLevelCascadeAttentionWrapper
    say(f"cascade {beams} beams prefix {prefix} {hq}/{hkv} d {d} {dtype} page {page}")
    r = random.Random(beams)
    tails = [r.randrange(0, 90) for _ in range(2 * beams)]
    total, ptr, ind, last, slots = lists([prefix, prefix + 13] + tails, page, r)
    codes, scale = cache(total, page, hkv, d, beams, spread=4)
    g = torch.Generator(device="cuda").manual_seed(d)
    q = torch.randn((2 * beams, hq, d), generator=g, device="cuda").to(dtype)
    cut = ptr[2]
    w = MultiLevelCascadeAttentionWrapper(2, workspace())
    w.plan([[0, beams, 2 * beams], list(range(2 * beams + 1))], [ptr[:3], [p - cut for p in ptr[2:]]], [ind[:cut], ind[cut:]],
           [last[:2], last[2:]], hq, hkv, d, page, causal=True, q_data_type=dtype, kv_data_type=F8)
    o, lse = w.run(q, codes, kv_scale=scale, return_lse=True)
    for i in r.sample(range(2 * beams), min(2 * beams, 24)):
        want, wl, tol = attend(q[i:i + 1], codes, scale, slots[i // beams] + slots[2 + i])
        close(o[i:i + 1], want, tol, f"beam {i}")
        lse_close(lse[i:i + 1], wl, d, f"beam {i}")


@pytest.mark.parametrize("page", [3, 8, 16])
@pytest.mark.parametrize("hq,hkv,d,dtype", HEADS)
@pytest.mark.parametrize("lens", [[(1, 0)], [(7, 9), (64, 0), (130, 31), (1, 300)], [(300, 0), (65, 500)], [(40, -13), (3, 0)]])
def test_causal_prefill(hq, hkv, d, dtype, page, lens):
    """(new tokens, cached ones); a negative number: fewer keys than queries, so the
    first rows see nothing."""
    from beam_engine_amd import BatchPrefillWithPagedKVCacheWrapper
    say(f"prefill {lens} {hq}/{hkv} d {d} {dtype} page {page}")
    r = random.Random(page + d)
    total, ptr, ind, last, slots = lists([n + c for n, c in lens], page, r)
    codes, scale = cache(total, page, hkv, d, page, spread=3)
    n = sum(a for a, _ in lens)
    g = torch.Generator(device="cuda").manual_seed(d)
    q = torch.randn((n, hq, d), generator=g, device="cuda").to(dtype)
    qo = [0]
    for a, _ in lens:
        qo.append(qo[-1] + a)
    for causal in (True, False):
        w = BatchPrefillWithPagedKVCacheWrapper(workspace(256))
        w.plan(qo, ptr, ind, last, hq, hkv, d, page, causal=causal, q_data_type=dtype, kv_data_type=F8)
        o, lse = w.run(q, codes, kv_scale=scale, return_lse=True)
        for i, (a, c) in enumerate(lens):
            sees = torch.arange(a, device="cuda") + c + 1 if causal else None
            want, wl, tol = attend(q[qo[i]:qo[i + 1]], codes, scale, slots[i], sees)
            close(o[qo[i]:qo[i + 1]], want, tol, f"prompt {i} causal {causal}")
            lse_close(lse[qo[i]:qo[i + 1]], wl, d, f"prompt {i}")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page", [5, 16])
def test_scales_far_apart(dtype, page):
    """Pages whose scales lie many binades apart: each value counts as what it stands for."""
    from beam_engine_amd import BatchDecodeWithPagedKVCacheWrapper
    say(f"scales far apart {dtype} page {page}")
    hq, hkv, d, n = 8, 2, 128, 4 * page + 1
    total, ptr, ind, last, slots = lists([n, n], page, random.Random(1))
    codes, scale = cache(total, page, hkv, d, 3)
    s = scale.view(torch.uint8)
    far = 20 if dtype == torch.float16 else 60
    g = torch.Generator(device="cuda").manual_seed(2)
    s[:, 1] = torch.randint(121 - far, 122, s[:, 1].shape, generator=g, device="cuda").to(torch.uint8)
    s[ind[0], 1] = 121 - far
    codes[ind[1], 0] = codes[ind[1], 0].view(torch.uint8).fill_(0).view(F8)
    q = torch.randn((2, hq, d), generator=g, device="cuda").to(dtype)
    # row 0 looks at the first page alone, whose values are the smallest
    k0 = codes[ind[0], 0, 0].double() * 2.0 ** (s[ind[0], 0].double() - 127)[:, None]
    q[0] = (k0 * 40.0).repeat_interleave(hq // hkv, 0).to(dtype)
    w = BatchDecodeWithPagedKVCacheWrapper(workspace())
    w.plan(ptr, ind, last, hq, hkv, d, page, q_data_type=dtype, kv_data_type=F8)
    o = w.run(q, codes, kv_scale=scale)
    for i in range(2):
        want, _, tol = attend(q[i:i + 1], codes, scale, slots[i])
        close(o[i:i + 1], want, tol, f"row {i}")


def test_void_slots_and_strides_and_streams():
    """NaN in void slots, in pages nobody names and behind the last sequence; strided q,
    out in a larger tensor, another stream; rows beyond the plan's stay as they were."""
    from beam_engine_amd import BatchPrefillWithPagedKVCacheWrapper
    say("void slots, strides, streams")
    hq, hkv, d, page, dtype = 16, 4, 128, 16, torch.bfloat16
    lens = [(5, 20), (70, 3)]
    total, ptr, ind, last, slots = lists([a + c for a, c in lens], page, random.Random(4), spare=6)
    codes, scale = cache(total, page, hkv, d, 5)
    live = torch.zeros(total * page, dtype=torch.bool)
    live[[t for s in slots for t in s]] = True
    raw = codes.view(torch.uint8).permute(0, 2, 1, 3, 4).contiguous().reshape(total * page, -1)
    raw[~live.cuda()] = 127
    codes = raw.reshape(total, page, 2, hkv, d).permute(0, 2, 1, 3, 4).contiguous().view(F8)
    n = 75
    g = torch.Generator(device="cuda").manual_seed(1)
    wide = torch.randn((n + 4, hq, d + 8), generator=g, device="cuda").to(dtype)
    q = wide[:, :, :d]
    out = torch.full((n + 4, hq, 2 * d), 3.0, dtype=dtype, device="cuda")
    w = BatchPrefillWithPagedKVCacheWrapper(workspace())
    w.plan([0, 5, 75], ptr, ind, last, hq, hkv, d, page, causal=True, q_data_type=dtype, kv_data_type=F8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        w.run(q, codes, kv_scale=scale, out=out[:, :, d:])
    torch.cuda.current_stream().wait_stream(side)
    for i, (lo, hi) in enumerate(((0, 5), (5, 75))):
        sees = torch.arange(hi - lo, device="cuda") + lens[i][1] + 1
        want, _, tol = attend(q[lo:hi].contiguous(), codes, scale, slots[i], sees)
        close(out[lo:hi, :, d:], want, tol, f"prompt {i}")
    assert bool((out[:, :, :d] == 3.0).all()) and bool((out[n:] == 3.0).all())


@pytest.mark.parametrize("hq,hkv,d", [(8, 8, 64), (32, 8, 128), (4, 1, 256)])
def test_nan_values_reach_the_rows_that_see_them(hq, hkv, d):
    """A NaN in V of a prompt's token: the queries from there on have it in that column,
    those before are as if it were not there.  NaN in K: the rows that see the token."""
    from beam_engine_amd import BatchPrefillWithPagedKVCacheWrapper
    say(f"NaN values {hq}/{hkv} d {d}")
    page, n, cached = 16, 150, 30
    total, ptr, ind, last, slots = lists([n + cached], page, random.Random(4))
    codes, scale = cache(total, page, hkv, d, 5)
    raw = codes.view(torch.uint8)
    raw[(raw & 127) == 127] = 3
    for sel, tok, h, c in ((1, 40, 0, 7), (1, 100, hkv - 1, d - 1), (1, 64, 0, 8), (0, 170, 0, 1)):
        raw[slots[0][tok] // page, sel, slots[0][tok] % page, h, c] = 127
    q = torch.randn((n, hq, d), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(torch.bfloat16)
    w = BatchPrefillWithPagedKVCacheWrapper(workspace())
    for cus in (None, 3):
        w._num_cus = cus
        w.plan([0, n], ptr, ind, last, hq, hkv, d, page, causal=True, q_data_type=torch.bfloat16, kv_data_type=F8)
        o = w.run(q, codes, kv_scale=scale)
        want, _, tol = attend(q, codes, scale, slots[0], torch.arange(n, device="cuda") + cached + 1)
        assert 0 < int(torch.isnan(want).sum()) < want.numel() // 2
        assert torch.equal(torch.isnan(o), torch.isnan(want))
        close(o, want, tol, f"cus {cus}")


def test_offsets_beyond_32_bits():
    """A pool of more than 2^32 code bytes: the append and attention at its end."""
    from beam_engine_amd import BatchDecodeWithPagedKVCacheWrapper, PageTable
    say("offsets beyond 32 bits")
    page, hkv, d, dtype = 16, 8, 128, torch.bfloat16
    pages = (5 << 30) // (2 * page * hkv * d)
    t = PageTable(1, page_size=page, max_num_pages=pages, head_num=hkv, head_dim=d, store_dtype=F8, compute_dtype=dtype)
    mine = [pages - 1, 0, pages // 2 + 1, pages - 2]
    n = 4 * page - 3
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn((n, hkv, d), generator=g, device="cuda").to(dtype) for _ in range(2))
    t.write_blocks_vectorized(0, i32([mine[i // page] for i in range(n)]), k, v, i32([i % page for i in range(n)]))
    t.check_errors()
    codes, scale = t.kv_cache_at_layer[0], t.kv_scale_at_layer[0]
    small = codes[mine].view(torch.uint8).cpu().numpy(), scale.view(torch.uint8)[mine].cpu().numpy()
    want = np.zeros_like(small[0]), np.zeros_like(small[1])
    kv8.append(*want, [i // page for i in range(n)], [i % page for i in range(n)], k.float().cpu().numpy(),
               v.float().cpu().numpy(), "bfloat16")
    assert np.array_equal(small[1], want[1])
    same_codes(small[0], want[0])
    assert torch.equal(t.dequantized(0)[mine].cpu().double(), torch.from_numpy(kv8.values(*want)))
    q = torch.randn((1, 32, d), generator=g, device="cuda").to(dtype)
    w = BatchDecodeWithPagedKVCacheWrapper(workspace())
    w.plan([0, 4], mine, [page - 3], 32, hkv, d, page, q_data_type=dtype, kv_data_type=F8)
    o = w.run(q, codes, kv_scale=scale)
    want, _, tol = attend(q, codes[mine], scale.view(torch.uint8)[mine].view(E8), list(range(n)))
    close(o, want, tol, "far pages")


# ------------------------------------------------------------------ each kernel
def blocks_of(w):
    return int(w._info.num_wg)


def planned(kind, qo, ptr, ind, last, hq, hkv, d, page, dtype, causal, **kw):
    """A prefill wrapper whose items of more than 64 rows are ``kind``: "blocks" (through a
    fixed layout, which says so), or "tiles" (none has more)."""
    from beam_engine_amd import BatchPrefillWithPagedKVCacheWrapper
    w = BatchPrefillWithPagedKVCacheWrapper(workspace(256))
    if kind == "blocks":
        w.use_fixed_layout(4096, max(1, qo[-1]), 4096, max(1, qo[-1]), 8192, max(1, qo[-1]), 128)
    else:
        w._no_blocks = True
    w.plan(qo, ptr, ind, last, hq, hkv, d, page, causal=causal, q_data_type=dtype, kv_data_type=F8, **kw)
    assert w.stats.kernel == "kv8" and (blocks_of(w) > 0) == (kind == "blocks")
    assert w.stats.launches[0] == ("attn_kv8_block_kernel" if kind == "blocks" else "attn_kv8_kernel")
    return w


@pytest.mark.parametrize("kind", ["tiles", "blocks"])
@pytest.mark.parametrize("sm_scale", [None, 0.0, -0.11])
@pytest.mark.parametrize("hq,hkv,d,dtype,page", [
    (32, 8, 128, torch.bfloat16, 16), (32, 8, 128, torch.float16, 8), (8, 8, 64, torch.float16, 48), (12, 2, 64, torch.bfloat16, 5),
    (40, 2, 128, torch.float16, 3)])
def test_tiles_and_blocks(kind, sm_scale, hq, hkv, d, dtype, page):
    """Prompts of every size through one kernel and the other: a group without queries, one
    without keys, rows that see nothing, NaN codes in void slots and in V."""
    say(f"{kind} {hq}/{hkv} d {d} {dtype} page {page} scale {sm_scale}")
    lens = [(200, 0), (0, 30), (33, 700), (40, -13), (3, 0), (65, 64), (5, -5), (17, 1100)]
    total, ptr, ind, last, slots = lists([a + c for a, c in lens], page, random.Random(page))
    codes, scale = cache(total, page, hkv, d, page, spread=3)
    raw = codes.view(torch.uint8)
    raw[(raw & 127) == 127] = 3
    live = torch.zeros(total * page, dtype=torch.bool)
    live[[t for s in slots for t in s]] = True
    void = ~live.reshape(total, page).cuda()
    raw.copy_(torch.where(void[:, None, :, None, None], torch.full_like(raw, 255), raw))
    t = slots[0][150]
    raw[t // page, 1, t % page, hkv - 1, d - 3] = 127          # seen by the first prompt's rows from 150 on
    qo = [0]
    for a, _ in lens:
        qo.append(qo[-1] + a)
    q = torch.randn((qo[-1], hq, d), generator=torch.Generator(device="cuda").manual_seed(d), device="cuda").to(dtype)
    for causal in (True, False):
        w = planned(kind, qo, ptr, ind, last, hq, hkv, d, page, dtype, causal, sm_scale=sm_scale)
        o, lse = w.run(q, codes, kv_scale=scale, return_lse=True)
        for i, (a, c) in enumerate(lens):
            if a == 0:
                continue
            sees = torch.arange(a, device="cuda") + c + 1 if causal else None
            want, wl, tol = attend(q[qo[i]:qo[i + 1]], codes, scale, slots[i], sees, sm_scale)
            close(o[qo[i]:qo[i + 1]], want, tol, f"prompt {i} causal {causal}")
            lse_close(lse[qo[i]:qo[i + 1]], wl, d, f"prompt {i}")


@pytest.mark.parametrize("hq,hkv,page", [(96, 1, 16), (128, 1, 8), (260, 4, 5)])
def test_groups_beyond_a_tile(hq, hkv, page):
    """GQA groups of more than 64 heads: blocks alone, whatever the plan."""
    from beam_engine_amd import BatchDecodeWithPagedKVCacheWrapper
    say(f"group {hq // hkv}")
    d, lens, dtype = 128, [1, 0, 17, 500, 2300], torch.bfloat16
    total, ptr, ind, last, slots = lists(lens, page, random.Random(1))
    codes, scale = cache(total, page, hkv, d, 3, spread=3)
    q = torch.randn((len(lens), hq, d), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    for no_blocks in (False, True):
        w = BatchDecodeWithPagedKVCacheWrapper(workspace())
        w._no_blocks = no_blocks
        w.plan(ptr, ind, last, hq, hkv, d, page, q_data_type=dtype, kv_data_type=F8)
        assert blocks_of(w) == w.stats.num_items
        o, lse = w.run(q, codes, kv_scale=scale, return_lse=True)
        for i in range(len(lens)):
            want, wl, tol = attend(q[i:i + 1], codes, scale, slots[i])
            close(o[i:i + 1], want, tol, f"len {lens[i]}")
            lse_close(lse[i:i + 1], wl, d, f"len {lens[i]}")


@pytest.mark.parametrize("page", [8, 16, 32])
@pytest.mark.parametrize("hq,hkv,d,dtype", [(32, 8, 128, torch.bfloat16), (8, 8, 64, torch.float16), (32, 2, 256, torch.bfloat16)])
def test_waves_of_short_items(hq, hkv, d, dtype, page):
    """Many short groups of at most 16 rows, a wave each where pages allow: every length
    around a step, several queries a group, NaN behind each group's last token."""
    from beam_engine_amd import BatchPrefillWithPagedKVCacheWrapper
    say(f"waves {hq}/{hkv} d {d} {dtype} page {page}")
    lens = [n for n in (1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 49, 64, 65, 100, 127, 128, 129)] * 3
    total, ptr, ind, last, slots = lists(lens, page, random.Random(page))
    codes, scale = cache(total, page, hkv, d, page, spread=3)
    raw = codes.view(torch.uint8)
    live = torch.zeros(total * page, dtype=torch.bool)
    live[[t for s in slots for t in s]] = True
    void = ~live.reshape(total, page).cuda()
    raw[(raw & 127) == 127] = 3
    raw.copy_(torch.where(void[:, None, :, None, None], torch.full_like(raw, 127), raw))
    per = max(1, 16 // (hq // hkv))
    qo = [0]
    for i in range(len(lens)):
        qo.append(qo[-1] + (i % per if i % 5 == 0 else 1 + i % per))
    q = torch.randn((qo[-1], hq, d), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    w = BatchPrefillWithPagedKVCacheWrapper(workspace())
    w.plan(qo, ptr, ind, last, hq, hkv, d, page, causal=False, q_data_type=dtype, kv_data_type=F8)
    if page % 16 == 0:
        assert w._info.num_tail_items >= len(lens) // 2
    else:
        assert w._info.num_tail_items == 0
    o, lse = w.run(q, codes, kv_scale=scale, return_lse=True)
    for i in range(len(lens)):
        if qo[i] == qo[i + 1]:
            continue
        want, wl, tol = attend(q[qo[i]:qo[i + 1]], codes, scale, slots[i])
        close(o[qo[i]:qo[i + 1]], want, tol, f"len {lens[i]}")
        lse_close(lse[qo[i]:qo[i + 1]], wl, d, f"len {lens[i]}")


def test_nothing_to_attend():
    """No queries at all, and queries without any key: zeros and an lse of -inf."""
    from beam_engine_amd import BatchDecodeWithPagedKVCacheWrapper
    say("nothing to attend")
    hq, hkv, d, page, dtype = 8, 2, 128, 16, torch.bfloat16
    codes, scale = cache(4, page, hkv, d, 1)
    w = BatchDecodeWithPagedKVCacheWrapper(workspace())
    for n in (0, 3):
        w.plan([0] * (n + 1), [], [0] * n, hq, hkv, d, page, q_data_type=dtype, kv_data_type=F8)
        o, lse = w.run(torch.ones((n, hq, d), dtype=dtype, device="cuda"), codes, kv_scale=scale, return_lse=True)
        assert o.shape == (n, hq, d) and not o.any() and bool(torch.isneginf(lse).all())


def test_a_small_workspace_takes_fewer_partial_rows():
    """A plan whose partial rows do not fit its workspace is made again with longer items;
    one that fits in no way is refused."""
    from beam_engine_amd import BatchDecodeWithPagedKVCacheWrapper
    say("small workspace")
    hq, hkv, d, page, dtype, n = 64, 8, 128, 16, torch.bfloat16, 9000
    total, ptr, ind, last, slots = lists([n, 3], page, random.Random(1))
    codes, scale = cache(total, page, hkv, d, 3)
    q = torch.randn((2, hq, d), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    wide = BatchDecodeWithPagedKVCacheWrapper(workspace())
    wide.plan(ptr, ind, last, hq, hkv, d, page, q_data_type=dtype, kv_data_type=F8)
    small = BatchDecodeWithPagedKVCacheWrapper(torch.empty(wide._need(wide._info) - 512, dtype=torch.uint8, device="cuda"))
    small.plan(ptr, ind, last, hq, hkv, d, page, q_data_type=dtype, kv_data_type=F8)
    assert 0 < small.stats.num_part_rows < wide.stats.num_part_rows
    for w in (wide, small):
        o = w.run(q, codes, kv_scale=scale)
        for i in range(2):
            want, _, tol = attend(q[i:i + 1], codes, scale, slots[i])
            close(o[i:i + 1], want, tol, f"rows {w.stats.num_part_rows}")
    with pytest.raises(MemoryError):
        tiny = BatchDecodeWithPagedKVCacheWrapper(torch.empty(2048, dtype=torch.uint8, device="cuda"))
        tiny.plan(ptr, ind, last, hq, hkv, d, page, q_data_type=dtype, kv_data_type=F8)


@pytest.mark.parametrize("tile_rows", [64, 128])
def test_two_graphs_of_one_plan(tile_rows):
    """A cascade of wide, narrow and short groups in a fixed layout, two layers captured as
    a graph each over one workspace, replayed in turn, again after each new plan, with
    eager work between: every replay gives its layer's result."""
    from beam_engine_amd import MultiLevelCascadeAttentionWrapper
    say(f"two graphs, {tile_rows} rows")
    hq, hkv, d, page, dtype, beams = 16, 4, 128, 16, torch.bfloat16, 40
    w = MultiLevelCascadeAttentionWrapper(2, workspace())
    w.use_fixed_layout(1024, beams, 1024, beams, 4096, beams, tile_rows)
    r = random.Random(2)
    pools = [cache(410, page, hkv, d, 10 + l, spread=3) for l in range(2)]
    q = torch.zeros((beams, hq, d), dtype=dtype, device="cuda")
    outs = [torch.zeros_like(q) for _ in range(2)]

    def plan(prefix, tails, groups):
        total, ptr, ind, last, slots = lists([prefix] * groups + tails, page, r)
        assert total <= 410
        cut = ptr[groups]
        edge = [i * beams // groups for i in range(groups + 1)]
        w.plan([edge, list(range(beams + 1))], [ptr[:groups + 1], [p - cut for p in ptr[groups:]]], [ind[:cut], ind[cut:]],
               [last[:groups], last[groups:]], hq, hkv, d, page, causal=True, q_data_type=dtype, kv_data_type=F8)
        return [slots[max(g for g in range(groups) if edge[g] <= b)] + slots[groups + b] for b in range(beams)]

    def run(layer):
        w.run(q, pools[layer][0], kv_scale=pools[layer][1], out=outs[layer])

    plan(600, [20] * beams, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(0)
        run(1)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for layer in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[layer]):
            run(layer)
    for turn, (prefix, tails, groups) in enumerate([(600, [20] * beams, 1), (1000, [r.randrange(0, 50) for _ in range(beams)], 2),
                                                   (33, [150] * beams, 1), (500, [0] * beams, 10), (640, [1] * beams, 1)]):
        where = plan(prefix, tails, groups)
        q.copy_(torch.randn(q.shape, generator=torch.Generator(device="cuda").manual_seed(turn), device="cuda"))
        for o in outs:
            o.fill_(7.0)
        for layer in (0, 1, 0):
            graphs[layer].replay()
            torch.cuda.synchronize()
            got = outs[layer].clone()
            run(layer)
            # (random codes hold some NaN)
            assert torch.equal(outs[layer].view(torch.int16), got.view(torch.int16)), f"turn {turn} layer {layer}"
        for layer in (0, 1):
            for b in (0, 1, beams // 2, beams - 1):
                want, _, tol = attend(q[b:b + 1], *pools[layer], where[b])
                close(outs[layer][b:b + 1], want, tol, f"turn {turn} layer {layer} beam {b}")


@pytest.mark.parametrize("kind", ["tiles", "blocks"])
def test_far_pages(kind):
    """Pages behind the first 2^32 bytes of a layer."""
    say(f"far pages, {kind}")
    page, hq, hkv, d, dtype = 16, 32, 8, 128, torch.bfloat16
    pages = (5 << 30) // (2 * page * hkv * d)
    codes = torch.zeros((pages, 2, page, hkv, d), dtype=torch.uint8, device="cuda").view(F8)
    scale = torch.zeros((pages, 2, hkv), dtype=torch.uint8, device="cuda").view(E8)
    n = 150
    mine = [pages - 1 - 7 * i for i in range(10)]
    few, s = cache(10, page, hkv, d, 1, spread=2)
    codes.view(torch.uint8)[mine], scale.view(torch.uint8)[mine] = few.view(torch.uint8), s.view(torch.uint8)
    q = torch.randn((n, hq, d), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    w = planned(kind, [0, n], [0, 10], mine, [n - 144], hq, hkv, d, page, dtype, True)
    o = w.run(q, codes, kv_scale=scale)
    want, _, tol = attend(q, few, s, list(range(n)), torch.arange(n, device="cuda") + 1)
    close(o, want, tol, "far pages")


def test_tree_entry_points():
    """The tree's own entry points on an 8-bit cache, which they refuse without its scales."""
    from beam_engine_amd import KVTreeNode
    from beam_engine_amd.fasttree import fasttree_decode, prepare_fasttree_metadata_for_paged_cache
    say("tree entry points")
    hq, hkv, d, page, dtype = 8, 2, 128, 16, torch.bfloat16
    codes, scale = cache(32, page, hkv, d, 4, spread=2)
    # a root of 40 tokens that two requests share, a tail of their own each
    spans = [(-1, 40, [0, 1]), (0, 21, [0]), (0, 5, [1])]           # parent, own tokens, requests
    nodes, pages = [], [[0, 1, 2], [5, 6], [9]]
    for i, (parent, n, reqs) in enumerate(spans):
        t = KVTreeNode()
        t.parent, t.id, t.seqlen, t.num_children, t.requests = parent, i, n + (40 if i else 0), 0 if i else 2, reqs
        nodes.append(t)
    slot = [[p * page + j for p in pg for j in range(page)][:n] for pg, (_, n, _) in zip(pages, spans)]
    paths = [slot[0] + slot[1], slot[0] + slot[2]]
    longest = max(map(len, paths))
    req = torch.tensor([p + [0] * (longest - len(p)) for p in paths])
    meta = prepare_fasttree_metadata_for_paged_cache(nodes, req, 2, hq, hkv, d, page_size=page, q_data_type=dtype, kv_data_type=F8)
    q = torch.randn((2, hq, d), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    with pytest.raises(ValueError, match="kv_scale"):
        fasttree_decode(q, codes, None, meta)
    o = fasttree_decode(q, codes, None, meta, kv_scale=scale)
    for b in range(2):
        want, _, tol = attend(q[b:b + 1], codes, scale, paths[b])
        close(o[b:b + 1], want, tol, f"request {b}")


# ------------------------------------------------------------------ together
def test_written_then_attended_then_captured():
    """Prompts appended and attended, a fork, and decode steps whose append and attention
    are one captured graph, replayed with eager work between: each replay gives the eager
    result on the same bytes."""
    from beam_engine_amd import BatchDecodeWithPagedKVCacheWrapper, BatchPrefillWithPagedKVCacheWrapper
    say("append + attention, eager and captured")
    hq, hkv, d, page, dtype, beams = 16, 4, 128, 16, torch.bfloat16, 4
    prompt, width = 43, (16 + 8) * 128
    g = torch.Generator(device="cuda").manual_seed(3)
    angle = torch.outer(torch.arange(256).double(), 10000.0 ** (-torch.arange(0, d, 2).double() / d))
    cos, sin = (f(torch.cat([angle, angle], -1)).to(dtype).cuda() for f in (torch.cos, torch.sin))
    t = table(32, page, hkv, d, dtype)
    mine = [t.allocate_block() for _ in range(3)]
    at = list(range(prompt))
    x = torch.randn((prompt, width), generator=g, device="cuda").to(dtype)
    q = t.write_rope_qkv(0, x, hq, torch.tensor(at).cuda(), cos, sin, i32([mine[i // page] for i in at]), i32([i % page for i in at]))
    w = BatchPrefillWithPagedKVCacheWrapper(workspace())
    w.plan([0, prompt], [0, 3], mine, [prompt - 32], hq, hkv, d, page, causal=True, q_data_type=dtype, kv_data_type=F8)
    codes, scale = t.kv_cache_at_layer[0], t.kv_scale_at_layer[0]
    slots = [mine[i // page] * page + i % page for i in at]
    want, _, tol = attend(q, codes, scale, slots, torch.arange(prompt, device="cuda") + 1)
    close(w.run(q, codes, kv_scale=scale), want, tol, "prompt")
    # every beam its own copy of the last, partial page
    tails = [t.copy_block(mine[2], prompt - 32) for _ in range(beams)]
    dec = BatchDecodeWithPagedKVCacheWrapper(workspace())
    qkv = torch.zeros((beams, width), dtype=dtype, device="cuda")
    pos = torch.zeros(beams, dtype=torch.long, device="cuda")
    pages, slot = i32(tails), i32([0] * beams)
    q_out, out = (torch.zeros((beams, hq, d), dtype=dtype, device="cuda") for _ in range(2))
    dec.use_fixed_layout(64, beams, 64, beams, 256, beams, 64)

    def plan(length):
        dec.plan([3 * i for i in range(beams + 1)], [p for b in range(beams) for p in mine[:2] + [tails[b]]],
                 [length - 32] * beams, hq, hkv, d, page, q_data_type=dtype, kv_data_type=F8)

    def step():
        t.write_rope_qkv(0, qkv, hq, pos, cos, sin, pages, slot, q_out=q_out)
        dec.run(q_out, codes, kv_scale=scale, out=out)

    plan(prompt + 1)
    pos.fill_(prompt)
    slot.fill_(prompt - 32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    kept = state(t)
    for length in range(prompt + 1, prompt + 5):
        plan(length)
        qkv.copy_((torch.randn((beams, width), generator=g, device="cuda") * (length - prompt)).to(dtype))
        pos.fill_(length - 1)
        slot.fill_(length - 1 - 32)
        x = qkv.float().cpu().numpy().reshape(beams, hq + 2 * hkv, d)
        table_row = cos[length - 1:length].float().cpu().numpy(), sin[length - 1:length].float().cpu().numpy()
        k = kv8.rotate(x[:, hq:hq + hkv], *table_row)
        graph.replay()
        torch.cuda.synchronize()
        kv8.append(*kept, tails, [length - 33] * beams, k, x[:, hq + hkv:], "bfloat16")
        got = state(t)
        assert np.array_equal(got[1], kept[1])
        same_codes(got[0], kept[0])
        captured = out.clone()
        for b in range(beams):
            where = [(mine[:2] + [tails[b]])[i // page] * page + i % page for i in range(length)]
            want, _, tol = attend(q_out[b:b + 1], codes, scale, where)
            close(captured[b:b + 1], want, tol, f"length {length} beam {b}")
        dec.run(q_out, codes, kv_scale=scale, out=out)
        assert torch.equal(out, captured)


def small_config():
    from beam_engine_amd.llama import LlamaConfig
    return LlamaConfig(num_hidden_layers=2, hidden_size=512, num_attention_heads=8, num_key_value_heads=2, head_dim=128,
                       intermediate_size=512, vocab_size=700, max_position_embeddings=512)


@pytest.mark.parametrize("kernel_type", ["cascade", "fasttree", "flat", "auto"])
def test_engine_on_an_8bit_cache(kernel_type):
    """Beam search over 18 steps, the whole step as one graph: each step's logits are the
    eager path's from the same state.  The two plans cut the keys differently, so an
    attention output may be two half steps of bf16 off, of its own size: 2^-7; each of
    the two layers passes that on and its products round once more: 2^-5 in the norm."""
    from beam_engine_amd import PageTable
    from beam_engine_amd.generator import BatchedBeamSearch
    from beam_engine_amd.llama import LlamaDecoder
    say(f"engine {kernel_type}")
    model = LlamaDecoder(small_config(), dtype=torch.bfloat16, seed=5)
    prompts = [[(7 * i + 13 * r) % 700 for i in range(45)] for r in range(2)]
    pt = PageTable(2, page_size=16, max_num_pages=256, head_num=2, head_dim=128, store_dtype=F8, compute_dtype=torch.bfloat16)
    gen = BatchedBeamSearch(model, pt, 4, kernel_type=kernel_type, graphs=True, workspace_bytes=32 << 20)
    gen.prefill(prompts)
    seen, select = [], gen._select
    gen._select = lambda logits: (seen.append(logits.float().clone()), select(logits))
    for step in range(18):
        gen.flush()
        kind, costs = gen._native_kind()
        levels, qids, wp, wpos, pos = gen.state.step_levels(kind, gen.include_self, costs)[:5]
        w = gen._plan(levels, kind == "cascade")
        assert w.stats.kernel == "kv8" and w.stats.launches[0].startswith("attn_kv8")
        want = model.decode(torch.tensor(np.asarray(qids), dtype=torch.long).cuda(), torch.tensor(np.asarray(pos), dtype=torch.long).cuda(),
                            i32(wp), i32(wpos), pt, lambda l, q, kv: w.run(q, kv, kv_scale=pt.kv_scale_at_layer[l])).float()
        gen.step()
        assert gen.step_graphed
        off = float((seen[-1] - want).norm() / want.norm())
        assert off < 2.0 ** -5, f"step {step}: {off}"
    res = gen.final_sequences()
    assert all(len(seqs) == 4 for seqs in res.values())


def test_prefill_logits_follow_the_cache():
    """The model's prompt logits on an 8-bit cache are those of a 16-bit model whose K and V
    went through the same rounding, to a few 16-bit steps."""
    from beam_engine_amd import PageTable
    from beam_engine_amd.llama import LlamaDecoder
    say("prefill logits")
    cfg = small_config()
    model = LlamaDecoder(cfg, dtype=torch.bfloat16, seed=6)
    ids = torch.randint(0, 700, (2, 70), generator=torch.Generator().manual_seed(1)).cuda()
    logits = {}
    for dt in (F8, torch.bfloat16):
        pt = PageTable(2, page_size=16, max_num_pages=32, head_num=2, head_dim=128, store_dtype=dt, compute_dtype=torch.bfloat16)
        pages = [[pt.allocate_block() for _ in range(5)] for _ in range(2)]
        logits[dt] = model.prefill(ids, pt, pages).double()
    # K and V are off by at most 2^-4 of themselves, a random part of it: the logits of
    # this model (two layers, attention a fraction of the residual) stay within a tenth
    off = (logits[F8] - logits[torch.bfloat16]).norm() / logits[torch.bfloat16].norm()
    assert 0 < float(off) < 0.1
