"""The 8-bit cache's checks of its arguments, on the host: the page table, the attention
wrappers' plans and the C entries refuse what the kernels do not take."""

import ctypes

import numpy as np
import pytest
import torch

from beam_engine_amd import PageTable, _lib

F8 = torch.float8_e4m3fn


def make(**kw):
    args = dict(page_size=8, max_num_pages=4, head_num=2, head_dim=64, device="cpu", store_dtype=F8)
    return PageTable(2, **{**args, **kw})


def test_table_has_codes_and_scales():
    t = make(compute_dtype=torch.float16)
    assert t.kv8 and t.kv_pool.dtype is F8 and t.compute_dtype is torch.float16
    assert t.kv_scale.shape == (2, 4, 2, 2) and t.kv_scale.dtype is torch.float8_e8m0fnu
    assert t.kv_scale_at_layer[1].data_ptr() == t.kv_scale[1].data_ptr()
    assert make().compute_dtype is torch.bfloat16
    plain = PageTable(1, max_num_pages=2, device="cpu")
    assert not plain.kv8 and plain.kv_scale is None and plain.kv_scale_at_layer == [None]
    assert plain.compute_dtype is torch.float16


@pytest.mark.parametrize("kw,what", [(dict(head_dim=96), "head_dim"), (dict(head_dim=32), "head_dim"),
                                     (dict(compute_dtype=torch.float32), "float32"), (dict(page_size=1025), "page size"),
                                     (dict(compute_dtype=F8), "rows")])
def test_table_refuses(kw, what):
    with pytest.raises(NotImplementedError, match=what):
        make(**kw)


def test_compute_dtype_belongs_to_8bit_tables():
    with pytest.raises(ValueError, match="compute_dtype"):
        PageTable(1, max_num_pages=2, device="cpu", store_dtype=torch.float16, compute_dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="8 bits"):
        PageTable(1, max_num_pages=2, device="cpu").dequantized()


def test_writes_check_types_and_devices():
    t = make()
    k = torch.zeros((3, 2, 64))
    idx = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="bfloat16"):
        t.write_blocks_vectorized(0, idx, k, k, idx)
    with pytest.raises(ValueError, match="device"):
        t.write_blocks_vectorized(0, idx, k.bfloat16(), k.bfloat16(), idx)
    with pytest.raises(ValueError, match="bfloat16"):
        t.write_rope_qkv(0, torch.zeros((3, 6 * 64)), 2, idx.long(), torch.zeros((9, 64)), torch.zeros((9, 64)), idx, idx)


# ------------------------------------------------------------------ plans
def plan(dtype=_lib.BE_BF16, flags=_lib.BE_PLAN_KV8, hq=8, hkv=2, d=128, page=16, lens=(40,), caps=None, cus=256):
    lib = _lib.load()
    npg = [-(-n // page) for n in lens]
    qo = np.arange(len(lens) + 1, dtype=np.int32)
    kvp = np.concatenate([[0], np.cumsum(npg)]).astype(np.int32)
    kvi = np.arange(kvp[-1], dtype=np.int32)
    last = np.array([n - (m - 1) * page if m else 0 for n, m in zip(lens, npg)], np.int32)
    level = (_lib.BeLevel * 1)(_lib.BeLevel(qo.ctypes.data, kvp.ctypes.data, kvi.ctypes.data, last.ctypes.data, len(lens)))
    info, buf = _lib.BeAttnPlanInfo(), np.zeros(1 << 16, np.int32)
    rc = lib.be_attn_plan(level, 1, len(lens), hq, hkv, d, page, max(1, len(kvi)), dtype, flags, cus, caps, buf.ctypes.data,
                          buf.size, ctypes.byref(info))
    return rc, info, buf


@pytest.mark.parametrize("kw", [dict(dtype=_lib.BE_F32), dict(page=1025), dict(hq=258, hkv=2), dict(d=96),
                                dict(flags=_lib.BE_PLAN_KV8 | _lib.BE_PLAN_FORCE_VALU),
                                dict(flags=_lib.BE_PLAN_KV8 | _lib.BE_PLAN_FUSED_MERGE),
                                dict(flags=_lib.BE_PLAN_KV8 | _lib.BE_PLAN_ROWS)])
def test_plan_refuses(kw):
    assert plan(**kw)[0] == _lib.BE_ERR_UNSUPPORTED


@pytest.mark.parametrize("hq,hkv,d,page", [(8, 8, 64, 1), (32, 8, 128, 16), (64, 1, 256, 5), (16, 2, 128, 1024)])
def test_plan_covers_every_token(hq, hkv, d, page):
    """Every group's tokens lie in its items once, and an item's pages fit the kernel's table."""
    lens = (1, 0, page, page + 1, 700, 5000)
    rc, info, buf = plan(hq=hq, hkv=hkv, d=d, page=page, lens=lens)
    assert rc == 0 and info.kernel == 4 and info.tile_rows in (16, 32, 64, 128)
    assert info.kv_bytes == 2 * sum(lens) * hkv * d
    items = buf[info.off_items:info.off_items + 8 * info.num_items].reshape(-1, 8)
    for i, n in enumerate(lens):
        mine = sorted((int(x[3]), int(x[4])) for x in items if x[0] == i)
        assert all(x[7] == x[3] // page for x in items)
        at = 0
        for b, c in mine:
            assert b == at and c > 0
            at += c
            assert (b + c - 1) // page - b // page + 1 <= 256
        assert at == n


def items_of(info, buf):
    return buf[info.off_items:info.off_items + 8 * info.num_items].reshape(-1, 8)


@pytest.mark.parametrize("page", [8, 16, 48])
def test_plan_names_who_takes_an_item(page):
    """Blocks first, one wave's items last; an item is a wave's by its rows, tokens and
    pages; NO_BLOCKS leaves blocks to groups that no tile holds."""
    lens = (5, 128, 129, 40, 0, 700)
    rc, info, buf = plan(hq=8, hkv=2, page=page, lens=lens)
    assert rc == 0 and info.num_wg == 0
    short = [x[4] <= 128 for x in items_of(info, buf)]
    if page % 16 == 0:
        assert info.num_tail_items == sum(short) and all(short[len(short) - sum(short):])
    else:
        assert info.num_tail_items == 0
    for flags in (_lib.BE_PLAN_KV8, _lib.BE_PLAN_KV8 | _lib.BE_PLAN_NO_BLOCKS):
        rc, info, buf = plan(hq=130, hkv=2, page=page, lens=lens, flags=flags)
        assert rc == 0 and info.num_wg == info.num_items and info.num_tail_items == 0 and info.tile_rows == 128
        assert all(x[7] == x[3] // page for x in items_of(info, buf))


def test_less_scratch_does_not_cut():
    rows = []
    for flags in (_lib.BE_PLAN_KV8, _lib.BE_PLAN_KV8 | _lib.BE_PLAN_LESS_SCRATCH):
        rc, info, _ = plan(hq=64, hkv=8, lens=(9000, 3), flags=flags)
        assert rc == 0
        rows.append(info.num_part_rows)
    assert rows[1] == 3 < rows[0]           # an item holds at most 4032 tokens of 16-token pages


def test_fixed_layout_keeps_its_rows():
    caps = _lib.BePlanCaps(64, 8, 64, 8, 64, 8, 64, 0)
    rc, info, _ = plan(lens=(100, 3, 0), caps=ctypes.byref(caps))
    assert rc == 0 and info.static_layout == 1 and info.tile_rows == 64 and info.grid_items == 64


def test_wrappers_refuse_other_types():
    from beam_engine_amd.attention import _PagedPlanner
    w = _PagedPlanner.__new__(_PagedPlanner)
    for q, kv in ((torch.float32, F8), (torch.bfloat16, torch.float16), ("float16", "float8_e5m2"), (F8, F8)):
        with pytest.raises(NotImplementedError):
            w._set_kv_type(q, kv)
    for q, kv, on in ((torch.bfloat16, F8, True), ("float16", "float8_e4m3fn", True), ("float16", torch.float16, False),
                      (torch.float32, None, False)):
        w._set_kv_type(q, kv)
        assert w._kv8 is on


# ------------------------------------------------------------------ C entries (nothing is launched)
def test_entries_refuse():
    lib = _lib.load()
    one, odd = 1 << 20, (1 << 20) + 8                       # addresses that no refused call reads
    ok = dict(kv=one, scale=one, dt=_lib.BE_BF16, pages=4, page=8, hkv=2, d=64, k=one, ksn=128, n=1)

    def append(**kw):
        a = {**ok, **kw}
        return lib.be_kv8_append(a["kv"], a["scale"], a["dt"], a["pages"], a["page"], a["hkv"], a["d"], one, one, a["k"],
                                 a["ksn"], 64, one, 128, 64, a["n"], None, None)

    assert append(n=0) == _lib.BE_OK
    for kw in (dict(kv=None), dict(scale=None), dict(dt=_lib.BE_F32), dict(pages=0), dict(page=0), dict(hkv=0), dict(kv=odd),
               dict(k=odd), dict(ksn=129), dict(n=-1)):
        assert append(**kw) == _lib.BE_ERR_INVALID, kw
    assert append(d=96) == _lib.BE_ERR_UNSUPPORTED

    def rope(qkv=one, sn=8 * 64, hq=4, q_out=one, n=1, maxp=16):
        return lib.be_kv8_rope_append(qkv, sn, _lib.BE_F16, n, hq, 2, 64, one, one, one, maxp, q_out, one, one, 4, 8, one, one,
                                      None, None)

    assert rope(n=0) == _lib.BE_OK
    for kw in (dict(qkv=odd), dict(sn=7 * 64), dict(sn=8 * 64 + 4), dict(hq=0), dict(q_out=odd), dict(q_out=None), dict(maxp=0)):
        assert rope(**kw) == _lib.BE_ERR_INVALID, kw

    def copy(stride=1 << 20, scales=1 << 10, layers=2, n=1):
        return lib.be_kv8_page_copy(one, stride, one, scales, layers, 4, 8, 2, 64, one, one, one, None, n, None, None)

    assert copy(n=0) == copy(layers=0) == _lib.BE_OK
    for kw in (dict(stride=64), dict(stride=(1 << 20) + 8), dict(scales=8), dict(n=-1), dict(layers=1 << 20)):
        assert copy(**kw) == _lib.BE_ERR_INVALID, kw
    assert lib.be_kv8_values(one, one, _lib.BE_F32, 4, 8, 2, 64, -1, one, None) == _lib.BE_ERR_INVALID
    assert lib.be_kv8_values(one, one, _lib.BE_F16, 4, 8, 2, 64, 2, one, None) == _lib.BE_ERR_INVALID
    assert lib.be_kv8_values(one, one, _lib.BE_F16, 4, 8, 2, 64, 0, odd, None) == _lib.BE_ERR_INVALID
    assert lib.be_kv8_values(one, one, _lib.BE_F16, 0, 8, 2, 64, 0, one, None) == _lib.BE_OK


def test_runs_name_their_cache():
    """An 8-bit plan does not run without scales, another plan not with them, and rows that
    do not start on 16 bytes are refused (nothing is launched)."""
    lib = _lib.load()
    _, info, _ = plan()
    one, odd = 1 << 20, (1 << 20) + 4
    run = (ctypes.byref(info), one, one)
    tail = (None, 1.0, 3, None)
    assert lib.be_attn_run(*run, one, 1024, 128, one, one, 1024, 128, *tail) == _lib.BE_ERR_INVALID
    assert lib.be_attn_run_kv8(*run, one, 1024, 128, one, None, one, 1024, 128, *tail) == _lib.BE_ERR_INVALID
    for q, kv, out, sn in ((odd, one, one, 1024), (one, odd, one, 1024), (one, one, odd, 1024), (one, one, one, 1022)):
        assert lib.be_attn_run_kv8(*run, q, sn, 128, kv, one, out, 1024, 128, *tail) == _lib.BE_ERR_INVALID
    rc, other, _ = plan(flags=0)
    assert rc == 0
    assert lib.be_attn_run_kv8(ctypes.byref(other), one, one, one, 1024, 128, one, one, one, 1024, 128, *tail) == _lib.BE_ERR_INVALID


def test_a_launch_has_its_limit():
    """Work items x KV heads beyond a grid are refused (nothing is launched)."""
    lib = _lib.load()
    _, info, _ = plan(hq=8, hkv=8)
    one = 1 << 20
    info.grid_items = 1 << 21
    rc = lib.be_attn_run_kv8(ctypes.byref(info), one, one, one, 1024, 128, one, one, one, 1024, 128, None, 1.0, 3, None)
    assert rc == _lib.BE_ERR_INVALID and b"exceed a launch" in lib.be_last_error()
