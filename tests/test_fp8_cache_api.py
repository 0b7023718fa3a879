"""The 8-bit KV cache without a GPU: refusals of its entry points, pool sizes, and
the order of the hand-offs in the built code."""

import os
import re
import sys

import numpy as np
import pytest
import torch

from test_merge_order import _hipcc, check_handoff, device_asm, kernels

import fp8_util
from mini_vllm.attention import _hip
from mini_vllm.attention import paged_attention_fp8 as fp8
from mini_vllm.cache.pool import KVCachePool, compute_num_gpu_blocks

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
BUF = 4096  # a stand-in address: every call here is refused before it is used


@pytest.fixture(scope="module")
def lib():
    return _hip.load()


# ------------------------------------------------------------- the C ABI --

PLAN = dict(slots=BUF, n=4, bs=16, nb=8, pos=None, max_pos=0, items=BUF, table=BUF, status=BUF,
            ws=None, ws_bytes=0, stream=None)
WRITE = dict(q=BUF, q_st=64, q_sh=64, qo=BUF, qo_st=64, qo_sh=64, k=BUF, k_st=64, k_sh=64, ko=BUF,
             ko_st=64, ko_sh=64, v=BUF, v_st=64, v_sh=64, kc=BUF, vc=BUF, scales=BUF, items=BUF,
             table=BUF, status=BUF, max_items=4, pos=BUF, cos=BUF, sin=BUF, table_st=64, max_pos=10,
             n=4, hq=2, hkv=1, d=64, bs=16, nb=8, dtype=2, stream=None)
DPLAN = dict(kv=BUF, kv64=1, bt=BUF, bt64=1, bt_st=4, n=2, width=4, bs=16, nb=8, hkv=1, d=64, cus=256,
             fixed=0, work=BUF, cap=512, ids=BUF, ids_cap=8192, counters=BUF, status=BUF, stream=None)
DECODE = dict(q=BUF, q_st=64, q_sh=64, kc=BUF, vc=BUF, scales=BUF, work=BUF, ids=BUF, ids_cap=64,
              groups=1, part=16, parts=1, counters=BUF, out=BUF, o_st=64, o_sh=64, scale=0.125, b=1,
              hq=2, hkv=1, d=64, bs=16, nb=8, dtype=2, ws=None, ws_bytes=0, stream=None)
PREFILL = dict(q=BUF, q_st=64, q_sh=64, k=BUF, k_st=64, k_sh=64, v=BUF, v_st=64, v_sh=64, kc=BUF,
               vc=BUF, scales=BUF, bt=BUF, i64=1, bt_st=4, seqs=BUF, n=1, work=BUF, groups=1,
               tokens=16, units=1, parts=1, out=BUF, o_st=64, o_sh=64, scale=0.125, hq=2, hkv=1, d=64,
               bs=16, nb=8, dtype=2, ws=None, ws_bytes=0, stream=None)
SLOTS = dict(bt=BUF, i64=1, bt_st=4, rows=1, width=4, seq_rows=BUF, cu=BUF, n=1, total=4, bs=16, nb=8,
             slots=BUF, bad=BUF, stream=None)
GATHER = dict(kc=BUF, vc=BUF, scales=BUF, slots=BUF, total=4, ok=BUF, ov=BUF, hkv=1, d=64, bs=16,
              nb=8, dtype=2, stream=None)
ENTRIES = {
    "mv_fp8_decode_plan": DPLAN, "mv_fp8_write_plan": PLAN, "mv_fp8_kv_cache_write": WRITE, "mv_fp8_paged_decode": DECODE,
    "mv_fp8_paged_prefill": PREFILL, "mv_fp8_prefix_slots": SLOTS, "mv_fp8_gather_kv": GATHER,
}
INVALID, UNSUPPORTED = _hip.MV_ERR_INVALID_ARGUMENT, _hip.MV_ERR_UNSUPPORTED
REFUSED = [
    ("mv_fp8_write_plan", dict(bs=8), UNSUPPORTED), ("mv_fp8_write_plan", dict(bs=512), UNSUPPORTED),
    ("mv_fp8_write_plan", dict(bs=48), UNSUPPORTED), ("mv_fp8_write_plan", dict(nb=0), INVALID),
    ("mv_fp8_write_plan", dict(nb=1 << 31), INVALID), ("mv_fp8_write_plan", dict(n=-1), INVALID),
    ("mv_fp8_write_plan", dict(status=None), INVALID), ("mv_fp8_write_plan", dict(slots=None), INVALID),
    ("mv_fp8_write_plan", dict(n=5000), INVALID),  # no workspace
    ("mv_fp8_kv_cache_write", dict(dtype=0), UNSUPPORTED),
    ("mv_fp8_kv_cache_write", dict(dtype=3), UNSUPPORTED),
    ("mv_fp8_kv_cache_write", dict(d=96), UNSUPPORTED), ("mv_fp8_kv_cache_write", dict(bs=1), UNSUPPORTED),
    ("mv_fp8_kv_cache_write", dict(hkv=0), INVALID), ("mv_fp8_kv_cache_write", dict(n=-1), INVALID),
    ("mv_fp8_kv_cache_write", dict(scales=None), INVALID),
    ("mv_fp8_kv_cache_write", dict(items=None), INVALID),
    ("mv_fp8_kv_cache_write", dict(sin=None), INVALID), ("mv_fp8_kv_cache_write", dict(pos=None), INVALID),
    ("mv_fp8_kv_cache_write", dict(max_pos=0), INVALID), ("mv_fp8_kv_cache_write", dict(qo=None), INVALID),
    ("mv_fp8_kv_cache_write", dict(cos=None), INVALID),  # a query without tables
    ("mv_fp8_kv_cache_write", dict(k=BUF + 2), INVALID), ("mv_fp8_kv_cache_write", dict(v_st=65), INVALID),
    ("mv_fp8_kv_cache_write", dict(table_st=65), INVALID),
    ("mv_fp8_decode_plan", dict(bs=8), UNSUPPORTED), ("mv_fp8_decode_plan", dict(d=96), UNSUPPORTED),
    ("mv_fp8_decode_plan", dict(n=-1), INVALID), ("mv_fp8_decode_plan", dict(hkv=0), INVALID),
    ("mv_fp8_decode_plan", dict(cus=0), INVALID), ("mv_fp8_decode_plan", dict(nb=0), INVALID),
    ("mv_fp8_decode_plan", dict(cap=1), INVALID), ("mv_fp8_decode_plan", dict(ids_cap=16), INVALID),
    ("mv_fp8_decode_plan", dict(status=None), INVALID), ("mv_fp8_decode_plan", dict(kv=None), INVALID),
    ("mv_fp8_decode_plan", dict(bt=None), INVALID), ("mv_fp8_decode_plan", dict(work=BUF + 4), INVALID),
    ("mv_fp8_decode_plan", dict(width=1 << 30), INVALID),
    ("mv_fp8_paged_decode", dict(dtype=0), UNSUPPORTED), ("mv_fp8_paged_decode", dict(d=32), UNSUPPORTED),
    ("mv_fp8_paged_decode", dict(bs=4), UNSUPPORTED), ("mv_fp8_paged_decode", dict(hq=17), UNSUPPORTED),
    ("mv_fp8_paged_decode", dict(hq=3, hkv=2), INVALID), ("mv_fp8_paged_decode", dict(scales=None), INVALID),
    ("mv_fp8_paged_decode", dict(ids_cap=3), INVALID), ("mv_fp8_paged_decode", dict(parts=2), INVALID),
    ("mv_fp8_paged_decode", dict(parts=2, ws=4096, ws_bytes=8), INVALID),
    ("mv_fp8_paged_decode", dict(parts=0), INVALID), ("mv_fp8_paged_decode", dict(groups=2, ids_cap=99), INVALID),
    ("mv_fp8_paged_decode", dict(q=BUF + 8), INVALID), ("mv_fp8_paged_decode", dict(out=BUF + 2), INVALID),
    ("mv_fp8_paged_decode", dict(o_st=63), INVALID),
    ("mv_fp8_paged_prefill", dict(dtype=0), UNSUPPORTED), ("mv_fp8_paged_prefill", dict(bs=8), UNSUPPORTED),
    ("mv_fp8_paged_prefill", dict(d=80), UNSUPPORTED), ("mv_fp8_paged_prefill", dict(scales=None), INVALID),
    ("mv_fp8_paged_prefill", dict(scales=BUF + 4), INVALID), ("mv_fp8_paged_prefill", dict(tokens=0), INVALID),
    ("mv_fp8_paged_prefill", dict(tokens=129), INVALID), ("mv_fp8_paged_prefill", dict(k=BUF + 4), INVALID),
    ("mv_fp8_paged_prefill", dict(parts=2), INVALID),
    ("mv_fp8_prefix_slots", dict(bs=8), UNSUPPORTED), ("mv_fp8_prefix_slots", dict(n=0), INVALID),
    ("mv_fp8_prefix_slots", dict(bad=None), INVALID), ("mv_fp8_prefix_slots", dict(bt=None), INVALID),
    ("mv_fp8_gather_kv", dict(dtype=0), UNSUPPORTED), ("mv_fp8_gather_kv", dict(d=100), UNSUPPORTED),
    ("mv_fp8_gather_kv", dict(total=-1), INVALID), ("mv_fp8_gather_kv", dict(slots=None), INVALID),
    ("mv_fp8_gather_kv", dict(ok=BUF + 8), INVALID),
]


@pytest.mark.parametrize("name,change,code", REFUSED)
def test_refused(lib, name, change, code):
    args = dict(ENTRIES[name])
    assert set(change) <= set(args)
    args.update(change)
    assert getattr(lib, name)(*args.values()) == code
    assert name.encode() in lib.mv_last_error() or b"mv_paged_prefill" in lib.mv_last_error()


def test_key_out_is_no_input(lib):
    """The append reads the key in two places at once: it is not rotated in place."""
    for change in (dict(ko=BUF), dict(ko=2 * BUF, v=2 * BUF)):
        args = dict(WRITE, **change)
        assert getattr(lib, "mv_fp8_kv_cache_write")(*args.values()) == INVALID
        assert b"key_out must not" in lib.mv_last_error()


def test_nothing_to_do(lib):
    assert lib.mv_fp8_kv_cache_write(*{**WRITE, "n": 0}.values()) == 0
    assert lib.mv_fp8_paged_decode(*{**DECODE, "groups": 0}.values()) == 0
    assert lib.mv_fp8_paged_prefill(*{**PREFILL, "groups": 0}.values()) == 0
    assert lib.mv_fp8_gather_kv(*{**GATHER, "total": 0}.values()) == 0


def test_workspaces(lib):
    assert lib.mv_fp8_write_plan_workspace_bytes(2048) == 0
    # at least twice as many entries as tokens, a key and an item each
    for n in (2049, 4096, 4097, 100000):
        assert lib.mv_fp8_write_plan_workspace_bytes(n) >= 2 * n * 8
    assert lib.mv_fp8_paged_decode_workspace_bytes(3, 14, 64, 1) == 0
    assert lib.mv_fp8_paged_decode_workspace_bytes(3, 14, 64, 5) >= 3 * 14 * 5 * (64 + 2) * 4


# --------------------------------------------------------- Python checks --


def _pool(bs=16, d=64, nb=4, hkv=2):
    c = torch.zeros(nb, hkv, bs, d).to(fp8.FP8_DTYPE)
    return c, c.clone(), torch.zeros(nb, hkv, 2)


def _check(kc, vc, sc, bs):
    return fp8._check_pool(kc, vc, sc, bs, "test")


def test_pool_checks():
    kc, vc, sc = _pool()
    with pytest.raises(AssertionError, match="must be cuda"):  # (all else is in order)
        _check(kc, vc, sc, 16)
    with pytest.raises(AssertionError, match="block_size"):
        _check(kc, vc, sc, 32)
    with pytest.raises(AssertionError, match="16 to 256"):
        _check(*_pool(bs=8), 8)
    with pytest.raises(AssertionError, match="head_dim"):
        _check(*_pool(d=32), 16)
    with pytest.raises(AssertionError, match="expected torch.float8"):
        _check(kc.to(torch.bfloat16), vc, sc, 16)
    with pytest.raises(AssertionError, match="kv_scales"):
        _check(kc, vc, sc[:, :, 0], 16)
    with pytest.raises(AssertionError, match="kv_scales"):
        _check(kc, vc, sc.double(), 16)
    with pytest.raises(AssertionError, match="contiguous"):
        _check(kc, vc, sc.transpose(0, 1).contiguous().transpose(0, 1), 16)


def test_pool_sizes():
    p = KVCachePool.allocate(3, 5, 32, 2, 64, torch.bfloat16, "cpu", cache_dtype=fp8.FP8_DTYPE)
    assert all(t.dtype is fp8.FP8_DTYPE and t.shape == (5, 2, 32, 64) for t in p.key_caches + p.value_caches)
    assert len(p.kv_scales) == 3 and all(s.shape == (5, 2, 2) and not s.any() for s in p.kv_scales)
    assert p.dtype is torch.bfloat16
    assert p.bytes_per_block_per_layer == 2 * 2 * 32 * 64 + 2 * 2 * 4
    held = sum(t.numel() * t.element_size() for t in p.key_caches + p.value_caches + p.kv_scales)
    assert p.total_bytes == held
    p.kv_scales[1].fill_(2.0)
    p.reset()
    assert not any(s.any() for s in p.kv_scales)
    plain = KVCachePool.allocate(3, 5, 32, 2, 64, torch.bfloat16, "cpu")
    assert plain.kv_scales is None and plain.bytes_per_block_per_layer == 4 * 2 * 32 * 64
    with pytest.raises(ValueError, match="cache_dtype"):
        KVCachePool.allocate(1, 4, 16, 2, 64, torch.bfloat16, "cpu", cache_dtype=torch.int8)
    assert compute_num_gpu_blocks(1, 2, 64, 16, torch.bfloat16, "cpu", cache_dtype=fp8.FP8_DTYPE) == 16


# ------------------------------------------------------------- the oracle --


def test_oracle_rounds_to_e4m3():
    """The oracle's rounding against every code and the midpoints between them."""
    codes = torch.arange(127, dtype=torch.uint8).view(fp8.FP8_DTYPE).double().numpy()
    assert np.array_equal(fp8_util.e4m3(codes), codes)
    mid = (codes[1:] + codes[:-1]) / 2
    want = np.where(np.arange(126) % 2 == 0, codes[:-1], codes[1:])  # ties to the even code
    assert np.array_equal(fp8_util.e4m3(mid), want)
    assert np.array_equal(fp8_util.e4m3(-np.nextafter(mid, 500)), -codes[1:])
    assert np.array_equal(fp8_util.e4m3(np.nextafter(mid, 0)), codes[:-1])
    assert np.isnan(fp8_util.e4m3(np.array([np.nan])))[0]


@pytest.mark.parametrize("amax,e", [(0.0, -110), (448.0, 0), (448.0001, 1), (447.9, 0), (224.0, -1),
                                    (1.75, -8), (1.0, -8), (2.0 ** -140, -110), (3.4e38, 120)])
def test_oracle_scale(amax, e):
    assert fp8_util.scale_exp(amax) == e


# ------------------------------------------------------- hand-off orders --


@pytest.mark.skipif(_hipcc() is None, reason="hipcc not installed")
@pytest.mark.parametrize("src,kernel,count", [
    ("fp8_decode.hip", "fp8_decode_kernel", 4),
    ("fp8_prefill.hip", "fp8_prefill_kernel", 16),
])
def test_partials_are_published_before_the_counter(src, kernel, count, tmp_path):
    ks = kernels(device_asm(src, tmp_path), kernel)
    assert len(ks) == count, sorted(ks)
    for name, ins in ks.items():
        check_handoff(name, ins)


@pytest.mark.skipif(_hipcc() is None, reason="hipcc not installed")
def test_plan_cells_are_cleared_before_they_are_claimed(tmp_path):
    """The one-group write plan: the table's -1 stores are acknowledged and every
    wave has met at a barrier before the first atomic on the table."""
    ks = kernels(device_asm("fp8_cache.hip", tmp_path), "fp8_write_plan_kernel")
    (ins,) = ks.values()
    claims = [i for i, x in enumerate(ins) if re.match(r"(global|flat)_atomic_smax", x)]
    assert claims, [x for x in ins if "atomic" in x]
    stores = [i for i in range(claims[0]) if ins[i].startswith("global_store")]
    between = ins[stores[-1] + 1:claims[0]]
    waits = [k for k, x in enumerate(between) if re.match(r"s_waitcnt\b.*\bvmcnt\(0\)", x)]
    assert waits and "s_barrier" in between[waits[0]:], between
