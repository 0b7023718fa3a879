"""The quantising append and the gather against the format's definition in 64
bits: codes and scales exactly."""

import numpy as np
import pytest
import torch

import fp8_util
from fp8_util import FP8
from gpu_util import DEV, bits, say
from mini_vllm.attention import paged_attention_fp8 as fp8
from mini_vllm.attention import paged_attention_gpu as gpu

pytestmark = pytest.mark.gpu


def _rows(t, hq, hkv, d, dtype, seed, scale=1.0):
    """q, k, v as column views of a fused QKV output."""
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(t, (hq + 2 * hkv) * d, generator=g) * scale).to(dtype).to(DEV)
    return (qkv[:, :hq * d].view(t, hq, d), qkv[:, hq * d:(hq + hkv) * d].view(t, hkv, d),
            qkv[:, (hq + hkv) * d:].view(t, hkv, d))


def _expected(kc, vc, scales, k, v, slots, bs):
    """The pool after the append: (code values, scales) in 64 bits."""
    out = []
    for j, (c, x) in enumerate(((kc, k), (vc, v))):
        codes = c.cpu().double().numpy()
        sc = scales[:, :, j].cpu().double().numpy().copy()
        fp8_util.append(codes, sc, x.cpu().double().numpy(), slots.tolist(), bs, x.dtype)
        out.append((codes, sc))
    return out


def _check(kc, vc, scales, want):
    torch.cuda.synchronize()
    for j, c in enumerate((kc, vc)):
        codes, sc = want[j]
        got = scales[:, :, j].cpu().double().numpy()
        assert np.array_equal(got, sc), (j, np.argwhere(got != sc)[:4])
        got = c.cpu().double().numpy()
        same = (got == codes) | (np.isnan(got) & np.isnan(codes))
        assert same.all(), (j, np.argwhere(~same)[:4], got[~same][:4], codes[~same][:4])


def _slots(seqs, bs, num_blocks, seed):
    """Slots of sequences (cached, new): blocks dealt at random, tokens in order."""
    it = iter(torch.randperm(num_blocks, generator=torch.Generator().manual_seed(seed)).tolist())
    out = []
    for cached, new in seqs:
        table = [next(it) for _ in range(-(-(cached + new) // bs))]
        out += [table[p // bs] * bs + p % bs for p in range(cached, cached + new)]
    return torch.tensor(out, dtype=torch.int64)


CASES = [
    # (sequences (cached, new), block size, kv heads, head_dim, dtype)
    ([(0, 1)], 16, 2, 64, torch.bfloat16),
    ([(15, 1), (16, 1), (31, 1), (700, 1)], 16, 1, 128, torch.float16),
    ([(5, 40), (0, 16), (33, 1)], 16, 2, 64, torch.float16),
    ([(c, 1) for c in range(70)], 16, 3, 64, torch.bfloat16),
    ([(7, 100), (0, 33)], 32, 4, 128, torch.bfloat16),
    ([(63, 130), (1, 1)], 64, 2, 64, torch.float16),
    ([(100, 300), (0, 128), (127, 1)], 128, 2, 128, torch.bfloat16),
    ([(255, 2), (0, 600), (513, 100)], 256, 1, 64, torch.bfloat16),
    ([(10, 2038), (3, 10)], 16, 1, 64, torch.bfloat16),    # 2048 tokens: the one-group plan's most
    ([(10, 2038), (3, 11)], 16, 1, 64, torch.bfloat16),    # one more
    ([(0, 4500), (77, 1200)], 64, 1, 128, torch.float16),
]


@pytest.mark.parametrize("i", range(len(CASES)))
def test_append_equals_the_definition(i):
    seqs, bs, hkv, d, dtype = CASES[i]
    say("append", i, seqs[:4], bs, hkv, d, dtype)
    num_blocks = sum(-(-(c + n) // bs) for c, n in seqs) + 3
    slots = _slots(seqs, bs, num_blocks, i)
    kc, vc, sc = fp8_util.random_pool(num_blocks, hkv, bs, d, i, DEV)
    _, k, v = _rows(len(slots), 1, hkv, d, dtype, i, scale=3.0)
    want = _expected(kc, vc, sc, k, v, slots, bs)
    fp8.hip_fp8_cache_write(k, v, kc, vc, sc, slots.to(DEV), bs)
    _check(kc, vc, sc, want)


def test_any_order_and_skipped_tokens():
    """Tokens of a block anywhere in the call, some skipped, int32 slots."""
    bs, num_blocks = 32, 40
    perm = torch.randperm(num_blocks * bs, generator=torch.Generator().manual_seed(3))[:500]
    perm[::7] = -1
    kc, vc, sc = fp8_util.random_pool(num_blocks, 2, bs, 64, 3, DEV)
    _, k, v = _rows(500, 2, 2, 64, torch.bfloat16, 4, scale=5.0)
    want = _expected(kc, vc, sc, k, v, perm, bs)
    fp8.hip_fp8_cache_write(k, v, kc, vc, sc, perm.to(torch.int32).to(DEV), bs)
    _check(kc, vc, sc, want)


@pytest.mark.parametrize("bs,d", [(16, 64), (16, 128), (64, 64), (256, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scales_grow_shrink_and_start_anew(bs, d, dtype):
    """One block over several calls: larger rows scale the earlier ones down, smaller
    ones leave the scale, place 0 starts anew (also over NaN codes), zeros."""
    say("grow", bs, d, dtype)
    kc, vc, sc = fp8_util.random_pool(3, 2, bs, d, 1, DEV)
    sc[2].zero_()  # never written
    kc.view(torch.uint8)[2] = 0x7F
    vc.view(torch.uint8)[2] = 0xFF
    for step, (places, size) in enumerate([((3,), 1.0), ((4, 5), 40.0), ((6,), 1e-3), ((7, 8, 9), 900.0),
                                           ((0, 1), 0.01), ((2,), 0.0), ((5, 0), 0.0), ((1,), 7.0)]):
        slots = torch.tensor([bs * b + o for b in (0, 2) for o in places])
        _, k, v = _rows(len(slots), 1, 2, d, dtype, step, scale=size)
        want = _expected(kc, vc, sc, k, v, slots, bs)
        fp8.hip_fp8_cache_write(k, v, kc, vc, sc, slots.to(DEV), bs)
        _check(kc, vc, sc, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_extreme_values(dtype):
    """Infinities and NaN (stored as NaN, no part in the scale), the type's largest
    and smallest values, exact borders of the scale."""
    bs, d = 16, 64
    info = torch.finfo(dtype)
    special = [float("inf"), -float("inf"), float("nan"), info.max, -info.max, info.tiny,
               info.smallest_normal / 4, 0.0, -0.0, 448.0, -449.0, 447.0, 240.0, 1.75, 1.7578125]
    kc, vc, sc = fp8_util.random_pool(len(special) + 1, 1, bs, d, 2, DEV)
    rows = torch.zeros(len(special), 1, d)
    for i, x in enumerate(special):
        rows[i, 0, :: 3] = x
        rows[i, 0, 1::3] = 0.37 if abs(x) < 1e3 else 1e4
    k = rows.to(dtype).to(DEV)
    v = rows.flip(2).to(dtype).to(DEV)
    slots = torch.tensor([bs * i for i in range(len(special))])
    want = _expected(kc, vc, sc, k, v, slots, bs)
    fp8.hip_fp8_cache_write(k, v, kc, vc, sc, slots.to(DEV), bs)
    _check(kc, vc, sc, want)
    # what is stored is a finite number of the row type, but for the NaN
    got, _ = fp8.gather_fp8_prefix_kv(kc, vc, sc, torch.arange(len(special), device=DEV)[None].t(),
                                      [1] * len(special), list(range(len(special))), bs, dtype)
    assert not torch.isinf(got).any()
    assert torch.isnan(got).any(2).any(1).tolist() == [not np.isfinite(x) for x in special]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bs,d,hq,hkv", [(16, 64, 14, 2), (32, 128, 4, 4), (256, 128, 6, 1)])
def test_rotation_on_the_way(bs, d, hq, hkv, dtype):
    """Rotated rows bit-identical to hip_rope_kv_cache_write's, and quantised
    exactly; the returned key covers skipped tokens too; tables wider than head_dim."""
    say("rope", bs, d, hq, hkv, dtype)
    seqs = [(0, 5), (40, 1), (9, 60)]
    t = sum(n for _, n in seqs)
    num_blocks = 16
    slots = _slots(seqs, bs, num_blocks, 5)
    slots[10] = -1
    positions = torch.cat([torch.arange(c, c + n) for c, n in seqs])
    g = torch.Generator().manual_seed(6)
    ang = torch.rand(80, d + 16, generator=g) * 6.28
    cos, sin = ang.cos().to(dtype).to(DEV), ang.sin().to(dtype).to(DEV)
    q, k, v = _rows(t, hq, hkv, d, dtype, 7)
    q0, k0 = gpu.hip_rope_kv_cache_write(q, k, None, positions.to(DEV), cos, sin)
    kc, vc, sc = fp8_util.random_pool(num_blocks, hkv, bs, d, 8, DEV)
    want = _expected(kc, vc, sc, fp8_util.rotated(k.cpu(), cos.cpu()[positions][:, :d], sin.cpu()[positions][:, :d]),
                     v, slots, bs)
    q1, k1 = fp8.hip_fp8_rope_kv_cache_write(q, k, v, positions.to(DEV), cos, sin, kc, vc, sc,
                                             slots.to(DEV), bs)
    _check(kc, vc, sc, want)
    assert torch.equal(bits(q0), bits(q1)) and torch.equal(bits(k0), bits(k1))
    # no query, no key back, sliced tables (another row stride), the plan given
    kc2, vc2, sc2 = fp8_util.random_pool(num_blocks, hkv, bs, d, 8, DEV)
    plan = fp8.plan_fp8_write(slots.to(DEV), bs, num_blocks, DEV, positions, 80)
    got = fp8.hip_fp8_rope_kv_cache_write(None, k, v, positions.to(DEV), cos[:, :d], sin[:, :d], kc2,
                                          vc2, sc2, slots.to(DEV), bs, return_key=False, plan=plan)
    assert got == (None, None)
    _check(kc2, vc2, sc2, want)


def test_no_tokens():
    kc, vc, sc = fp8_util.random_pool(2, 2, 16, 64, 0, DEV)
    before = kc.clone(), sc.clone()
    empty = torch.empty(0, 2, 64, dtype=torch.bfloat16, device=DEV)
    none = torch.empty(0, dtype=torch.int64, device=DEV)
    fp8.hip_fp8_cache_write(empty, empty, kc, vc, sc, none, 16)
    table = torch.ones(4, 64, dtype=torch.bfloat16, device=DEV)
    q, k = fp8.hip_fp8_rope_kv_cache_write(empty, empty, empty, none, table, table, kc, vc, sc, none, 16)
    assert q.shape == k.shape == (0, 2, 64)
    skipped = torch.full((5,), -1, device=DEV)
    rows = torch.ones(5, 2, 64, dtype=torch.bfloat16, device=DEV)
    fp8.hip_fp8_cache_write(rows, rows, kc, vc, sc, skipped, 16)
    torch.cuda.synchronize()
    assert torch.equal(kc.view(torch.uint8), before[0].view(torch.uint8)) and torch.equal(sc, before[1])


@pytest.mark.parametrize("t", [8, 3000])
def test_metadata_errors(t):
    """Both forms of the plan; nothing is written by a refused call."""
    bs, num_blocks = 16, 256
    kc, vc, sc = fp8_util.random_pool(num_blocks, 1, bs, 64, 0, DEV)
    before = kc.view(torch.uint8).clone()
    rows = torch.ones(t, 1, 64, dtype=torch.float16, device=DEV)
    slots = torch.arange(t)
    bad = slots.clone()
    bad[3], bad[5] = bs * num_blocks, -2
    with pytest.raises(IndexError, match="2 slot"):
        fp8.hip_fp8_cache_write(rows, rows, kc, vc, sc, bad.to(DEV), bs)
    dup = slots.clone()
    dup[7] = dup[2]
    with pytest.raises(AssertionError, match="Duplicate"):
        fp8.hip_fp8_cache_write(rows, rows, kc, vc, sc, dup.to(DEV), bs)
    pos = torch.arange(t)
    table = torch.ones(t - 1, 64, dtype=torch.float16, device=DEV)
    with pytest.raises(IndexError, match="1 position"):
        fp8.hip_fp8_rope_kv_cache_write(None, rows, rows, pos.to(DEV), table, table, kc, vc, sc,
                                        slots.to(DEV), bs)
    plan = fp8.plan_fp8_write(slots, bs, num_blocks, DEV)
    with pytest.raises(AssertionError, match="another step or pool"):
        fp8.hip_fp8_cache_write(rows[1:], rows[1:], kc, vc, sc, slots[1:].to(DEV), bs, plan=plan)
    with pytest.raises(AssertionError, match="dtype"):
        fp8.hip_fp8_cache_write(rows.float(), rows.float(), kc, vc, sc, slots.to(DEV), bs)
    with pytest.raises(AssertionError, match="positions were checked"):
        fp8.hip_fp8_rope_kv_cache_write(None, rows, rows, pos.to(DEV), table, table, kc, vc, sc,
                                        slots.to(DEV), bs, plan=plan)
    torch.cuda.synchronize()
    assert torch.equal(kc.view(torch.uint8), before)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bs,d,hkv,lens", [(16, 64, 2, [1, 0, 17, 300]), (256, 128, 3, [255, 257, 3]),
                                           (32, 64, 1, [5000])])
def test_gather(bs, d, hkv, lens, dtype):
    say("gather", bs, d, hkv, lens, dtype)
    need = [-(-n // bs) for n in lens]
    num_blocks = sum(need) + 2
    kc, vc, sc = fp8_util.random_pool(num_blocks, hkv, bs, d, 1, DEV)
    perm = torch.randperm(num_blocks, generator=torch.Generator().manual_seed(2)).tolist()
    table = torch.full((len(lens) + 1, max(need)), -1)
    for i, n in enumerate(need):
        table[i + 1, :n] = torch.tensor([perm.pop() for _ in range(n)], dtype=torch.int64)
    rows = [i + 1 for i in range(len(lens))]
    for bt in (table, table.to(DEV), table.to(torch.int32).to(DEV)):
        k, v = fp8.gather_fp8_prefix_kv(kc, vc, sc, bt, lens, rows, bs, dtype)
        torch.cuda.synchronize()
        for j, (got, codes) in enumerate(((k, kc), (v, vc))):
            val = fp8_util.values(codes, sc, j).transpose(1, 2)  # [blocks, bs, H, D]
            want = torch.cat([val[table[r, : -(-n // bs)]].flatten(0, 1)[:n] for r, n in zip(rows, lens)])
            assert torch.equal(got.cpu().double(), want)
    with pytest.raises(IndexError, match="insufficient"):
        fp8.gather_fp8_prefix_kv(kc, vc, sc, table, [n + bs for n in lens], rows, bs, dtype)
    with pytest.raises(IndexError, match="insufficient"):
        fp8.gather_fp8_prefix_kv(kc, vc, sc, table, [-1], [1], bs, dtype)
    k, _ = fp8.gather_fp8_prefix_kv(kc, vc, sc, table, [0], [1], bs, dtype)
    assert k.shape == (0, hkv, d)
