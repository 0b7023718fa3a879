"""Decode and prefill attention over the 8-bit cache: against 64-bit attention over
the values the codes stand for (tolerances derived in fp8_util.attend), and
prefill bit-identical to the 16-bit kernel over the dequantised pool."""

import pytest
import torch

import fp8_util
from gpu_util import DEV, bits, say
from mini_vllm.attention import paged_attention_fp8 as fp8
from mini_vllm.attention import paged_attention_gpu as gpu

pytestmark = pytest.mark.gpu


def _tables(lens, bs, seed, extra=3):
    need = [-(-n // bs) for n in lens]
    num_blocks = sum(need) + extra
    perm = torch.randperm(num_blocks, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lens), max(max(need), 1)), -1)
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor([perm.pop() for _ in range(n)], dtype=torch.int64)
    return table, num_blocks


def _poison(kc, vc, table, lens, bs):
    """NaN codes in every place that no sequence attends."""
    held = torch.zeros(kc.shape[0], bs, dtype=torch.bool)
    for row, n in zip(table, lens):
        for j in range(-(-n // bs)):
            held[row[j], : min(bs, n - j * bs)] = True
    dead = (~held)[:, None, :, None].expand(kc.shape).to(DEV)
    for c in (kc, vc):
        c.view(torch.uint8)[dead] = 0x7F


def _sequence(codes, scales, j, row, n, bs):
    """Tokens 0 .. n - 1 of a sequence, what their codes stand for: [n, H, D] on the CPU."""
    blocks = row[: -(-n // bs)].to(DEV)
    held = codes.view(torch.uint8)[blocks].view(fp8_util.FP8)
    return fp8_util.values(held, scales[blocks], j).transpose(1, 2).flatten(0, 1)[:n]


def _check_decode(out, q, kc, vc, sc, table, lens, bs, only=None):
    torch.cuda.synchronize()
    for b, n in enumerate(lens):
        if only is not None and b not in only:
            continue
        k = _sequence(kc, sc, 0, table[b], n, bs)
        v = _sequence(vc, sc, 1, table[b], n, bs)
        want, tol = fp8_util.attend(q[b:b + 1].cpu().double(), k, v, n - 1, q.dtype)
        err = (out[b:b + 1].cpu().double() - want).abs()
        assert (err <= tol).all(), (b, n, (err / tol).max().item())


DECODE = [
    # (lengths, block size, q heads, kv heads, head_dim, dtype)
    ([1], 16, 14, 2, 64, torch.bfloat16),
    ([1, 2, 15, 16, 17, 31, 33, 64, 65], 16, 14, 2, 64, torch.float16),
    ([1, 127, 128, 129, 700], 16, 28, 4, 128, torch.bfloat16),
    ([5, 300, 1000], 32, 8, 8, 64, torch.bfloat16),
    ([63, 64, 66, 2000], 64, 16, 1, 128, torch.float16),
    ([1, 129, 1100], 128, 9, 3, 64, torch.float16),
    ([255, 257, 3000, 12], 256, 6, 6, 128, torch.bfloat16),
    ([8000, 3], 16, 16, 1, 64, torch.bfloat16),         # a long one cut into many pieces
    ([9001], 256, 4, 1, 128, torch.float16),
    ([37 * i + 1 for i in range(150)], 16, 4, 2, 64, torch.bfloat16),
]


@pytest.mark.parametrize("i", range(len(DECODE)))
def test_decode(i):
    lens, bs, hq, hkv, d, dtype = DECODE[i]
    say("decode", i, lens[:6], bs, hq, hkv, d, dtype)
    table, num_blocks = _tables(lens, bs, i)
    kc, vc, sc = fp8_util.random_pool(num_blocks, hkv, bs, d, i, DEV)
    _poison(kc, vc, table, lens, bs)
    q = torch.randn(len(lens), hq, d, generator=torch.Generator().manual_seed(i)).to(dtype).to(DEV)
    for bt, kv in ((table.to(DEV), torch.tensor(lens, device=DEV)),
                   (table.to(torch.int32).to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV))):
        out = fp8.hip_fp8_decode_attention(q, kc, vc, sc, bt, kv, bs)
        _check_decode(out, q, kc, vc, sc, table, lens, bs, only=None if len(lens) < 20 else (0, 1, 70, 149))
    again = fp8.hip_fp8_decode_attention(q, kc, vc, sc, bt, kv, bs)
    assert torch.equal(bits(out), bits(again))


@pytest.mark.parametrize("bs,units,n", [(16, 700, 8170), (32, 520, 9000), (256, 520, 20000)])
def test_decode_pieces_longer_than_a_window(bs, units, n):
    """So many sequences that a piece is a whole sequence of more than 64 tiles per
    wave; they share their blocks."""
    say("window", bs, units, n)
    lens = [n - 13 * (i % 5) for i in range(units)]
    table, num_blocks = _tables([n], bs, 1)
    kc, vc, sc = fp8_util.random_pool(num_blocks, 1, bs, 64, 1, DEV)
    rows = table.expand(units, -1).contiguous()
    q = torch.randn(units, 5, 64, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(DEV)
    plan = fp8.plan_fp8_decode(rows.to(DEV), torch.tensor(lens, device=DEV), bs, num_blocks, DEV, 64, 1)
    assert plan.plan.partition_tokens > 64 * 64, plan.plan.partition_tokens
    out = fp8.hip_fp8_decode_attention(q, kc, vc, sc, rows.to(DEV), torch.tensor(lens, device=DEV), bs,
                                       plan=plan)
    _check_decode(out, q, kc, vc, sc, rows, lens, bs, only=(0, 3, units - 1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["sharp", "late", "below"])
def test_decode_moving_reference(kind, dtype):
    """Scores that force the reference to move: far apart, one late key far above the
    rest, all far below zero."""
    say("reference", kind, dtype)
    lens, bs, hq, hkv, d = [700, 77], 16, 8, 2, 64
    table, num_blocks = _tables(lens, bs, 4)
    g = torch.Generator().manual_seed(5)
    q = torch.randn(2, hq, d, generator=g) * (8.0 if kind == "sharp" else 1.0)
    q = q.to(dtype).to(DEV)
    kc, vc, sc = fp8_util.random_pool(num_blocks, hkv, bs, d, 5, DEV)
    if kind != "sharp":
        # every key a multiple of one direction (per kv head), the last one far along it
        u = q.view(2, hkv, hq // hkv, d).float().mean(2)
        for b in range(2):
            for p in range(lens[b]):
                blk, o = table[b, p // bs], p % bs
                mult = -40.0 if kind == "below" else (60.0 if p == lens[b] - 2 else 0.5)
                row = (u[b] / u[b].norm(dim=1, keepdim=True) * mult).clamp(-400, 400)
                kc[blk, :, o] = row.to(fp8_util.FP8)
        sc[:, :, 0] = 1.0
    out = fp8.hip_fp8_decode_attention(q, kc, vc, sc, table.to(DEV), torch.tensor(lens, device=DEV), bs)
    _check_decode(out, q, kc, vc, sc, table, lens, bs)


def test_decode_scales_far_apart():
    """Blocks whose V scales differ by 2^40, and extreme scales of the format."""
    lens, bs, hq, hkv, d = [200], 16, 4, 1, 64
    table, num_blocks = _tables(lens, bs, 4)
    for dtype, exps in ((torch.bfloat16, (-100, -60, 0, 3)), (torch.float16, (-20, -9, 0, 4))):
        say("scales", dtype)
        kc, vc, sc = fp8_util.random_pool(num_blocks, hkv, bs, d, 6, DEV)
        for i in range(num_blocks):
            sc[i, :, 1] = 2.0 ** exps[i % len(exps)]
        q = torch.randn(1, hq, d, generator=torch.Generator().manual_seed(7)).to(dtype).to(DEV)
        out = fp8.hip_fp8_decode_attention(q, kc, vc, sc, table.to(DEV), torch.tensor(lens, device=DEV), bs)
        _check_decode(out, q, kc, vc, sc, table, lens, bs)


def test_decode_strided_query_and_errors():
    lens, bs, hq, hkv, d = [33, 50], 16, 4, 2, 64
    table, num_blocks = _tables(lens, bs, 4)
    kc, vc, sc = fp8_util.random_pool(num_blocks, hkv, bs, d, 6, DEV)
    bt, kv = table.to(DEV), torch.tensor(lens, device=DEV)
    wide = torch.randn(2, hq + 3, d, generator=torch.Generator().manual_seed(7)).to(torch.bfloat16).to(DEV)
    for q in (wide[:, 1:1 + hq], wide[:, :hq].transpose(0, 1).contiguous().transpose(0, 1)):
        out = fp8.hip_fp8_decode_attention(q, kc, vc, sc, bt, kv, bs)
        assert out.is_contiguous()
        _check_decode(out, q, kc, vc, sc, table, lens, bs)
    q = wide[:, :hq]
    with pytest.raises(ValueError, match="kv_len"):
        fp8.hip_fp8_decode_attention(q, kc, vc, sc, bt, torch.tensor([33, 0], device=DEV), bs)
    with pytest.raises(IndexError, match="insufficient"):
        fp8.hip_fp8_decode_attention(q, kc, vc, sc, bt, torch.tensor([33, 500], device=DEV), bs)
    with pytest.raises(IndexError, match="not pool blocks"):
        fp8.hip_fp8_decode_attention(q, kc, vc, sc, bt + num_blocks, kv, bs)
    with pytest.raises(AssertionError, match="dtype"):
        fp8.hip_fp8_decode_attention(q.float(), kc, vc, sc, bt, kv, bs)
    with pytest.raises(AssertionError, match="divisible"):
        fp8.hip_fp8_decode_attention(wide[:, :3], kc, vc, sc, bt, kv, bs)
    plan = fp8.plan_fp8_decode(bt, kv, bs, num_blocks, DEV, d, hkv)
    with pytest.raises(AssertionError, match="another step or pool"):
        fp8.hip_fp8_decode_attention(q[:1], kc, vc, sc, bt[:1], kv[:1], bs, plan=plan)
    none = fp8.hip_fp8_decode_attention(q[:0], kc, vc, sc, bt[:0], kv[:0], bs)
    assert none.shape == (0, hq, d)


# ------------------------------------------------------------- prefill ----

PREFILL = [
    # (chunks (cached, new), block size, q heads, kv heads, head_dim, dtype)
    ([(0, 1)], 16, 14, 2, 64, torch.bfloat16),
    ([(1, 1), (16, 1), (15, 3), (17, 40)], 16, 14, 2, 64, torch.float16),
    ([(37, 50), (0, 9), (130, 70)], 16, 28, 4, 128, torch.bfloat16),
    ([(1536, 512)] * 2, 16, 14, 2, 64, torch.bfloat16),
    ([(700, 300), (5, 700)], 32, 28, 4, 128, torch.float16),
    ([(3001, 200)], 64, 8, 8, 64, torch.bfloat16),          # keys cut into parts
    ([(2050, 130), (256, 1)], 256, 16, 1, 128, torch.bfloat16),
    ([(1000, 500)] * 12, 16, 14, 2, 64, torch.float16),     # 256 rows per work group
    ([(900, 504)] * 7, 128, 28, 4, 128, torch.bfloat16),    # the same at head_dim 128
    ([(33000, 40)], 16, 4, 1, 64, torch.bfloat16),          # prefix ids in two windows
]


def _prefill_inputs(i):
    seqs, bs, hq, hkv, d, dtype = PREFILL[i]
    cached = [c for c, _ in seqs]
    table, num_blocks = _tables(cached, bs, i)
    kc, vc, sc = fp8_util.random_pool(num_blocks, hkv, bs, d, i, DEV)
    _poison(kc, vc, table, cached, bs)
    t = sum(n for _, n in seqs)
    g = torch.Generator().manual_seed(i + 50)
    qkv = torch.randn(t + 2, (hq + 2 * hkv) * d, generator=g).to(dtype).to(DEV)
    q = qkv[:, :hq * d].view(t + 2, hq, d)
    k = qkv[:, hq * d:(hq + hkv) * d].view(t + 2, hkv, d)
    v = qkv[:, (hq + hkv) * d:].view(t + 2, hkv, d)
    return table, num_blocks, kc, vc, sc, q, k, v


@pytest.mark.parametrize("i", range(len(PREFILL)))
def test_prefill(i):
    seqs, bs, hq, hkv, d, dtype = PREFILL[i]
    say("prefill", i, seqs[:4], bs, hq, hkv, d, dtype)
    table, num_blocks, kc, vc, sc, q, k, v = _prefill_inputs(i)
    cached, new = [c for c, _ in seqs], [n for _, n in seqs]
    rows = list(range(len(seqs)))
    out = fp8.hip_fp8_prefill_attention(q, k, v, kc, vc, sc, table.to(DEV), rows, cached, new, bs)
    assert out.shape == (sum(new), hq, d)
    # the 16-bit kernel over the values the codes stand for: the same bits
    pool = [(c.float() * sc[:, :, j, None, None]).to(dtype) for j, c in enumerate((kc, vc))]
    same = gpu.hip_prefill_attention(q, k, v, *pool, table.to(DEV), rows, cached, new, bs)
    assert torch.equal(bits(out), bits(same))
    torch.cuda.synchronize()
    start = 0
    for b, (c, n) in enumerate(seqs[:3]):
        kk = torch.cat([_sequence(kc, sc, 0, table[b], c, bs), k[start:start + n].cpu().double()])
        vv = torch.cat([_sequence(vc, sc, 1, table[b], c, bs), v[start:start + n].cpu().double()])
        picks = sorted({0, n // 3, n - 1})
        for r in picks:
            want, tol = fp8_util.attend(q[start + r:start + r + 1].cpu().double(), kk[:c + r + 1],
                                        vv[:c + r + 1], c + r, dtype)
            err = (out[start + r:start + r + 1].cpu().double() - want).abs()
            assert (err <= tol).all(), (b, r, (err / tol).max().item())
        start += n
    plan = fp8.plan_fp8_prefill(table.to(DEV), rows, cached, new, bs, num_blocks, hq, hkv, d, dtype, DEV)
    again = fp8.hip_fp8_prefill_attention(q, k, v, kc, vc, sc, table.to(DEV), rows, cached, new, bs,
                                          plan=plan)
    assert torch.equal(bits(out), bits(again))


@pytest.mark.parametrize("bs,hq,hkv,d,new", [(16, 14, 2, 64, 2), (16, 14, 2, 64, 37), (32, 7, 1, 128, 2),
                                             (64, 14, 2, 128, 37)])
def test_prefill_every_prefix_end(bs, hq, hkv, d, new):
    """Prefixes that end at every place of two stages of keys: the bits of the 16-bit
    kernel over the values the codes stand for, few sequences at a time and all at once."""
    dtype = torch.bfloat16
    cached = list(range(0, 260, 1 if new == 2 else 3))
    table, num_blocks = _tables(cached, bs, d)
    kc, vc, sc = fp8_util.random_pool(num_blocks, hkv, bs, d, new, DEV)
    _poison(kc, vc, table, cached, bs)
    pool = [(c.float() * sc[:, :, j, None, None]).to(dtype) for j, c in enumerate((kc, vc))]
    g = torch.Generator().manual_seed(d + new)
    t = len(cached) * new
    q = torch.randn(t, hq, d, generator=g).to(dtype).to(DEV)
    k, v = (torch.randn(t, hkv, d, generator=g).to(dtype).to(DEV) for _ in range(2))
    table = table.to(DEV)
    for first, count in ((0, len(cached)), (5, 40), (60, 25)):
        rows, lens = list(range(first, first + count)), cached[first:first + count]
        part = slice(first * new, (first + count) * new)
        got = fp8.hip_fp8_prefill_attention(q[part], k[part], v[part], kc, vc, sc, table, rows, lens,
                                            [new] * count, bs)
        want = gpu.hip_prefill_attention(q[part], k[part], v[part], *pool, table, rows, lens, [new] * count, bs)
        assert not torch.isnan(got).any() and torch.equal(bits(got), bits(want)), (first, count)


def test_prefill_errors():
    table, num_blocks, kc, vc, sc, q, k, v = _prefill_inputs(1)
    seqs, bs, hq, hkv, d, dtype = PREFILL[1]
    cached, new = [c for c, _ in seqs], [n for _, n in seqs]
    rows = list(range(len(seqs)))

    def call(cached=cached, new=new, table=table, q=q, k=k, v=v, **kw):
        return fp8.hip_fp8_prefill_attention(q, k, v, kc, vc, sc, table.to(DEV), rows, cached, new, bs, **kw)

    with pytest.raises(IndexError, match="insufficient"):
        call(cached=[c + 64 for c in cached])
    with pytest.raises(IndexError, match="insufficient"):
        call(cached=[-1, 1, 1, 1])
    with pytest.raises(IndexError, match="insufficient"):
        call(table=table + num_blocks)
    with pytest.raises(AssertionError, match="chunk tokens"):
        call(new=[n + 100 for n in new])
    with pytest.raises(AssertionError, match="dtype"):
        call(q=q.float(), k=k.float(), v=v.float())
    plan = fp8.plan_fp8_prefill(table.to(DEV), rows, cached, new, bs, num_blocks, hq + hkv, hkv, d, dtype, DEV)
    with pytest.raises(AssertionError, match="another step or pool"):
        call(plan=plan)
    assert call(cached=[0] * 4, new=[0] * 4).shape == (0, hq, d)
