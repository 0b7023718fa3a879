"""The 8-bit cache's decode plan: every token of every (sequence, kv head) in exactly
one piece, the pieces' block ids, the launch's bounds; and its choices where
they are plain."""

import random

import pytest
import torch

from gpu_util import DEV, say
from mini_vllm.attention import _hip
from mini_vllm.attention import paged_attention_fp8 as fp8
from mini_vllm.attention import paged_attention_gpu as gpu

pytestmark = pytest.mark.gpu


def _batch(lens, bs, seed, extra_cols=0):
    need = [-(-n // bs) for n in lens]
    num_blocks = 4096
    g = torch.Generator().manual_seed(seed)
    table = torch.full((len(lens), max(max(need), 1) + extra_cols), -1)
    for i, n in enumerate(need):  # (blocks may be shared between sequences)
        table[i, :n] = torch.randint(0, num_blocks, (n,), generator=g)
    return table, num_blocks


def _check(plan, lens, table, bs, hkv, fixed=False):
    p = plan.plan
    work = p.work.view(-1, 8).cpu()
    stride = ((p.partition_tokens + bs - 1) // bs + 1 + 3) // 4 * 4
    ids = p.block_ids.cpu()
    seen = {}
    most = 0
    for slot in range(p.num_groups):
        b, h, piece, pieces, t0, t1 = work[slot, :6].tolist()
        if b < 0:
            assert fixed
            continue
        assert 0 <= b < len(lens) and 0 <= h < hkv and 0 <= piece < pieces <= p.max_parts
        assert t0 % 16 == 0 and t0 < t1 <= lens[b] and t1 - t0 <= p.partition_tokens
        assert t1 == lens[b] or t1 % 16 == 0
        seen.setdefault((b, h), []).append((piece, pieces, t0, t1))
        first, n = t0 // bs, (t1 - 1) // bs - t0 // bs + 1
        assert n <= stride
        if h == 0:
            assert torch.equal(ids[slot * stride:slot * stride + n].long(), table[b, first:first + n].long())
        most = max(most, t1 - t0)
    assert set(seen) == {(b, h) for b in range(len(lens)) if lens[b] > 0 for h in range(hkv)}
    for (b, h), pieces in seen.items():
        pieces.sort()
        assert [x[0] for x in pieces] == list(range(len(pieces))) and all(x[1] == len(pieces) for x in pieces)
        assert pieces[0][2] == 0 and pieces[-1][3] == lens[b]
        assert all(a[3] == c[2] for a, c in zip(pieces, pieces[1:]))
    assert not p.counters.any()
    return most


def _lens(kind, r):
    return {"one": [1], "short": [r.randint(1, 40) for _ in range(9)],
            "serving": [r.randint(128, 2048) for _ in range(64)],
            "long": [r.randint(8192, 32768) for _ in range(6)],
            "skewed": [20000] + [r.randint(1, 200) for _ in range(255)],
            "many": [r.randint(1, 900) for _ in range(900)],
            "crowd": [r.randint(1, 100) for _ in range(3000)],
            "equal": [1024] * 128}[kind]


@pytest.mark.parametrize("kind", ["one", "short", "serving", "long", "skewed", "many", "crowd", "equal"])
@pytest.mark.parametrize("bs,hkv,d", [(16, 2, 64), (64, 1, 128), (256, 3, 64)])
def test_plan_covers_every_token_once(kind, bs, hkv, d):
    r = random.Random(kind)
    lens = _lens(kind, r)
    say("plan", kind, bs, hkv)
    table, num_blocks = _batch(lens, bs, 1, extra_cols=3)
    for ints in (torch.int64, torch.int32):
        plan = fp8.plan_fp8_decode(table.to(ints).to(DEV), torch.tensor(lens, dtype=ints, device=DEV), bs,
                                   num_blocks, DEV, d, hkv)
        most = _check(plan, lens, table, bs, hkv)
        assert most <= plan.plan.partition_tokens < most + 16


def test_plan_cuts_where_it_pays():
    """Uncut where the launch is short or balanced as it is, cut where one sequence
    would outlast the rest."""
    def parts(lens, d=64, hkv=2):
        table, num_blocks = _batch(lens, 16, 1)
        p = fp8.plan_fp8_decode(table.to(DEV), torch.tensor(lens, device=DEV), 16, num_blocks, DEV, d, hkv)
        return p.plan.max_parts, p.plan.num_groups

    assert parts([512] * 64) == (1, 128)
    assert parts([1024] * 128) == (1, 256)
    assert parts([700]) == (1, 2)
    assert parts([20000])[0] > 8
    r = random.Random(0)
    assert parts([r.randint(512, 4096) for _ in range(128)], 128, 4)[0] == 1
    assert parts([6000] + [300] * 255)[0] > 1


def test_captured_plan_of_fixed_size():
    """The plan of a captured launch over changing lengths and tables: unused
    entries marked, lengths out of range left out and reported."""
    bs, hkv, d = 16, 2, 64
    table, num_blocks = _batch([2000] * 5, bs, 1)
    bt, kv = table.to(DEV), torch.tensor([2000] * 5, device=DEV)
    fp8.plan_fp8_decode(bt, kv, bs, num_blocks, DEV, d, hkv)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = fp8.plan_fp8_decode(bt, kv, bs, num_blocks, DEV, d, hkv)
    gid = gpu.last_capture_id()
    for lens in ([2000] * 5, [1, 1, 1, 1, 1], [1999, 5, 700, 16, 17]):
        kv.copy_(torch.tensor(lens))
        graph.replay()
        gpu.check_deferred(gid)
        _check(plan, lens, table, bs, hkv, fixed=True)
    kv.copy_(torch.tensor([5, 0, 3000, 8, -4]))
    graph.replay()
    with pytest.raises(ValueError, match="min=-4"):
        gpu.check_deferred(gid)
    _check(plan, [5, 0, 0, 8, 0], table, bs, hkv, fixed=True)
    kv.copy_(torch.tensor([5, 6, 7, 8, 9]))
    bt[2, 0] = num_blocks
    graph.replay()
    with pytest.raises(IndexError, match="1 entr"):
        gpu.check_deferred(gid)
    gpu.clear_deferred(gid)


def test_bounds_hold_for_any_length():
    """mv_fp8_decode_plan_bounds against the plans of random batches (the check of
    capacities is on the host: a plan that exceeded them would be refused)."""
    import ctypes

    lib = _hip.load()
    r = random.Random(5)
    for _ in range(12):
        n, bs, hkv = r.choice([1, 3, 40, 300]), r.choice([16, 32, 256]), r.choice([1, 2, 8])
        lens = [r.choice([1, r.randint(1, 6000), r.randint(1, 200)]) for _ in range(n)]
        table, num_blocks = _batch(lens, bs, 2)
        out = (ctypes.c_int64 * 4)()
        assert lib.mv_fp8_decode_plan_bounds(n, table.shape[1], bs, hkv, 256, 0, out) == 0
        plan = fp8.plan_fp8_decode(table.to(DEV), torch.tensor(lens, device=DEV), bs, num_blocks, DEV, 64, hkv)
        p = plan.plan
        stride = ((p.partition_tokens + bs - 1) // bs + 1 + 3) // 4 * 4
        assert p.num_groups <= out[0] and p.max_parts <= out[2] and p.num_groups * stride <= out[3]
        _check(plan, lens, table, bs, hkv)
