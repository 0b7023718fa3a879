"""The 8-bit cache through the backend: steps of prefill chunks and decode tokens, as
the runner mixes them, eager and captured; streams; plans used side by side."""

import types

import pytest
import torch

import fp8_util
from gpu_util import DEV, bits, say
from mini_vllm.attention import AttentionBackend
from mini_vllm.attention import paged_attention_fp8 as fp8
from mini_vllm.attention import paged_attention_gpu as gpu
from mini_vllm.model_runner.base import AttentionGroup, AttentionMetadata, ModelConfig

pytestmark = pytest.mark.gpu


def _backend(hq, hkv, d, dtype, num_blocks, bs, layers=2):
    cfg = ModelConfig(num_layers=layers, num_heads=hq, num_kv_heads=hkv, head_dim=d, dtype=dtype)
    be = AttentionBackend.create(cfg, backend="hip")
    pool = be.allocate_pool(layers, num_blocks, bs, hkv, d, dtype, DEV, cache_dtype=fp8.FP8_DTYPE)
    for t in pool.key_caches + pool.value_caches:
        t.view(torch.uint8).fill_(0x7F)  # (uninitialised memory may hold NaN)
    return be, pool


def _rope(d, dtype, n=4096):
    inv = 1.0 / (1e4 ** (torch.arange(0, d, 2, dtype=torch.float64) / d))
    ang = torch.arange(n, dtype=torch.float64)[:, None] * inv
    ang = torch.cat([ang, ang], dim=1)
    return types.SimpleNamespace(cos=ang.cos().to(dtype).to(DEV), sin=ang.sin().to(dtype).to(DEV))


def _meta(pre, dec, tables, bs):
    """Metadata of prefill chunks [(sequence, cached, new)] and decode rows
    [(sequence, cached)]: (metadata, slots, positions)."""
    groups, slots, positions = [], [], []
    for kind, rows in (("prefill_gpu", pre), ("decode_gpu", [(s, c, 1) for s, c in dec])):
        if not rows:
            continue
        before = torch.tensor([c for _, c, _ in rows], device=DEV)
        new = torch.tensor([n for _, _, n in rows], device=DEV)
        groups.append(AttentionGroup(list(range(len(rows))), kind, before, new, before + new))
        for s, c, n in rows:
            positions += range(c, c + n)
            slots += [int(tables[s, p // bs]) * bs + p % bs for p in range(c, c + n)]
    meta = AttentionMetadata(groups=groups, block_size=bs)
    if pre:
        meta.prefill_block_tables = tables[[s for s, _, _ in pre]].to(DEV)
    if dec:
        meta.decode_block_tables = tables[[s for s, _ in dec]].to(DEV)
    return meta, torch.tensor(slots, device=DEV), torch.tensor(positions, device=DEV)


class _Model:
    """The definition over the same steps, 64 bits on the CPU, one layer."""

    def __init__(self, num_blocks, hkv, bs, d, dtype):
        self.k = torch.zeros(num_blocks, hkv, bs, d, dtype=torch.float64).numpy()
        self.v, self.bs, self.dtype = self.k.copy(), bs, dtype
        self.sc = torch.zeros(2, num_blocks, hkv, dtype=torch.float64).numpy()

    def write(self, k, v, slots):
        fp8_util.append(self.k, self.sc[0], k.double().numpy(), slots.tolist(), self.bs, self.dtype)
        fp8_util.append(self.v, self.sc[1], v.double().numpy(), slots.tolist(), self.bs, self.dtype)

    def rows(self, j, table, n):
        c = torch.from_numpy((self.k, self.v)[j] * self.sc[j][:, :, None, None])
        return c[table[: -(-n // self.bs)]].transpose(1, 2).flatten(0, 1)[:n]


@pytest.mark.parametrize("hq,hkv,d,bs,dtype", [(14, 2, 64, 16, torch.bfloat16), (8, 2, 128, 32, torch.float16)])
def test_steps_through_the_backend(hq, hkv, d, bs, dtype):
    """Chunks of two prompts, then mixed steps, then decode steps by each of the
    backend's methods, over two layers: the pool exactly the definition's, the
    attention within its tolerance."""
    num_blocks, layers = 40, 2
    be, pool = _backend(hq, hkv, d, dtype, num_blocks, bs, layers)
    rope = _rope(d, dtype)
    perm = torch.randperm(num_blocks, generator=torch.Generator().manual_seed(1))
    tables = perm[: 3 * 12].view(3, 12)
    model = [_Model(num_blocks, hkv, bs, d, dtype) for _ in range(layers)]
    steps = [([(0, 0, 37), (1, 0, 5)], [], "rope"), ([(0, 37, 30)], [(1, 5)], "rope"),
             ([(2, 0, 50)], [(0, 67), (1, 6)], "rope"), ([], [(0, 68), (1, 7), (2, 50)], "calls"),
             ([], [(0, 69), (1, 8), (2, 51)], "write"), ([], [(0, 70), (1, 9), (2, 52)], "sublayer")]
    g = torch.Generator().manual_seed(2)
    for step, (pre, dec, form) in enumerate(steps):
        say("step", step, form)
        meta, slots, positions = _meta(pre, dec, tables, bs)
        t, p = slots.numel(), sum(n for _, _, n in pre)
        for layer in range(layers):
            size = 1.0 if step < 4 else 6.0  # (later tokens larger: blocks are rescaled)
            qkv = (torch.randn(t, (hq + 2 * hkv) * d, generator=g) * size).to(dtype).to(DEV)
            q = qkv[:, :hq * d].view(t, hq, d)
            k = qkv[:, hq * d:(hq + hkv) * d].view(t, hkv, d)
            v = qkv[:, (hq + hkv) * d:].view(t, hkv, d)
            pos = positions.cpu()
            kr, qr = k.cpu(), q.cpu()
            if form in ("rope", "sublayer"):
                kr, qr = (fp8_util.rotated(x.cpu(), rope.cos.cpu()[pos], rope.sin.cpu()[pos]) for x in (k, q))
            outs = []
            if form == "rope":
                q2, k2 = be.rope_write_kv_cache(layer, q, k, v, positions, rope, slots, return_key=True)
                assert torch.equal(bits(q2.cpu()), bits(qr)) and torch.equal(bits(k2.cpu()), bits(kr))
                if pre:
                    outs.append(be.prefill_attention(layer, q2[:p], k2[:p], v[:p], meta, pool))
                if dec:
                    outs.append(be.decode_attention(layer, q2[p:], meta, pool))
            elif form == "calls":
                be.write_kv_cache(layer, k, v, slots)
                outs.append(be.decode_attention(layer, q, meta, pool))
            elif form == "write":
                outs.append(be.decode_attention_with_write(layer, q, k, v, slots, meta, pool))
            else:
                outs.append(be.decode_attention_with_rope_write(layer, q, k, v, positions, rope, slots,
                                                                meta, pool))
            torch.cuda.synchronize()
            m = model[layer]
            m.write(kr, v.cpu(), slots.cpu())
            for j, c in enumerate((pool.key_caches[layer], pool.value_caches[layer])):
                assert torch.equal(pool.kv_scales[layer][:, :, j].cpu().double(), torch.from_numpy(m.sc[j]))
                for s, c_len, n in pre + [(s, c, 1) for s, c in dec]:
                    got = c.view(torch.uint8)[tables[s].to(DEV)].view(fp8.FP8_DTYPE).cpu().double()
                    want = torch.from_numpy((m.k, m.v)[j])[tables[s]]
                    held = c_len + n
                    assert torch.equal(got.transpose(1, 2).flatten(0, 1)[:held],
                                       want.transpose(1, 2).flatten(0, 1)[:held])
            out, at = torch.cat(outs).cpu().double(), 0
            for s, c, n in pre + [(s, c, 1) for s, c in dec]:
                is_dec = (s, c) in dec
                held = c + 1 if is_dec else c
                kk, vv = m.rows(0, tables[s], held), m.rows(1, tables[s], held)
                if not is_dec:  # the chunk's own keys are its 16-bit rows
                    kk = torch.cat([kk, kr[at:at + n].double()])
                    vv = torch.cat([vv, v[at:at + n].cpu().double()])
                want, tol = fp8_util.attend(qr[at:at + n].double(), kk, vv, c, dtype)
                assert ((out[at:at + n] - want).abs() <= tol).all(), (s, c, n)
                at += n


def test_captured_decode_step():
    """Append and decode of two layers captured once, replayed over steps with new
    tokens, lengths and slots in the same tensors: each replay equals the eager calls on
    a pool of their own; bad metadata is reported afterwards."""
    hq, hkv, d, bs, dtype, b, num_blocks = 14, 2, 64, 16, torch.bfloat16, 5, 60
    be, pool = _backend(hq, hkv, d, dtype, num_blocks, bs)
    be2, pool2 = _backend(hq, hkv, d, dtype, num_blocks, bs)
    rope = _rope(d, dtype)
    tables = torch.randperm(num_blocks, generator=torch.Generator().manual_seed(3))[:b * 10].view(b, 10)
    lens = [3, 17, 31, 64, 100]
    g = torch.Generator().manual_seed(4)
    rows = torch.randn(2, sum(lens), 2, hkv, d, generator=g).to(dtype).to(DEV)
    slots0 = torch.tensor([int(tables[s, p // bs]) * bs + p % bs for s in range(b) for p in range(lens[s])],
                          device=DEV)
    for bk in (be, be2):
        for layer in range(2):
            bk.write_kv_cache(layer, rows[layer, :, 0], rows[layer, :, 1], slots0)
    meta, slots, positions = _meta([], [(s, lens[s]) for s in range(b)], tables, bs)
    kv = meta.groups[0].kv_len_after
    qkv = torch.empty(2, b, (hq + 2 * hkv) * d, dtype=dtype, device=DEV)

    def split(x):
        return (x[:, :hq * d].view(b, hq, d), x[:, hq * d:(hq + hkv) * d].view(b, hkv, d),
                x[:, (hq + hkv) * d:].view(b, hkv, d))

    def step(bk, pl, m, sl, ps):
        return [bk.decode_attention_with_rope_write(i, *split(qkv[i]), ps, rope, sl, m, pl) for i in range(2)]

    def fill(n):
        qkv.copy_(torch.randn(qkv.shape, generator=g) * (1 + n))

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(be, pool, meta, slots, positions)  # warm-up: also the first step's append
    torch.cuda.current_stream().wait_stream(side)
    eager = step(be2, pool2, *_meta([], [(s, lens[s]) for s in range(b)], tables, bs))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(be, pool, meta, slots, positions)
    gid = gpu.last_capture_id()
    for n in range(1, 5):
        say("replay", n)
        cur = [x + n for x in lens]
        m2, sl, ps = _meta([], list(enumerate(cur)), tables, bs)
        fill(n)
        slots.copy_(sl)
        positions.copy_(ps)
        kv.copy_(m2.groups[0].kv_len_after)
        graph.replay()
        gpu.check_deferred(gid)
        eager = step(be2, pool2, m2, sl, ps)
        torch.cuda.synchronize()
        for layer in range(2):
            assert torch.equal(bits(outs[layer]), bits(eager[layer]))
            assert torch.equal(pool.kv_scales[layer], pool2.kv_scales[layer])
    kv[2] = 0
    graph.replay()
    with pytest.raises(ValueError, match="kv_len"):
        gpu.check_deferred(gid)
    kv[2] = 40
    slots[1] = slots[0]
    graph.replay()
    with pytest.raises(AssertionError, match="Duplicate"):
        gpu.check_deferred(gid)
    slots[1] = num_blocks * bs + 5
    graph.replay()
    with pytest.raises(IndexError, match="out of range"):
        gpu.check_deferred(gid)
    gpu.clear_deferred(gid)


def test_captured_prefill():
    """A captured chunk's prefill with its lengths on the device, replayed with other
    lengths, equals the eager call; a plan made before the capture too."""
    hq, hkv, d, bs, dtype, num_blocks = 14, 2, 64, 16, torch.float16, 64
    kc, vc, sc = fp8_util.random_pool(num_blocks, hkv, bs, d, 1, DEV)
    table = torch.randperm(num_blocks, generator=torch.Generator().manual_seed(3))[:40].view(2, 20).to(DEV)
    g = torch.Generator().manual_seed(4)
    q = torch.randn(96, hq, d, generator=g).to(dtype).to(DEV)
    k, v = (torch.randn(96, hkv, d, generator=g).to(dtype).to(DEV) for _ in range(2))
    cached, new = torch.tensor([50, 7], device=DEV), torch.tensor([60, 36], device=DEV)

    def call(c, n, **kw):
        return fp8.hip_fp8_prefill_attention(q, k, v, kc, vc, sc, table, [0, 1], c, n, bs, **kw)

    first = call(cached, new)
    plan = fp8.plan_fp8_prefill(table, [0, 1], cached, new, bs, num_blocks, hq, hkv, d, dtype, DEV)
    graph, planned = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(cached, new)
    gid = gpu.last_capture_id()
    with torch.cuda.graph(planned):
        out2 = call(cached, new, plan=plan)
    planned.replay()
    torch.cuda.synchronize()
    assert torch.equal(bits(out2), bits(first))
    for c, n in (([50, 7], [60, 36]), ([0, 300], [1, 95]), ([123, 16], [48, 48])):
        cached.copy_(torch.tensor(c))
        new.copy_(torch.tensor(n))
        graph.replay()
        gpu.check_deferred(gid)
        assert torch.equal(bits(out), bits(call(c, n))), (c, n)
    cached[1] = 321
    graph.replay()
    with pytest.raises(IndexError, match="insufficient"):
        gpu.check_deferred(gid)
    gpu.clear_deferred(gid)


def test_two_plans_on_two_streams():
    """Calls with plans of their own on two streams at once, pieces merged in each."""
    bs, hq, hkv, d, dtype = 16, 14, 2, 64, torch.bfloat16
    sets = []
    for i, n in enumerate((6000, 5001)):
        num_blocks = -(-n // bs)
        kc, vc, sc = fp8_util.random_pool(num_blocks, hkv, bs, d, i, DEV)
        bt, kv = torch.arange(num_blocks, device=DEV)[None], torch.tensor([n], device=DEV)
        q = torch.randn(1, hq, d, generator=torch.Generator().manual_seed(i)).to(dtype).to(DEV)
        plan = fp8.plan_fp8_decode(bt, kv, bs, num_blocks, DEV, d, hkv)
        assert plan.plan.max_parts > 1
        want = fp8.hip_fp8_decode_attention(q, kc, vc, sc, bt, kv, bs)
        sets.append((q, kc, vc, sc, bt, kv, plan, want, torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, (q, kc, vc, sc, bt, kv, plan, _, stream) in enumerate(sets):
            with torch.cuda.stream(stream):
                outs[i].append(fp8.hip_fp8_decode_attention(q, kc, vc, sc, bt, kv, bs, plan=plan))
    torch.cuda.synchronize()
    for i, s in enumerate(sets):
        assert all(torch.equal(bits(o), bits(s[7])) for o in outs[i])


def test_metadata_changed_in_place_is_planned_again():
    bs, hq, hkv, d, dtype, num_blocks = 16, 4, 2, 64, torch.bfloat16, 8
    kc, vc, sc = fp8_util.random_pool(num_blocks, hkv, bs, d, 1, DEV)
    kc2, vc2, sc2 = kc.clone(), vc.clone(), sc.clone()
    slots = torch.tensor([3, 20], device=DEV)
    k, v = (torch.randn(2, hkv, d, device=DEV).to(dtype) for _ in range(2))
    fp8.hip_fp8_cache_write(k, v, kc, vc, sc, slots, bs)
    slots.add_(32)
    fp8.hip_fp8_cache_write(k, v, kc, vc, sc, slots, bs)
    for s in ([3, 20], [35, 52]):
        fp8.hip_fp8_cache_write(k, v, kc2, vc2, sc2, torch.tensor(s, device=DEV), bs)
    torch.cuda.synchronize()
    assert torch.equal(kc.view(torch.uint8), kc2.view(torch.uint8)) and torch.equal(sc, sc2)
    gpu.invalidate_cached_metadata()
    bt, kv = torch.arange(8, device=DEV).view(2, 4), torch.tensor([30, 64], device=DEV)
    q = torch.randn(2, hq, d, device=DEV).to(dtype)
    fp8.hip_fp8_decode_attention(q, kc, vc, sc, bt, kv, bs)
    kv.copy_(torch.tensor([5, 6]))
    got = fp8.hip_fp8_decode_attention(q, kc, vc, sc, bt, kv, bs)
    want = fp8.hip_fp8_decode_attention(q, kc, vc, sc, bt.clone(), kv.clone(), bs)
    assert torch.equal(bits(got), bits(want))


def test_backend_refusals():
    cfg = ModelConfig(num_layers=1, num_heads=2, num_kv_heads=1, head_dim=64)
    be = AttentionBackend.create(cfg, backend="hip")
    for dtype, bs, cache in ((torch.float32, 16, fp8.FP8_DTYPE), (torch.bfloat16, 8, fp8.FP8_DTYPE),
                             (torch.bfloat16, 512, fp8.FP8_DTYPE), (torch.bfloat16, 16, torch.int8),
                             (torch.bfloat16, 16, torch.float16)):
        with pytest.raises(RuntimeError, match="not supported"):
            be.allocate_pool(1, 4, bs, 1, 64, dtype, DEV, cache_dtype=cache)
    pool = be.allocate_pool(1, 4, 16, 1, 64, torch.bfloat16, DEV, cache_dtype=torch.bfloat16)
    assert pool.kv_scales is None and pool.key_caches[0].dtype is torch.bfloat16


@pytest.mark.parametrize("form", ["plan", "step"])
def test_native_calls_equal_the_wrappers(form, monkeypatch):
    """Three layers of a step through the native calls and with them off: the same
    bits; what is not the plain case (strided K, another stream) is left to the
    wrapper and gives them too."""
    hq, hkv, d, bs, dtype, num_blocks = 14, 2, 64, 16, torch.bfloat16, 40
    tables = torch.randperm(num_blocks, generator=torch.Generator().manual_seed(1))[:24].view(2, 12)
    rope = _rope(d, dtype)
    meta, slots, positions = _meta([(0, 20, 50), (1, 0, 9)], [], tables, bs)
    bt, kv = tables.to(DEV), torch.tensor([70, 9], device=DEV)
    rows, cached, new = [0, 1], [20, 0], [50, 9]
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(59, h, d, generator=g).to(dtype).to(DEV) for h in (hq, hkv, hkv))
    odd = torch.empty(59, hkv, d + 4, dtype=dtype, device=DEV)[:, :, :d]
    odd.copy_(k)  # (rows that are not 16-byte aligned)
    results = []
    for native in (True, False):
        if not native:
            monkeypatch.setattr(fp8._hip, "native_fp8", None)
        assert (fp8._hip.native_fp8 is not None) == native
        kc, vc, sc = fp8_util.random_pool(num_blocks, hkv, bs, d, 1, DEV)
        plans = [None] * 4
        if form == "plan":
            plans = [fp8.plan_fp8_write(slots, bs, num_blocks, DEV, positions, rope.cos.shape[0]),
                     fp8.plan_fp8_decode(bt, kv, bs, num_blocks, DEV, d, hkv),
                     fp8.plan_fp8_prefill(bt, rows, cached, new, bs, num_blocks, hq, hkv, d, dtype, DEV),
                     fp8.plan_fp8_gather(bt, [70, 9], rows, bs, num_blocks, DEV)]
        outs = []
        for layer, (stream, key) in enumerate([(None, k), (None, k), (torch.cuda.Stream(), k), (None, odd)]):
            torch.cuda.synchronize()
            with torch.cuda.stream(stream) if stream else torch.cuda.stream(torch.cuda.current_stream()):
                qr, kr = fp8.hip_fp8_rope_kv_cache_write(q, key, v, positions, rope.cos, rope.sin, kc, vc, sc,
                                                         slots, bs, plan=plans[0])
                outs += [qr, kr, fp8.hip_fp8_prefill_attention(qr, kr, v, kc, vc, sc, bt, rows, cached, new,
                                                               bs, plan=plans[2])]
                outs.append(fp8.hip_fp8_decode_attention(qr[:2], kc, vc, sc, bt, kv, bs, plan=plans[1]))
                outs += fp8.gather_fp8_prefix_kv(kc, vc, sc, bt, [70, 9], rows, bs, dtype, plan=plans[3])
            torch.cuda.synchronize()
        results.append(outs)
        gpu.invalidate_cached_metadata()
    assert len(results[0]) == len(results[1]) == 24
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(*results))


def _decode_set(n, seed, hq=14, hkv=2, d=64, bs=16, dtype=torch.bfloat16):
    num_blocks = -(-n // bs)
    kc, vc, sc = fp8_util.random_pool(num_blocks, hkv, bs, d, seed, DEV)
    q = torch.randn(1, hq, d, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)
    return q, kc, vc, sc, torch.arange(num_blocks, device=DEV)[None], torch.tensor([n], device=DEV), bs


def test_one_steps_calls_on_two_streams():
    """Two layers of a step on a stream each, at once, without a plan given: neither
    merges in the other's workspace."""
    layers = [list(_decode_set(6000, i)) for i in range(2)]
    layers[1][4:6] = layers[0][4:6]  # the step's table and lengths
    want = []
    for layer in layers:
        gpu.invalidate_cached_metadata()
        want.append(fp8.hip_fp8_decode_attention(*layer))
    streams = [torch.cuda.Stream() for _ in layers]
    torch.cuda.synchronize()
    gpu.invalidate_cached_metadata()
    outs = [[], []]
    for i, stream in enumerate(streams):
        with torch.cuda.stream(stream):
            for _ in range(20):
                outs[i].append(fp8.hip_fp8_decode_attention(*layers[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(bits(o), bits(want[i])) for o in outs[i])


def test_plan_first_used_on_another_stream():
    layer = _decode_set(6000, 3)
    want = fp8.hip_fp8_decode_attention(*layer)
    kc, bt, kv, bs = layer[1], *layer[4:]
    plan = fp8.plan_fp8_decode(bt, kv, bs, kc.shape[0], DEV, kc.shape[3], kc.shape[1])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        first = fp8.hip_fp8_decode_attention(*layer, plan=plan)
    torch.cuda.current_stream().wait_stream(side)
    second = fp8.hip_fp8_decode_attention(*layer, plan=plan)
    del plan  # (its memory waits for the calls)
    with torch.cuda.stream(side):
        junk = [torch.full((1 << 20,), 7, dtype=torch.uint8, device=DEV) for _ in range(4)]
    torch.cuda.synchronize()
    assert torch.equal(bits(first), bits(want)) and torch.equal(bits(second), bits(want)), len(junk)


def test_plan_of_a_capture_serves_it_only():
    layer = _decode_set(300, 5)
    kc, vc, sc, bt, kv, bs = layer[1:]
    nb, hkv, _, d = kc.shape
    slots = torch.tensor([16, 17], device=DEV)
    k, v = (torch.randn(2, hkv, d, device=DEV).to(torch.bfloat16) for _ in range(2))
    pool = [x.clone() for x in (kc, vc, sc)]
    fp8.hip_fp8_cache_write(k, v, *pool, slots, bs)
    want = fp8.hip_fp8_decode_attention(layer[0], *pool, bt, kv, bs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        write = fp8.plan_fp8_write(slots, bs, nb, DEV)
        decode = fp8.plan_fp8_decode(bt, kv, bs, nb, DEV, d, hkv)
        fp8.hip_fp8_cache_write(k, v, kc, vc, sc, slots, bs, plan=write)
        out = fp8.hip_fp8_decode_attention(*layer, plan=decode)
    gid = gpu.last_capture_id()
    with pytest.raises(RuntimeError, match="that capture only"):
        fp8.hip_fp8_cache_write(k, v, kc, vc, sc, slots, bs, plan=write)
    with pytest.raises(RuntimeError, match="that capture only"):
        fp8.hip_fp8_decode_attention(*layer, plan=decode)
    for _ in range(3):
        graph.replay()
        gpu.check_deferred(gid)
        assert torch.equal(bits(out), bits(want))
    gpu.clear_deferred(gid)


def test_pools_past_4_gib():
    """Blocks whose offsets pass 32 bits: every call equals the same one on a small pool."""
    hq, hkv, d, bs, dtype = 4, 2, 128, 16, torch.bfloat16
    num_blocks = (5 << 30) // (hkv * bs * d)
    far = [num_blocks - 1, 3, (4 << 30) // (hkv * bs * d), num_blocks - 2, (2 << 30) // (hkv * bs * d) + 1]
    g = torch.Generator().manual_seed(1)
    n, new = 70, 9
    k, v = (torch.randn(n, hkv, d, generator=g).to(dtype).to(DEV) for _ in range(2))
    q = torch.randn(new, hq, d, generator=g).to(dtype).to(DEV)
    got = []
    for blocks, count in ((list(range(5)), 5), (far, num_blocks)):
        kc, vc = (torch.zeros(count, hkv, bs, d, dtype=torch.uint8, device=DEV).view(fp8.FP8_DTYPE) for _ in range(2))
        sc = torch.zeros(count, hkv, 2, device=DEV)
        table = torch.tensor([blocks], device=DEV)
        slots = torch.tensor([blocks[p // bs] * bs + p % bs for p in range(n)], device=DEV)
        fp8.hip_fp8_cache_write(k, v, kc, vc, sc, slots, bs)
        fp8.hip_fp8_cache_write(3 * k[-2:], v[-2:], kc, vc, sc, slots[-2:], bs)
        res = [fp8.hip_fp8_decode_attention(q[:1], kc, vc, sc, table, torch.tensor([n], device=DEV), bs),
               fp8.hip_fp8_prefill_attention(q, k[:new], v[:new], kc, vc, sc, table, [0], [n], [new], bs),
               *fp8.gather_fp8_prefix_kv(kc, vc, sc, table, [n], [0], bs, dtype)]
        at = torch.tensor(blocks, device=DEV)
        res += [kc.view(torch.uint8)[at], vc.view(torch.uint8)[at], sc[at]]
        assert (sc[at] > 0).all()
        torch.cuda.synchronize()
        got.append([r.cpu() for r in res])
        del kc, vc, sc
    for x, y in zip(*got):
        assert torch.equal(x, y)


def test_a_plan_keeps_its_own_metadata():
    """Metadata tensors that change after an eager plan was made do not change its calls."""
    hq, hkv, d, bs, dtype, nb = 14, 2, 64, 16, torch.bfloat16, 8
    rope = _rope(d, dtype, 64)
    kc, vc, sc = fp8_util.random_pool(nb, hkv, bs, d, 1, DEV)
    g = torch.Generator().manual_seed(2)
    q = torch.randn(3, hq, d, generator=g).to(dtype).to(DEV)
    k, v = (torch.randn(3, hkv, d, generator=g).to(dtype).to(DEV) for _ in range(2))
    slots, positions = torch.tensor([40, 41, 42], device=DEV), torch.tensor([8, 9, 10], device=DEV)
    table, kv = torch.tensor([[2, 5]], device=DEV), torch.tensor([27], device=DEV)
    plans = (fp8.plan_fp8_write(slots, bs, nb, DEV, positions, 64),
             fp8.plan_fp8_decode(table, kv, bs, nb, DEV, d, hkv),
             fp8.plan_fp8_prefill(table, [0], [24], [3], bs, nb, hq, hkv, d, dtype, DEV),
             fp8.plan_fp8_gather(table, [27], [0], bs, nb, DEV))

    def run(write=None, decode=None, prefill=None, gather=None):
        pool = [x.clone() for x in (kc, vc, sc)]
        qr, kr = fp8.hip_fp8_rope_kv_cache_write(q, k, v, positions, rope.cos, rope.sin, *pool, slots, bs,
                                                 plan=write)
        return [pool[0].view(torch.uint8), pool[1].view(torch.uint8), pool[2], qr, kr,
                fp8.hip_fp8_decode_attention(q[:1], *pool, table, kv, bs, plan=decode),
                fp8.hip_fp8_prefill_attention(qr, kr, v, *pool, table, [0], [24], [3], bs, plan=prefill),
                *fp8.gather_fp8_prefix_kv(*pool, table, [27], [0], bs, dtype, plan=gather)]

    want = run()
    for t, x in ((slots, [7, 8, 9]), (positions, [60, 61, 62]), (table, [[6, 7]]), (kv, [3])):
        t.copy_(torch.tensor(x))
    got = run(*plans)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("t", [70, 3000])
def test_captured_append_of_a_prompt(t):
    """An append captured once (its plan in one launch or four), replayed with other
    slots and rows, eager work between the replays."""
    hkv, d, bs, dtype, nb = 2, 64, 32, torch.bfloat16, 128
    g = torch.Generator().manual_seed(t)
    kc, vc, sc = fp8_util.random_pool(nb, hkv, bs, d, 1, DEV)
    slots = torch.arange(t, device=DEV) + 5
    k, v = (torch.empty(t, hkv, d, dtype=dtype, device=DEV) for _ in range(2))

    def fill():
        for x in (k, v):
            x.copy_(torch.randn(x.shape, generator=g) * 3)

    fill()
    own = [x.clone() for x in (kc, vc, sc)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fp8.hip_fp8_cache_write(k, v, kc, vc, sc, slots, bs)
    gid = gpu.last_capture_id()
    for n in range(4):
        fill()
        order = torch.randperm(nb * bs, generator=g)[:t] if n % 2 else torch.arange(t) + 32 * n + n
        slots.copy_(order)
        slots[t // 2] = -1
        graph.replay()
        gpu.check_deferred(gid)
        fp8.hip_fp8_cache_write(k, v, *own, slots.clone(), bs)
        torch.cuda.synchronize()
        for a, b in zip((kc, vc), own):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        assert torch.equal(sc, own[2])
    gpu.clear_deferred(gid)
