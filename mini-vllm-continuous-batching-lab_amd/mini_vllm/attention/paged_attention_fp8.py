"""The 8-bit KV cache on the HIP kernels: append, decode, prefill, gather.

The counterparts of ``paged_attention_gpu``'s entry points over pools of e4m3
codes (``torch.float8_e4m3fn``) with one scale per pool block and kv head, half
the bytes of a 16-bit pool:

* ``hip_fp8_cache_write`` (``hip_cache_write``)
* ``hip_fp8_rope_kv_cache_write`` (``hip_rope_kv_cache_write``)
* ``hip_fp8_decode_attention`` (``hip_decode_attention``)
* ``hip_fp8_prefill_attention`` (``hip_prefill_attention``)
* ``gather_fp8_prefix_kv`` (``gather_prefix_kv``)

``AttentionBackendGPU`` calls them for a pool allocated with
``cache_dtype=torch.float8_e4m3fn``. The reference's cache holds the model's type
only.

Format. ``key_cache`` and ``value_cache`` are ``[num_blocks, num_kv_heads,
block_size, head_dim]`` codes and ``kv_scales`` ``[num_blocks, num_kv_heads, 2]``
fp32 (K's, V's): an entry stands for ``code * scale``. A scale is a power of two
(2^-110 or more), 0 for a block never written, so a new pool's scales are zeroed.
What a code stands for is a number of the model's own 16-bit type. Rows are
fp16 or bf16, ``block_size`` a power of two from 16 to 256, ``head_dim`` 64 or
128; anything else is refused.

Plans. What the layers of a step share (the tokens' blocks, the work lists) is
planned once, checked on the device and read back (one synchronisation); the
plan keeps no reference to the metadata, which may change afterwards:
``plan_fp8_write``, ``plan_fp8_decode``, ``plan_fp8_prefill``,
``plan_fp8_gather``. The entry points take such a plan as ``plan``, made from the
same metadata; without one they make it, and find it again for the step's other
layers by their unmodified metadata tensors, as ``paged_attention_gpu`` does. A
plan may be used on any stream; a decode or prefill plan holds the workspace of
its merge, so calls with the same one have to be ordered among themselves (calls
with plans of their own, or without ``plan`` on different streams, need not be).
While a stream is being captured into a graph, a call without a plan records the
planning too, and its checks raise from ``check_deferred()``; a plan made outside
the graph has to outlive it, and one made inside serves that capture only.
"""

from __future__ import annotations

import contextlib
import ctypes
from dataclasses import dataclass, field
from typing import Optional, Sequence, Tuple

import torch

from . import _hip
from . import paged_attention_gpu as _gpu

FP8_DTYPE = torch.float8_e4m3fn
FP8_ROW_DTYPES = (torch.float16, torch.bfloat16)
FP8_BLOCK_SIZES = (16, 32, 64, 128, 256)

__all__ = [
    "FP8_DTYPE",
    "Fp8DecodePlan",
    "Fp8GatherPlan",
    "Fp8PrefillPlan",
    "Fp8WritePlan",
    "gather_fp8_prefix_kv",
    "hip_fp8_cache_write",
    "hip_fp8_decode_attention",
    "hip_fp8_prefill_attention",
    "hip_fp8_rope_kv_cache_write",
    "plan_fp8_decode",
    "plan_fp8_gather",
    "plan_fp8_prefill",
    "plan_fp8_write",
]


def _indexed(device: torch.device) -> torch.device:
    if device.index is None:
        return torch.device(device.type, torch.cuda.current_device())
    return device


def _on(device: torch.device):
    """The device as the current one (a launch goes to the current device)."""
    if torch.cuda.current_device() == device.index:
        return contextlib.nullcontext()
    return torch.cuda.device(device)


@dataclass
class _Plan:
    """What every plan keeps: its device, the buffers its calls read (complete
    when an eager plan is returned) and the stream they were allocated on."""

    device: torch.device
    buffers: Tuple[torch.Tensor, ...]
    stream: int = 0
    capture: int = 0
    words: Optional[bytes] = None  # for the native calls (on the plan's own stream)

    def _used(self, raw_stream: int) -> None:
        """The buffers' memory is not reused before this call is done, where it
        runs on another stream than theirs. (A graph keeps no plan alive.)"""
        if raw_stream != self.stream and not _gpu._capturing():
            current = torch.cuda.current_stream(self.device)
            for t in self.buffers:
                t.record_stream(current)

    def _check_capture(self) -> None:
        """A plan recorded into a graph holds nothing until that graph is replayed."""
        if self.capture and self.capture != _gpu._capture_id(self.device):
            raise RuntimeError("the plan was made inside a graph's capture: it serves that capture only")


def _seen_plan(name: str, *tensors):
    """The plan that an earlier layer of this eager step made for these, unmodified,
    metadata tensors, looked up natively (None: not known here)."""
    entry, lookup = getattr(_gpu._state, name, None), _hip.native
    if entry is None or lookup is None or not lookup.seen(entry[0].refs, entry[0].versions, *tensors):
        return None
    return None if _gpu._capturing() else entry[1]


def _check_pool(key_cache: torch.Tensor, value_cache: torch.Tensor, kv_scales: torch.Tensor,
                block_size: int, who: str) -> Tuple[int, int, int]:
    """(num_blocks, num_kv_heads, head_dim) of an 8-bit pool."""
    num_blocks, num_kv_heads, bs, head_dim = shape = key_cache.shape
    assert key_cache.dtype is FP8_DTYPE and value_cache.dtype is FP8_DTYPE, (
        f"{who}: caches {key_cache.dtype} / {value_cache.dtype}, expected {FP8_DTYPE}"
    )
    assert value_cache.shape == shape, f"{who}: key_cache {tuple(shape)} != {tuple(value_cache.shape)}"
    assert bs == block_size, f"block_size {block_size} != cache dim2 {bs}"
    assert block_size in FP8_BLOCK_SIZES, (
        f"{who}: block_size {block_size} not supported (a power of 2 from 16 to 256)"
    )
    assert head_dim in _gpu.SUPPORTED_HEAD_DIMS, f"head_dim {head_dim} not supported (only 64, 128)"
    assert kv_scales.dtype is torch.float32 and kv_scales.shape == (num_blocks, num_kv_heads, 2), (
        f"{who}: kv_scales {kv_scales.dtype} {tuple(kv_scales.shape)}, expected float32 "
        f"({num_blocks}, {num_kv_heads}, 2)"
    )
    assert key_cache.is_contiguous() and value_cache.is_contiguous() and kv_scales.is_contiguous(), (
        "cache must be contiguous"
    )
    device = key_cache.device
    assert device.type == "cuda", f"key_cache.device must be cuda, got {device}"
    assert value_cache.device == device and kv_scales.device == device
    return num_blocks, num_kv_heads, head_dim


def _check_rows(x: torch.Tensor, name: str, dtype: torch.dtype, device: torch.device) -> None:
    assert x.dtype is dtype and x.device == device, (
        f"{name} {x.dtype} on {x.device}, expected {dtype} on {device}"
    )


def _i64(x: torch.Tensor, device: torch.device) -> torch.Tensor:
    return x.to(device=device, dtype=torch.int64).contiguous()


# ============================================================================
# Append
# ============================================================================


@dataclass
class Fp8WritePlan(_Plan):
    """A step's new tokens by block (``mv_fp8_write_plan``)."""

    num_tokens: int = 0
    block_size: int = 0
    num_blocks: int = 0
    max_positions: int = 0                    # 0: positions not checked
    positions: Optional[torch.Tensor] = None  # on the device, int64
    max_items: int = 0                        # touched blocks (captured: their bound)


def plan_fp8_write(
    slot_mapping: torch.Tensor,
    block_size: int,
    num_blocks: int,
    device: torch.device,
    positions: Optional[torch.Tensor] = None,
    max_positions: int = 0,
) -> Fp8WritePlan:
    """Group a step's new tokens by the pool block of their slot and check them.

    ``slot_mapping`` ``[T]``: pool slots, -1 skips a token. With ``positions``
    ``[T]`` they are checked against rotary tables of ``max_positions`` rows.
    Raises ``IndexError`` for slots or positions out of range and
    ``AssertionError`` for duplicate slots, as ``hip_cache_write`` does; while a
    graph is being captured ``check_deferred()`` raises them.
    """
    device = _indexed(torch.device(device))
    assert block_size in FP8_BLOCK_SIZES, (
        f"block_size {block_size} not supported (a power of 2 from 16 to 256)"
    )
    n = slot_mapping.numel()
    assert slot_mapping.shape == (n,), f"slot_mapping {tuple(slot_mapping.shape)}"
    if positions is not None:
        assert positions.shape == (n,), f"positions {tuple(positions.shape)} != ({n},)"
        assert max_positions > 0
    lib = _hip.load()
    with _on(device):
        capture = _gpu._capture_id(device)
        slots = _i64(slot_mapping, device)
        pos = None if positions is None else _i64(positions, device)
        if pos is positions and pos is not None and not capture:
            pos = pos.clone()  # (the plan's own: the calls read it)
        ws_bytes = lib.mv_fp8_write_plan_workspace_bytes(n)
        # status, items, table and the hash table of large steps in one buffer
        words = _hip.MV_FP8_PLAN_WORDS + n
        words += -words % 4
        buf = torch.empty(words + n * block_size + ws_bytes // 4, dtype=torch.int32, device=device)
        base = buf.data_ptr()
        table_at = base + 4 * words
        _hip.check(
            lib.mv_fp8_write_plan(
                slots.data_ptr(), n, block_size, num_blocks, _gpu._ptr(pos), max_positions,
                base + 4 * _hip.MV_FP8_PLAN_WORDS, table_at, base,
                table_at + 4 * n * block_size if ws_bytes else None, ws_bytes, _gpu._stream(device),
            ),
            "mv_fp8_write_plan",
        )
        status = buf[:_hip.MV_FP8_PLAN_WORDS]
        plan = Fp8WritePlan(device, (buf, slots) if pos is None else (buf, slots, pos),
                            _gpu._stream(device), capture, num_tokens=n, block_size=block_size,
                            num_blocks=num_blocks, max_positions=max_positions if pos is not None else 0,
                            positions=pos, max_items=n)

        def raise_write(st) -> None:
            if st[_hip.MV_FP8_PLAN_OUT_OF_RANGE]:
                raise IndexError(
                    f"slot_mapping has {st[_hip.MV_FP8_PLAN_OUT_OF_RANGE]} slot(s) out of range "
                    f"[0, {num_blocks * block_size}) (-1 marks a skipped token)"
                )
            if st[_hip.MV_FP8_PLAN_REPEATED]:
                raise AssertionError(
                    f"Duplicate slots in slot_mapping: {st[_hip.MV_FP8_PLAN_REPEATED]} token(s) "
                    f"repeat another's slot. The HIP cache write forbids duplicate slots."
                )
            if st[_hip.MV_FP8_PLAN_POSITIONS]:
                raise IndexError(f"{st[_hip.MV_FP8_PLAN_POSITIONS]} position(s) outside the rotary "
                                 f"tables [0, {max_positions})")

        if capture:
            _gpu._defer(capture, raise_write, status)
        else:
            st = status.tolist()
            raise_write(st)
            plan.max_items = st[_hip.MV_FP8_PLAN_ITEMS]
        plan.words = _hip.fp8_write_words(
            base + 4 * _hip.MV_FP8_PLAN_WORDS, table_at, base, plan.max_items, _gpu._ptr(pos), n,
            block_size, num_blocks, plan.max_positions, device.index)
    return plan


def _write_plan(slot_mapping, block_size, num_blocks, device, positions, max_positions):
    """``plan_fp8_write``, found again for the step's other layers."""
    capture = _gpu._capture_id(device)
    name = "fp8_write_graph" if capture else "fp8_write"
    tensors = (slot_mapping,) if positions is None else (slot_mapping, positions)
    extra = (block_size, num_blocks, device, max_positions, capture)
    plan = _gpu._cache_get(name, tensors, extra)
    if plan is None:
        plan = plan_fp8_write(slot_mapping, block_size, num_blocks, device, positions, max_positions)
        _gpu._cache_put(name, tensors, extra, plan)
    return plan


def _append(who, query, key, value, positions, cos, sin, key_cache, value_cache, kv_scales,
            slot_mapping, block_size, return_key, plan):
    native = _hip.native_fp8
    known = plan
    if known is None:
        known = _seen_plan("fp8_write", *((slot_mapping,) if cos is None else (slot_mapping, positions)))
    if (known is not None and native is not None and not known.capture
            and slot_mapping.shape == (known.num_tokens,)):
        stream = _gpu._stream(known.device)
        if stream == known.stream and (cos is None or known.max_positions):
            done = native.write(known.words, query, key, value, cos, sin, key_cache, value_cache,
                                kv_scales, block_size, return_key, stream)
            if done is not None:
                if type(done) is int:
                    _hip.check(done, "mv_fp8_kv_cache_write")
                return done
    num_blocks, num_kv_heads, head_dim = _check_pool(key_cache, value_cache, kv_scales, block_size, who)
    device, dtype = key_cache.device, key.dtype
    num_tokens = key.shape[0]
    assert key.shape == (num_tokens, num_kv_heads, head_dim), (
        f"key {tuple(key.shape)} does not match cache {tuple(key_cache.shape)}"
    )
    assert key.shape == value.shape, f"key {key.shape} != value {value.shape}"
    assert slot_mapping.shape == (num_tokens,)
    assert dtype in FP8_ROW_DTYPES, f"dtype {dtype} not supported (fp16, bf16)"
    _check_rows(key, "key", dtype, device)
    _check_rows(value, "value", dtype, device)
    rope = cos is not None
    num_q_heads = max_pos = 0
    if rope:
        assert positions.shape == (num_tokens,), f"positions {tuple(positions.shape)} != ({num_tokens},)"
        assert cos.dim() == 2 and cos.shape == sin.shape and cos.shape[1] >= head_dim, (
            f"rotary tables {tuple(cos.shape)} / {tuple(sin.shape)} do not cover head_dim {head_dim}"
        )
        _check_rows(cos, "cos", dtype, device)
        _check_rows(sin, "sin", dtype, device)
        max_pos = cos.shape[0]
        if query is not None:
            assert query.dim() == 3 and query.shape[0] == num_tokens and query.shape[2] == head_dim, (
                f"query {tuple(query.shape)} does not match key {tuple(key.shape)}"
            )
            _check_rows(query, "query", dtype, device)
            num_q_heads = query.shape[1]
    with _on(device):
        if plan is None:
            plan = _write_plan(slot_mapping, block_size, num_blocks, device,
                               positions if rope else None, max_pos)
        assert (plan.num_tokens, plan.block_size, plan.num_blocks, plan.device) == (
            num_tokens, block_size, num_blocks, device), "the plan is of another step or pool"
        plan._check_capture()
        assert not rope or plan.max_positions == max_pos, (
            f"the plan's positions were checked against {plan.max_positions} rows, not {max_pos}"
        )
        q_out = k_out = None
        qp = qo = ko = 0
        q_st = q_sh = qo_st = qo_sh = ko_st = ko_sh = 0
        if query is not None:
            query, qp, q_st, q_sh = _gpu._row_args(query)
            q_out = torch.empty_like(query, memory_format=torch.contiguous_format)
            qo = q_out.data_ptr()
            qo_st, qo_sh, _ = q_out.stride()
        if return_key:
            k_out = torch.empty_like(key, memory_format=torch.contiguous_format)
            ko = k_out.data_ptr()
            ko_st, ko_sh, _ = k_out.stride()
        if num_tokens == 0:
            return q_out, k_out
        key, kp, k_st, k_sh = _gpu._row_args(key)
        value, vp, v_st, v_sh = _gpu._row_args(value)
        table_st = 0
        if rope:
            c_st, s_st = cos.stride(), sin.stride()
            if (c_st[1] != 1 or s_st[1] != 1 or c_st[0] != s_st[0] or c_st[0] % 8
                    or cos.data_ptr() % 16 or sin.data_ptr() % 16):
                cos, sin = cos[:, :head_dim].contiguous(), sin[:, :head_dim].contiguous()
            table_st = cos.stride(0)
        stream = _gpu._stream(device)
        plan._used(stream)
        base = plan.buffers[0].data_ptr()
        words = _hip.MV_FP8_PLAN_WORDS + num_tokens
        _hip.check(
            _hip.load().mv_fp8_kv_cache_write(
                qp or None, q_st, q_sh, qo or None, qo_st, qo_sh, kp, k_st, k_sh, ko or None, ko_st,
                ko_sh, vp, v_st, v_sh, key_cache.data_ptr(), value_cache.data_ptr(),
                kv_scales.data_ptr(), base + 4 * _hip.MV_FP8_PLAN_WORDS,
                base + 4 * (words + -words % 4), base, plan.max_items,
                plan.positions.data_ptr() if rope else None, cos.data_ptr() if rope else None,
                sin.data_ptr() if rope else None, table_st, max_pos, num_tokens, num_q_heads,
                num_kv_heads, head_dim, block_size, num_blocks, _hip.MV_DTYPE[dtype], stream,
            ),
            "mv_fp8_kv_cache_write",
        )
    return q_out, k_out


def hip_fp8_cache_write(
    key: torch.Tensor,
    value: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    kv_scales: torch.Tensor,
    slot_mapping: torch.Tensor,
    block_size: int,
    *,
    plan: Optional[Fp8WritePlan] = None,
) -> None:
    """Quantise a step's new K/V rows into one layer's 8-bit paged cache.

    ``key`` / ``value`` ``[T, num_kv_heads, head_dim]`` (fp16 or bf16, strided
    views without a copy) go to the slots of ``slot_mapping`` (-1 skips a token).
    For each block that gets a row, and each kv head of K and of V: the scale
    becomes the smallest power of two (2^-110 or more) that holds the call's
    finite values in the block as codes of at most 448, or stays what it was if
    that is larger; the rows' codes are ``x / scale`` rounded to nearest even. Where the
    scale grows, the block's other codes are scaled to it and rounded. A row at a
    block's first place starts the block anew: its old scale does not count, and
    places the call does not write hold nothing. Values that are not finite are stored
    as NaN (the code has no infinity); magnitudes over 61440 (fp16) or 240 *
    2^120 (bf16), whose code would stand for a value outside the type, as that.
    Errors as ``hip_cache_write``; ``plan``: ``plan_fp8_write`` of these slots.
    """
    _append("hip_fp8_cache_write", None, key, value, None, None, None, key_cache, value_cache,
            kv_scales, slot_mapping, block_size, False, plan)


def hip_fp8_rope_kv_cache_write(
    query: Optional[torch.Tensor],
    key: torch.Tensor,
    value: torch.Tensor,
    positions: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    kv_scales: torch.Tensor,
    slot_mapping: torch.Tensor,
    block_size: int,
    *,
    return_key: bool = True,
    plan: Optional[Fp8WritePlan] = None,
) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """``hip_rope_kv_cache_write`` into an 8-bit cache, in one launch: the query
    and the key rotated (bit-identical to it), the rotated key, as the 16-bit
    type holds it, and the value quantised (``hip_fp8_cache_write``).

    Returns ``(query_rot, key_rot)``, new tensors; ``query_rot`` is None without
    a query, ``key_rot`` None without ``return_key`` (a chunk's prefill attention
    reads it). ``plan``: ``plan_fp8_write`` of these slots and positions
    (``max_positions`` the tables' rows).
    """
    assert positions is not None and cos is not None and sin is not None
    return _append("hip_fp8_rope_kv_cache_write", query, key, value, positions, cos, sin, key_cache,
                   value_cache, kv_scales, slot_mapping, block_size, return_key, plan)


# ============================================================================
# Decode
# ============================================================================


@dataclass
class Fp8DecodePlan(_Plan):
    """A decode step's work list (``mv_fp8_decode_plan``) and its merge
    workspaces per query-head count."""

    plan: _gpu.DecodePlan = None
    key: tuple = ()  # (num_seqs, block_size, num_blocks, head_dim, num_kv_heads)
    owner: Optional[torch.cuda.Stream] = None  # `stream`
    workspaces: dict = field(default_factory=dict)

    def workspace(self, num_q_heads: int, head_dim: int) -> Optional[torch.Tensor]:
        if num_q_heads not in self.workspaces:
            n = _hip.load().mv_fp8_paged_decode_workspace_bytes(
                self.key[0], num_q_heads, head_dim, self.plan.max_parts)
            ws = torch.empty(n, dtype=torch.uint8, device=self.device) if n else None
            self.workspaces[num_q_heads] = ws
            if ws is not None:
                if _gpu._stream(self.device) != self.stream and not _gpu._capturing():
                    ws.record_stream(self.owner)  # (calls on the plan's stream do not)
                self.buffers += (ws,)
        return self.workspaces[num_q_heads]


def plan_fp8_decode(
    block_table: torch.Tensor,
    kv_len_after: torch.Tensor,
    block_size: int,
    num_blocks: int,
    device: torch.device,
    head_dim: int,
    num_kv_heads: int,
) -> Fp8DecodePlan:
    """The work list of a decode step over an 8-bit pool, with ``plan_decode``'s
    errors: ``ValueError`` for lengths below 1, ``IndexError`` for tables that do
    not cover them or hold something else than pool blocks."""
    device = _indexed(torch.device(device))
    assert block_size in FP8_BLOCK_SIZES, (
        f"block_size {block_size} not supported (a power of 2 from 16 to 256)"
    )
    assert head_dim in _gpu.SUPPORTED_HEAD_DIMS, f"head_dim {head_dim} not supported (only 64, 128)"
    assert block_table.dim() == 2 and block_table.shape[0] == kv_len_after.shape[0]
    lib = _hip.load()
    with _on(device):
        capture = _gpu._capture_id(device)
        bt, kv = _gpu._decode_metadata(block_table, kv_len_after, device)
        num_seqs, max_blocks = bt.shape
        cus = torch.cuda.get_device_properties(device).multi_processor_count
        bounds = (ctypes.c_int64 * 4)()
        _hip.check(lib.mv_fp8_decode_plan_bounds(num_seqs, max_blocks, block_size, num_kv_heads, cus,
                                                 int(bool(capture)), bounds),
                   "mv_fp8_decode_plan_bounds")
        cap, most_tokens, most_parts, n_ids = bounds
        # work list, block ids, counters and status words in one buffer, each part
        # 16-byte aligned
        n_work, n_ids = 8 * max(cap, 1), -(-max(n_ids, 4) // 4) * 4
        n_units = max(num_seqs * num_kv_heads, 1)
        n_cnt = -(-n_units // 4) * 4
        buf = torch.empty(n_work + n_ids + n_cnt + _hip.MV_PLAN_WORDS, dtype=torch.int32, device=device)
        base = buf.data_ptr()
        _hip.check(
            lib.mv_fp8_decode_plan(
                _gpu._ptr(kv), int(kv.dtype == torch.int64), bt.data_ptr() if bt.numel() else None,
                int(bt.dtype == torch.int64), bt.stride(0), num_seqs, max_blocks, block_size,
                num_blocks, num_kv_heads, head_dim, cus, int(bool(capture)), base, cap,
                base + 4 * n_work, n_ids, base + 4 * (n_work + n_ids),
                base + 4 * (n_work + n_ids + n_cnt), _gpu._stream(device),
            ),
            "mv_fp8_decode_plan",
        )
        status = buf[n_work + n_ids + n_cnt:]

        def raise_plan(st) -> None:
            if st[_hip.MV_PLAN_BAD_KV_LEN]:
                raise ValueError(
                    f"kv_len_after must be >= 1 for all decode sequences, "
                    f"got min={st[_hip.MV_PLAN_MIN_KV_LEN]}"
                )
            if st[_hip.MV_PLAN_INSUFFICIENT]:
                raise IndexError(
                    f"block_table with {max_blocks} blocks per row (block_size={block_size}) is "
                    f"insufficient to cover kv_len_after for {st[_hip.MV_PLAN_INSUFFICIENT]} "
                    f"sequence(s)"
                )
            if st[_hip.MV_PLAN_BAD_BLOCK]:
                raise IndexError(
                    f"block_table has {st[_hip.MV_PLAN_BAD_BLOCK]} entr(ies) within kv_len_after "
                    f"that are not pool blocks [0, {num_blocks})"
                )

        if capture:
            _gpu._defer(capture, raise_plan, status)
            groups, parts, tokens = cap, most_parts, most_tokens
        else:
            st = status.tolist()
            raise_plan(st)
            groups, parts, tokens = (st[_hip.MV_PLAN_NUM_ITEMS], st[_hip.MV_PLAN_MAX_PARTS],
                                     st[_hip.MV_PLAN_PARTITION_TOKENS])
        made = _gpu.DecodePlan(buf[:n_work], buf[n_work:n_work + n_ids],
                               buf[n_work + n_ids:n_work + n_ids + n_units], groups, parts, tokens)
        return Fp8DecodePlan(device, (buf,), _gpu._stream(device), capture, plan=made,
                             key=(num_seqs, block_size, num_blocks, head_dim, num_kv_heads),
                             owner=torch.cuda.current_stream(device))


def hip_fp8_decode_attention(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    kv_scales: torch.Tensor,
    block_table: torch.Tensor,
    kv_len_after: torch.Tensor,
    block_size: int,
    *,
    plan: Optional[Fp8DecodePlan] = None,
) -> torch.Tensor:
    """``hip_decode_attention`` over an 8-bit cache.

    ``query`` ``[B, num_q_heads, head_dim]`` (fp16 or bf16) attends the first
    ``kv_len_after[b]`` tokens of its row of ``block_table``; returns the same
    shape in the query's type. Products with K and V are those of the values the
    codes stand for; softmax statistics and sums are held in fp32, the weights
    rounded to the query's type for the product with V. Errors as there;
    ``plan``: ``plan_fp8_decode`` of this table and these lengths.
    """
    native = _hip.native_fp8
    known = plan if plan is not None else _seen_plan("fp8_decode", block_table, kv_len_after)
    if known is not None and native is not None and known.words is not None and not known.capture:
        stream = _gpu._stream(known.device)
        if stream == known.stream:
            output = native.decode(known.words, query, key_cache, value_cache, kv_scales, block_table,
                                   kv_len_after, block_size, stream)
            if output is not None:
                if type(output) is int:
                    _hip.check(output, "mv_fp8_paged_decode")
                return output
    num_blocks, num_kv_heads, head_dim = _check_pool(key_cache, value_cache, kv_scales, block_size,
                                                     "hip_fp8_decode_attention")
    num_seqs, num_q_heads, q_dim = query.shape
    device, dtype = key_cache.device, query.dtype
    assert q_dim == head_dim, f"query head_dim {q_dim} != cache {head_dim}"
    assert num_q_heads % num_kv_heads == 0, (
        f"num_q_heads {num_q_heads} not divisible by num_kv_heads {num_kv_heads}"
    )
    assert num_q_heads // num_kv_heads <= _gpu.MAX_QUERY_HEADS_PER_KV_HEAD, (
        f"{num_q_heads // num_kv_heads} query heads per kv head "
        f"(max {_gpu.MAX_QUERY_HEADS_PER_KV_HEAD})"
    )
    assert dtype in FP8_ROW_DTYPES, f"dtype {dtype} not supported (fp16, bf16)"
    _check_rows(query, "query", dtype, device)
    assert block_table.shape[0] == num_seqs
    assert kv_len_after.shape == (num_seqs,)
    with _on(device):
        output = torch.empty_like(query, memory_format=torch.contiguous_format)
        if num_seqs == 0:
            return output
        stream = _gpu._stream(device)
        if plan is None:
            capture = _gpu._capture_id(device)
            name = "fp8_decode_graph" if capture else "fp8_decode"
            extra = (block_size, num_blocks, device, head_dim, num_kv_heads, capture, stream)
            plan = _gpu._cache_get(name, (block_table, kv_len_after), extra)
            if plan is None:
                plan = plan_fp8_decode(block_table, kv_len_after, block_size, num_blocks, device,
                                       head_dim, num_kv_heads)
                _gpu._cache_put(name, (block_table, kv_len_after), extra, plan)
        assert plan.key == (num_seqs, block_size, num_blocks, head_dim, num_kv_heads) and (
            plan.device == device), "the plan is of another step or pool"
        plan._check_capture()
        p = plan.plan
        if p.num_groups == 0:
            return output
        plan._used(stream)
        ws = plan.workspace(num_q_heads, head_dim)
        query, qp, q_st, q_sh = _gpu._row_args(query)
        o_st, o_sh, _ = output.stride()
        split = (p.work.data_ptr(), p.block_ids.data_ptr(), p.block_ids.numel(), p.num_groups,
                 p.partition_tokens, p.max_parts, p.counters.data_ptr())
        shape = (float(head_dim ** -0.5), num_seqs, num_q_heads, num_kv_heads, head_dim, block_size,
                 num_blocks, _hip.MV_DTYPE[dtype])
        space = (_gpu._ptr(ws), ws.numel() if ws is not None else 0)
        _hip.check(
            _hip.load().mv_fp8_paged_decode(
                qp, q_st, q_sh, key_cache.data_ptr(), value_cache.data_ptr(), kv_scales.data_ptr(),
                *split, output.data_ptr(), o_st, o_sh, *shape, *space, stream,
            ),
            "mv_fp8_paged_decode",
        )
        # the step's other layers (the same query heads) launch from these words
        plan.words = _hip.fp8_decode_words(*split, *shape, *space, device.index)
    return output


# ============================================================================
# Prefill
# ============================================================================


@dataclass
class Fp8PrefillPlan(_Plan):
    """A step's prefill work list (``paged_attention_gpu``'s prefill plan)."""

    plan: tuple = ()
    num_seqs: int = 0
    total: int = 0
    key: tuple = ()  # (block_size, num_blocks, num_q_heads, num_kv_heads, head_dim, dtype)


def plan_fp8_prefill(
    block_table: torch.Tensor,
    seq_indices: Sequence[int],
    cached_len_before,
    query_len,
    block_size: int,
    num_blocks: int,
    num_q_heads: int,
    num_kv_heads: int,
    head_dim: int,
    dtype: torch.dtype,
    device: torch.device,
) -> Fp8PrefillPlan:
    """The work list of a step's chunks (``hip_fp8_prefill_attention``'s
    arguments of the same names). ``IndexError`` ("insufficient") for a table that
    cannot cover a prefix and for negative lengths. Not while a graph is being
    captured: there the attention call plans on the device."""
    device = _indexed(torch.device(device))
    assert block_size in FP8_BLOCK_SIZES, (
        f"block_size {block_size} not supported (a power of 2 from 16 to 256)"
    )
    assert head_dim in _gpu.SUPPORTED_HEAD_DIMS, f"head_dim {head_dim} not supported (only 64, 128)"
    assert dtype in FP8_ROW_DTYPES, f"dtype {dtype} not supported (fp16, bf16)"
    rows = [int(r) for r in seq_indices]
    with _on(device):
        if _gpu._capture_id(device):
            raise RuntimeError("plan_fp8_prefill: not while a graph is being captured "
                               "(hip_fp8_prefill_attention plans on the device there)")
        cached, qlens = _gpu._host_lengths(cached_len_before, query_len)
        assert len(rows) == len(cached) == len(qlens)
        if block_table.device == device:
            block_table = block_table.clone()  # (the plan's own: the calls read it)
        made = _gpu._prefill_plan_make(block_table, rows, cached, qlens, block_size, num_blocks,
                                       num_q_heads, num_kv_heads, head_dim, dtype, device)
        bt, meta, work, ws = made[0], made[1], made[2], made[7]
        torch.cuda.current_stream(device).synchronize()  # (complete, for whatever stream uses it)
        return Fp8PrefillPlan(
            device, tuple(t for t in (bt, meta, work, ws) if t is not None), _gpu._stream(device),
            words=made[8], plan=made, num_seqs=len(rows), total=sum(qlens),
            key=(block_size, num_blocks, num_q_heads, num_kv_heads, head_dim, dtype))


def _prefill_native(plan, query, key, value, key_cache, value_cache, kv_scales, block_size):
    """The call's checks and launch in native code (None: not the plain case)."""
    native = _hip.native_fp8
    stream = _gpu._stream(plan.device)
    if native is None or stream != plan.stream:
        return None
    out = native.prefill(plan.words, query, key, value, key_cache, value_cache, kv_scales, plan.total,
                         block_size, stream)
    if type(out) is int:
        _hip.check(out, "mv_fp8_paged_prefill")
    return out


def hip_fp8_prefill_attention(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    kv_scales: torch.Tensor,
    block_table: torch.Tensor,
    seq_indices: Sequence[int],
    cached_len_before,
    query_len,
    block_size: int,
    *,
    plan: Optional[Fp8PrefillPlan] = None,
) -> torch.Tensor:
    """``hip_prefill_attention`` over an 8-bit cache: chunk tokens attend their
    cached prefix as its codes stand for it and the chunk's own 16-bit rows. The
    result is that call's over the dequantised pool. Arguments and errors as
    there; ``plan``: ``plan_fp8_prefill`` of this table and these lengths.
    """
    out = None if plan is None else _prefill_native(plan, query, key, value, key_cache, value_cache,
                                                    kv_scales, block_size)
    if out is not None:
        return out
    num_blocks, num_kv_heads, head_dim = _check_pool(key_cache, value_cache, kv_scales, block_size,
                                                     "hip_fp8_prefill_attention")
    total_q, num_q_heads, q_dim = query.shape
    device, dtype = key_cache.device, query.dtype
    assert q_dim == head_dim and key.shape[1:] == (num_kv_heads, head_dim) and value.shape == key.shape
    assert dtype in FP8_ROW_DTYPES, f"dtype {dtype} not supported (fp16, bf16)"
    for x, name in ((query, "query"), (key, "key"), (value, "value")):
        _check_rows(x, name, dtype, device)
    rows = [int(r) for r in seq_indices] if plan is None else None
    with _on(device):
        stream = _gpu._stream(device)
        if plan is None and _gpu._capture_id(device):
            assert key.shape[0] >= total_q
            total = total_q
            if total == 0 or not rows:
                return torch.empty(total, num_q_heads, head_dim, dtype=dtype, device=device)
            made = _gpu._prefill_device_plan(
                block_table, rows, cached_len_before, query_len, total_q, block_size, num_blocks,
                num_q_heads, num_kv_heads, head_dim, dtype, device, _gpu._capture_id(device))
            n = len(rows)
        else:
            if plan is None:
                cached, qlens = _gpu._host_lengths(cached_len_before, query_len)
                extra = (tuple(rows), tuple(cached), tuple(qlens), block_size, num_blocks,
                         num_q_heads, num_kv_heads, head_dim, dtype, device, stream)
                plan = _gpu._cache_get("fp8_prefill", (block_table,), extra)
                if plan is None:
                    plan = plan_fp8_prefill(block_table, rows, cached, qlens, block_size, num_blocks,
                                            num_q_heads, num_kv_heads, head_dim, dtype, device)
                    _gpu._cache_put("fp8_prefill", (block_table,), extra, plan)
                else:
                    out = _prefill_native(plan, query, key, value, key_cache, value_cache, kv_scales,
                                          block_size)
                    if out is not None:
                        return out
            assert plan.key == (block_size, num_blocks, num_q_heads, num_kv_heads, head_dim, dtype) and (
                plan.device == device), "the plan is of another step or pool"
            total, made, n = plan.total, plan.plan, plan.num_seqs
            assert total <= total_q and total <= key.shape[0], (
                f"{total} chunk tokens, query has {total_q} rows, key {key.shape[0]}"
            )
            plan._used(stream)
        out = torch.empty(total, num_q_heads, head_dim, dtype=dtype, device=device)
        if total == 0:
            return out
        q, qp, q_st, q_sh = _gpu._row_args(query)
        k, kp, k_st, k_sh = _gpu._row_args(key)
        v, vp, v_st, v_sh = _gpu._row_args(value)
        bt, meta, work, n_work, tokens, units, max_parts, ws = made[:8]
        has_bt = bt.numel() > 0
        o_st, o_sh, _ = out.stride()
        _hip.check(
            _hip.load().mv_fp8_paged_prefill(
                qp, q_st, q_sh, kp, k_st, k_sh, vp, v_st, v_sh, key_cache.data_ptr(),
                value_cache.data_ptr(), kv_scales.data_ptr(), bt.data_ptr() if has_bt else None,
                int(bt.dtype == torch.int64), bt.stride(0) if has_bt else 0, meta.data_ptr(), n,
                work.data_ptr(), n_work, tokens, units, max_parts, out.data_ptr(), o_st, o_sh,
                float(head_dim ** -0.5), num_q_heads, num_kv_heads, head_dim, block_size, num_blocks,
                _hip.MV_DTYPE[dtype], _gpu._ptr(ws), ws.numel() if ws is not None else 0, stream,
            ),
            "mv_fp8_paged_prefill",
        )
    return out


# ============================================================================
# Gather
# ============================================================================


@dataclass
class Fp8GatherPlan(_Plan):
    """The pool slots of every prefix token, sequence by sequence."""

    total: int = 0
    key: tuple = ()  # (block_size, num_blocks)


def plan_fp8_gather(
    block_table: torch.Tensor,
    cached_len_before: Sequence[int],
    seq_indices: Sequence[int],
    block_size: int,
    num_blocks: int,
    device: torch.device,
) -> Fp8GatherPlan:
    """Look the prefixes' tokens up in the block table. ``IndexError``
    ("insufficient") where a row cannot cover its prefix or an entry it needs is
    not a pool block, and for negative lengths. Not while a graph is being captured."""
    device = _indexed(torch.device(device))
    assert block_size in FP8_BLOCK_SIZES, (
        f"block_size {block_size} not supported (a power of 2 from 16 to 256)"
    )
    lens = [int(c) for c in cached_len_before]
    rows = [int(s) for s in seq_indices]
    assert len(lens) == len(rows)
    if any(n < 0 for n in lens):
        raise IndexError(f"block_table insufficient: negative prefix lengths {lens}")
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    total = cu[-1]
    with _on(device):
        if _gpu._capture_id(device):
            raise RuntimeError("plan_fp8_gather: not while a graph is being captured")
        bt = block_table
        if bt.dim() != 2:
            bt = bt.reshape(-1, bt.shape[-1] if bt.dim() else 0)
        bt = bt.to(device)
        if bt.dtype not in (torch.int32, torch.int64):
            bt = bt.to(torch.int64)
        bt = bt.contiguous()
        meta = torch.tensor([*rows, *cu], dtype=torch.int64).to(device)
        slots = torch.empty(max(total, 1), dtype=torch.int64, device=device)
        bad = torch.empty(1, dtype=torch.int32, device=device)
        has_bt = bt.numel() > 0
        _hip.check(
            _hip.load().mv_fp8_prefix_slots(
                bt.data_ptr() if has_bt else None, int(bt.dtype == torch.int64),
                bt.stride(0) if has_bt else 0, bt.shape[0] if has_bt else 0,
                bt.shape[1] if has_bt else 0, meta.data_ptr(), meta.data_ptr() + 8 * len(rows),
                len(rows), total, block_size, num_blocks, slots.data_ptr(), bad.data_ptr(),
                _gpu._stream(device),
            ),
            "mv_fp8_prefix_slots",
        )
        if total and bad.item():
            raise IndexError(
                f"block_table insufficient to cover the cached prefixes: {bad.item()} token(s) "
                f"without a pool block"
            )
        words = _hip.fp8_gather_words(slots.data_ptr(), total, block_size, num_blocks, device.index)
        return Fp8GatherPlan(device, (slots,), _gpu._stream(device), words=words, total=total,
                             key=(block_size, num_blocks))


def gather_fp8_prefix_kv(
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    kv_scales: torch.Tensor,
    block_table: torch.Tensor,
    cached_len_before: Sequence[int],
    seq_indices: Sequence[int],
    block_size: int,
    dtype: torch.dtype,
    *,
    plan: Optional[Fp8GatherPlan] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """``gather_prefix_kv`` from an 8-bit cache: K and V
    ``[sum(cached_len_before), num_kv_heads, head_dim]`` in ``dtype`` (fp16 or
    bf16, the type the cache was written in), ``code * scale`` exactly. Errors as
    there; ``plan``: ``plan_fp8_gather`` of this table and these lengths.
    """
    native = _hip.native_fp8
    if plan is not None and native is not None and dtype in FP8_ROW_DTYPES:
        stream = _gpu._stream(plan.device)
        if stream == plan.stream:
            out = native.gather(plan.words, key_cache, value_cache, kv_scales, block_size,
                                dtype is torch.float16, stream)
            if out is not None:
                if type(out) is int:
                    _hip.check(out, "mv_fp8_gather_kv")
                return out
    num_blocks, num_kv_heads, head_dim = _check_pool(key_cache, value_cache, kv_scales, block_size,
                                                     "gather_fp8_prefix_kv")
    assert dtype in FP8_ROW_DTYPES, f"dtype {dtype} not supported (fp16, bf16)"
    device = key_cache.device
    with _on(device):
        if plan is None:
            plan = plan_fp8_gather(block_table, cached_len_before, seq_indices, block_size,
                                   num_blocks, device)
        assert plan.key == (block_size, num_blocks) and plan.device == device, (
            "the plan is of another step or pool"
        )
        total = plan.total
        out_k = torch.empty(total, num_kv_heads, head_dim, dtype=dtype, device=device)
        out_v = torch.empty_like(out_k)
        if total == 0:
            return out_k, out_v
        stream = _gpu._stream(device)
        plan._used(stream)
        _hip.check(
            _hip.load().mv_fp8_gather_kv(
                key_cache.data_ptr(), value_cache.data_ptr(), kv_scales.data_ptr(),
                plan.buffers[0].data_ptr(), total, out_k.data_ptr(), out_v.data_ptr(), num_kv_heads,
                head_dim, block_size, num_blocks, _hip.MV_DTYPE[dtype], stream,
            ),
            "mv_fp8_gather_kv",
        )
    return out_k, out_v
