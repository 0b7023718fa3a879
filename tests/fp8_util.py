"""The 8-bit KV cache's definition in 64 bits (not a test module).

Written from the format alone (numpy, explicit loops over blocks): e4m3 with 3
fraction bits, normal from 2^-6, at most 448; one power-of-two scale per (block,
kv head) for K and for V.
"""

from __future__ import annotations

import math

import numpy as np
import torch

FP8 = torch.float8_e4m3fn
# half a step of a rounding, relative to the value
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LIMIT = {torch.bfloat16: 240.0 * 2.0 ** 120, torch.float16: 61440.0}


def e4m3(y: np.ndarray) -> np.ndarray:
    """Values rounded to the nearest e4m3 number, ties to even (|y| <= 448 or NaN)."""
    a = np.abs(y)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.where(a > 0, np.floor(np.log2(np.where(a > 0, a, 1.0))), -6.0)
    # (log2 may round up to an integer just below a power of two)
    e = np.where(np.exp2(e) > a, e - 1, e)
    step = np.exp2(np.maximum(e, -6.0) - 3)
    return np.copysign(np.rint(a / step) * step, y)


def scale_exp(amax: float) -> int:
    """The smallest e >= -110 with amax <= 448 * 2^e."""
    e = -110
    if amax > 0:
        e = max(e, math.ceil(math.log2(amax / 448.0)) - 1)
        while amax > 448.0 * 2.0 ** e:
            e += 1
    return e


def append(codes, scales, rows, slots, block_size, dtype):
    """Rows [T, H, D] (64-bit) into codes [blocks, H, bs, D] (values of the codes)
    and scales [blocks, H], in place."""
    by_block: dict = {}
    for t, s in enumerate(slots):
        if s >= 0:
            by_block.setdefault(s // block_size, []).append((s % block_size, t))
    for blk, places in by_block.items():
        anew = any(o == 0 for o, _ in places)
        off = [o for o, _ in places]
        for h in range(codes.shape[1]):
            x = np.stack([rows[t, h] for _, t in places])
            x = np.where(np.isfinite(x), np.clip(x, -LIMIT[dtype], LIMIT[dtype]), np.nan)
            amax = float(np.nanmax(np.abs(np.nan_to_num(x, nan=0.0))))
            old = 0.0 if anew else scales[blk, h]
            new = max(old, 2.0 ** scale_exp(amax))
            if 0 < old < new:
                codes[blk, h] = e4m3(codes[blk, h] * (old / new))
            codes[blk, h, off] = e4m3(x / new)
            scales[blk, h] = new


def rotated(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x cos + rotate_half(x) sin with every operation rounded to x's type (CPU)."""
    h = x.shape[-1] // 2

    def r(y):
        return y.float().to(x.dtype).double()

    a, c, s = x.double(), cos.double()[:, None], sin.double()[:, None]
    half = torch.cat([-a[..., h:], a[..., :h]], dim=-1)
    return r(r(a * c) + r(half * s)).to(x.dtype)


def random_pool(num_blocks, hkv, block_size, d, seed, dev, spread=3.0):
    """(key codes, value codes, scales) of a pool with blocks of different
    magnitudes and K with large channels; every code finite."""
    g = torch.Generator().manual_seed(seed)
    caches, scales = [], torch.empty(num_blocks, hkv, 2)
    for j in range(2):
        size = torch.exp2((torch.rand(num_blocks, hkv, 1, 1, generator=g) - 0.5) * spread)
        x = torch.randn(num_blocks, hkv, block_size, d, generator=g) * size
        if j == 0:
            x[..., ::19] *= 6
        e = torch.ceil(torch.log2(x.abs().amax((2, 3)) / 448) + 1e-6)
        scales[:, :, j] = torch.exp2(e)
        caches.append((x / scales[:, :, j, None, None]).to(FP8))
    return caches[0].to(dev), caches[1].to(dev), scales.to(dev)


def values(codes: torch.Tensor, scales: torch.Tensor, j: int) -> torch.Tensor:
    """What the codes stand for, in 64 bits: [blocks, H, bs, D]."""
    return codes.cpu().double() * scales[:, :, j, None, None].cpu().double()


def attend(q, k, v, first, dtype):
    """Query i of q [T, Hq, D] over keys 0 .. first + i of k, v [N, Hkv, D], all
    64-bit; (result, how far a kernel may be off).

    The kernel's weights are p_j = 2^(s_j - m) with s_j an fp32 sum of D products:
    off by at most 2 D 2^-23 sum |q k| scale (each addition of a chain of D rounds
    once, the products are exact; a factor 2 for the order) plus the fp32 rounding of
    scale, s and m, 2^-21 max |s|; then rounded to the row type (u = half a step) and
    divided by the sum of the rounded weights. A relative error r of every weight moves
    the result by at most r sum w_j |v_j - o| <= 2 r max |v|; the result is rounded
    once more, u |o| (twice that where the pieces' sums, in fp32, are joined)."""
    t, hq, d = q.shape
    n, hkv, _ = k.shape
    rep = hq // hkv
    out, tol = torch.empty_like(q), torch.empty_like(q)
    u = HALF[dtype]
    keys = torch.arange(n)
    for h in range(hq):
        kk, vv = k[:, h // rep], v[:, h // rep]
        s = (q[:, h] @ kk.T) / math.sqrt(d)
        mag = (q[:, h].abs() @ kk.abs().T) / math.sqrt(d)
        seen = keys[None] <= torch.arange(t)[:, None] + first
        s = s.masked_fill(~seen, -math.inf)
        w = torch.softmax(s, dim=1)
        o = w @ vv
        off = torch.where(seen, 2 * d * 2.0 ** -23 * mag + 2.0 ** -21 * s.abs().nan_to_num(posinf=0.0), 0.0)
        vmax = torch.stack([vv[: first + i + 1].abs().amax() for i in range(t)])[:, None]
        r = u + 2 * off.amax(1, keepdim=True)
        out[:, h] = o
        tol[:, h] = 2 * r * vmax + u * o.abs() + 2.0 ** -20 * vmax
    return out, tol
