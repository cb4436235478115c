"""Oracle of the quantised paged KV cache, in numpy.

What the format specifies to the bit (codes, params, index, selected pages) is
computed in the fp32 steps that the specification names; what it computes
(values, attention) in 64 bits.  Blocks are unpacked from and compared as the
raw bytes of the pool.
"""
from __future__ import annotations

import numpy as np

GROUP = 64
TINY = np.float32(2.0 ** -100)
F32 = np.float32


# ------------------------------------------------------------------ dtype bits
def to_bits(x, dtype: str) -> np.ndarray:
    """float32 values -> uint16 bit patterns of dtype, rounded to nearest even."""
    x = np.asarray(x, F32)
    if dtype == "float16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bits(b, dtype: str) -> np.ndarray:
    """uint16 bit patterns -> float32 values."""
    b = np.ascontiguousarray(b, np.uint16)
    if dtype == "float16":
        return b.view(np.float16).astype(F32)
    return (b.astype(np.uint32) << 16).view(F32)


def round_to(x, dtype: str) -> np.ndarray:
    return from_bits(to_bits(x, dtype), dtype)


def _toward(x, dtype: str, up: bool) -> np.ndarray:
    """x >= 0 rounded up (or down) to dtype."""
    b = to_bits(x, dtype)
    near = from_bits(b, dtype)
    step = (near < x) if up else (near > x)
    return from_bits((b.astype(np.int32) + np.where(step, 1 if up else -1, 0)).astype(np.uint16), dtype)


# ------------------------------------------------------------------- quantiser
def quantise(x, bits: int, dtype: str):
    """x [..., D] (float32 values of dtype) -> codes uint8 [..., D], scale, min float32 [..., D/64]."""
    n = F32(2 ** bits - 1)
    g = np.asarray(x, F32).reshape(*x.shape[:-1], -1, GROUP)
    with np.errstate(all="ignore"):
        lo, hi = g.min(-1), g.max(-1)
        want = (hi * F32(0.5) - lo * F32(0.5)) * F32(2.0 / float(n))
        up, down = _toward(want, dtype, True), _toward(want, dtype, False)
        # in 64 bits: n*up alone may pass fp32's largest where the sum does not
        past = np.isinf(round_to((np.float64(n) * up + lo).astype(F32), dtype))
        scale = np.where(past, down, up).astype(F32)
        scale = np.where(scale < TINY, F32(0), scale)
        inv = F32(1) / (scale * F32(0.5))
        c = np.rint((g * F32(0.5) - lo[..., None] * F32(0.5)) * inv[..., None])
    c = np.where(scale[..., None] == 0, 0, np.clip(c, 0, n))
    bad = ~np.isfinite(g).all(-1)
    c = np.where(bad[..., None], 0, c).astype(np.uint8).reshape(x.shape)
    nan = F32(np.nan)
    return c, np.where(bad, nan, scale), np.where(bad, nan, lo)


def values(codes, scale, lo) -> np.ndarray:
    """What codes [..., D] stand for, in 64 bits and not rounded."""
    s = np.repeat(np.asarray(scale, np.float64), GROUP, -1)
    m = np.repeat(np.asarray(lo, np.float64), GROUP, -1)
    return codes.astype(np.float64) * s + m


def read_back(codes, scale, lo, dtype: str) -> np.ndarray:
    """The read-back values (one fp32 multiply-add, rounded once to dtype)."""
    # a code times a scale is exact in 32 bits, so rounding the 64-bit sum to 32
    # bits is the fused multiply-add (the sum itself is exact, or far from a tie)
    with np.errstate(all="ignore"):
        return round_to(values(codes, scale, lo).astype(F32), dtype)


def unpack(data, page: int, D: int, bits: int, dtype: str):
    """Pool bytes [..., block] -> per side (codes [..., page, D], scale, min [..., page, D/64])."""
    row, ng = D * bits // 8, D // GROUP
    lead = data.shape[:-1]
    out = []
    for side in (0, 1):
        c = data[..., side * page * row:(side + 1) * page * row].reshape(*lead, page, row)
        if bits == 4:
            c = np.stack((c & 15, c >> 4), -1).reshape(*lead, page, D)
        at = 2 * page * row + side * page * ng * 4
        p = np.ascontiguousarray(data[..., at:at + page * ng * 4]).view(np.uint16)
        p = from_bits(p, dtype).reshape(*lead, page, ng, 2)
        out.append((c, p[..., 0], p[..., 1]))
    return out


# ----------------------------------------------------------------------- index
def signed8(x, axes):
    """(int codes, fp32 scale) of float32 x over `axes`."""
    with np.errstate(all="ignore"):
        top = np.abs(x).max(axes, keepdims=True).astype(F32)
        ok = np.isfinite(top)
        scale = np.where(ok, top * F32(1.0 / 127.0), F32(np.nan)).astype(F32)
        c = np.clip(np.rint(x.astype(F32) * (F32(1) / scale)), -127, 127)
        c = np.where(scale >= TINY, c, 0)
    return c.astype(np.int8), scale


def bounds(k):
    """Index codes [2, D] and scale of a page's read-back keys k [tokens, D]."""
    c, s = signed8(np.stack((k.min(0), k.max(0))).astype(F32), (0, 1))
    return c, s[0, 0]


def select(q, index, index_scale, count: int, top_k: int) -> np.ndarray:
    """Pages of one (sequence, KV head): q [G, D], index [count, 2, D], index_scale [count]."""
    out = np.full(top_k, -1, np.int32)
    if count == 0:
        return out
    q8, sq = signed8(np.asarray(q, F32), (1,))
    q8, idx = q8.astype(np.int64), index.astype(np.int64)
    dot = np.maximum(q8[:, None] * idx[None, :, 0], q8[:, None] * idx[None, :, 1]).sum(-1)
    with np.errstate(all="ignore"):
        score = (dot.astype(F32) * sq) * np.asarray(index_scale, F32)[None]
    score = np.where(np.isnan(score), F32(np.inf), score).max(0)
    score[-1] = np.inf
    best = sorted(range(count), key=lambda p: (-score[p], p))[:top_k]
    out[:len(best)] = sorted(best)
    return out


# ------------------------------------------------------------------- attention
def attend(q, k, v, scale: float):
    """(O, L) of q [G, D] over k, v [n, D] in 64 bits; n may be 0."""
    q = np.asarray(q, np.float64)
    if len(k) == 0:
        return np.zeros(q.shape), np.full(q.shape[0], -np.inf)
    s = q @ k.T * scale
    m = s.max(-1, keepdims=True)
    p = np.exp(s - m)
    l = p.sum(-1, keepdims=True)
    return (p / l) @ v, (m + np.log(l))[:, 0]
