"""The quantised decode path in numpy, from its definitions: rows and products in 8-bit
integers, the 4-bit cache of keys and values (its codes, its place in a page, its values)
and attention over it in binary64.  Divisions that the definitions round to fp32 are numpy's
IEEE fp32 divisions."""
from __future__ import annotations

import numpy as np

PAGE, GROUP = 64, 64
NAMES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize_rows(x: np.ndarray):
    """int8 rows and fp32 scales of fp32 rows.  A scale of few units of 2^-149 may have been rounded down by up to
    a third: quotients past 127 are held there."""
    x = np.asarray(x, np.float32)
    finite = np.isfinite(x).all(-1)
    top = np.abs(np.where(finite[:, None], x, 0.0)).max(-1).astype(np.float32)
    scale = top / np.float32(127.0)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.clip(np.rint(x / scale[:, None]), -127.0, 127.0)
    q = np.where(finite[:, None] & (scale[:, None] > 0.0), q, 0.0)
    return q.astype(np.int8), np.where(finite, scale, np.float32(np.nan)).astype(np.float32)


def int8_product(a, w, a_scale, w_scale) -> np.ndarray:
    """In binary64 (sums of whole numbers below 2^53: exact)."""
    c = a.astype(np.float64) @ w.astype(np.float64).T
    return c * (a_scale.astype(np.float64)[:, None] * w_scale.astype(np.float64)[None, :])


def kv4_quantise(x: np.ndarray):
    """Codes uint8 [..., D] and steps (the upper halves of fp32) uint16 [..., D / 64] of fp32 values."""
    x = np.asarray(x, np.float32)
    g = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    finite = np.isfinite(g).all(-1)
    g = np.where(finite[..., None], g, np.float32(0.0))
    t = np.abs(g).max(-1) / np.float32(6.0)
    step = ((t.view(np.uint32) + np.uint32(0x3FFFF)) & np.uint32(0xFFFC0000)).view(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        y = np.where(step[..., None] > 0.0, g / step[..., None], np.float32(0.0))
    # nearest name, a tie to the even place
    distance = np.abs(np.abs(y.astype(np.float64))[..., None] - NAMES)
    near = distance == distance.min(-1, keepdims=True)
    first = near.argmax(-1)
    tie = near.sum(-1) == 2
    place = np.where(tie & (first % 2 == 1), first + 1, first).astype(np.uint8)
    codes = np.where(np.signbit(y), place + 8, place).astype(np.uint8)
    steps = np.where(finite, step.view(np.uint32) >> 16, 0x7FC0).astype(np.uint16)
    return codes.reshape(x.shape), steps


def kv4_values(codes: np.ndarray, steps: np.ndarray) -> np.ndarray:
    """What codes and steps stand for, binary64 (exact)."""
    step = (steps.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    v = NAMES[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    return (v.reshape(*steps.shape, GROUP) * step[..., None]).reshape(codes.shape)


def key_order(dim: int) -> np.ndarray:
    """The channel whose code lies at each place of a key row."""
    block = min(dim, 128)
    per_quarter = block // 32
    place = np.arange(dim)
    word, within = place % block // 8, place % 8
    h, s = word // per_quarter, word % per_quarter
    return place // block * block + 32 * s + 8 * h + within


class Cache:
    """A pool of pages as the device holds it, filled token by token."""

    def __init__(self, pages: int, heads: int, dim: int, fill: np.ndarray):
        self.heads, self.dim = heads, dim
        self.block = PAGE * dim + 4 * dim
        self.pool = np.ascontiguousarray(fill, np.uint8).reshape(pages, heads, self.block).copy()

    def store(self, page: int, slot: int, k: np.ndarray, v: np.ndarray) -> None:
        """k and v: one token's fp32 [heads, D]."""
        half, groups = PAGE * self.dim // 2, self.dim // GROUP
        kc, ks = kv4_quantise(k)
        vc, vs = kv4_quantise(v)
        kc = kc[:, key_order(self.dim)]
        row = slice(slot * self.dim // 2, (slot + 1) * self.dim // 2)
        self.pool[page, :, :half][:, row] = kc[:, 0::2] | (kc[:, 1::2] << 4)
        self.pool[page, :, half:2 * half][:, row] = vc[:, 0::2] | (vc[:, 1::2] << 4)
        params = self.pool[page, :, 2 * half:].view(np.uint16).reshape(self.heads, 2, groups, PAGE)
        params[:, 0, :, slot] = ks
        params[:, 1, :, slot] = vs


def attention(q, k, v, position: int, scale: float, window: int = 0):
    """One row's heads: q [q_heads, D] over k and v [tokens, heads, D] (binary64).  Returns the output and, for
    error bounds, sum_t p_t |v_t| and the largest sum_d |q_d k_td| scale of each head."""
    q_heads, dim = q.shape
    group = q_heads // k.shape[1]
    low = max(0, position - window + 1) if window else 0
    out, size = np.zeros((q_heads, dim)), np.zeros((q_heads, dim))
    reach = np.zeros(q_heads)
    if position < 0:
        return out, size, reach
    for h in range(q_heads):
        kh, vh = k[low:position + 1, h // group], v[low:position + 1, h // group]
        s = kh @ q[h] * scale
        with np.errstate(invalid="ignore"):
            p = np.exp(s - s.max())
            p /= p.sum()
            out[h], size[h] = p @ vh, p @ np.abs(vh)
            reach[h] = (np.abs(kh) @ np.abs(q[h])).max() * scale
    return out, size, reach
