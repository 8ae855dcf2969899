"""The rest of a decoder's step in numpy, from its definitions in binary64: weights in 4 bits (codes, steps, their
place in the packed matrix, values), products with them, a mixture-of-experts layer, rotary positions, and the residual
sum with norms.  Divisions that the definitions round to fp32 are numpy's IEEE fp32 divisions.

Beside a result some functions give a bound on what fp32 arithmetic may be off by, from the sizes of what is added:
`chain` is the number of roundings, each at most 2^-23 of the sum of magnitudes, that a sum of products goes through."""
from __future__ import annotations

import numpy as np

from oracle.quantised import NAMES

U = 2.0 ** -24  # half a step of fp32


def w4_quantise(w: np.ndarray, group: int):
    """Codes uint8 [n, k] and steps (upper halves of fp32) uint16 [n, ceil(k / group)] of fp32 weights."""
    n, k = w.shape
    groups = -(-k // group)
    g = np.zeros((n, groups * group), np.float32)
    g[:, :k] = w
    g = g.reshape(n, groups, group)
    finite = np.isfinite(g).all(-1)
    g = np.where(finite[..., None], g, np.float32(0.0))
    t = np.abs(g).max(-1) / np.float32(6.0)
    step = ((t.view(np.uint32) + np.uint32(0x3FFFF)) & np.uint32(0xFFFC0000)).view(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        y = np.where(step[..., None] > 0.0, g / step[..., None], np.float32(0.0))
    # nearest name, a tie to the even place: counting the borders that a magnitude has passed
    a = np.abs(y)
    place = sum((a > b).astype(np.uint8) for b in (0.25, 1.25, 2.5, 5.0)) + sum(
        (a >= b).astype(np.uint8) for b in (0.75, 1.75, 3.5))
    codes = np.where(np.signbit(y), place + 8, place).astype(np.uint8).reshape(n, -1)[:, :k]
    return codes, np.where(finite, step.view(np.uint32) >> 16, 0x7FC0).astype(np.uint16)


def w4_values(codes: np.ndarray, steps: np.ndarray, group: int) -> np.ndarray:
    """What codes and steps stand for, binary64 (exact)."""
    step = (steps.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    v = NAMES[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    return v * np.repeat(step, group, axis=1)[:, :codes.shape[1]]


def w4_pack(codes: np.ndarray, steps: np.ndarray, group: int) -> np.ndarray:
    """The bytes of the packed matrix, code by code from the layout's definition."""
    n, k = codes.shape
    tiles_n, tiles_k, per = -(-n // 16), -(-k // 128), 128 // group
    nibbles = np.zeros(tiles_n * tiles_k * 2048, np.uint8)
    i, j = np.meshgrid(np.arange(n), np.arange(k), indexing="ij")
    tile, column = (i // 16) * tiles_k + j // 128, j % 128
    s, quarter, within = column // 32, column % 32 // 8, column % 8
    nibbles[tile * 2048 + 32 * (16 * quarter + i % 16) + 8 * s + within] = codes
    out_steps = np.zeros((tiles_n * tiles_k, 16, per), np.uint16)
    i, g = np.meshgrid(np.arange(n), np.arange(steps.shape[1]), indexing="ij")
    out_steps[(i // 16) * tiles_k + g // per, i % 16, g % per] = steps
    return np.concatenate((nibbles[0::2] | (nibbles[1::2] << 4), out_steps.reshape(-1).view(np.uint8)))


def product(x: np.ndarray, w: np.ndarray):
    """x w^T and the sums of magnitudes, binary64."""
    x, w = x.astype(np.float64), w.astype(np.float64)
    with np.errstate(invalid="ignore"):
        return x @ w.T, np.abs(x) @ np.abs(w).T


def activation(g: np.ndarray, gelu: bool) -> np.ndarray:
    z = 2.0 * np.sqrt(2.0 / np.pi) * (g + 0.044715 * g ** 3) if gelu else g
    with np.errstate(over="ignore"):
        return g / (1.0 + np.exp(-z))


def route(x: np.ndarray, router: np.ndarray, top_k: int, renormalise: bool):
    """Experts int32 and weights binary64 [tokens, top_k]."""
    logits = x.astype(np.float64) @ router.astype(np.float64).T
    chosen = np.argsort(-np.where(np.isnan(logits), -np.inf, logits), axis=1, kind="stable")[:, :top_k].astype(np.int32)
    with np.errstate(invalid="ignore"):
        p = np.exp(logits - logits.max(1, keepdims=True))
        picked = np.take_along_axis(p, chosen, 1)
        return chosen, picked / (picked if renormalise else p).sum(1, keepdims=True)


def mixture(x, chosen, weights, gate, up, down, gelu: bool, chain: float, carried: float):
    """The layer's output for given experts and weights, and a bound on fp32's part of its error.  gate, up, down:
    [experts][n, k] values; `carried`: how far relative to it a hidden value is off when it enters the second product."""
    x = x.astype(np.float64)
    out, bound = np.zeros(x.shape), np.zeros(x.shape)
    for t in range(x.shape[0]):
        for e, p in zip(chosen[t], weights[t]):
            g, gs = product(x[t:t + 1], gate[e])
            u, us = product(x[t:t + 1], up[e])
            eg, eu = chain * 2 * U * gs, chain * 2 * U * us
            a = activation(g, gelu)
            # the slope of either activation is below 1.13; its argument and exponential a few roundings
            ea = 1.13 * eg + np.abs(a) * (16 + 8 * np.abs(g) + 8 * np.abs(g) ** 3 * gelu) * U
            h = a * u
            eh = ea * (np.abs(u) + eu) + np.abs(a) * eu + np.abs(h) * (2 * U + carried)
            y, ys = product(h, down[e])
            out[t] += p * y[0]
            bound[t] += p * (chain * 2 * U * ys[0] + (eh @ np.abs(down[e]).T)[0] * (1 + chain * 2 * U)) + (
                (len(chosen[t]) + 4) * U) * p * np.abs(y[0])
    return out, bound


def rope(x: np.ndarray, positions: np.ndarray, turns: np.ndarray, rotary: int, pairs: bool, magnitude: float):
    """x [rows, heads, dim] turned, and a bound: the fraction of a turn is rounded to fp32 (2^-26 of a turn, and the
    product of position and turns to 2^-53 of itself), sine and cosine within two units, and five roundings follow."""
    half = rotary // 2
    exact = positions.astype(np.longdouble)[:, None] * turns.astype(np.longdouble)
    fraction = (exact - np.rint(exact)).astype(np.float64)
    angle = 2.0 * np.pi * fraction
    cos, sin = (magnitude * np.cos(angle))[:, None], (magnitude * np.sin(angle))[:, None]
    off = abs(magnitude) * (2 * np.pi * (2.0 ** -26 + np.abs(exact.astype(np.float64)) * 2.0 ** -53) + 9 * U)[:, None]
    out, bound = x.astype(np.float64), np.zeros(x.shape)
    first = np.arange(half) * 2 if pairs else np.arange(half)
    second = first + 1 if pairs else first + half
    a, b = out[..., first].copy(), out[..., second].copy()
    out[..., first], out[..., second] = a * cos - b * sin, b * cos + a * sin
    bound[..., first] = bound[..., second] = (np.abs(a) + np.abs(b)) * off
    return out, bound


def residual_norm(h, y=None, post=None, gate=None, gate_tanh=False, pre=None, scale=None, shift=None, rows_per_vector=1,
                  residual_scale=1.0, weight_offset=0.0, eps=1e-6):
    """h' and out, and bounds on fp32's part of their errors."""
    wide = lambda v: None if v is None else v.astype(np.float64)  # noqa: E731
    h, y, post, gate, pre, scale, shift = (wide(v) for v in (h, y, post, gate, pre, scale, shift))
    vector = np.arange(h.shape[0]) // rows_per_vector
    inverse = lambda v: 1.0 / np.sqrt((v * v).mean(1, keepdims=True) + eps)  # noqa: E731
    bound = np.zeros(h.shape)
    if y is not None:
        f = np.full(h.shape, residual_scale)
        if post is not None:
            f = f * inverse(y) * (weight_offset + post)
        if gate is not None:
            f = f * (np.tanh(gate) if gate_tanh else gate)[vector]
        add = y * f
        h = h + add
        bound = 10 * U * np.abs(add) + U * np.abs(h)
    with np.errstate(invalid="ignore", divide="ignore"):
        r = inverse(h)
        out = h * r
        rel = np.sqrt((bound * bound).sum(1, keepdims=True) / np.maximum((h * h).sum(1, keepdims=True), 1e-300)) + 3 * U
    w = np.ones(h.shape[1]) if pre is None else weight_offset + pre
    out_bound = np.abs(w) * (r * bound + np.abs(out) * (rel + 3 * U))
    out = out * w
    if scale is not None:
        factor = (1.0 + scale)[vector]
        out, out_bound = out * factor, out_bound * np.abs(factor) + np.abs(out) * U * (1 + 3 * np.abs(factor))
    if shift is not None:
        out = out + shift[vector]
        out_bound = out_bound + U * np.abs(out)
    return h, out, bound, out_bound
