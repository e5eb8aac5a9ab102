"""The attention operators in numpy, 64 bits, with how far fp32 arithmetic and
the roundings the kernels make may be from it, value by value."""
import math

import numpy as np

from lunaflux_amd import synth

U32, UBF = 2.0 ** -24, 2.0 ** -8  # half a step, relative: fp32, bf16


def cache_values(codes, kind):
    """fp64 values of cached elements (bf16 bits, or e4m3 codes in steps of the scale)."""
    return (synth.bf16_values(codes) if kind == "bf16" else synth.e4m3_decode(codes)).astype(np.float64)


def decode(q, keys, values, scale):
    """q [G, D] against keys, values [n, D] (fp64): (out [G, D], tolerance).

    Scores: products of bf16 values are exact in fp32, so the sum of D of them
    and the scaling err by at most (D + 3) u sum|q k| scale; exp2 and its
    argument's rounding by (2 + |z|) 2^-23. With e their sum, a weight is off by
    the factor 1 + 2 e, and by 1 + 2^-8 as a bf16 value; both leave an
    average of the values, which moves by at most that times sum p |v - out|,
    twice for the normalization. The fp32 sums over n keys (products of bf16
    values, joined in any order, rescaled at most once a key) err by 2 (n + 8) u
    sum p |v|. Then one rounding to bf16."""
    if len(keys) == 0:
        return np.zeros_like(q), np.zeros_like(q)
    z = q @ keys.T * scale
    p = np.exp(z - z.max(axis=1, keepdims=True))
    p /= p.sum(axis=1, keepdims=True)
    out = p @ values
    reach = (np.abs(q) @ np.abs(keys).T).max(axis=1, keepdims=True) * abs(scale)
    spread = np.abs(z - z.max(axis=1, keepdims=True)).max(axis=1, keepdims=True) + np.abs(z).max(axis=1, keepdims=True)
    e = (q.shape[1] + 3) * U32 * reach + (2 + 1.5 * spread) * 2 * U32
    apart = np.stack([(p[r][:, None] * np.abs(values - out[r])).sum(axis=0) for r in range(len(q))])
    size = p @ np.abs(values)
    tol = 2 * (UBF + 2 * e) * 1.02 * apart + 2 * (len(keys) + 8) * U32 * size
    return out, tol + (np.abs(out) + tol) * UBF + 1e-38


def turned(u, positions, rotary):
    """u [M, heads, D] rotated by positions [M, axes]."""
    half = len(rotary.turns)
    i = np.arange(half)
    a, b = (i, i + half) if rotary.pairing == "half" else (2 * i, 2 * i + 1)
    turn = positions[:, rotary.axis].astype(np.float64) * rotary.turns
    angle = 2 * math.pi * (turn - np.round(turn))
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    out = u.copy()
    out[..., a] = u[..., a] * c - u[..., b] * s
    out[..., b] = u[..., b] * c + u[..., a] * s
    return out


def heads(x, g, epsilon, positions, rotary):
    """Rows x [M, heads, D] normalized (epsilon None: not) and rotated (rotary
    None: not): (values, fp32 tolerance). The mean of D squares errs by
    (D + 2) u, half of that under the root; root, reciprocal and the two
    products by u each (2.5 u for the division); the angle, pi (1 + u) of a
    fraction of a turn, by pi u and sincos by 2^-22: together 2^-21 of |a| + |b|,
    with the rotation's own products."""
    dim = x.shape[2]
    u, rel = x, 0.0
    if epsilon is not None:
        u = x / np.sqrt((x * x).mean(axis=2, keepdims=True) + epsilon) * g
        rel = (dim / 2 + 8) * U32
    tol = np.abs(u) * rel
    if rotary is not None:
        half = len(rotary.turns)
        i = np.arange(half)
        a, b = (i, i + half) if rotary.pairing == "half" else (2 * i, 2 * i + 1)
        both = (np.abs(u[..., a]) + np.abs(u[..., b])) * (rel + 2.0 ** -21)
        tol = tol.copy()
        tol[..., a] = tol[..., b] = both
        u = turned(u, positions, rotary)
    return u, tol


def rounded_bf16(tol, value):
    return tol + (np.abs(value) + tol) * UBF + 1e-38


def rounded_e4m3(tol, value):
    """In steps of the scale, |value| <= 448: half a step is 2^-4 of the value, or 2^-10 below 2^-6."""
    return tol + np.maximum((np.abs(value) + tol) * 2.0 ** -4, 2.0 ** -10)
