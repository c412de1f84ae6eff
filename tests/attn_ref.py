"""Attention over a paged cache and rotary positions from their definitions in 64
bits, in numpy on the CPU, and the tolerance that the kernels' roundings leave."""
from __future__ import annotations

import numpy as np
import torch

EPS = {torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10}


def f64(t):
    return t.detach().cpu().double().numpy()


def rotated(x, positions, freqs, rot, interleaved, amplitude):
    """x [t, heads, dim] -> f64, and the largest magnitude that entered each value."""
    y = f64(x).copy()
    z = np.exp(1j * positions.cpu().double().numpy()[:, None] * f64(freqs)[None]) * amplitude
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    w = (y[:, :, a] + 1j * y[:, :, b]) * z[:, None, :]
    size = np.abs(y)
    size[:, :, a] = size[:, :, b] = np.abs(y[:, :, a]) + np.abs(y[:, :, b])
    y[:, :, a], y[:, :, b] = w.real, w.imag
    return y, size * abs(amplitude)


def intervals(p, length, start, window, prefix, causal):
    """Keys [lo, hi) that the token at position p sees."""
    if p < 0:
        return 0, 0
    lo = max(start, p - window + 1 if window else 0, 0)
    return lo, min(length, max(p + 1, prefix)) if causal else length


def attention(q, keys, values, seen, p, scale, softcap=0.0, slope=None):
    """One query row q [dim] over keys, values [length, dim] (f64), of which it sees
    [lo, hi): (out, sum of p |v|, what bounds a probability's relative error in f32)."""
    lo, hi = seen
    if lo >= hi:
        return np.zeros(values.shape[1]), np.zeros(values.shape[1]), 0.0
    k, v = keys[lo:hi], values[lo:hi]
    s = scale * (k @ q)
    size = abs(scale) * (np.abs(k) @ np.abs(q)).max()
    if softcap:
        s = softcap * np.tanh(s / softcap)
        size += 4 * softcap  # 1 - 2 / (e + 1): a few steps of f32 of the cap
    if slope is not None:
        b = slope * np.abs(p - np.arange(lo, hi))
        s = s - b
        size += np.abs(b).max()
    with np.errstate(all="ignore"):
        w = np.exp(s - s.max())
        w = w / w.sum()
        return w @ v, w @ np.abs(v), size + np.abs(s).max()


def bound(out, absolute, size, dim, length, dtype, exact_p):
    """How far a kernel may be from `attention`.  The output's rounding; each
    probability's (unless kept in twice the bits) times |v|; f32: a score's product
    of dim terms and its few further steps move a probability by 2^-23 (dim + 8)
    of the sizes that enter the score, numerator and denominator; sums of `length`
    terms.  f16 keeps probabilities above 2^-40 of the largest, and has values
    below 2^-14 in steps of 2^-24."""
    half = EPS[dtype] / 2
    p = 2.0 ** -16 if exact_p else half
    f32 = 2.0 ** -23 * ((dim + 8) * size + 2 * length + 64)
    return half * np.abs(out) * (1 + 2 * f32) + (p + 2 * f32) * absolute + 2.0 ** -25


def gathered(cache, table, length, head):
    """f64 [length, dim] of one sequence and kv head, through the table."""
    page = cache.shape[1]
    j = torch.arange(length)
    rows = cache.cpu()[table.cpu().long()[j // page], j % page, head]
    return rows.double().numpy()
