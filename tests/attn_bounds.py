"""attn_ref's attention with a tolerance that follows each key's own error to the
output: what moves key j's score by e_j moves the output by p_j e_j (v_j - out), so a
term that enters a score once counts once, and a key of no weight not at all."""
from __future__ import annotations

import numpy as np

import attn_ref as R

F32 = 2.0 ** -23  # twice an f32 rounding: a step of the matrix unit or of a hardware exp2 or reciprocal


def cap_error(s, softcap):
    """Of softcap * tanh(s / softcap), absolutely.  Caps up to 128, cap - 2 cap / (e + 1):
    e's argument (2 roundings and exp2) moves it by at most cap F32, e + 1 and the
    reciprocal by 1.5 F32 of 2 cap, the sum and the cap by F32 of cap: 5 cap F32.  Above,
    where |s| < cap / 4, s times a series: 8 roundings of s; elsewhere cap < 4.1 |out|:
    21 F32 of it."""
    return 5 * softcap * F32 if softcap <= 128 else 21 * np.abs(softcap * np.tanh(s / softcap)) * F32


def attention(q, keys, values, seen, p, scale, softcap, slope, dtype, decode, rounded=None):
    """One query row: (out, tolerance), [dim] each.  `rounded`: what a probability is
    rounded by, relative to the largest, in place of the exact one (then the first
    returned is not the definition)."""
    lo, hi = seen
    if lo >= hi:
        return np.zeros(values.shape[1]), np.zeros(values.shape[1])
    k, v = keys[lo:hi], values[lo:hi]
    n, dim = v.shape
    s = scale * (k @ q)
    error = dim * abs(scale) * (np.abs(k) @ np.abs(q)) * F32  # the product's sum
    if softcap:
        error = error + cap_error(s, softcap)
        s = softcap * np.tanh(s / softcap)
    if slope is not None:
        b = slope * np.abs(p - np.arange(lo, hi))
        error = error + (2 * np.abs(b) + np.abs(s)) * F32  # the slope's rounding to units of 1 / log2(e), the bias' and the sum's
        s = s - b
    top = s.max()
    error = error + (2 * np.abs(s) + 2 * abs(top) + 2) * F32  # the factor, the reference, their difference, exp2
    w = np.exp(s - top)
    if rounded is not None:
        w = rounded(w)
    w = w / w.sum()
    out = w @ v
    far = np.abs(v - out)
    half = R.EPS[dtype] / 2
    tol = half * np.abs(out) + 1.1 * ((w * error) @ far)
    if dtype != R.torch.bfloat16 or not decode:  # prefill adds up the rounded probabilities, decode the ones before
        tol = tol + half * (w @ (np.abs(v) if decode else far))
    else:
        tol = tol + 2.0 ** -16 * (w @ np.abs(v))
    tol = tol + (n + 64) * F32 * (w @ np.abs(v) + np.abs(out))  # sums of n terms, parts and waves
    if dtype == R.torch.float16:  # probabilities of 2^15 at the largest (prefill 2^7 to 2^15), in steps of 2^-24 below 2^-14
        tol = tol + 2.0 ** (-40 if decode else -32) * w.max() * (np.abs(v).sum(0) + n * np.abs(out)) + 2.0 ** -25
    return out, tol * (1 + 2.0 ** -10)
