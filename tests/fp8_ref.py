"""The block-scaled e4m3 operators from their definitions in 64 bits (numpy),
and how far an f32 kernel's outputs may be from them."""
from __future__ import annotations

import math

import numpy as np

BLOCK = 128
# the values of codes 0 .. 126 (0x7F is NaN); 0x80 is the sign
VALUES = np.array([math.ldexp(c % 8 + (8 if c >= 8 else 0), max(c // 8, 1) - 10) for c in range(127)])
MIDDLES = (VALUES[1:] + VALUES[:-1]) / 2


def kb(k):
    return -(-k // BLOCK)


def decode(codes):
    """e4m3 bytes -> f64 values."""
    codes = np.asarray(codes, dtype=np.uint8)
    v = np.append(VALUES, np.nan)[codes & 0x7F]
    return np.where(codes & 0x80, -v, v)


def encode(v):
    """f64 -> the nearest e4m3 byte (ties to the even code), |v| <= 448; NaN -> 0x7F."""
    v = np.asarray(v, dtype=np.float64)
    a = np.abs(v)
    low, high = np.searchsorted(MIDDLES, a, side="left"), np.searchsorted(MIDDLES, a, side="right")
    code = np.where(low % 2 == 0, low, high)
    code = np.where(np.isnan(v), 0x7F, code)
    return (code | (np.signbit(v) & ~np.isnan(v)) * 0x80).astype(np.uint8)


def quantize(x):
    """(codes [m, k] uint8, scales [m, kb] f32) of f32 / f64 rows."""
    x = np.asarray(x, dtype=np.float64)
    m, k = x.shape
    codes, scales = np.zeros((m, k), np.uint8), np.zeros((m, kb(k)), np.float32)
    for b in range(kb(k)):
        part = x[:, b * BLOCK:(b + 1) * BLOCK]
        bad = ~np.isfinite(part).all(axis=1)
        amax = np.where(bad, 0.0, np.abs(np.where(np.isfinite(part), part, 0.0)).max(axis=1))
        s = np.maximum((amax / 448.0).astype(np.float32), np.float32(2.0 ** -126))
        with np.errstate(invalid="ignore"):
            c = encode(part / s.astype(np.float64)[:, None])
        codes[:, b * BLOCK:(b + 1) * BLOCK] = np.where(bad[:, None], 0x7F, c)
        scales[:, b] = np.where(bad, np.float32(np.nan), s)
    return codes, scales


def spread(scales, rows, cols):
    """Block scales [.., .., KB] -> one per element [rows, cols]."""
    return np.repeat(np.repeat(scales.astype(np.float64), BLOCK, axis=0)[:rows], BLOCK, axis=1)[:, :cols]


def product(xq, xs, w, ws):
    """(sum, sum of absolute values) of the scaled products, f64 [m, n]."""
    m, k = xq.shape
    a = decode(xq) * np.repeat(xs.astype(np.float64), BLOCK, axis=1)[:, :k]
    b = decode(w) * spread(ws, w.shape[0], k)
    return a @ b.T, np.abs(a) @ np.abs(b).T


def product_tol(k, absolute, exact=True):
    """How far an f32 product of K columns may be from `product`.  A block's 128
    exact products are added in f32, each addition at most one last place off
    (2^-23 of the sum of absolute values, truncation included); a block's sum is
    scaled (two roundings) and added to the f32 accumulator, and at most 16
    partial accumulators are joined: KB + 18 more roundings of 2^-24.  With the
    8-bit matrix instruction (not `exact`) the 8 products of a group are first
    cut at 2^-13 of the largest of them: 8 * 2^-13 of the sum of absolute values."""
    window = 0.0 if exact else 2.0 ** -10
    return (window + BLOCK * 2.0 ** -23 + (kb(k) + 18) * 2.0 ** -24) * absolute


def bf16_half_step(y):
    """Half a bf16 step, relative to the value."""
    return np.abs(y) * 2.0 ** -8


def silu(g):
    return g / (1.0 + np.exp(-g))


def swiglu(g, u, tol_g, tol_u):
    """(silu(g) * u, its tolerance): |silu'| <= 1.1, and 2^-21 relative for exp,
    divide and the products in f32."""
    h = silu(g) * u
    return h, 1.1 * tol_g * (np.abs(u) + tol_u) + (np.abs(silu(g))) * tol_u + np.abs(h) * 2.0 ** -21 + 1e-37
