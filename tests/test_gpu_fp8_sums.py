"""What the e4m3 products add up to where products cancel: f32 outputs keep every
product, whatever stands beside it."""
from __future__ import annotations

import numpy as np
import pytest

import fp8_ref as R
from r9v_amd import ffi
from test_gpu_fp8 import acts, codes, dev
from test_gpu_fp8_moe import call, check, check_both, reference, routing

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

# Groups of 8 neighbouring columns: a large product, of alternating sign from group
# to group, and seven of its 2^-14.8: the large ones cancel, and a sum that keeps 14
# bits of a group's largest product loses all that is left.
BIG = 64.0


def cancelling(rows, k):
    """Weight codes [rows, k] to be met by cancelling_x."""
    w = np.ones(k)
    w[::8] = np.where(np.arange(k // 8) % 2, -BIG, BIG)
    return np.repeat(R.encode(w)[None], rows, axis=0)


def cancelling_x(rows, k):
    x = np.ones((rows, k), np.float32)
    x[:, ::8] = 448.0  # a scale of 1: the codes are the values
    return x * np.exp2(np.arange(rows) % 3)[:, None].astype(np.float32)


def same(e, *codes_and_scales):
    return tuple(np.repeat(a[None], e, axis=0) for a in codes_and_scales)


def positive_codes(seed, n, k):
    r = np.random.default_rng(seed)
    return R.encode(np.clip(100 * np.abs(r.standard_normal((n, k))), 0, 448))


@pytest.mark.parametrize("t,e,shared", [(33, 3, 0), (70, 3, 1), (90, 40, 1), (300, 2, 0), (700, 3, 1)])
def test_gate_and_up_products_that_cancel(t, e, shared):
    dm, dff = 256, 256
    gu = cancelling(2 * dff, dm)
    gus = np.full((2 * dff // 128, dm // 128), 2.0 ** -7, np.float32)
    dn, dns = positive_codes(1, dm, dff), np.full((dm // 128, dff // 128), 2.0 ** -8, np.float32)
    ex = same(e + shared, gu, gus, dn, dns)
    x = cancelling_x(t, dm)
    ids, wts = routing(2, t, e, 2)
    y, tol, _ = reference(x, ids, wts, *ex, shared, exact=True)
    assert np.max(tol / np.abs(y)) < 0.9  # a sum without the small products, zero, is none of these
    check(call(x, ids, wts, ex, shared=shared), y, tol, False)


@pytest.mark.parametrize("t,e,shared", [(33, 3, 0), (70, 3, 1), (90, 40, 1), (300, 2, 0), (700, 3, 1)])
def test_down_products_that_cancel(t, e, shared):
    """h by its up rows, of one product each: 448 : 1, as cancelling_x."""
    dm, dff = 128, 256
    one = np.zeros((dff, dm))
    one[:, 0] = 1.0
    up = one.copy()
    up[::8, 0] = 448.0
    gu = R.encode(np.concatenate([one, up]))
    gus = np.ones((2 * dff // 128, dm // 128), np.float32)
    dn, dns = cancelling(dm, dff), np.ones((dm // 128, dff // 128), np.float32)
    ex = same(e + shared, gu, gus, dn, dns)
    x = np.ones((t, dm), np.float32) * np.exp2(np.arange(t) % 3)[:, None].astype(np.float32)
    ids, wts = routing(3, t, e, 2)
    y, tol, _ = reference(x, ids, wts, *ex, shared, exact=True)
    assert np.max(tol / np.abs(y)) < 0.9
    check(call(x, ids, wts, ex, shared=shared), y, tol, False)


@pytest.mark.parametrize("m", [4, 40, 200, 600])
def test_dense_products_that_cancel(m):
    n, k = 300, 528
    x, w, ws = cancelling_x(m, k), cancelling(n, k), np.full((R.kb(n), R.kb(k)), 0.5, np.float32)
    xq, xs = R.quantize(x)
    p, a = R.product(xq, xs, w, ws)
    tol = R.product_tol(k, a)
    assert np.max(tol / np.abs(p)) < 0.9
    check(ffi.matmul_fp8(codes(w), dev(ws), dev(x)), p, tol, False)


def cancelling_experts(t):
    """Two experts whose outputs differ in a hundredth, with weights 1 and -1.  A block of h
    is one value, so that its codes are 448 whatever the last bits, and the down weights are
    small whole numbers times a power of two, 2^-14 apart between rows: every sum is exact."""
    dm, dff = 256, 128
    r = np.random.default_rng(4)
    rows = [r.integers(1, 4, (1, dm)).repeat(dff, axis=0) for _ in range(2)]
    gu, gus = R.encode(np.concatenate(rows)), np.full((2, 2), 2.0 ** -9, np.float32)
    dn = r.integers(1, 9, (dm, dff)).astype(np.float64)
    other = dn.copy()
    other[:, ::16] += 1
    size = np.where(np.arange(dm) % 2, 2.0 ** -9, 32.0)[:, None]
    dns = np.full((2, 1), 2.0 ** -7, np.float32)
    ex = (np.stack([gu, gu]), np.stack([gus, gus]), np.stack([R.encode(dn * size), R.encode(other * size)]), np.stack([dns, dns]))
    x = np.abs(acts(6, t, dm))
    ids, wts = np.tile(np.array([0, 1], np.int32), (t, 1)), np.tile(np.array([1, -1], np.float32), (t, 1))
    return x, ids, wts, ex


@pytest.mark.parametrize("t", [40, 150])
def test_experts_that_cancel(t):
    """bf16 outputs of many tokens are off by 2^-11 of each |w o| and 2^-25 of its 128
    columns' largest, not by a share of what is left; f32 ones are not."""
    x, ids, wts, ex = cancelling_experts(t)
    y, tol, half = reference(x, ids, wts, *ex, 0, exact=True)
    assert np.max(tol / np.abs(y)) < 2.0 ** -6 and (t <= 64 or np.min(half / np.abs(y)) > 2.0 ** -5)
    check_both(x, ids, wts, ex, (y, tol, half))
