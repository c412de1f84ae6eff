"""K past 64 steps of each product kernel, where it loads its block scales anew:
8192 columns in the tiles, 16384 and 32768 in the small ones of two and four
blocks a step."""
from __future__ import annotations

import numpy as np
import pytest

import fp8_ref as R
from r9v_amd import ffi
from test_gpu_fp8 import acts, bytes_of, check, codes, dev, on_gpu, weights
from test_gpu_fp8_moe import check_both, experts, reference, routing

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

# m, n, K, f32 outputs, gated, the kernel that the sizes choose
CASES = [(4100, 2100, 8336, False, False, "fp8_tile_kernel<256, 256, 2, false, false>"),
         (1030, 4100, 8208, False, True, "fp8_tile_kernel<256, 256, 2, true, false>"),
         (4100, 4100, 8336, True, True, "fp8_tile_kernel<128, 256, 2, true, true>"),
         (1100, 2050, 8208, False, False, "fp8_tile_kernel<64, 128, 2, false, false>"),
         (520, 1030, 16656, False, True, "fp8_thin_kernel<64, 128, 2, 2, 2, true, false>"),
         (520, 1030, 16656, True, True, "fp8_thin_kernel<64, 128, 2, 2, 2, true, true>"),
         (300, 700, 33040, False, False, "fp8_thin_kernel<64, 64, 2, 1, 4, false, false>"),
         (300, 700, 33040, True, False, "fp8_thin_kernel<64, 64, 2, 1, 4, false, true>"),
         (70, 200, 18432, True, False, "fp8_thin_kernel<64, 64, 2, 1, 4, false, true>"),
         (20, 72, 33040, True, True, "fp8_stream_kernel<2, 2, 8, 0, true>"),
         (5, 200, 18432, False, False, "fp8_stream_kernel<1, 2, 8, 0, false>")]


@pytest.mark.parametrize("m,n,k,f32,gated,kernel", CASES)
def test_matmul_of_long_rows(m, n, k, f32, gated, kernel):
    """All columns of rows from the first, a middle and the last tile."""
    q, s = ffi.quantize_fp8(on_gpu(acts(1, m, k)))
    w, ws = weights(2, n, k)
    rows = sorted({0, 1, m // 2, m - 2, m - 1})
    xq, xs = bytes_of(q)[rows], s.cpu().numpy()[rows]
    exact = f32 or m <= 32
    p, a = R.product(xq, xs, w, ws)
    tol = R.product_tol(k, a, exact)
    if gated:
        w2, ws2 = weights(3, n, k)
        p2, a2 = R.product(xq, xs, w2, ws2)
        p, tol = R.swiglu(p, p2, tol, R.product_tol(k, a2, exact))
        w, ws = np.concatenate([w, w2]), np.concatenate([ws, ws2])
    y = ffi.matmul_fp8(codes(w), dev(ws), q, x_scales=s, swiglu=gated, out_dtype=ffi.F32 if f32 else ffi.BF16)
    check(y[rows], p, tol, not f32)


@pytest.mark.parametrize("t", [5, 70])
@pytest.mark.parametrize("dm,dff", [(8320, 128), (128, 8320)])
def test_experts_of_long_rows(t, dm, dff):
    x, ids, wts, ex = acts(4, t, dm), *routing(5, t, 3, 2), experts(6, 3, dm, dff)
    check_both(x, ids, wts, ex, reference(x, ids, wts, *ex, 0, exact=t <= 64))


@pytest.mark.parametrize("m", [3, 40])
def test_quantize_of_long_rows(m):
    x = acts(7, m, 33040)
    q, s = ffi.quantize_fp8(on_gpu(x))
    want_q, want_s = R.quantize(x)
    assert np.array_equal(s.cpu().numpy(), want_s) and np.array_equal(R.decode(bytes_of(q)), R.decode(want_q))
