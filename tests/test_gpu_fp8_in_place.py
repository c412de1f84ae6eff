"""Outputs over operands where that is allowed, and refused where it is not."""
from __future__ import annotations

import numpy as np
import pytest

from r9v_amd import ffi
from test_gpu_fp8 import acts, codes, dev, on_gpu, weights
from test_gpu_fp8_moe import experts, routing

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("n", [256, 201])
@pytest.mark.parametrize("m", [5, 40, 300])
def test_an_f32_output_may_be_its_residual(m, n):
    x = on_gpu(acts(1, m, 256))
    w, ws = weights(2, n, 256)
    w, ws = codes(w), dev(ws)
    r = dev(np.random.default_rng(3).standard_normal((m, n)).astype(np.float32))
    want = ffi.matmul_fp8(w, ws, x, residual=r)
    assert ffi.matmul_fp8(w, ws, x, residual=r, y=r) is r and torch.equal(r, want)


@pytest.mark.parametrize("m", [5, 40])
def test_an_output_may_not_be_its_input(m):
    x = on_gpu(acts(4, m, 256), "f32")
    w, ws = weights(5, 256, 256)
    before = x.clone()
    with pytest.raises(ffi.R9vxError, match="y must not overlap"):
        ffi.matmul_fp8(codes(w), dev(ws), x, y=x)
    assert torch.equal(x, before)


@pytest.mark.parametrize("t", [6, 150])
def test_the_experts_output_may_be_their_input(t):
    x, ex = on_gpu(acts(6, t, 256)), experts(7, 5, 256, 128)
    ids, wts = routing(8, t, 5, 2)
    args = (dev(ids), dev(wts), codes(ex[0]), dev(ex[1]), codes(ex[2]), dev(ex[3]))
    want = ffi.moe_ffn_fp8(x, *args, out_dtype=ffi.BF16)
    assert ffi.moe_ffn_fp8(x, *args, out_dtype=ffi.BF16, y=x) is x and torch.equal(x, want)
