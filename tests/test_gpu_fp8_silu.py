"""The gated epilogue's silu over the range of its argument, seen through an up
operand that makes its smallest values ordinary numbers."""
from __future__ import annotations

import numpy as np
import pytest

import fp8_ref as R
from r9v_amd import ffi
from test_gpu_fp8 import codes, dev

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def gated(v, up_scale, n=40, out=ffi.F32, bucket=None):
    """(silu(g) * u, g, u) of rows whose one value v gives g = v and u = v * up_scale (both
    as the kernel has them: one product and two f32 roundings)."""
    m, k = v.size, 144
    x = np.zeros((m, k), np.float32)
    x[:, 3] = v
    w = np.zeros((2 * n, k))
    w[:, 3] = 1.0
    ws = np.ones((2 * R.kb(n), R.kb(k)), np.float32)
    ws[R.kb(n):] = up_scale
    y = ffi.matmul_fp8(codes(R.encode(w)), dev(ws), dev(x), swiglu=True, out_dtype=out, m_bucket=bucket)
    xq, xs = R.quantize(x)
    c = R.decode(xq)[:, 3]
    s = xs[:, 0]
    return y.float().cpu().numpy().astype(np.float64), c * s.astype(np.float64), c * (s * np.float32(up_scale)).astype(np.float64)


def silu64(g):
    e = np.exp(-np.abs(g))
    return np.where(g < 0, g * e, g) / (1 + e)


RANGES = {"all": (np.concatenate([-np.geomspace(1e-30, 84, 150), np.geomspace(1e-30, 1e30, 150)]), 1e-3),
          "small": (-np.linspace(84, 91, 300), 1e35), "denormal": (-np.linspace(91, 106, 300), 1e35)}


@pytest.mark.parametrize("m", [10, 30, 300])
@pytest.mark.parametrize("name", RANGES)
def test_silu_keeps_its_relative_error(name, m):
    """2^-20 of silu and 2^-24 for each of: g (2), u (2), the product, the store; g's
    error moves silu by at most (1 + |g|) of it, relatively.  Below 2^-126 silu is off
    by 2^-149 as well."""
    v, up = RANGES[name]
    for at in range(0, v.size, m):
        y, g, u = gated(v[at:at + m].astype(np.float32), up, bucket=m)
        want = silu64(g) * u
        tol = np.abs(want) * (2.0 ** -20 + (2 * (1 + np.abs(np.minimum(g, 0))) + 4) * 2.0 ** -24) + 2.0 ** -149 * (1 + np.abs(u))
        over = np.abs(want) > np.finfo(np.float32).max  # no f32 number: an infinity
        assert np.isposinf(y[over]).all()
        bad = np.abs(y - want[:, None])[~over] > tol[~over, None]
        assert not bad.any(), (name, g[~over][bad.any(axis=1)][:5])


def test_far_gates():
    v = np.array([-1e30, -3000, -300, -200, 300, 1e30], np.float32)
    y, g, u = gated(v, 1.0)
    assert (y[:4] == 0).all() and np.allclose(y[4:], (g * u)[4:, None].astype(np.float32), rtol=2.0 ** -20)
