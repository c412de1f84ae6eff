"""The tolerance of tests/attn_bounds.py on the CPU: it holds for probabilities of the
kernels' precision and not for coarser ones."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import attn_bounds as B  # noqa: E402
import attn_ref as R  # noqa: E402
from attn_cases import DT  # noqa: E402
from attn_scores import CASES, WINDOW, inputs  # noqa: E402


def rounding(dtype):
    return lambda w: torch.from_numpy(w).to(dtype).double().numpy()


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("kw", CASES, ids=str)
@pytest.mark.parametrize("dim", [64, 192])
def test_f16_probabilities_rounded_to_bf16_are_not_within_it(dim, kw, decode):
    q, k, v = inputs(dim, "f16", 1, 300, 8)
    missed = 0
    for h in range(8):
        slope = 0.5 / (1 + h) if kw.get("slopes") else None
        args = (R.f64(q)[0, h], R.f64(k)[:, 0], R.f64(v)[:, 0], (300 - WINDOW, 300), 299, kw.get("scale", dim ** -0.5), kw.get("softcap", 0.0), slope, DT["f16"], decode)
        want, tol = B.attention(*args)
        good = B.attention(*args, rounded=rounding(torch.float16))[0]
        assert (np.abs(good - want) <= tol).all()
        coarse = B.attention(*args, rounded=rounding(torch.bfloat16))[0]
        missed += int((np.abs(coarse - want) > tol).any())
    assert missed >= 4


def test_an_f32_of_the_short_form_is_not_within_it_at_large_caps():
    """1 - 2 / (e + 1) in f32 throughout, at the caps that take the series."""
    f = np.float32
    s = np.linspace(-4, 4, 1001)
    for cap, holds in ((0.3, True), (20.0, True), (50.0, True), (128.0, True), (1e4, False), (1e7, False)):
        with np.errstate(over="ignore"):
            e = np.exp2((s.astype(f) * f(2 * 1.4426950408889634 / cap)).astype(f)).astype(f)
            short = f(cap) - f(2 * cap) / (e + f(1))
        err = np.abs(short.astype(np.float64) - cap * np.tanh(s / cap))
        assert (err <= B.cap_error(s, cap) + B.F32).all() == holds, cap
