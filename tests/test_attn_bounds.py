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
