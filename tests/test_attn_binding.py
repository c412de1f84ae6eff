"""The attention binding on the CPU: the numbers it takes and what it keeps of its calls."""
from __future__ import annotations

import fractions

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from r9v_amd import attn, ffi  # noqa: E402
from test_attn_abi import CALLS, on_cpu, spy  # noqa: E402, F401

NUMBERS = [0.25, 1, np.float64(0.25), 1 / np.sqrt(128), np.float32(0.25), np.float16(0.1), np.int64(3), fractions.Fraction(1, 4)]


@pytest.mark.parametrize("x", NUMBERS, ids=lambda x: type(x).__name__)
def test_numbers_of_any_type_are_taken(x, on_cpu, monkeypatch):  # noqa: F811
    monkeypatch.setattr(attn.ffi, "_fp8_operands", lambda *o: 0)
    assert attn._number("scale", x) == attn._bits(float(x))
    with on_cpu:
        for name, kw in (("decode", dict(scale=x)), ("prefill", dict(softcap=x)), ("rope", dict(amplitude=x))):
            CALLS[name](**kw)


@pytest.mark.parametrize("x", [True, None, "1", 1j, torch.ones(()), np.array(1.0), np.bool_(True), [1.0]], ids=lambda x: type(x).__name__)
def test_what_is_no_number_is_refused(x):
    with pytest.raises(ffi.R9vxError, match="is no number"):
        attn._number("softcap", x)


def test_plans_are_of_these_calls_alone(on_cpu, monkeypatch):  # noqa: F811
    """A caller that never repeats a size leaves what the e4m3 calls keep."""
    monkeypatch.setattr(attn.ffi, "_fp8_operands", lambda *o: 0)
    kept = {("a static", i): i for i in range(4000)}
    monkeypatch.setattr(ffi, "_fp8_statics", dict(kept))
    monkeypatch.setattr(attn, "_plans", {}, raising=False)
    with on_cpu:
        for i in range(5000):
            CALLS["rope"](amplitude=1.0 + i)
    assert ffi._fp8_statics == kept and 0 < len(attn._plans) <= 4096
