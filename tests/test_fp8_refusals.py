"""Refusals and figures of the e4m3 entry points on the CPU (test_fp8_abi.py's arguments)."""
from __future__ import annotations

import ctypes

import pytest

from r9v_amd import ffi
from test_fp8_abi import ALIGN, FAKE, INVALID, NULL, lib, mm, moe, refused, route


def test_moe_launch_ex():
    st, a = moe(t=0, x=None, y=None, workspace=None)
    ref = ctypes.byref
    assert lib.r9vx_moe_ffn_fp8_launch_ex(ref(st), ref(a), None, 1, None) == 0
    assert lib.r9vx_moe_ffn_fp8_launch_ex(None, None, None, 0, None) == NULL
    st, a = moe()
    assert lib.r9vx_moe_ffn_fp8_launch_ex(ref(st), ref(a), ctypes.c_void_p(FAKE + 2), 0, None) == ALIGN
    assert "status word" in lib.r9vx_last_error().decode()


def apart(*names):
    """Addresses 2^28 from each other."""
    return {n: FAKE + (i << 28) for i, n in enumerate(names)}


MM = apart("w", "w_scales", "x", "y", "workspace")
Y = MM["y"]  # 4 rows of 200 f32: 3200 bytes


@pytest.mark.parametrize("kw,text", [
    (dict(x=Y), "y must not overlap"), (dict(x=Y + 3184), "y must not overlap"), (dict(x=Y - 4 * 512 + 16), "y must not overlap"),
    (dict(w=Y), "y must not overlap"), (dict(w=Y - 200 * 256 + 16), "y must not overlap"), (dict(w_scales=Y + 16), "y must not overlap"),
    (dict(epilogue=ffi.EPILOGUE_BIAS, bias=Y + 16), "y must not overlap"),
    (dict(epilogue=ffi.EPILOGUE_RESIDUAL, residual=Y + 16), "y must not overlap"),
    (dict(epilogue=ffi.EPILOGUE_RESIDUAL, residual=Y, out_dtype=ffi.BF16), "y must not overlap"),
    (dict(epilogue=ffi.EPILOGUE_SWIGLU, w=Y - 2 * 200 * 256 + 16), "y must not overlap"),
    (dict(in_dtype=ffi.E4M3, x_scales=Y + 64), "y must not overlap"),
    (dict(m_bucket=40, workspace=Y - 256), "workspace must not overlap"), (dict(m_bucket=40, workspace=MM["x"]), "workspace must not overlap")])
def test_matmul_operands_apart(kw, text):
    refused(lib.r9vx_matmul_fp8_launch, *mm(**{**MM, "y": Y & ~255, **kw}), code=INVALID, text=text)


MOE = apart("x", "expert_ids", "weights", "w_gate_up", "w_gate_up_scales", "w_down", "w_down_scales", "y", "workspace")


@pytest.mark.parametrize("kw,text", [
    (dict(expert_ids=MOE["y"] + 64), "y must not overlap"), (dict(weights=MOE["y"]), "y must not overlap"),
    (dict(y=MOE["workspace"] + 256), "workspace must not overlap"), (dict(x=MOE["workspace"] + 256), "workspace must not overlap"),
    (dict(expert_ids=MOE["workspace"]), "workspace must not overlap"), (dict(weights=MOE["workspace"]), "workspace must not overlap")])
def test_moe_operands_apart(kw, text):
    refused(lib.r9vx_moe_ffn_fp8_launch, *moe(**{**MOE, **kw}), code=INVALID, text=text)


ROUTE = apart("logits", "bias", "expert_ids", "weights")


@pytest.mark.parametrize("kw", [dict(expert_ids=ROUTE["logits"] + 4 * 64 * 4 - 4), dict(weights=ROUTE["logits"]),
                                dict(weights=ROUTE["expert_ids"] + 64), dict(weights=ROUTE["bias"]), dict(expert_ids=ROUTE["bias"] + 252)])
def test_route_operands_apart(kw):
    st, a = route(**{**ROUTE, "has_bias": 1, **kw})
    assert lib.r9vx_moe_route_group_launch(ctypes.byref(st), ctypes.byref(a), None, None) == INVALID
    assert "must not overlap" in lib.r9vx_last_error().decode()
