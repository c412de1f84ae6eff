"""Refusals and figures of the e4m3 entry points on the CPU (test_fp8_abi.py's arguments)."""
from __future__ import annotations

import ctypes

from r9v_amd import ffi
from test_fp8_abi import ALIGN, FAKE, NULL, lib, moe


def test_moe_launch_ex():
    st, a = moe(t=0, x=None, y=None, workspace=None)
    ref = ctypes.byref
    assert lib.r9vx_moe_ffn_fp8_launch_ex(ref(st), ref(a), None, 1, None) == 0
    assert lib.r9vx_moe_ffn_fp8_launch_ex(None, None, None, 0, None) == NULL
    st, a = moe()
    assert lib.r9vx_moe_ffn_fp8_launch_ex(ref(st), ref(a), ctypes.c_void_p(FAKE + 2), 0, None) == ALIGN
    assert "status word" in lib.r9vx_last_error().decode()
