"""The block-scaled e4m3 entry points on the CPU: struct layouts and host-side
refusals (made before any device call), and the figures they report."""
from __future__ import annotations

import ctypes
import pathlib
import subprocess

import pytest

from r9v_amd import ffi

ROOT = pathlib.Path(__file__).resolve().parent.parent
FAKE = 1 << 20  # aligned, never dereferenced: every call below is refused or has no rows
INVALID, UNSUPPORTED, NULL, ALIGN, WORKSPACE = -1, -2, -3, -4, -5


class Lib:
    """The library, loaded by the first test: at collection it would bind its HIP runtime ahead of torch's."""

    def __getattr__(self, name):
        if not name.startswith("r9vx_"):  # pytest asks every object of a module for its own attributes
            raise AttributeError(name)
        return getattr(ffi.load(), name)


lib = Lib()

STRUCTS = {"r9vx_moe_ffn_fp8_static": ffi.MoeFfnFp8Static, "r9vx_moe_ffn_fp8_args": ffi.MoeFfnFp8Args,
           "r9vx_moe_route_group_static": ffi.MoeRouteGroupStatic, "r9vx_quantize_fp8_args": ffi.QuantizeFp8Args, "r9vx_matmul_fp8_static": ffi.MatmulFp8Static,
           "r9vx_matmul_fp8_args": ffi.MatmulFp8Args}


def refused(fn, *structs, code, text):
    rc = fn(*[None if s is None else ctypes.byref(s) for s in structs], None)
    assert rc == code, (rc, lib.r9vx_last_error())
    assert text in lib.r9vx_last_error().decode()


def test_struct_layouts(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "r9vx_fp8.h"', "int main(void){"]
    for name, cls in STRUCTS.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    (tmp_path / "s.c").write_text("\n".join([*lines, "return 0;}"]))
    subprocess.run(["gcc", "-std=c11", "-I", str(ROOT / "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for cls in STRUCTS.values():
        want += [ctypes.sizeof(cls), *(getattr(cls, f).offset for f, _ in cls._fields_)]
    assert got == want


def quant(**kw):
    a = dict(x=FAKE, q=FAKE + (1 << 16), scales=FAKE + (2 << 16), m=4, k=256, in_dtype=ffi.BF16)
    a.update(kw)
    return ffi.QuantizeFp8Args(**a)


@pytest.mark.parametrize("kw,code,text", [
    (dict(k=0), INVALID, "multiple of 16"), (dict(k=136), INVALID, "multiple of 16"), (dict(k=(1 << 20) + 16), UNSUPPORTED, "2^20"),
    (dict(in_dtype=ffi.F16), UNSUPPORTED, "in_dtype 1"), (dict(in_dtype=ffi.E4M3), UNSUPPORTED, "in_dtype"),
    (dict(x=None), NULL, "required"), (dict(q=None), NULL, "required"), (dict(scales=None), NULL, "required"),
    (dict(x=FAKE + 8), ALIGN, "16-byte"), (dict(scales=FAKE + (2 << 16) + 2), ALIGN, "4-byte"),
    (dict(q=FAKE + 1024), INVALID, "overlap"), (dict(scales=FAKE + (1 << 16)), INVALID, "overlap"),
    (dict(m=1 << 41), INVALID, "2^40")])
def test_quantize_refusals(kw, code, text):
    refused(lib.r9vx_quantize_fp8_launch, quant(**kw), code=code, text=text)


def test_quantize_without_rows_or_arguments():
    assert lib.r9vx_quantize_fp8_launch(ctypes.byref(quant(m=0, x=None, q=None, scales=None)), None) == 0
    assert lib.r9vx_quantize_fp8_launch(None, None) == NULL


def mm(**kw):
    st = dict(m_bucket=8, n=200, k=256, in_dtype=ffi.BF16, out_dtype=ffi.F32, epilogue=ffi.EPILOGUE_NONE)
    a = dict(w=FAKE, w_scales=FAKE, x=FAKE, y=FAKE, workspace=FAKE, m=4)
    for k, v in kw.items():
        (st if k in st else a)[k] = v
    return ffi.MatmulFp8Static(**st), ffi.MatmulFp8Args(**a)


@pytest.mark.parametrize("kw,code,text", [
    (dict(k=100), INVALID, "multiple of 16"), (dict(n=0), INVALID, "n must be positive"), (dict(n=(1 << 26) + 1), UNSUPPORTED, "2^26"),
    (dict(m_bucket=1 << 25), UNSUPPORTED, "m_bucket"), (dict(m=9), INVALID, "exceeds m_bucket"),
    (dict(in_dtype=ffi.F16), UNSUPPORTED, "in_dtype"), (dict(in_dtype=ffi.I8), UNSUPPORTED, "in_dtype"),
    (dict(out_dtype=ffi.E4M3), UNSUPPORTED, "out_dtype"), (dict(epilogue=4), UNSUPPORTED, "epilogue 4"),
    (dict(w=None), NULL, "w and w_scales"), (dict(w_scales=None), NULL, "w and w_scales"), (dict(x=None), NULL, "x is NULL"),
    (dict(y=None), NULL, "y is NULL"), (dict(in_dtype=ffi.E4M3), NULL, "x_scales"), (dict(x_scales=FAKE), INVALID, "x_scales"),
    (dict(epilogue=ffi.EPILOGUE_BIAS), NULL, "bias"), (dict(bias=FAKE), INVALID, "bias given"),
    (dict(epilogue=ffi.EPILOGUE_RESIDUAL), NULL, "residual"), (dict(residual=FAKE), INVALID, "residual given"),
    (dict(w=FAKE + 4), ALIGN, "16-byte"), (dict(w_scales=FAKE + 1), ALIGN, "4-byte"), (dict(m_bucket=17, workspace=None), WORKSPACE, "workspace"),
    (dict(k=8192, workspace=None), WORKSPACE, "workspace"), (dict(workspace=FAKE + 16), ALIGN, "256-byte")])
def test_matmul_refusals(kw, code, text):
    refused(lib.r9vx_matmul_fp8_launch, *mm(**kw), code=code, text=text)


def test_matmul_reports_every_problem():
    refused(lib.r9vx_matmul_fp8_launch, *mm(k=100, n=0, w=None, epilogue=9), code=INVALID, text="epilogue 9")
    msg = lib.r9vx_last_error().decode()
    assert "multiple of 16" in msg and "n must be positive" in msg and "w and w_scales" in msg


def test_matmul_without_rows_needs_no_operands():
    st, _ = mm()
    assert lib.r9vx_matmul_fp8_launch(ctypes.byref(st), ctypes.byref(ffi.MatmulFp8Args()), None) == 0
    assert lib.r9vx_matmul_fp8_launch(None, None, None) == NULL


def test_figures():
    st, _ = mm(m_bucket=64, n=200, k=272)
    assert ffi.matmul_fp8_workspace_bytes(st) >= 64 * 272 + 64 * 3 * 4
    assert lib.r9vx_matmul_fp8_static_bytes(ctypes.byref(st), 5) == 200 * 272 + 4 * 2 * 3 + 5 * 272 * 2 + 5 * 200 * 4
    assert lib.r9vx_matmul_fp8_static_flops(ctypes.byref(st), 5) == 2 * 5 * 200 * 272
    st.in_dtype, st.epilogue, st.out_dtype = ffi.E4M3, ffi.EPILOGUE_SWIGLU, ffi.BF16
    assert lib.r9vx_matmul_fp8_static_bytes(ctypes.byref(st), 5) == 2 * (200 * 272 + 4 * 2 * 3) + 5 * (272 + 12) + 5 * 200 * 2
    assert lib.r9vx_matmul_fp8_static_flops(ctypes.byref(st), 5) == 4 * 5 * 200 * 272
    st.k = 100
    assert ffi.matmul_fp8_workspace_bytes(st) == 0 and lib.r9vx_matmul_fp8_static_bytes(ctypes.byref(st), 5) == 0


def test_python_calls_refuse_host_tensors():
    torch = pytest.importorskip("torch")
    x = torch.zeros(4, 256)
    with pytest.raises(ffi.R9vxError):
        ffi.quantize_fp8(x)
    with pytest.raises(ffi.R9vxError):
        ffi.matmul_fp8(torch.zeros(8, 256, dtype=torch.uint8), torch.ones(1, 2), x)


def route(**kw):
    st = dict(t_bucket=8, e_total=64, top_k=8, scoring=1, renormalize=1, n_group=8, topk_group=4, group_score=1,
              scale_bits=0x3F800000, has_bias=0)
    a = dict(logits=FAKE, bias=None, expert_ids=FAKE, weights=FAKE, t=4)
    for k, v in kw.items():
        (st if k in st else a)[k] = v
    return ffi.MoeRouteGroupStatic(**st), ffi.MoeRouteArgs(**a)


@pytest.mark.parametrize("kw,code,text", [
    (dict(e_total=0), INVALID, "E must be"), (dict(e_total=1032), UNSUPPORTED, "exceeds 1024"), (dict(top_k=0), INVALID, "top_k"),
    (dict(top_k=33), UNSUPPORTED, "top_k=33"), (dict(n_group=0), INVALID, "multiple of n_group"),
    (dict(n_group=7), INVALID, "multiple of n_group"), (dict(e_total=1024, n_group=128), UNSUPPORTED, "n_group=128"),
    (dict(topk_group=0), INVALID, "topk_group"), (dict(topk_group=9), INVALID, "topk_group"),
    (dict(t_bucket=(1 << 24) + 1), UNSUPPORTED, "2^24"), (dict(top_k=9, topk_group=1), INVALID, "exceeds the 8 experts"), (dict(n_group=64, topk_group=16), INVALID, "at least two"),
    (dict(group_score=2), UNSUPPORTED, "group_score 2"), (dict(scoring=2), UNSUPPORTED, "scoring 2"), (dict(t=9), INVALID, "t_bucket"),
    (dict(logits=None), NULL, "required"), (dict(expert_ids=None), NULL, "required"), (dict(weights=None), NULL, "required"),
    (dict(has_bias=1), NULL, "bias is NULL"), (dict(bias=FAKE), INVALID, "bias given"), (dict(scale_bits=0), INVALID, "scale"),
    (dict(scale_bits=0x7F800000), INVALID, "scale"), (dict(logits=FAKE + 2), ALIGN, "4-byte")])
def test_route_group_refusals(kw, code, text):
    st, a = route(**kw)
    assert lib.r9vx_moe_route_group_launch(ctypes.byref(st), ctypes.byref(a), None, None) == code
    assert text in lib.r9vx_last_error().decode()


def test_route_group_other_calls():
    st, a = route(t=0, logits=None)
    assert lib.r9vx_moe_route_group_launch(ctypes.byref(st), ctypes.byref(a), None, None) == 0
    assert lib.r9vx_moe_route_group_launch(None, None, None, None) == NULL
    st, a = route()
    assert lib.r9vx_moe_route_group_launch(ctypes.byref(st), ctypes.byref(a), ctypes.c_void_p(FAKE + 1), None) == ALIGN
    assert lib.r9vx_moe_route_group_static_bytes(ctypes.byref(st), 5) == 5 * 64 * 4 + 5 * 8 * 8
    assert lib.r9vx_moe_route_group_static_flops(ctypes.byref(st), 5) == 5 * (6 * 64 + 3 * 8)


def moe(**kw):
    st = dict(t_bucket=8, e_local=16, k_topk=4, dm=256, dff=384, out_dtype=ffi.F32, shared_experts=1)
    a = dict(x=FAKE, expert_ids=FAKE, weights=FAKE, w_gate_up=FAKE, w_gate_up_scales=FAKE, w_down=FAKE, w_down_scales=FAKE,
             y=FAKE, workspace=FAKE, t=5)
    for k, v in kw.items():
        (st if k in st else a)[k] = v
    return ffi.MoeFfnFp8Static(**st), ffi.MoeFfnFp8Args(**a)


@pytest.mark.parametrize("kw,code,text", [
    (dict(e_local=0), INVALID, "E must be"), (dict(e_local=1025), UNSUPPORTED, "exceeds 1024"), (dict(k_topk=0), INVALID, "top-k"),
    (dict(k_topk=33), UNSUPPORTED, "top-k 33"), (dict(dm=0), INVALID, "dm=0"), (dict(dm=192), INVALID, "dm=192"),
    (dict(dff=64), INVALID, "dff=64"), (dict(dff=1 << 17), UNSUPPORTED, "2^16"), (dict(shared_experts=65), UNSUPPORTED, "65 shared"),
    (dict(t_bucket=1 << 24), UNSUPPORTED, "2^32"), (dict(t_bucket=(1 << 23) + 1, k_topk=1), UNSUPPORTED, "2^23"), (dict(t_bucket=1 << 23, k_topk=16, dm=128), UNSUPPORTED, "2^26"),
    (dict(out_dtype=ffi.F16), UNSUPPORTED, "out_dtype"), (dict(t=9), INVALID, "t_bucket"), (dict(x=None), NULL, "required"),
    (dict(expert_ids=None), NULL, "required"), (dict(weights=None), NULL, "required"), (dict(y=None), NULL, "required"),
    (dict(w_gate_up=None), NULL, "scales are required"), (dict(w_gate_up_scales=None), NULL, "scales are required"),
    (dict(w_down=None), NULL, "scales are required"), (dict(w_down_scales=None), NULL, "scales are required"),
    (dict(workspace=None), WORKSPACE, "workspace"), (dict(workspace=FAKE + 64), ALIGN, "256-byte"), (dict(x=FAKE + 2), ALIGN, "16-byte"),
    (dict(w_down_scales=FAKE + 2), ALIGN, "4-byte")])
def test_moe_refusals(kw, code, text):
    refused(lib.r9vx_moe_ffn_fp8_launch, *moe(**kw), code=code, text=text)


def test_moe_other_calls_and_figures():
    st, a = moe(t=0, x=None, y=None, workspace=None)
    assert lib.r9vx_moe_ffn_fp8_launch(ctypes.byref(st), ctypes.byref(a), None) == 0
    assert lib.r9vx_moe_ffn_fp8_launch(None, None, None) == NULL
    assert lib.r9vx_moe_ffn_fp8_status(ctypes.byref(st), None, None, None) == NULL
    expert = 3 * 256 * 384 + 12 * 2 * 3
    assert lib.r9vx_moe_ffn_fp8_expert_bytes(ctypes.byref(st)) == expert
    assert lib.r9vx_moe_ffn_fp8_static_bytes(ctypes.byref(st), 5) == 17 * expert + 5 * 256 * 6 + 20 * 8
    assert lib.r9vx_moe_ffn_fp8_static_flops(ctypes.byref(st), 5) == 6 * 25 * 256 * 384
    assert ffi.ffn_fp8_workspace_bytes(st) > 0
    st.dm = 100
    assert ffi.ffn_fp8_workspace_bytes(st) == 0 and lib.r9vx_moe_ffn_fp8_static_bytes(ctypes.byref(st), 5) == 0
