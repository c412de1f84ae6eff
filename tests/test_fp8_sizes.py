"""Sizes past 32 bits from Python: refused by name, not taken modulo 2^32 (on the
CPU, with tensors that have no memory)."""
from __future__ import annotations

import pytest

from r9v_amd import ffi

torch = pytest.importorskip("torch")
BIG = 1 << 32
BF, F, I, U8 = torch.bfloat16, torch.float32, torch.int32, torch.uint8


def meta(*shape, dtype=F):
    return torch.empty(shape, dtype=dtype, device="meta")


class Library:
    """Notes every call that gets through."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: 0 if name.endswith("_bytes") else self.calls.append(name) or 0


@pytest.fixture
def lib(monkeypatch):
    lib = Library()
    monkeypatch.setattr(ffi, "load", lambda: lib)
    monkeypatch.setattr(ffi, "_fp8_operands", lambda *o: 0)
    monkeypatch.setattr(ffi, "_raw_stream", lambda device, s: 0)
    monkeypatch.setattr(ffi, "_fp8_statics", {})
    return lib


def experts(t, dm, k=2):
    return (meta(t, dm, dtype=BF), meta(t, k, dtype=I), meta(t, k), meta(4, 256, dm, dtype=U8), meta(4, 2, dm // 128),
            meta(4, dm, 128, dtype=U8), meta(4, dm // 128, 1))


CALLS = {
    "quantize k": lambda b: ffi.quantize_fp8(meta(1, b + 16, dtype=BF)),
    "matmul k": lambda b: ffi.matmul_fp8(meta(8, b + 128, dtype=U8), meta(1, b // 128 + 1), meta(1, b + 128, dtype=BF)),
    "matmul n": lambda b: ffi.matmul_fp8(meta(b + 16, 16, dtype=U8), meta(b // 128 + 1, 1), meta(1, 16, dtype=BF)),
    "matmul m": lambda b: ffi.matmul_fp8(meta(8, 16, dtype=U8), meta(1, 1), meta(b + 3, 16, dtype=BF), m_bucket=8),
    "matmul m_bucket": lambda b: ffi.matmul_fp8(meta(8, 16, dtype=U8), meta(1, 1), meta(3, 16, dtype=BF), m_bucket=b + 8),
    "route t": lambda b: ffi.moe_route_group(meta(b + 1, 4), 2, 2, 1, t_bucket=8),
    "route e_total": lambda b: ffi.moe_route_group(meta(1, b + 4), 2, 2, 1),
    "route n_group": lambda b: ffi.moe_route_group(meta(1, 4), 2, b + 2, 1),
    "route topk_group": lambda b: ffi.moe_route_group(meta(1, 4), 2, 2, b + 1),
    "route scoring": lambda b: ffi.moe_route_group(meta(1, 4), 2, 2, 1, scoring=b),
    "route negative": lambda b: ffi.moe_route_group(meta(1, 4), 2, 2, 1, group_score=b - 1 if b == 0 else -b),
    "moe t": lambda b: ffi.moe_ffn_fp8(*experts(b + 1, 128), t_bucket=8),
    "moe dm": lambda b: ffi.moe_ffn_fp8(*experts(1, b + 128)),
}


@pytest.mark.parametrize("name", CALLS)
def test_sizes_past_32_bits_are_refused(name, lib):
    if name != "route negative":
        CALLS[name](0)
        assert len(lib.calls) == 1
    with pytest.raises(ffi.R9vxError, match="32 bits"):
        CALLS[name](BIG)
    assert len(lib.calls) <= 1
