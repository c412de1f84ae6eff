"""Where the binding's calls allocate: what a call on a stream of the caller's
writes comes from that stream's pool, and returned tensors also wait for the
stream that will read them.  On the CPU, with streams and library stood in for."""
from __future__ import annotations

import contextlib
import types
from functools import partial

import pytest

from r9v_amd import ffi, gguf

torch = pytest.importorskip("torch")
from torch.utils._python_dispatch import TorchDispatchMode  # noqa: E402


def stream(n):
    return types.SimpleNamespace(cuda_stream=n, synchronize=lambda: None)


RAW_STREAM = ffi._raw_stream  # the binding's own; the calls below run with a stand-in


class Allocations(TorchDispatchMode):
    """(name, stream that is current) of every operator that makes or fills memory."""

    def __init__(self):
        super().__init__()
        self.seen, self.kept, self.current = [], [], 0

    @contextlib.contextmanager
    def on(self, s):
        before, self.current = self.current, s.cuda_stream
        yield
        self.current = before

    def __torch_dispatch__(self, func, types_, args=(), kwargs=None):
        if func._schema.name.split("::")[1] in ("empty", "empty_strided", "new_empty", "zeros", "new_zeros", "zero_", "fill_", "_local_scalar_dense"):
            self.seen.append((func._schema.name, self.current))
        return func(*args, **(kwargs or {}))


class Library:
    """Every entry point succeeds and touches nothing."""

    def __getattr__(self, name):
        return lambda *a: 4096 if name.endswith(("_bytes", "_blocks")) else 0


@pytest.fixture
def spy(monkeypatch):
    mode = Allocations()
    monkeypatch.setattr(ffi, "load", Library)
    monkeypatch.setattr(ffi, "_need_gpu", lambda *t: torch)
    monkeypatch.setattr(ffi, "_fp8_operands", lambda *o: 0)
    monkeypatch.setattr(ffi, "_raw_stream", lambda device, s: 0)
    monkeypatch.setattr(ffi, "_fp8_statics", {})
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, device=None, **kw: empty(*a, **kw))  # "cuda" too
    monkeypatch.setattr(torch.cuda, "stream", mode.on)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: stream(mode.current))
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: mode.kept.append((t.data_ptr(), s.cuda_stream)), raising=False)
    return mode


def z(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


B, I, U8 = torch.bfloat16, torch.int32, torch.uint8
FILE = types.SimpleNamespace(_h=None, tensor=lambda name: types.SimpleNamespace(dtype=8, nbytes=340, block_bytes=34))
CALLS = {
    "matmul": partial(ffi.matmul, z(8), ffi.Q4_K, 16, 256, z(20, 256, dtype=B)),
    "dequantize": partial(ffi.dequantize, z(144, dtype=U8), ffi.Q4_K, 1, 256),
    "repack": partial(ffi.repack, z(34, dtype=U8), ffi.Q8_0, 1, 32),
    "repack_iq3s": partial(ffi.repack, z(110, dtype=U8), ffi.IQ3_S, 1, 256),
    "validate_weights": partial(ffi.validate_weights, z(144, dtype=U8), ffi.Q4_K, 1, 256),
    "moe_route": partial(ffi.moe_route, z(4, 16), 2),
    "router_repack": partial(ffi.router_repack, z(16, 64)),
    "moe_route_hidden": partial(ffi.moe_route_hidden, z(4, 64, dtype=B), z(1024), 2),
    "moe_ffn": partial(ffi.moe_ffn, z(4, 256, dtype=B), z(4, 2, dtype=I), z(4, 2), z(8), z(8), 4, 256),
    "moe_sort": partial(ffi.moe_sort, z(4, 2, dtype=I), 4),
    "moe_route_group": partial(ffi.moe_route_group, z(4, 16), 2, 4, 2),
    "quantize_fp8": partial(ffi.quantize_fp8, z(4, 256, dtype=B)),
    "matmul_fp8": partial(ffi.matmul_fp8, z(16, 256, dtype=U8), z(1, 2), z(20, 256, dtype=B)),
    "moe_ffn_fp8": partial(ffi.moe_ffn_fp8, z(4, 128, dtype=B), z(4, 2, dtype=I), z(4, 2), z(3, 256, 128, dtype=U8), z(3, 2, 1),
                           z(3, 128, 128, dtype=U8), z(3, 1, 1)),
    "probe_stream": partial(ffi.probe_stream, z(64)),
    "probe_mfma": partial(ffi.probe_mfma, 2, 1),
    "probe_matmul_tiles": partial(ffi.probe_matmul_tiles, z(8), ffi.Q4_K, 16, 256, z(20, 256, dtype=B), 1, 1),
    "gguf.upload": partial(gguf.upload, FILE, b"0", "w"),
    "gguf.upload_gate_up": partial(gguf.upload_gate_up, FILE, b"0", "g", FILE, b"0", "u"),
    "gguf.upload_split": partial(gguf.upload_split, FILE, b"0", "w"),
    "gguf.upload_gate_up_split": partial(gguf.upload_gate_up_split, FILE, b"0", "g", FILE, b"0", "u"),
}


@pytest.mark.parametrize("name", CALLS)
def test_memory_of_a_call_belongs_to_its_stream(name, spy):
    with spy:
        CALLS[name]()
    assert spy.seen and {s for _, s in spy.seen} == {0} and spy.kept == []
    del spy.seen[:]
    with spy:
        out = CALLS[name](stream=stream(7))
    assert spy.seen and {s for _, s in spy.seen} == {7}, spy.seen
    for t in out if isinstance(out, tuple) else (out,):
        if isinstance(t, torch.Tensor):
            assert (t.data_ptr(), 0) in spy.kept


def test_every_call_with_a_stream_is_here():
    """But for those that only write where they are told, or read a status back."""
    import inspect

    told = {"moe_ffn_noalloc", "probe_moe_stage", "status_read", "moe_route_status", "moe_route_hidden_status", "moe_ffn_status",
            "moe_ffn_fp8_status"}
    names = {n for m in (ffi, gguf) for n, f in inspect.getmembers(m, inspect.isfunction)
             if f.__module__ == m.__name__ and not n.startswith("_") and "stream" in inspect.signature(f).parameters}
    assert names == told | {n.split(".")[-1] for n in CALLS if n != "repack_iq3s"}


@pytest.mark.parametrize("name", ["moe_route_group", "quantize_fp8", "matmul_fp8", "moe_ffn_fp8"])
def test_a_stream_of_another_device_is_refused(name, spy, monkeypatch):
    monkeypatch.setattr(ffi, "_raw_stream", RAW_STREAM)
    here, other = stream(7), stream(8)
    here.device, other.device = torch.device("cuda", 0), torch.device("cuda", 1)
    CALLS[name](stream=here)
    with pytest.raises(ffi.R9vxError, match="stream is of cuda:1"):
        CALLS[name](stream=other)
