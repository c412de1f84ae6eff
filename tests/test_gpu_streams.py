"""Calls on a stream of the caller's: the memory they take, and their results."""
from __future__ import annotations

import numpy as np
import pytest

from r9v_amd import ffi
from test_gpu_fp8 import acts, codes, dev, on_gpu, weights

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


class Recorder:
    """The library, with products that are noted instead of launched."""

    def __init__(self):
        self.lib, self.made = ffi.load(), []

    def __getattr__(self, name):
        return getattr(self.lib, name)

    def r9vx_matmul_fp8_launch(self, st, args, stream):
        self.made.append({args._obj.y, args._obj.workspace})
        return 0


def test_a_call_takes_no_memory_that_the_current_stream_may_still_write(monkeypatch):
    """The blocks of a call on the current stream are free when it returns, and its
    kernels may still be queued: a call on another stream may not get them."""
    w, ws = weights(1, 64, 256)
    w, ws, x = codes(w), dev(ws), on_gpu(acts(2, 40, 256))
    lib = Recorder()
    monkeypatch.setattr(ffi, "load", lambda: lib)
    side = torch.cuda.Stream()
    ffi.matmul_fp8(w, ws, x)
    ffi.matmul_fp8(w, ws, x, stream=side)
    ffi.matmul_fp8(w, ws, x)
    here, there, again = lib.made
    assert here == again  # freed blocks are taken again
    assert len(there) == 2 and not here & there


def test_results_on_another_stream():
    w, ws = weights(3, 200, 528)
    w, ws, x = codes(w), dev(ws), on_gpu(acts(4, 70, 528))
    side = torch.cuda.Stream()
    want = ffi.matmul_fp8(w, ws, x)
    q, s = ffi.quantize_fp8(x)
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        ffi.matmul_fp8(w, ws, x)  # its blocks are freed with its kernels queued
        got = ffi.matmul_fp8(w, ws, x, stream=side)
        gq, gs = ffi.quantize_fp8(x, stream=side)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want) and torch.equal(gs, s) and torch.equal(gq.view(torch.uint8), q.view(torch.uint8))


def test_bad_weights_are_counted_on_their_stream():
    wire = np.zeros((8, 144), np.uint8)
    wire[3, :2] = [0x00, 0x7C]  # an infinite scale
    side = torch.cuda.Stream()
    w = dev(wire)
    side.wait_stream(torch.cuda.current_stream())
    assert ffi.validate_weights(w, ffi.Q4_K, 8, 256) == 1 and ffi.validate_weights(w, ffi.Q4_K, 8, 256, stream=side) == 1
