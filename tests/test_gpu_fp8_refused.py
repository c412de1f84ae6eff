"""What a caller sees of experts' calls that were refused."""
from __future__ import annotations

import pytest

from r9v_amd import ffi
from test_gpu_fp8 import acts
from test_gpu_fp8_moe import call, experts, routing

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("out", [ffi.F32, ffi.BF16])
@pytest.mark.parametrize("t", [1, 7, 200])
def test_a_refused_calls_own_output_is_nan_and_its_bits_are_kept(t, out):
    x, ex = acts(9, t, 128), experts(10, 5, 128, 128)
    ids, wts = routing(11, t, 4, 2)
    worse = ids.copy()
    worse[t // 2, 1] = 4
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    want = call(x, ids, wts, ex, shared=1, out_dtype=out, status=status)
    assert ffi.status_read(status) == 0 and torch.isfinite(want).all()
    for _ in range(2):
        assert torch.isnan(call(x, worse, wts, ex, shared=1, out_dtype=out)).all()
    y = torch.full_like(want, 7.0)
    assert call(x, worse, wts, ex, shared=1, out_dtype=out, status=status, y=y) is y and (y == 7.0).all()
    assert torch.equal(call(x, ids, wts, ex, shared=1, out_dtype=out, status=status), want)
    assert ffi.status_read(status) == ffi.STATUS_BAD_EXPERT  # no later launch clears it


def test_a_captured_call_reports_into_its_word():
    t = 6
    x, ex = acts(12, t, 128), experts(13, 4, 128, 128)
    ids, wts = routing(14, t, 4, 2)
    from test_gpu_fp8 import codes, dev, on_gpu

    gx, gi, gw = on_gpu(x), dev(ids), dev(wts)
    w = (codes(ex[0]), dev(ex[1]), codes(ex[2]), dev(ex[3]))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    want = ffi.moe_ffn_fp8(gx, gi, gw, *w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ffi.moe_ffn_fp8(gx, gi, gw, *w, status=status)
    good = gi.clone()
    for bad in (False, True, False, True):
        gi.copy_(good)
        if bad:
            gi[3, 0] = 99
        status.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert ffi.status_read(status) == (ffi.STATUS_BAD_EXPERT if bad else 0)
        assert torch.isnan(y).all() if bad else torch.equal(y, want)
