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


@pytest.mark.parametrize("out", [ffi.F32, ffi.BF16])
@pytest.mark.parametrize("t,k,shared", [(6, 2, 0), (5, 1, 1), (150, 2, 1), (700, 3, 0)])
def test_a_row_that_the_router_refused_stays_alone(t, k, shared, out):
    from test_gpu_fp8 import codes, dev, on_gpu

    x, ex = acts(15, t, 256), experts(16, 8 + shared, 256, 128)
    w = (codes(ex[0]), dev(ex[1]), codes(ex[2]), dev(ex[3]))
    logits = torch.randn(t, 8, generator=torch.Generator().manual_seed(t)).cuda()
    clean = ffi.moe_ffn_fp8(on_gpu(x), *ffi.moe_route_group(logits, k, 4, 2), *w, shared=shared, out_dtype=out)
    assert torch.isfinite(clean).all()
    bad = [0, 3, t - 1]
    logits[bad, 1] = float("nan")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ids, wts = ffi.moe_route_group(logits, k, 4, 2, status=status)
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = ffi.moe_ffn_fp8(on_gpu(x), ids, wts, *w, shared=shared, out_dtype=out, y=torch.empty_like(clean), status=word)
    rest = [i for i in range(t) if i not in bad]
    assert ffi.status_read(status) == ffi.STATUS_NONFINITE and ffi.status_read(word) == 0
    assert torch.isnan(y[bad]).all() and torch.equal(y[rest], clean[rest])
    assert torch.isnan(ffi.moe_ffn_fp8(on_gpu(x), torch.full_like(ids, -1), wts, *w, shared=shared, out_dtype=out)).all()
    if k > 1:  # one id of a token is no refused row
        ids[1, 0] = -1
        y.fill_(7.0)
        ffi.moe_ffn_fp8(on_gpu(x), ids, wts, *w, shared=shared, out_dtype=out, y=y, status=word)
        assert ffi.status_read(word) == ffi.STATUS_BAD_EXPERT and (y == 7.0).all()
