"""moe_ffn_fp8 on the GPU against its definition in 64 bits, and the router,
the experts and a dense projection as one chain."""
from __future__ import annotations

import numpy as np
import pytest

import fp8_ref as R
from r9v_amd import ffi
from test_gpu_fp8 import acts, bf16, codes, dev, on_gpu, weights

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def requantized(h, tol):
    """(values of h's codes times their scales, how far a kernel's may be from them)
    for rows h [m, dff] that a kernel has within tol: next to the middle of two codes
    it may take either, and its scale is within the relative error of the block's largest."""
    m, dff = h.shape
    q, s = R.quantize(h.astype(np.float32))  # h is f32 in the kernel too
    s = np.repeat(s.astype(np.float64), R.BLOCK, axis=1)[:, :dff]
    amax = np.repeat(np.abs(h).reshape(m, -1, R.BLOCK).max(axis=2), R.BLOCK, axis=1)
    top = np.repeat(tol.reshape(m, -1, R.BLOCK).max(axis=2), R.BLOCK, axis=1)
    ds = (top + 2.0 ** -23 * amax) / np.maximum(amax, 1e-300)
    tol = tol + np.abs(h) * 2.0 ** -23
    v = R.decode(q)
    lo = R.decode(R.encode(np.clip(np.maximum(np.abs(h) - tol, 0) / s * (1 - ds), 0, 448)))
    hi = R.decode(R.encode(np.clip((np.abs(h) + tol) / s * (1 + ds), 0, 448)))
    off = np.maximum(hi - np.abs(v), np.abs(v) - lo) * s + np.abs(v) * s * ds
    return q, s, v * s, off


def expert(xq, xs, gu, gus, dn, dns, exact):
    """(o, tolerance) of one expert's rows."""
    dff, dm = gu.shape[0] // 2, gu.shape[1]
    half = gus.shape[0] // 2
    g, ag = R.product(xq, xs, gu[:dff], gus[:half])
    u, au = R.product(xq, xs, gu[dff:], gus[half:])
    h, tol = R.swiglu(g, u, R.product_tol(dm, ag, exact), R.product_tol(dm, au, exact))
    _, _, v, off = requantized(h, tol)
    w = R.decode(dn) * R.spread(dns, dn.shape[0], dff)
    a = (np.abs(v) + off) @ np.abs(w).T
    return v @ w.T, off @ np.abs(w).T + R.product_tol(dff, a, exact)


def reference(x, ids, wts, gu, gus, dn, dns, shared, exact):
    t, dm = x.shape
    e = gu.shape[0] - shared
    xq, xs = R.quantize(x)
    y, tol, total, half = np.zeros((t, dm)), np.zeros((t, dm)), np.zeros((t, dm)), np.zeros((t, dm))
    for i in range(e + shared):
        tok, slot = np.nonzero(ids == i) if i < e else (np.arange(t), None)
        if tok.size == 0:
            continue
        o, d = expert(xq[tok], xs[tok], gu[i], gus[i], dn[i], dns[i], exact)
        w = wts[tok, slot].astype(np.float64)[:, None] if slot is not None else 1.0
        np.add.at(y, tok, w * o)
        np.add.at(tol, tok, np.abs(w) * d)
        size = np.abs(o) + d
        np.add.at(total, tok, np.abs(w) * size)
        # bf16 outputs of many tokens keep o in f16, scaled by a power of two that brings the largest
        # of 128 columns into [1, 2): half a step is 2^-11 of a normal number, 2^-25 below 2^-14
        top = np.maximum.reduceat(size, np.arange(0, dm, 128), axis=1)
        top = np.repeat(top, 128, axis=1)
        np.add.at(half, tok, np.abs(w) * (size * 2.0 ** -11 + top * 2.0 ** -25))
    # o is weighted and added in f32
    return y, tol + total * (ids.shape[1] + shared + 3) * 2.0 ** -23, half if t > 64 else 0.0 * half


def check_both(x, ids, wts, ex, want, **kw):
    y, tol, half = want
    check(call(x, ids, wts, ex, **kw), y, tol, False)
    check(call(x, ids, wts, ex, out_dtype=ffi.BF16, **kw), y, tol + half, True)


def experts(seed, e, dm, dff, whole=False):
    r = np.random.default_rng(seed)
    if whole:
        one = R.encode(np.array([0.0, 1, -1, 2, -2]))
        gu, dn = one[r.integers(0, 5, (e, 2 * dff, dm))], one[r.integers(0, 5, (e, dm, dff))]
    else:
        gu, dn = (R.encode(np.clip(100 * r.standard_normal(s), -448, 448)) for s in ((e, 2 * dff, dm), (e, dm, dff)))
    gus = (0.0005 * np.exp(0.3 * r.standard_normal((e, 2 * dff // 128, dm // 128)))).astype(np.float32)
    dns = (0.0005 * np.exp(0.3 * r.standard_normal((e, dm // 128, dff // 128)))).astype(np.float32)
    return gu, gus, dn, dns


def routing(seed, t, e, k, skew=0.0):
    r = np.random.default_rng(seed)
    l = r.standard_normal((t, e)) + skew * r.standard_normal(e)
    ids = np.argsort(-l, axis=1)[:, :k].astype(np.int32)
    return ids, r.random((t, k)).astype(np.float32)


def call(x, ids, wts, ex, **kw):
    gu, gus, dn, dns = ex
    return ffi.moe_ffn_fp8(on_gpu(x), dev(ids), dev(wts), codes(gu), dev(gus), codes(dn), dev(dns), **kw)


def check(got, want, tol, bf):
    got = got.float().cpu().numpy().astype(np.float64)
    tol = tol + (R.bf16_half_step(np.abs(want) + tol) if bf else 0) + 1e-30
    err = np.abs(got - want)
    assert np.isfinite(got).all()
    assert (err <= tol).all(), f"{(err > tol).sum()} of {err.size}, worst {np.max(err / tol):.2f}"


SHAPES = [(1, 4, 1, 128, 128, 0), (5, 16, 3, 256, 384, 1), (8, 8, 8, 384, 128, 2), (33, 4, 2, 128, 256, 0), (64, 40, 5, 256, 128, 1),
          (70, 3, 2, 256, 256, 1), (300, 6, 2, 128, 384, 0), (530, 2, 1, 384, 128, 1), (700, 9, 4, 256, 128, 0)]


@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("t,e,k,dm,dff,shared", SHAPES)
def test_moe_ffn_fp8(t, e, k, dm, dff, shared, whole):
    r = np.random.default_rng(t)
    x = r.integers(-1, 2, (t, dm)).astype(np.float32) if whole else acts(t, t, dm)
    ids, wts = routing(t + 1, t, e, k, 0.7)
    ex = experts(t + 2, e + shared, dm, dff, whole)
    check_both(x, ids, wts, ex, reference(x, ids, wts, *ex, shared, exact=whole or t <= 64), shared=shared)


@pytest.mark.parametrize("t", [20, 300])
def test_all_tokens_to_one_expert_and_repeated_experts(t):
    x = acts(3, t, 256)
    ex = experts(4, 7, 256, 128)
    ids = np.full((t, 2), 5, np.int32)
    wts = np.random.default_rng(5).random((t, 2)).astype(np.float32)
    check_both(x, ids, wts, ex, reference(x, ids, wts, *ex, 0, exact=t <= 64))


@pytest.mark.parametrize("bucket", [8, 64, 400])
def test_a_rows_bits_do_not_depend_on_its_batch(bucket):
    t, e, k, dm, dff = min(bucket, 330), 6, 2, 256, 256
    x, ex = acts(6, t, dm), experts(7, e + 1, dm, dff)
    ids, wts = routing(8, t, e, k)
    full = call(x, ids, wts, ex, shared=1, t_bucket=bucket)
    again = call(x, ids, wts, ex, shared=1, t_bucket=bucket)
    assert torch.equal(full, again)
    for i in (0, t // 2, t - 1):
        assert torch.equal(call(x[i:i + 1], ids[i:i + 1], wts[i:i + 1], ex, shared=1, t_bucket=bucket)[0], full[i])
    back = call(x[::-1].copy(), ids[::-1].copy(), wts[::-1].copy(), ex, shared=1, t_bucket=bucket)
    assert torch.equal(back.flip(0), full)


@pytest.mark.parametrize("t", [7, 200])
def test_bad_expert_refuses_the_call(t):
    x, ex = acts(9, t, 128), experts(10, 4, 128, 128)
    ids, wts = routing(11, t, 4, 2)
    st = ffi.ffn_fp8_static(t, 4, 2, 128, 128)
    ws = torch.empty(ffi.ffn_fp8_workspace_bytes(st), dtype=torch.uint8, device="cuda")
    y = torch.full((t, 128), 7.0, device="cuda")
    for bad in (4, -1):
        worse = ids.copy()
        worse[t // 2, 1] = bad
        call(x, worse, wts, ex, y=y, workspace=ws)
        assert ffi.moe_ffn_fp8_status(st, ws) == ffi.STATUS_BAD_EXPERT and (y == 7.0).all()
    call(x, ids, wts, ex, y=y, workspace=ws)
    assert ffi.moe_ffn_fp8_status(st, ws) == 0 and not (y == 7.0).any()


def test_bad_token_stays_alone():
    for t in (6, 150):
        x, ex = acts(12, t, 256), experts(13, 5, 256, 128)
        ids, wts = routing(14, t, 5, 2)
        clean = call(x, ids, wts, ex)
        x[2, 9] = np.inf
        y = call(x, ids, wts, ex)
        rest = [i for i in range(t) if i != 2]
        assert torch.isnan(y[2]).all() and torch.equal(y[rest], clean[rest])


@pytest.mark.parametrize("t", [6, 150])
def test_an_outputs_infinity_stays_alone(t):
    """One weight row of NaN codes and one whose sums pass f32: only their columns lose their values."""
    x, ids, wts = acts(23, t, 256), *routing(24, t, 3, 2)
    gu, gus, dn, dns = experts(25, 3, 256, 128)
    clean = call(x, ids, wts, (gu, gus, dn, dns), out_dtype=ffi.BF16).float()
    dn, dns = dn.copy(), dns.copy()
    dn[:, 7] = 0x7F
    dns[:, 1] = 3e38
    y = call(x, ids, wts, (gu, gus, dn, dns), out_dtype=ffi.BF16).float()
    assert torch.isnan(y[:, 7]).all() and not torch.isfinite(y[:, 128:]).all()
    keep = [i for i in range(128) if i != 7]
    # the same but for f16's step below 2^-14 of a block's largest, which column 7 may have been:
    # 2^-25 of it before and after, from two experts, and a bf16 step where that crosses a middle
    off = 0.0 if t <= 64 else clean[:, keep].abs() * 2.0 ** -7 + clean[:, :128].abs().amax() * 2.0 ** -20
    assert ((y[:, keep] - clean[:, keep]).abs() <= off).all()


def test_rows_behind_the_last_are_left():
    x, ex = acts(15, 9, 128), experts(16, 4, 128, 128)
    ids, wts = routing(17, 9, 4, 2)
    y = torch.full((12, 128), 3.0, device="cuda")
    call(x, ids, wts, ex, y=y[:9], t_bucket=16)
    assert (y[9:] == 3.0).all() and not (y[:9] == 3.0).any()


def layer(x, logits, bias, ex, w, ws, out=None):
    """A layer's tail as an engine runs it: route, experts, projection onto the residual."""
    ids, wts = ffi.moe_route_group(logits, 4, 4, 2, bias=bias, scale=2.5)
    gu, gus, dn, dns = ex
    y = ffi.moe_ffn_fp8(x, ids, wts, gu, gus, dn, dns, shared=1, out_dtype=ffi.BF16)
    q, s = ffi.quantize_fp8(y)
    return ffi.matmul_fp8(w, ws, q, x_scales=s, residual=x.float(), y=out)


@pytest.mark.parametrize("t", [3, 90])
def test_route_experts_and_projection_together(t):
    e, dm, dff = 16, 256, 128
    r = np.random.default_rng(t)
    x, ex = acts(18, t, dm), experts(19, e + 1, dm, dff)
    w, ws = weights(20, dm, dm)
    logits, bias = r.standard_normal((t, e)).astype(np.float32), (0.1 * r.standard_normal(e)).astype(np.float32)
    gpu_ex = (codes(ex[0]), dev(ex[1]), codes(ex[2]), dev(ex[3]))
    args = (on_gpu(x), dev(logits), dev(bias), gpu_ex, codes(w), dev(ws))
    got = layer(*args)
    # each step's operands from the GPU's own previous step, its arithmetic from the definition
    ids, wts = ffi.moe_route_group(args[1], 4, 4, 2, bias=args[2], scale=2.5)
    want_y, tol_y, half = reference(x, ids.cpu().numpy(), wts.cpu().numpy(), *ex, 1, exact=t <= 64)
    y = ffi.moe_ffn_fp8(args[0], ids, wts, *gpu_ex, shared=1, out_dtype=ffi.BF16)
    check(y, want_y, tol_y + half, True)
    q, s = R.quantize(y.float().cpu().numpy())
    p, a = R.product(q, s, w, ws)
    p = p + x
    check(got, p, R.product_tol(dm, a) + np.abs(p) * 2.0 ** -24, False)
    # on another stream, and captured and replayed with eager work between the replays
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(layer(*args), got)
    torch.cuda.current_stream().wait_stream(side)
    out = torch.empty_like(got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(*args, out=out)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, got) and torch.equal(layer(*args), got)


def test_stream_argument():
    x, ex = acts(21, 40, 128), experts(22, 4, 128, 128)
    ids, wts = routing(23, 40, 4, 2)
    want = call(x, ids, wts, ex)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = call(x, ids, wts, ex, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
