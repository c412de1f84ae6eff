"""quantize_fp8 and matmul_fp8 on the GPU against their definitions in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import fp8_ref as R
from r9v_amd import ffi, synth

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def codes(a):
    return dev(a).view(torch.float8_e4m3fn)


def bytes_of(t):
    return t.view(torch.uint8).cpu().numpy()


def bf16(a):
    """f32 values that bf16 holds."""
    return synth.bf16_bits_to_f32(synth.to_bf16_bits(np.asarray(a, np.float32)))


def acts(seed, m, k, dtype="bf16"):
    r = np.random.default_rng(seed)
    x = r.standard_normal((m, k)).astype(np.float32) * np.where(r.random(k) < 0.02, 20, 1).astype(np.float32)
    return bf16(x) if dtype == "bf16" else x


def on_gpu(x, dtype="bf16"):
    return dev(x).to(torch.bfloat16) if dtype == "bf16" else dev(x)


def weights(seed, n, k):
    """Random finite codes, every bit pattern among them, and scales of both signs."""
    r = np.random.default_rng(seed)
    w = r.integers(0, 256, (n, k), dtype=np.uint8)
    w[(w & 0x7F) == 0x7F] = 0x7E
    s = (0.002 * np.exp(r.standard_normal((R.kb(n), R.kb(k)))) * np.where(r.random((R.kb(n), R.kb(k))) < 0.1, -1, 1)).astype(np.float32)
    return w, s


# ------------------------------------------------------------------ quantize

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m,k", [(1, 16), (1, 128), (3, 144), (5, 2048), (7, 1040), (257, 112), (33, 4096)])
def test_quantize_every_code_and_scale(m, k, dtype):
    x = acts(m * 1000 + k, m, k, dtype)
    x[0, :min(k, 16)] = 0.0
    q, s = ffi.quantize_fp8(on_gpu(x, dtype))
    want_q, want_s = R.quantize(x)
    assert np.array_equal(s.cpu().numpy(), want_s)
    assert np.array_equal(R.decode(bytes_of(q)), R.decode(want_q))


def test_quantize_middles_between_codes():
    """Quotients that are exactly between two codes, one f32 step to either side
    of them, and every code: the largest value 448 makes the scale 1."""
    mids = R.MIDDLES.astype(np.float32)
    v = np.concatenate([R.VALUES.astype(np.float32), mids, np.nextafter(mids, np.float32(0)), np.nextafter(mids, np.float32(1e9))])
    v = np.concatenate([v, -v])
    blocks = -(-v.size // 127)
    x = np.full((blocks, 128), 448.0, np.float32)
    x[:, :127].flat[:v.size] = v
    q, s = ffi.quantize_fp8(dev(x))
    assert (s.cpu().numpy() == 1.0).all()
    assert np.array_equal(R.decode(bytes_of(q)), R.decode(R.quantize(x)[0]))


def test_quantize_quotients_next_to_middles():
    """bf16 values in ratios of few bits over scales that f32 rounds: thousands of
    quotients lie within one f32 step of a middle without being one."""
    r = np.random.default_rng(5)
    top = bf16(np.abs(r.standard_normal(4096)) + 0.1)
    ratio = r.choice(R.MIDDLES[8:], (4096, 127)) / 448.0
    x = bf16(np.concatenate([top[:, None].astype(np.float64) * ratio, top[:, None]], axis=1))
    q, s = ffi.quantize_fp8(on_gpu(x))
    want_q, want_s = R.quantize(x)
    assert np.array_equal(s.cpu().numpy(), want_s)
    assert np.array_equal(R.decode(bytes_of(q)), R.decode(want_q))


def test_quantize_small_large_and_bad_blocks():
    x = np.zeros((12, 256), np.float32)
    r = np.random.default_rng(6)
    for i, e in enumerate([-149, -140, -130, -126, -118, -100, -64, 60, 119]):
        x[i] = np.ldexp(r.standard_normal(256), e).astype(np.float32)
    x[9] = np.float32(3.4028235e38)
    x[10, 7], x[11, 200] = np.nan, -np.inf
    q, s = ffi.quantize_fp8(dev(x))
    want_q, want_s = R.quantize(x)
    assert np.array_equal(s.cpu().numpy(), want_s, equal_nan=True)
    assert np.array_equal(R.decode(bytes_of(q)), R.decode(want_q), equal_nan=True)


def test_quantize_leaves_what_is_behind_the_rows():
    q = torch.full((9, 144), 0x55, dtype=torch.uint8, device="cuda")
    s = torch.full((9, 2), 7.0, device="cuda")
    ffi.quantize_fp8(on_gpu(acts(1, 4, 144)), q=q[:4], scales=s[:4])
    assert (q[4:] == 0x55).all() and (s[4:] == 7.0).all()


# ------------------------------------------------------------------ matmul

def check(got, want, tol, bf):
    got = got.float().cpu().numpy().astype(np.float64)
    tol = tol + (R.bf16_half_step(np.abs(want) + tol) if bf else np.abs(want) * 2.0 ** -24)
    err = np.abs(got - want)
    assert np.isfinite(got).all()
    assert (err <= tol).all(), f"{(err > tol).sum()} of {err.size} out of tolerance, worst {np.max(err / tol):.2f}"


def run(m, n, k, dtype="bf16", out="f32", epilogue="none", bucket=None, seed=1):
    x = acts(seed, m, k, "f32" if dtype == "f32" else "bf16")
    xq, xs = R.quantize(x)
    r = np.random.default_rng(seed + 2)
    bias = r.standard_normal(n).astype(np.float32) if epilogue == "bias" else None
    res = r.standard_normal((m, n)).astype(np.float32) if epilogue == "residual" else None
    w, ws = weights(seed + 1, n, k)
    p, a = R.product(xq, xs, w, ws)
    exact = out == "f32" or (bucket or m) <= 32
    tol = R.product_tol(k, a, exact)
    if epilogue == "swiglu":
        w2, ws2 = weights(seed + 3, n, k)
        p2, a2 = R.product(xq, xs, w2, ws2)
        p, tol = R.swiglu(p, p2, tol, R.product_tol(k, a2, exact))
        w, ws = np.concatenate([w, w2]), np.concatenate([ws, ws2])
    for extra in (bias, res):
        if extra is not None:
            p = p + extra
            tol = tol + np.abs(p) * 2.0 ** -24
    xg, sg = (codes(xq), dev(xs)) if dtype == "e4m3" else (on_gpu(x, dtype), None)
    y = ffi.matmul_fp8(codes(w), dev(ws), xg, x_scales=sg, out_dtype=ffi.BF16 if out == "bf16" else ffi.F32,
                       bias=None if bias is None else dev(bias), residual=None if res is None else dev(res),
                       swiglu=epilogue == "swiglu", m_bucket=bucket)
    check(y, p, tol, out == "bf16")
    return y


SHAPES = [(1, 16, 16), (1, 1, 128), (3, 130, 272), (5, 5120, 2048), (16, 257, 640), (17, 96, 1152), (31, 200, 144),
          (48, 1408, 1024), (64, 66, 256), (65, 300, 400), (255, 129, 256), (256, 256, 128), (257, 512, 1040), (600, 700, 368)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matmul_sizes(m, n, k):
    run(m, n, k)


@pytest.mark.parametrize("epilogue", ["none", "bias", "residual", "swiglu"])
@pytest.mark.parametrize("dtype", ["bf16", "f32", "e4m3"])
@pytest.mark.parametrize("m,n,k", [(5, 200, 400), (40, 72, 656), (300, 390, 272)])
def test_matmul_types_and_epilogues(m, n, k, dtype, epilogue):
    run(m, n, k, dtype, "bf16" if m == 40 else "f32", epilogue)


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(1, 72, 144), (16, 130, 256), (40, 300, 400), (64, 64, 2048), (200, 260, 640), (513, 384, 1168)])
def test_small_whole_numbers_are_exact(m, n, k, out):
    """Codes 0, +-1, +-2 and scales that are powers of two: every sum is a whole
    number of few bits, so every path gives it exactly (bf16 outputs: rounded once)."""
    r = np.random.default_rng(m + n + k)
    one = R.encode(np.array([0.0, 1, -1, 2, -2]))
    xq, w = one[r.integers(0, 5, (m, k))], one[r.integers(0, 5, (n, k))]
    xs = np.exp2(r.integers(-2, 3, (m, R.kb(k)))).astype(np.float32)
    ws = np.exp2(r.integers(-2, 3, (R.kb(n), R.kb(k)))).astype(np.float32)
    want = R.product(xq, xs, w, ws)[0].astype(np.float32)
    if out == "bf16":
        want = bf16(want)
    y = ffi.matmul_fp8(codes(w), dev(ws), codes(xq), x_scales=dev(xs), out_dtype=ffi.BF16 if out == "bf16" else ffi.F32)
    assert np.array_equal(y.float().cpu().numpy(), want)


@pytest.mark.parametrize("m,out", [(1800, "f32"), (1878, "f32"), (1900, "f32"), (1800, "bf16"), (1878, "bf16"), (1942, "bf16"), (2020, "bf16")])
def test_last_tile_of_every_height(m, out):
    """The large tiles' last rows: up to a quarter, a half, three quarters and all of a tile."""
    run(m, 4352, 2048, "e4m3", out, "none")


@pytest.mark.parametrize("epilogue", ["none", "swiglu"])
@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(256, 256, 128), (300, 520, 272), (600, 700, 368), (70, 4100, 1040), (130, 2050, 656),
                                   (520, 2112, 1168), (1100, 2000, 400), (4096, 1030, 272)])
def test_matmul_tiles(m, n, k, out, epilogue):
    """Rows and columns that end inside tiles of every kind, K inside a step."""
    run(m, n, k, out=out, epilogue=epilogue)


@pytest.mark.parametrize("bucket", [64, 300])
def test_matmul_fewer_rows_than_the_bucket(bucket):
    for m in (1, 33, bucket):
        run(m, 144, 528, bucket=bucket)


def test_nan_codes_past_a_ragged_row_do_not_leak():
    """The columns behind a ragged K are the next row's first ones: NaN codes there
    reach no output but that row's own."""
    for m in (4, 40, 200):
        k, n = 144, 40
        x = acts(9, m, k)
        w, ws = weights(10, n, k)
        w[1::2, :112] = 0x7F
        y = ffi.matmul_fp8(codes(w), dev(ws), on_gpu(x)).cpu().numpy()
        assert np.isnan(y[:, 1::2]).all() and np.isfinite(y[:, ::2]).all()


@pytest.mark.parametrize("m", [4, 40, 200])
def test_a_rows_bits_do_not_depend_on_its_batch(m):
    k, n = 528, 300
    x = acts(13, m, k)
    w, ws = weights(14, n, k)
    wg, sg = codes(w), dev(ws)
    for out in (ffi.F32, ffi.BF16):
        full = ffi.matmul_fp8(wg, sg, on_gpu(x), out_dtype=out)
        assert torch.equal(ffi.matmul_fp8(wg, sg, on_gpu(x), out_dtype=out), full)
        for i in (0, m // 2, m - 1):
            assert torch.equal(ffi.matmul_fp8(wg, sg, on_gpu(x[i:i + 1]), out_dtype=out, m_bucket=m)[0], full[i])
        assert torch.equal(ffi.matmul_fp8(wg, sg, on_gpu(x[::-1].copy()), out_dtype=out).flip(0), full)


@pytest.mark.parametrize("m", [4, 40, 200])
def test_bad_rows_stay_alone(m):
    x = acts(11, m, 256)
    w, ws = weights(12, 100, 256)
    clean = ffi.matmul_fp8(codes(w), dev(ws), on_gpu(x)).cpu().numpy()
    bad = x.copy()
    bad[1, 3], bad[3, 200] = np.nan, np.inf
    y = ffi.matmul_fp8(codes(w), dev(ws), on_gpu(bad)).cpu().numpy()
    rest = [i for i in range(m) if i not in (1, 3)]
    assert np.isnan(y[[1, 3]]).all() and np.array_equal(y[rest], clean[rest])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m,k", [(1, 4096), (5, 272), (16, 2048), (16, 4096), (3, 16)])
def test_in_call_quantization_is_quantize_fp8s(m, k, dtype):
    """Few rows are quantized by the workgroups that read them, others by a launch: the same bits."""
    x = acts(31, m, k, dtype)
    x[0, :16] = 0.0
    x[m - 1, k - 1] = np.inf
    w, ws = weights(32, 200, k)
    xg = on_gpu(x, dtype)
    q, s = ffi.quantize_fp8(xg)
    want = ffi.matmul_fp8(codes(w), dev(ws), q, x_scales=s)
    got = ffi.matmul_fp8(codes(w), dev(ws), xg)
    assert torch.isnan(got[m - 1]).all() and torch.equal(got[:m - 1], want[:m - 1])
