"""attn.rope_kv and attn.rope against the definition in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import attn_ref as R  # noqa: E402
from r9v_amd import attn, ffi  # noqa: E402

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
HALF = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}


def inputs(t, heads, kv, dim, x, out, page, seed, start=0):
    g = torch.Generator().manual_seed(seed)
    rows = torch.randn(t, (heads + 2 * kv) * dim, generator=g).to(DT[x]).cuda()
    q, k, v = rows.split((heads * dim, kv * dim, kv * dim), 1)
    pages = -(-t // page) + 2
    caches = [torch.randn(pages, page, kv, dim, generator=g).to(DT[out]).cuda() for _ in range(2)]
    slots = torch.randperm(pages * page, generator=g)[:t].cuda()
    pos = torch.arange(start, start + t, dtype=torch.int32, device="cuda")
    return q.view(t, heads, dim), k.view(t, kv, dim), v.view(t, kv, dim), pos, caches[0], caches[1], slots


def near(got, want, size, out, position=0):
    """One rounding; cosine, sine and the two products in f32: 2^-21 of what enters;
    the angle's few roundings in f64, 2^-51 of an angle of at most `position`;
    f16's steps below 2^-14."""
    tol = HALF[out] * np.abs(want) * (1 + 2.0 ** -20) + (2.0 ** -21 + 2.0 ** -51 * position) * size + 2.0 ** -25
    err = np.abs(R.f64(got) - want)
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("t,heads,kv,dim,rot,x,out,interleaved,start,amplitude", [
    (1, 1, 1, 16, 16, "bf16", "bf16", False, 0, 1.0), (1, 16, 2, 256, 64, "bf16", "bf16", False, 5119, 1.0), (5, 32, 8, 128, 128, "f32", "bf16", True, 1000003, 1.2),
    (3, 5, 1, 96, 48, "f16", "f16", False, (1 << 31) - 4, 1.0), (77, 7, 7, 64, 32, "f32", "f16", True, 3, 0.5), (1100, 4, 2, 128, 112, "bf16", "bf16", True, 1 << 20, 1.0),
    (2, 3, 2, 512, 512, "f16", "f16", True, 9, -1.0), (33, 2, 3, 80, 80, "bf16", "bf16", False, -20, 1.0), (4, 1, 1, 24, 16, "f32", "bf16", False, 100, 0.0)])
def test_rope_kv(t, heads, kv, dim, rot, x, out, interleaved, start, amplitude):
    q, k, v, pos, kc, vc, slots = inputs(t, heads, kv, dim, x, out, 16, 7, start)
    freqs, _ = attn.rope_freqs(rot, base=500000.0)
    before = R.f64(kc).reshape(-1, kv, dim), R.f64(vc).reshape(-1, kv, dim)
    got = attn.rope_kv(q, k, v, pos, freqs, kc, vc, slots, interleaved=interleaved, amplitude=amplitude)
    want, size = R.rotated(q, pos, freqs, rot, interleaved, amplitude)
    want[..., rot:], size[..., rot:] = R.f64(q)[..., rot:], 0
    far = float(pos.abs().max())
    near(got, want, size, out, far)
    want, size = R.rotated(k, pos, freqs, rot, interleaved, amplitude)
    want[..., rot:], size[..., rot:] = R.f64(k)[..., rot:], 0
    at = slots.cpu().numpy()
    kk, vv = kc.reshape(-1, kv, dim), vc.reshape(-1, kv, dim)
    near(kk[slots], want, size, out, far)
    near(vv[slots], R.f64(v), 0 * size, out)
    rest = np.setdiff1d(np.arange(len(kk)), at)
    assert np.array_equal(R.f64(kk)[rest], before[0][rest]) and np.array_equal(R.f64(vv)[rest], before[1][rest])


@pytest.mark.parametrize("x", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_alone_and_in_place(x, interleaved):
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(40, 6, 128, generator=g).to(DT[x]).cuda()
    data = wide[:, 1:4]
    pos = torch.randint(0, 1 << 21, (40,), generator=g).int().cuda()
    freqs, amp = attn.rope_freqs(96, scaling="yarn", factor=4.0, original_length=4096)
    got = attn.rope(data, pos, freqs, interleaved=interleaved, amplitude=amp)
    want, size = R.rotated(data, pos, freqs, 96, interleaved, amp)
    want[..., 96:], size[..., 96:] = R.f64(data)[..., 96:], 0
    near(got, want, size, x, 1 << 21)
    rest = wide[:, [0, 4, 5]].clone()
    assert attn.rope(data, pos, freqs, interleaved=interleaved, amplitude=amp, out=data) is data
    assert torch.equal(data, got) and torch.equal(wide[:, [0, 4, 5]], rest)


def test_q_in_place_among_a_projections_rows():
    q, k, v, pos, kc, vc, slots = inputs(9, 4, 2, 64, "bf16", "bf16", 16, 8)
    freqs, _ = attn.rope_freqs(64)
    kc2, vc2 = kc.clone(), vc.clone()
    want = attn.rope_kv(q, k, v, pos, freqs, kc2, vc2, slots)
    attn.rope_kv(q, k, v, pos, freqs, kc, vc, slots, q_out=q)
    assert torch.equal(q, want) and torch.equal(kc, kc2) and torch.equal(vc, vc2)


def test_slots_that_are_not_written():
    q, k, v, pos, kc, vc, slots = inputs(6, 4, 2, 64, "bf16", "bf16", 8, 9)
    freqs, _ = attn.rope_freqs(64)
    whole = attn.rope_kv(q, k, v, pos, freqs, kc.clone(), vc.clone(), slots)
    for bad, word in ((-1, 0), (-2, ffi.STATUS_BAD_SLOT), (kc.shape[0] * 8, ffi.STATUS_BAD_SLOT), (1 << 40, ffi.STATUS_BAD_SLOT), (-(1 << 63), ffi.STATUS_BAD_SLOT)):
        s = slots.clone()
        s[2] = bad
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        k1, v1, k2, v2 = kc.clone(), vc.clone(), kc.clone(), vc.clone()
        out = attn.rope_kv(q, k, v, pos, freqs, k1, v1, s, status=status)
        assert ffi.status_read(status) == word and torch.equal(out, whole)
        keep = [0, 1, 3, 4, 5]
        attn.rope_kv(q[keep], k[keep], v[keep], pos[keep], freqs, k2, v2, slots[keep])
        assert torch.equal(k1, k2) and torch.equal(v1, v2)


def test_nan_and_infinity_stay_in_their_columns():
    q, k, v, pos, kc, vc, slots = inputs(4, 2, 1, 64, "bf16", "bf16", 8, 10, start=77)
    freqs, _ = attn.rope_freqs(32)
    clean = attn.rope_kv(q, k, v, pos, freqs, kc, vc, slots)
    q = q.clone()
    q[1, 0, 3], q[2, 1, 60] = float("nan"), float("inf")
    out = attn.rope_kv(q, k, v, pos, freqs, kc, vc, slots)
    assert out[1, 0, [3, 19]].isnan().all() and out[2, 1, 60] == float("inf")
    out[1, 0, [3, 19]], out[2, 1, 60] = clean[1, 0, [3, 19]], clean[2, 1, 60]
    assert torch.equal(out, clean)


def test_captured_and_replayed():
    q, k, v, pos, kc, vc, slots = inputs(5, 8, 2, 128, "f32", "bf16", 16, 11)
    freqs, _ = attn.rope_freqs(128)
    out = torch.empty(5, 8, 128, dtype=torch.bfloat16, device="cuda")
    attn.rope_kv(q, k, v, pos, freqs, kc, vc, slots, q_out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        attn.rope_kv(q, k, v, pos, freqs, kc, vc, slots, q_out=out)
    for step in range(3):
        pos += 1
        slots.copy_((slots + 1) % (kc.shape[0] * 16))
        kc.zero_(), vc.zero_()
        g.replay()
        k2, v2 = torch.zeros_like(kc), torch.zeros_like(vc)
        want = attn.rope_kv(q, k, v, pos, freqs, k2, v2, slots)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(kc, k2) and torch.equal(vc, v2)
