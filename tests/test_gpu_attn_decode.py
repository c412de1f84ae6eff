"""attn.decode against the definition in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import attn_ref as R  # noqa: E402
from attn_cases import DT, ints, pool, queries  # noqa: E402
from r9v_amd import attn, ffi  # noqa: E402

pytestmark = pytest.mark.gpu


def check(out, q, k, v, table, lengths, softcap=0.0, slopes=None, window=0, starts=None, scale=None, skip=()):
    b, new, heads, dim = q.shape
    group = heads // k.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    got, qq = R.f64(out), R.f64(q)
    sl = None if slopes is None else slopes.cpu().double().numpy()
    for i in range(b):
        if i in skip:
            continue
        n = int(lengths[i])
        for kvh in range(k.shape[2]):
            kk, vv = R.gathered(k, table[i], n, kvh), R.gathered(v, table[i], n, kvh)
            for h in range(kvh * group, (kvh + 1) * group):
                for t in range(new):
                    p = n - new + t
                    seen = R.intervals(p, n, 0 if starts is None else int(starts[i]), window, 0, True)
                    want, size, s = R.attention(qq[i, t, h], kk, vv, seen, p, scale, softcap, None if sl is None else sl[h])
                    tol = R.bound(want, size, s, dim, n, q.dtype, q.dtype == torch.bfloat16)
                    err = np.abs(got[i, t, h] - want)
                    assert (err <= tol).all(), (i, h, t, float(np.nanmax(err / tol)), err.max())


CASES = [  # lengths, new, kv, group, dim, page, type
    ([1], 1, 1, 1, 64, 8, "bf16"), ([0, 3, 0, 32, 33], 1, 2, 4, 128, 16, "bf16"), ([31, 64, 65, 127, 128, 129], 1, 1, 7, 64, 32, "f16"),
    ([517], 1, 2, 8, 256, 64, "bf16"), ([700, 5], 5, 2, 8, 256, 16, "bf16"), ([300, 1, 2], 4, 3, 3, 96, 8, "f16"),
    ([1000], 8, 1, 16, 128, 128, "bf16"), ([2049, 2048, 7], 1, 4, 1, 192, 256, "f16"), ([400, 90], 3, 2, 5, 192, 32, "bf16"),
    ([5000], 1, 1, 4, 64, 16, "f16"), ([260, 259], 2, 8, 12, 128, 64, "f16"), ([7], 8, 2, 2, 96, 8, "bf16"), ([40] * 70, 1, 4, 2, 64, 8, "bf16")]


@pytest.mark.parametrize("lengths,new,kv,group,dim,page,kind", CASES)
def test_lengths_and_heads(lengths, new, kv, group, dim, page, kind):
    k, v, table = pool(lengths, page, kv, dim, DT[kind], 11)
    q = queries((len(lengths), new, kv * group, dim), DT[kind], 12)
    out = attn.decode(q, k, v, table, ints(lengths))
    check(out, q, k, v, table, lengths)


@pytest.mark.parametrize("kw", [dict(softcap=20.0), dict(softcap=0.3), dict(slopes=True), dict(window=1), dict(window=70), dict(window=1 << 31),
                                dict(starts=[0, 100, 900, 37]), dict(softcap=5.0, slopes=True, window=333, starts=[3, 0, 599, 601]), dict(scale=0.5),
                                dict(scale=0.0), dict(scale=-0.2)])
@pytest.mark.parametrize("new,dim,kind", [(1, 128, "bf16"), (5, 64, "f16")])
def test_scores_and_masks(kw, new, dim, kind):
    lengths = [800, 130, 600, 37]
    k, v, table = pool(lengths, 16, 2, dim, DT[kind], 21)
    q = queries((4, new, 6, dim), DT[kind], 22)
    more = dict(kw)
    if "slopes" in kw:
        more["slopes"] = torch.linspace(0.5, 0.01, 6, device="cuda")
    if "starts" in kw:
        more["starts"] = ints(kw["starts"])
    out = attn.decode(q, k, v, table, ints(lengths), **more)
    check(out, q, k, v, table, lengths, **{**more, "starts": kw.get("starts")})


@pytest.mark.parametrize("layout", ["heads", "together"])
def test_strides(layout):
    lengths = [77, 300]
    k, v, table = pool(lengths, 32, 3, 96, torch.bfloat16, 31, layout)
    wide = torch.full((2, 40), -5, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    q = queries((2, 2, 6, 96), torch.bfloat16, 32, strided=True)
    whole = torch.full((2, 2, 8, 96), 9.0, dtype=torch.bfloat16, device="cuda")
    out = attn.decode(q, k, v, wide, ints(lengths), out=whole[:, :, 1:7], len_bucket=300)
    check(out, q, k, v, table, lengths)
    assert (whole[:, :, 0] == 9.0).all() and (whole[:, :, 7] == 9.0).all()


def test_a_buckets_row_has_the_same_bits_in_any_batch():
    lengths = [3000, 45, 800]
    k, v, table = pool(lengths, 16, 2, 128, torch.bfloat16, 41)
    q = queries((3, 2, 8, 128), torch.bfloat16, 42)
    whole = attn.decode(q, k, v, table, ints(lengths), b_bucket=4, len_bucket=3000)
    for i in range(3):
        one = attn.decode(q[i:i + 1], k, v, table[i:i + 1], ints(lengths[i:i + 1]), b_bucket=4, len_bucket=3000)
        assert torch.equal(one[0], whole[i])


def test_a_key_that_drafts_do_not_all_see_may_be_nan_or_infinite():
    """Each draft's own key is seen by it and those behind it alone."""
    lengths = [200, 333]
    for bad, where in ((float("nan"), "v"), (float("inf"), "v"), (float("nan"), "k"), (float("-inf"), "v")):
        k, v, table = pool(lengths, 16, 1, 64, torch.float16, 51)
        q = queries((2, 4, 2, 64), torch.float16, 52)
        p = lengths[1] - 2  # seen by the last two of four tokens
        cache = v if where == "v" else k
        clean = attn.decode(q, k, v, table, ints(lengths))
        cache[table[1, p // 16].long(), p % 16, 0, 5] = bad
        out = attn.decode(q, k, v, table, ints(lengths))
        assert torch.equal(out[0], clean[0]) and torch.equal(out[1, :2], clean[1, :2])
        hit = out[1, 2:]
        if where == "k":
            assert hit.isnan().all()
        else:
            assert not hit[..., 5].isfinite().any() and torch.equal(hit[..., 6:], clean[1, 2:, :, 6:])


@pytest.mark.parametrize("length", [40, 4000])
def test_scores_that_are_no_softmax(length):
    """A NaN row of q, +infinity, and -infinity alone; the other heads as they were."""
    k, v, table = pool([length], 16, 1, 64, torch.bfloat16, 61)
    q = queries((1, 1, 4, 64), torch.bfloat16, 62)
    clean = attn.decode(q, k, v, table, ints([length]))
    k[:, :, :, 0] = torch.where(k[:, :, :, 0].isnan(), float("nan"), 1.0)
    q[..., 0] = 0.0
    clean = attn.decode(q, k, v, table, ints([length]))
    q[0, 0, 0, 3] = float("nan")
    q[0, 0, 1, 0] = float("inf")
    q[0, 0, 2, 0] = float("-inf")
    out = attn.decode(q, k, v, table, ints([length]))
    assert out[0, 0, :3].isnan().all() and torch.equal(out[0, 0, 3], clean[0, 0, 3])


def test_bad_pages_and_lengths():
    lengths = [100, 90, 80, 70, 2000]
    k, v, table = pool(lengths, 16, 2, 128, torch.bfloat16, 71)
    q = queries((5, 1, 4, 128), torch.bfloat16, 72)
    clean = attn.decode(q, k, v, table, ints(lengths))
    for word, change in ((ffi.STATUS_BAD_PAGE, (1, 3, k.shape[0])), (ffi.STATUS_BAD_PAGE, (1, 0, -1)), (ffi.STATUS_BAD_PAGE, (1, 5, 1 << 30)),
                         (ffi.STATUS_BAD_LENGTH, -1), (ffi.STATUS_BAD_LENGTH, table.shape[1] * 16 + 1), (ffi.STATUS_BAD_LENGTH, -(1 << 31))):
        t, n = table.clone(), list(lengths)
        if word == ffi.STATUS_BAD_PAGE:
            t[change[0], change[1]] = change[2]
        else:
            n[1] = change
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = attn.decode(q, k, v, t, ints(n), status=status)
        assert ffi.status_read(status) == word
        assert out[1].isnan().all()
        keep = [0, 2, 3, 4]
        assert torch.equal(out[keep], clean[keep])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    bad = table.clone()
    bad[0, :3] = -7  # pages before the window, given up
    out = attn.decode(q, k, v, bad, ints(lengths), window=50, status=status)
    assert ffi.status_read(status) == 0 and torch.equal(out, attn.decode(q, k, v, table, ints(lengths), window=50))


def test_rows_behind_the_batch_are_left():
    k, v, table = pool([50, 60], 16, 1, 64, torch.bfloat16, 81)
    q = queries((2, 1, 2, 64), torch.bfloat16, 82)
    whole = torch.full((4, 1, 2, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    attn.decode(q, k, v, table, ints([50, 60]), out=whole[:2], b_bucket=4)
    assert (whole[2:] == 3.0).all()
    empty = attn.decode(q[:0], k, v, table[:0], ints([]))
    assert empty.shape == (0, 1, 2, 64)


def test_a_cache_past_32_bits_of_elements():
    """Pages 2^31 elements apart."""
    lengths, page, kv, dim = [40, 23], 16, 1, 64
    k, v, table = pool(lengths, page, kv, dim, torch.bfloat16, 91)
    step = 1 << 31
    big = torch.empty((k.shape[0] - 1) * step + 2 * page * kv * dim, dtype=torch.bfloat16, device="cuda")
    at = [torch.as_strided(big, k.shape, (step, kv * dim, dim, 1), o) for o in (0, page * kv * dim)]
    at[0].copy_(k), at[1].copy_(v)
    q = queries((2, 1, 4, dim), torch.bfloat16, 92)
    out = attn.decode(q, at[0], at[1], table, ints(lengths))
    assert torch.equal(out, attn.decode(q, k, v, table, ints(lengths)))


def test_captured_and_replayed_with_new_lengths():
    """One workspace for two graphs, each replayed in turn with eager calls between."""
    k, v, table = pool([3000, 1500], 16, 2, 128, torch.bfloat16, 101)
    q = queries((2, 1, 8, 128), torch.bfloat16, 102)
    lengths = ints([3000, 1500])
    st = ffi.AttnStatic(2, 1, 3008, 8, 2, 128, 16, ffi.BF16, 1, 0, attn._bits(128 ** -0.5), 0)
    need = attn.decode_workspace_bytes(st)
    assert need > 0
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    outs, graphs = [torch.empty_like(q) for _ in range(2)], []
    calls = [lambda: attn.decode(q, k, v, table, lengths, out=outs[0], workspace=ws),
             lambda: attn.decode(q, k, v, table, lengths, out=outs[1], workspace=ws, window=900)]
    for call in calls:
        call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        graphs.append(g)
    for n in ([3000, 1500], [1, 0], [2999, 64], [3000, 1500]):
        lengths.copy_(ints(n))
        for i, g in enumerate(graphs):
            outs[i].zero_()
            g.replay()
        eager = [attn.decode(q, k, v, table, lengths, window=w) for w in (0, 900)]
        torch.cuda.synchronize()
        assert torch.equal(outs[0], eager[0]) and torch.equal(outs[1], eager[1])


def test_on_a_stream_of_its_own():
    k, v, table = pool([3000], 16, 2, 64, torch.float16, 111)
    q = queries((1, 1, 8, 64), torch.float16, 112)
    n = ints([3000])
    want = attn.decode(q, k, v, table, n)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = attn.decode(q, k, v, table, n, stream=s)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, want)


@pytest.mark.parametrize("lengths,new,kv,group,dim,kind", [([900, 33, 2100, 0], 4, 2, 8, 256, "bf16"), ([1, 1500, 64, 310], 6, 2, 6, 192, "f16"),
                                                           ([520, 17, 6, 95], 8, 2, 7, 256, "f16"), ([40, 2000, 31, 33], 3, 2, 6, 192, "bf16")])
def test_wide_heads_of_many_rows_with_room_for_long_sequences(lengths, new, kv, group, dim, kind):
    """A table of 16384 places: what picks the kernel is the room, not the lengths."""
    k, v, table = pool(lengths, 64, kv, dim, DT[kind], 121)
    wide = torch.full((len(lengths), 256), -9, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    q = queries((len(lengths), new, kv * group, dim), DT[kind], 122)
    out = attn.decode(q, k, v, wide, ints(lengths))
    check(out, q, k, v, table, lengths)
    out = attn.decode(q, k, v, wide, ints(lengths), scale=-0.1, starts=ints([20, 0, 64, 3]), softcap=9.0)
    check(out, q, k, v, table, lengths, scale=-0.1, starts=[20, 0, 64, 3], softcap=9.0)


def test_a_long_tail_of_small_probabilities():
    """One key far above 3000 that weigh 2^-16 of it each: below the steps of an f16 probability of 1, a twentieth of the sum."""
    for kind, new in (("f16", 1), ("bf16", 1), ("f16", 3)):
        k, v, table = pool([3001], 16, 1, 64, DT[kind], 131)
        k.mul_(0.0), k.nan_to_num_(0.0)
        k[table[0, 5].long(), 7, 0, 0] = 1.0
        q = torch.zeros(1, new, 2, 64, dtype=DT[kind], device="cuda")
        q[..., 0] = 11.0
        out = attn.decode(q, k, v, table, ints([3001]), scale=1.0)
        check(out, q, k, v, table, [3001], scale=1.0)
