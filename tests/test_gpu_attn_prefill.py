"""attn.prefill against the definition in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import attn_ref as R  # noqa: E402
from attn_cases import DT, ints, pool, queries  # noqa: E402
from r9v_amd import attn, ffi  # noqa: E402

pytestmark = pytest.mark.gpu


def offsets_of(new):
    return ints(np.concatenate(([0], np.cumsum(new))).tolist())


def check(out, q, k, v, table, lengths, new, causal=True, softcap=0.0, slopes=None, window=0, starts=None, prefix=None, scale=None, rows=None):
    """Every row, or `rows` of them spread over each sequence."""
    _, heads, dim = q.shape
    group = heads // k.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    got, qq = R.f64(out), R.f64(q)
    sl = None if slopes is None else slopes.cpu().double().numpy()
    st = None if starts is None else starts.cpu().numpy()
    first = 0
    for i, (n, m) in enumerate(zip(lengths, new)):
        picked = range(m) if rows is None or m <= rows else sorted(set(np.linspace(0, m - 1, rows).astype(int).tolist()))
        for kvh in range(k.shape[2]):
            kk, vv = R.gathered(k, table[i], n, kvh), R.gathered(v, table[i], n, kvh)
            for h in range(kvh * group, (kvh + 1) * group):
                for t in picked:
                    p = n - m + t
                    seen = R.intervals(p, n, 0 if st is None else int(st[first + t]), window, 0 if prefix is None else int(prefix[i]), causal)
                    want, size, s = R.attention(qq[first + t, h], kk, vv, seen, p, scale, softcap, None if sl is None else sl[h])
                    tol = R.bound(want, size, s, dim, n, q.dtype, False)
                    err = np.abs(got[first + t, h] - want)
                    assert (err <= tol).all(), (i, h, t, float(np.nanmax(err / tol)), err.max())
        first += m


CASES = [  # cached before, new tokens, kv, group, dim, page, type
    ([0], [1], 1, 1, 64, 8, "bf16"), ([0], [17], 2, 8, 256, 64, "bf16"), ([0, 5, 0], [0, 3, 0], 1, 2, 128, 16, "f16"),
    ([0, 0, 0, 0], [31, 32, 33, 64], 2, 1, 128, 16, "bf16"), ([40, 0, 63, 64], [65, 127, 128, 129], 1, 3, 96, 32, "f16"),
    ([700], [50], 2, 4, 128, 8, "bf16"), ([1000, 3], [9, 100], 1, 7, 192, 128, "bf16"), ([200], [130], 3, 2, 64, 256, "f16"),
    ([33], [77], 1, 5, 256, 16, "f16"), ([0] * 40, [3] * 40, 1, 4, 64, 8, "bf16"), ([4000], [2], 1, 16, 128, 64, "bf16")]


@pytest.mark.parametrize("before,new,kv,group,dim,page,kind", CASES)
def test_lengths_and_heads(before, new, kv, group, dim, page, kind):
    lengths = [a + b for a, b in zip(before, new)]
    k, v, table = pool(lengths, page, kv, dim, DT[kind], 13)
    q = queries((sum(new), kv * group, dim), DT[kind], 14)
    out = attn.prefill(q, k, v, table, ints(lengths), offsets_of(new))
    check(out, q, k, v, table, lengths, new)


def test_a_long_prompt():
    k, v, table = pool([2300], 64, 1, 128, torch.bfloat16, 15)
    q = queries((2300, 2, 128), torch.bfloat16, 16)
    out = attn.prefill(q, k, v, table, ints([2300]), offsets_of([2300]))
    check(out, q, k, v, table, [2300], [2300], rows=300)


@pytest.mark.parametrize("kw", [dict(softcap=20.0), dict(slopes=True), dict(window=1), dict(window=70), dict(causal=False), dict(causal=False, window=50),
                                dict(prefix=[0, 200, 40]), dict(prefix=[1 << 30, 13, -3]), dict(docs=50), dict(docs=1), dict(docs=64, window=20),
                                dict(softcap=5.0, slopes=True, window=111, prefix=[30, 100, 70], docs=90), dict(causal=False, docs=33), dict(scale=-0.3)])
@pytest.mark.parametrize("dim,kind", [(128, "bf16"), (64, "f16"), (192, "f16")])
def test_scores_and_masks(kw, dim, kind):
    before, new = [64, 0, 7], [150, 220, 40]
    lengths = [a + b for a, b in zip(before, new)]
    k, v, table = pool(lengths, 16, 2, dim, DT[kind], 23)
    q = queries((sum(new), 4, dim), DT[kind], 24)
    more = {n: x for n, x in kw.items() if n != "docs"}
    if "slopes" in kw:
        more["slopes"] = torch.linspace(0.5, 0.01, 4, device="cuda")
    if "docs" in kw:
        more["starts"] = ints([b + t - t % kw["docs"] for b, n in zip(before, new) for t in range(n)])
    call = dict(more, prefix=ints(kw["prefix"])) if "prefix" in kw else more
    out = attn.prefill(q, k, v, table, ints(lengths), offsets_of(new), **call)
    check(out, q, k, v, table, lengths, new, rows=60, **more)


def test_rows_that_see_nothing_are_zero():
    new = [100]
    k, v, table = pool([100], 16, 1, 64, torch.bfloat16, 33)
    q = queries((100, 2, 64), torch.bfloat16, 34)
    starts = [0] * 100
    for t in range(20, 60):
        starts[t] = 100 if t % 2 else 1 << 30  # past the row itself
    out = attn.prefill(q, k, v, table, ints([100]), offsets_of(new), starts=ints(starts))
    assert (out[20:60] == 0).all()
    check(out, q, k, v, table, [100], new, starts=ints(starts))
    out = attn.prefill(q, k, v, table, ints([40]), offsets_of(new))  # 60 rows without a place
    assert (out[:60] == 0).all()
    check(out, q, k, v, table, [40], new)
    assert (attn.prefill(q, k, v, table, ints([0]), offsets_of(new)) == 0).all()


@pytest.mark.parametrize("layout", ["heads", "together"])
def test_strides_and_rows_behind(layout):
    new, lengths = [70, 31], [100, 31]
    k, v, table = pool(lengths, 32, 3, 96, torch.bfloat16, 35, layout)
    q = queries((120, 6, 96), torch.bfloat16, 36, strided=True)
    whole = torch.full((120, 8, 96), 9.0, dtype=torch.bfloat16, device="cuda")
    for off in (offsets_of(new), offsets_of(new) + 5):  # rows before the first sequence too
        whole.fill_(9.0)
        out = attn.prefill(q, k, v, table, ints(lengths), off, out=whole[:, 1:7])
        o = int(off[0])
        check(out[o:o + 101], q[o:o + 101], k, v, table, lengths, new)
        assert (whole[:, 0] == 9.0).all() and (whole[:, 7] == 9.0).all() and (whole[:o] == 9.0).all() and (whole[o + 101:] == 9.0).all()


@pytest.mark.parametrize("before,t_bucket", [(0, 400), (3000, 64)])
def test_a_buckets_row_has_the_same_bits_in_any_batch(before, t_bucket):
    new = [30, 9, 20]
    lengths = [n + before for n in new]
    k, v, table = pool(lengths, 16, 2, 128, torch.bfloat16, 43)
    q = queries((59, 8, 128), torch.bfloat16, 44)
    kw = dict(b_bucket=4, t_bucket=t_bucket, len_bucket=table.shape[1] * 16)
    whole = attn.prefill(q, k, v, table, ints(lengths), offsets_of(new), **kw)
    first = 0
    for i, n in enumerate(new):
        one = attn.prefill(q[first:first + n], k, v, table[i:i + 1], ints(lengths[i:i + 1]), offsets_of([n]), **kw)
        assert torch.equal(one, whole[first:first + n])
        first += n


@pytest.mark.parametrize("dim,before", [(64, 0), (128, 0), (128, 2500), (256, 0)])
@pytest.mark.parametrize("bad,where", [(float("nan"), "v"), (float("inf"), "v"), (float("nan"), "k"), (float("inf"), "k")])
def test_a_key_that_not_all_rows_see_may_be_nan_or_infinite(bad, where, dim, before):
    """Rows before it (causal), rows past its window and rows of other documents keep their bits."""
    new = [150, 60]
    lengths = [150 + before, 60]
    k, v, table = pool(lengths, 16, 1, dim, torch.float16, 53)
    q = queries((210, 2, dim), torch.float16, 54)
    starts = ints([0 if t < 100 else before + 100 for t in range(150)] + [0] * 60)
    for kw in (dict(), dict(window=30), dict(starts=starts)):
        k2, v2 = k.clone(), v.clone()
        p = before + 70
        (v2 if where == "v" else k2)[table[0, p // 16].long(), p % 16, 0, 5] = bad
        clean = attn.prefill(q, k, v, table, ints(lengths), offsets_of(new), **kw)
        out = attn.prefill(q, k2, v2, table, ints(lengths), offsets_of(new), **kw)
        hit = [t for t in range(70, 150) if ("window" not in kw or t < 100) and ("starts" not in kw or t < 100)]
        rest = [t for t in range(210) if t not in hit]
        assert torch.equal(out[rest], clean[rest])
        assert clean.isfinite().all()
        if where == "v":
            assert not out[hit][..., 5].isfinite().any()
            other = [c for c in range(dim) if c != 5]
            assert torch.equal(out[hit][..., other], clean[hit][..., other])
        elif bad != bad:
            assert out[hit].isnan().all()


def test_scores_that_are_no_softmax():
    for n in (60, 3000):
        k, v, table = pool([n], 16, 1, 64, torch.bfloat16, 63)
        k[:, :, :, 0] = torch.where(k[:, :, :, 0].isnan(), float("nan"), 1.0)
        q = queries((10, 4, 64), torch.bfloat16, 64)
        q[..., 0] = 0.0
        clean = attn.prefill(q, k, v, table, ints([n]), offsets_of([10]))
        q[4, 0, 3] = float("nan")
        q[5, 1, 0] = float("inf")
        q[6, 2, 0] = float("-inf")
        out = attn.prefill(q, k, v, table, ints([n]), offsets_of([10]))
        for t, h in ((4, 0), (5, 1), (6, 2)):
            assert out[t, h].isnan().all()
            out[t, h] = clean[t, h]
        assert torch.equal(out, clean)


def test_bad_pages_lengths_and_offsets():
    new, lengths = [40, 50, 60], [100, 50, 2000]
    k, v, table = pool(lengths, 16, 2, 128, torch.bfloat16, 73)
    q = queries((150, 4, 128), torch.bfloat16, 74)
    clean = attn.prefill(q, k, v, table, ints(lengths), offsets_of(new))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    attn.prefill(q, k, v, table, ints(lengths), offsets_of(new), status=status)
    assert ffi.status_read(status) == 0
    for page in (k.shape[0], -1, 1 << 30):
        t = table.clone()
        t[0, 5] = page  # keys 80 .. 95: seen from row 20 of the first sequence on
        status.zero_()
        out = attn.prefill(q, k, v, t, ints(lengths), offsets_of(new), status=status)
        assert ffi.status_read(status) == ffi.STATUS_BAD_PAGE
        assert out[20:40].isnan().all() and torch.equal(out[:20], clean[:20]) and torch.equal(out[40:], clean[40:])
    for n in (-1, table.shape[1] * 16 + 1, -(1 << 31)):
        status.zero_()
        out = attn.prefill(q, k, v, table, ints([100, n, 2000]), offsets_of(new), status=status)
        assert ffi.status_read(status) == ffi.STATUS_BAD_LENGTH
        assert out[40:90].isnan().all() and torch.equal(out[:40], clean[:40]) and torch.equal(out[90:], clean[90:])
    for off in ([0, 40, 90, 151], [0, 40, 30, 150], [-1, 40, 90, 150], [0, 40, 90, 1 << 30], [0, -(1 << 31), (1 << 31) - 1, 150]):
        status.zero_()
        attn.prefill(q, k, v, table, ints(lengths), ints(off), status=status)
        assert ffi.status_read(status) & ffi.STATUS_BAD_LENGTH


def test_captured_and_replayed_with_new_lengths():
    k, v, table = pool([3000, 1500], 16, 2, 128, torch.bfloat16, 103)
    q = queries((64, 8, 128), torch.bfloat16, 104)
    lengths, off = ints([3000, 1500]), offsets_of([40, 24])
    out = torch.empty_like(q)
    attn.prefill(q, k, v, table, lengths, off, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        attn.prefill(q, k, v, table, lengths, off, out=out)
    for n, m in (([3000, 1500], [40, 24]), ([3000, 1500], [1, 63]), ([2000, 7], [60, 0]), ([64, 0], [64, 0])):
        lengths.copy_(ints(n)), off.copy_(offsets_of(m))
        out.fill_(7.0)
        g.replay()
        eager = attn.prefill(q, k, v, table, lengths, off, out=torch.full_like(q, 7.0))
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_on_a_stream_of_its_own():
    k, v, table = pool([3000], 16, 2, 64, torch.float16, 113)
    q = queries((20, 8, 64), torch.float16, 114)
    n, off = ints([3000]), offsets_of([20])
    want = attn.prefill(q, k, v, table, n, off)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = attn.prefill(q, k, v, table, n, off, stream=s)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, want)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("score", [11.0, 17.0])
def test_a_long_tail_of_small_probabilities(kind, score):
    """One key far above 3000 that weigh 2^-16 (2^-24) of it each, which an f16 probability of 1 would not resolve."""
    k, v, table = pool([3001], 16, 1, 64, DT[kind], 131)
    k.mul_(0.0), k.nan_to_num_(0.0)
    k[table[0, 5].long(), 7, 0, 0] = 1.0
    q = torch.zeros(4, 2, 64, dtype=DT[kind], device="cuda")
    q[..., 0] = score
    out = attn.prefill(q, k, v, table, ints([3001]), offsets_of([4]), scale=1.0)
    check(out, q, k, v, table, [3001], [4], scale=1.0)


# Buckets of 6 heads on 2 of kv that pick two halves of the keys a workgroup: of each of several parts, and alone.
HALVES = [1152, 4138]


@pytest.mark.parametrize("t_bucket", HALVES)
@pytest.mark.parametrize("dim,kind", [(64, "bf16"), (96, "f16"), (128, "bf16"), (192, "bf16"), (256, "f16")])
def test_halves_of_the_keys(dim, kind, t_bucket):
    before, new = [1100, 0, 60], [70, 33, 0]
    lengths = [a + b for a, b in zip(before, new)]
    k, v, table = pool(lengths, 16, 2, dim, DT[kind], 141)
    q = queries((sum(new), 6, dim), DT[kind], 142)
    slopes = torch.linspace(0.3, 0.01, 6, device="cuda")
    starts = ints([t // 40 * 40 for t in range(70)] + [0] * 20 + [12] * 13)
    for kw in (dict(), dict(window=300), dict(causal=False), dict(softcap=10.0, slopes=slopes, window=33), dict(starts=starts, prefix=ints([1140, 5, 3]))):
        out = attn.prefill(q, k, v, table, ints(lengths), offsets_of(new), b_bucket=3, t_bucket=t_bucket, **kw)
        check(out, q, k, v, table, lengths, new, rows=20, **kw)


@pytest.mark.parametrize("t_bucket", HALVES)
@pytest.mark.parametrize("length", [1, 31, 64, 65, 128, 129, 500, 513])
def test_halves_of_few_keys(length, t_bucket):
    """From no tile for the second half on."""
    for dim in (128, 256):
        k, v, table = pool([length, 1500], 16, 2, dim, torch.bfloat16, 151)
        q = queries((min(length, 9), 6, dim), torch.bfloat16, 152)
        out = attn.prefill(q, k, v, table[:1], ints([length]), offsets_of([len(q)]), b_bucket=3, t_bucket=t_bucket)
        check(out, q, k, v, table[:1], [length], [len(q)])


@pytest.mark.parametrize("t_bucket", HALVES)
def test_halves_with_faults(t_bucket):
    """NaN where a row sees it or not, pages that are not there, in either half; captured and replayed."""
    before, new = [1000, 0], [60, 100]
    lengths, dim = [1060, 100], 128
    k, v, table = pool(lengths, 16, 2, dim, torch.float16, 161)
    q = queries((160, 6, dim), torch.float16, 162)
    table = torch.cat((table, torch.full((2, 30), -1, dtype=torch.int32, device="cuda")), 1)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    n, off, out = ints(lengths), offsets_of(new), torch.zeros_like(q)

    def call(values, pages, y=None):
        return attn.prefill(q, k, values, pages, n, off, window=500, out=y, status=status, b_bucket=3, t_bucket=t_bucket)

    clean = call(v, table)
    check(clean, q, k, v, table, lengths, new, window=500, rows=20)
    assert ffi.status_read(status) == 0
    for p in (530, 540, 700, 1030, 1059):
        v2 = v.clone()
        v2[table[0, p // 16].long(), p % 16, :, 7] = float("inf")
        y = call(v2, table)
        sees = [t for t in range(60) if 1000 + t >= p > 500 + t]
        rest = [t for t in range(160) if t not in sees]
        assert torch.equal(y[rest], clean[rest]) and (not sees or not y[sees][..., 7].isfinite().any())
        assert torch.equal(y[..., 8:], clean[..., 8:])
    assert ffi.status_read(status) == 0
    for page in (40, 50, 60, 66):
        t2 = table.clone()
        t2[0, page] = k.shape[0]
        status.zero_()
        y = call(v, t2)
        assert ffi.status_read(status) == ffi.STATUS_BAD_PAGE
        sees = [t for t in range(60) if 16 * page <= 1000 + t and 16 * page + 15 > 500 + t]
        rest = [t for t in range(160) if t not in sees]
        assert y[sees].isnan().all() and torch.equal(y[rest], clean[rest])
    status.zero_()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(v, table, out)
    for lens in (lengths, [60, 100], [1060, 100]):
        n.copy_(ints(lens))
        out.zero_()
        g.replay()
        want = call(v, table)
        assert torch.equal(out, want)
    assert torch.equal(out, clean) and ffi.status_read(status) == 0
