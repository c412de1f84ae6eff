"""Scores, caps and biases of attn.decode and attn.prefill against the definition in 64
bits, with a tolerance that follows each key's own error (tests/attn_bounds.py), on
rows that see six keys."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import attn_bounds as B  # noqa: E402
import attn_ref as R  # noqa: E402
from attn_cases import DT, ints, pool, queries  # noqa: E402
from attn_scores import CASES, WINDOW  # noqa: E402
from r9v_amd import attn  # noqa: E402

pytestmark = pytest.mark.gpu


def check(out, q, k, v, table, lengths, new, decode, scale=None, softcap=0.0, slopes=None, window=0):
    """out and q [rows, heads, dim], the sequences' rows one after another."""
    _, heads, dim = q.shape
    group = heads // k.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    got, qq = R.f64(out), R.f64(q)
    first = 0
    for i, (n, m) in enumerate(zip(lengths, new)):
        for kvh in range(k.shape[2]):
            kk, vv = R.gathered(k, table[i], n, kvh), R.gathered(v, table[i], n, kvh)
            for h in range(kvh * group, (kvh + 1) * group):
                slope = None if slopes is None else float(slopes[h])
                for t in range(m):
                    p = n - m + t
                    want, tol = B.attention(qq[first + t, h], kk, vv, R.intervals(p, n, 0, window, 0, True), p, scale, softcap, slope, q.dtype, decode)
                    err = np.abs(got[first + t, h] - want)
                    assert (err <= tol).all(), (i, h, t, float(np.nanmax(err / tol)), err.max())
        first += m


@pytest.mark.parametrize("kw", CASES, ids=str)
@pytest.mark.parametrize("dim,kind", [(64, "f16"), (128, "f16"), (128, "bf16"), (256, "f16")])
def test_decode(kw, dim, kind):
    lengths, new = [800, 130, 600, 3], 2
    k, v, table = pool(lengths, 16, 2, dim, DT[kind], 171)
    q = queries((4, new, 6, dim), DT[kind], 172)
    more = dict(kw, window=WINDOW)
    if "slopes" in kw:
        more["slopes"] = torch.linspace(0.5, 0.05, 6, device="cuda")
    out = attn.decode(q, k, v, table, ints(lengths), **more)
    check(out.view(-1, 6, dim), q.view(-1, 6, dim), k, v, table, lengths, [new] * 4, True, **more)


@pytest.mark.parametrize("kw", CASES, ids=str)
@pytest.mark.parametrize("dim,kind", [(64, "f16"), (96, "bf16"), (128, "f16"), (192, "f16"), (256, "bf16")])
def test_prefill(kw, dim, kind):
    lengths, new = [150, 33, 400], [60, 33, 7]
    k, v, table = pool(lengths, 16, 2, dim, DT[kind], 173)
    q = queries((100, 4, dim), DT[kind], 174)
    more = dict(kw, window=WINDOW)
    if "slopes" in kw:
        more["slopes"] = torch.linspace(0.5, 0.05, 4, device="cuda")
    out = attn.prefill(q, k, v, table, ints(lengths), ints(np.concatenate(([0], np.cumsum(new))).tolist()), **more)
    check(out, q, k, v, table, lengths, new, False, **more)


@pytest.mark.parametrize("softcap", [50.0, 1e4, 1e7])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_caps_of_many_keys(softcap, kind):
    """Every key seen, in parts that are joined; scores of up to 50, so that the caps of 50 are reached."""
    k, v, table = pool([2000], 16, 1, 128, DT[kind], 175)
    q = queries((1, 2, 4, 128), DT[kind], 176)
    for scale in (0.09, 1.0):
        out = attn.decode(q, k, v, table, ints([2000]), softcap=softcap, scale=scale)
        check(out[0], q[0], k, v, table, [2000], [2], True, softcap=softcap, scale=scale)
        out = attn.prefill(q[0], k, v, table, ints([2000]), ints([0, 2]), softcap=softcap, scale=scale)
        check(out, q[0], k, v, table, [2000], [2], False, softcap=softcap, scale=scale)


@pytest.mark.parametrize("new", [1, 3])
@pytest.mark.parametrize("score", [17.0, 21.0, 23.0])
def test_a_tail_whose_values_are_large(score, new):
    """One key of value 0, and those behind it that weigh 2^-24 to 2^-33 of it and have values of 60000."""
    for length in (384, 3000):
        k, v, table = pool([length], 16, 1, 64, torch.float16, 177)
        k.mul_(0.0), k.nan_to_num_(0.0)
        v.mul_(0.0).nan_to_num_(0.0).add_(60000.0)
        page = table[0, 0].long()
        k[page, 7, 0, 0] = 1.0
        v[page, 7] = 0.0
        q = torch.zeros(1, new, 2, 64, dtype=torch.float16, device="cuda")
        q[..., 0] = score
        out = attn.decode(q, k, v, table, ints([length]), scale=1.0)
        check(out[0], q[0], k, v, table, [length], [new], True, scale=1.0)
        out = attn.prefill(q[0], k, v, table, ints([length]), ints([0, new]), scale=1.0)
        check(out, q[0], k, v, table, [length], [new], False, scale=1.0)
