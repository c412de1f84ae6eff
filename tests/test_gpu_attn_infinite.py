"""Infinite values that a row sees: an infinite value of any probability is the sum,
two of opposite signs or a NaN make it a NaN, and other columns keep their bits."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from attn_cases import DT, ints, pool, queries  # noqa: E402
from r9v_amd import attn  # noqa: E402

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


def at(table, p, page=16):
    return table[0, p // page].long(), p % page


def calls(q, k, v, table, n, **kw):
    """decode's and prefill's outputs of the last q.shape[0] tokens of n."""
    new = q.shape[0]
    return {"decode": attn.decode(q[None], k, v, table, ints([n]), **kw)[0], "prefill": attn.prefill(q, k, v, table, ints([n]), ints([0, new]), **kw)}


def plant(v, table, columns):
    """columns: {column: [(position, value)]}"""
    v = v.clone()
    for c, places in columns.items():
        for p, x in places:
            page, place = at(table, p)
            v[page, place, 0, c] = x
    return v


COLUMNS = {1: [(0, INF)], 2: [(37, -INF)], 3: [(5, INF), (90, INF)], 4: [(5, INF), (90, -INF)], 6: [(40, NAN)], 7: [(40, NAN), (41, INF)]}
WANT = {1: INF, 2: -INF, 3: INF, 4: NAN, 6: NAN, 7: NAN}


@pytest.mark.parametrize("length", [91, 3000])
@pytest.mark.parametrize("new", [1, 3])
@pytest.mark.parametrize("dim,kind", [(64, "bf16"), (64, "f16"), (128, "bf16"), (256, "bf16"), (192, "f16")])
def test_infinite_values_that_all_rows_see(dim, kind, new, length):
    k, v, table = pool([length], 16, 1, dim, DT[kind], 181)
    q = queries((new, 4, dim), DT[kind], 182)
    if new > 1:
        length -= 1  # position 90 is then the last one before the last row: some rows do not see it
    clean = calls(q, k, v, table, length)
    for name, out in calls(q, k, plant(v, table, COLUMNS), table, length).items():
        rest = [c for c in range(dim) if c not in COLUMNS]
        assert torch.equal(out[..., rest], clean[name][..., rest]), name
        for t in range(new):
            for c, want in WANT.items():
                sees = [x for p, x in COLUMNS[c] if p <= length - new + t]
                want = sum(sees) if sees else None
                got = out[t, :, c]
                if want is None:
                    assert torch.equal(got, clean[name][t, :, c])
                elif want != want:
                    assert got.isnan().all(), (name, t, c, got)
                else:
                    assert (got == want).all(), (name, t, c, got)


@pytest.mark.parametrize("far", [3.0, 30.0, 90.0, 400.0])
@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("length", [100, 3000])
def test_infinite_values_of_small_probability(length, kind, first, far):
    """The key's score is `far` below the others', which come behind it or before it."""
    k, v, table = pool([length], 16, 1, 64, DT[kind], 183)
    k.nan_to_num_(0.0).mul_(0.0)
    k[..., 0] = 1.0
    p = 3 if first else length - 5
    k[at(table, p)[0], at(table, p)[1], 0, 0] = 0.0
    q = torch.zeros(2, 2, 64, dtype=DT[kind], device="cuda")
    q[..., 0] = far
    v2 = plant(v, table, {9: [(p, -INF)]})
    clean = calls(q, k, v, table, length, scale=1.0)
    for name, out in calls(q, k, v2, table, length, scale=1.0).items():
        assert (out[..., 9] == -INF).all(), (name, out[..., 9])
        rest = [c for c in range(64) if c != 9]
        assert torch.equal(out[..., rest], clean[name][..., rest]), name
