"""moe_route_group on the GPU against its definition in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

from r9v_amd import ffi

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def reference(logits, k, groups, topk_group, bias=None, sigmoid=True, top2=True, renormalize=True, scale=1.0):
    l = logits.astype(np.float64)
    t, e = l.shape
    with np.errstate(over="ignore"):
        if sigmoid:
            s = 1.0 / (1.0 + np.exp(-l))
        else:
            p = np.exp(l - l.max(axis=1, keepdims=True))
            s = p / p.sum(axis=1, keepdims=True)
    c = s + (0.0 if bias is None else bias.astype(np.float64))
    per = np.sort(c.reshape(t, groups, -1), axis=2)[:, :, ::-1]
    score = per[:, :, :2 if top2 else 1].sum(axis=2)
    kept = np.argsort(-score, axis=1, kind="stable")[:, :topk_group]
    mask = np.zeros((t, groups), bool)
    np.put_along_axis(mask, kept, True, axis=1)
    c = np.where(np.repeat(mask, e // groups, axis=1), c, -np.inf)
    ids = np.argsort(-c, axis=1, kind="stable")[:, :k]
    w = np.take_along_axis(s, ids, axis=1)
    if renormalize:
        w = w / w.sum(axis=1, keepdims=True)
    return ids, w * scale


def check(logits, k, groups, topk_group, bias=None, sigmoid=True, top2=True, renormalize=True, scale=1.0):
    want_i, want_w = reference(logits, k, groups, topk_group, bias, sigmoid, top2, renormalize, scale)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ids, w = ffi.moe_route_group(dev(logits), k, groups, topk_group, bias=None if bias is None else dev(bias),
                                 scoring=ffi.SCORING_SIGMOID if sigmoid else ffi.SCORING_SOFTMAX,
                                 group_score=ffi.GROUP_TOP2 if top2 else ffi.GROUP_MAX, renormalize=renormalize, scale=scale,
                                 status=status)
    assert np.array_equal(ids.cpu().numpy(), want_i)
    # one rounding to f32 of weights whose f32 parts are each within a few steps of 2^-24;
    # below 2^-126 f32 numbers stand 2^-149 apart, so half of that is a rounding there
    w = w.cpu().numpy()
    assert np.allclose(w, want_w, rtol=8 * 2.0 ** -24, atol=2.0 ** -150)
    assert ffi.status_read(status) == 0


SHAPES = [(1, 8, 1, 1, 1), (5, 256, 8, 4, 8), (3, 1024, 32, 5, 32), (7, 60, 4, 2, 6), (33, 160, 8, 3, 6), (2, 64, 1, 1, 8),
          (4, 512, 8, 3, 10), (9, 1024, 1, 1, 32), (6, 130, 2, 1, 3), (5, 128, 64, 7, 9), (300, 72, 3, 3, 4), (2, 2, 1, 1, 2),
          (3, 1000, 50, 1, 20)]


@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("top2", [False, True])
@pytest.mark.parametrize("t,e,groups,topk_group,k", SHAPES)
def test_route_group(t, e, groups, topk_group, k, top2, sigmoid, biased):
    r = np.random.default_rng(t * 7 + e + k)
    logits = (2 * r.standard_normal((t, e))).astype(np.float32)
    bias = (0.1 * r.standard_normal(e)).astype(np.float32) if biased else None
    check(logits, k, groups, topk_group, bias, sigmoid, top2, renormalize=t % 2 == 1, scale=2.5)


@pytest.mark.parametrize("sigmoid", [False, True])
def test_equal_scores_go_to_the_lower_index(sigmoid):
    logits = np.zeros((4, 96), np.float32)
    logits[1, 40:] = 1.0
    logits[2] = np.repeat(np.arange(8)[::-1], 12) % 3
    logits[3, ::5] = 2.0
    for bias in (None, np.zeros(96, np.float32), np.full(96, -0.5, np.float32)):
        for top2 in (False, True):
            check(logits, 9, 8, 3, bias, sigmoid, top2)
            check(logits, 12, 1, 1, bias, sigmoid, False)


@pytest.mark.parametrize("sigmoid", [False, True])
def test_scores_that_f32_cannot_tell_apart(sigmoid):
    """Biases that undo the scores' differences to 1e-9: f32 sums of them tie or
    swap, f64 ones do not."""
    r = np.random.default_rng(8)
    t, e = 64, 128
    row = r.standard_normal(e).astype(np.float32)
    s = 1 / (1 + np.exp(-row.astype(np.float64))) if sigmoid else np.exp(row.astype(np.float64)) / np.exp(row.astype(np.float64)).sum()
    bias = (0.75 - s).astype(np.float32)
    logits = np.repeat(row[None], t, axis=0)
    logits += (np.arange(t)[:, None] * 2.0 ** -20).astype(np.float32) * (r.random((t, e)) < 0.3)
    for groups, topk_group, top2 in ((1, 1, False), (8, 3, True), (8, 3, False)):
        check(logits, 8, groups, topk_group, bias, sigmoid, top2)


def test_masked_experts_and_far_logits():
    r = np.random.default_rng(9)
    logits = (30 * r.standard_normal((16, 64))).astype(np.float32)
    bias = np.zeros(64, np.float32)
    bias[r.random(64) < 0.6] = -np.finfo(np.float32).max
    check(logits, 8, 8, 2, bias)
    check(logits, 8, 8, 8, bias, top2=False)
    check(logits, 4, 4, 1, None, sigmoid=False, top2=False)


def test_bad_rows_are_refused_alone():
    r = np.random.default_rng(10)
    logits = r.standard_normal((9, 128)).astype(np.float32)
    want_i, want_w = reference(logits, 8, 4, 2)
    bad = logits.copy()
    bad[2, 5], bad[4, 127], bad[8, 0] = np.nan, np.inf, -np.inf
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ids, w = ffi.moe_route_group(dev(bad), 8, 4, 2, status=status)
    ids, w = ids.cpu().numpy(), w.cpu().numpy()
    assert ffi.status_read(status) == ffi.STATUS_NONFINITE
    rest = [0, 1, 3, 5, 6, 7]
    assert np.array_equal(ids[rest], want_i[rest]) and (ids[[2, 4, 8]] == -1).all() and (w[[2, 4, 8]] == 0).all()
    # every score of a row underflows: a zero sum
    low = logits.copy()
    low[3] = -1000.0
    ids, w = ffi.moe_route_group(dev(low), 8, 4, 2, status=status)
    assert ffi.status_read(status) == ffi.STATUS_NONFINITE | ffi.STATUS_DEGENERATE  # or-ed into what is there
    assert (ids[3] == -1).all() and (ids[2] >= 0).all()
    ids, w = ffi.moe_route_group(dev(low), 8, 4, 2, renormalize=False)
    assert (ids[3] >= 0).all() and (w[3] == 0).all()
    ids, _ = ffi.moe_route_group(dev(bad), 8, 4, 2)  # no status word
    assert (ids[2] == -1).all()


def test_bad_bias_refuses_every_row():
    logits, bias = np.zeros((3, 16), np.float32), np.zeros(16, np.float32)
    bias[9] = np.nan
    ids, _ = ffi.moe_route_group(dev(logits), 4, 2, 1, bias=dev(bias))
    assert (ids == -1).all()


def test_rows_behind_the_last_are_left():
    ids = torch.full((6, 4), 77, dtype=torch.int32, device="cuda")
    w = torch.full((6, 4), 7.0, device="cuda")
    ffi.moe_route_group(dev(np.random.default_rng(1).standard_normal((4, 32)).astype(np.float32)), 4, 4, 2, ids=ids[:4], weights=w[:4])
    assert (ids[4:] == 77).all() and (w[4:] == 7.0).all() and (ids[:4] < 32).all()


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("biased", [False, True])
def test_many_rows(sigmoid, biased):
    r = np.random.default_rng(12)
    logits = (3 * r.standard_normal((1531, 192))).astype(np.float32)
    bias = (0.3 * r.standard_normal(192)).astype(np.float32) if biased else None
    check(logits, 6, 12, 5, bias, sigmoid)
    check(logits, 6, 12, 5, bias, sigmoid, top2=False, renormalize=False)


def neighbours(start, n, step=1):
    """n f32 values, `step` representable steps apart."""
    return (np.float32(start).view(np.int32) + step * np.arange(n, dtype=np.int32)).view(np.float32)


@pytest.mark.parametrize("start", [1e-30, 0.1, 3.0, 15.9, 20.0, 25.0, 31.0, 36.0, 40.0, 80.0, -3.0, -15.9, -80.0, -590.0, -700.0])
def test_neighbouring_logits(start):
    """Logits that f64 scores tell apart, or round to one value (sigmoid near 1)."""
    r = np.random.default_rng(13)
    logits = np.stack([r.permutation(neighbours(start, 64, step)) for step in (1, 1, 2, 5, 40, 300)])
    for groups, topk_group in ((1, 1), (8, 3)):
        check(logits, 8, groups, topk_group, None, sigmoid=True, top2=False)
    check(logits, 8, 1, 1, None, sigmoid=False, top2=False)


def test_group_sums_that_cancel():
    """A group's two keys of a thousand and of opposite signs: their sum is small, its error is not."""
    r = np.random.default_rng(14)
    logits = r.standard_normal((200, 16)).astype(np.float32)
    bias = np.tile(np.array([1000.0, -1000.0], np.float32), 8) + r.standard_normal(16).astype(np.float32) * np.float32(2e-4)
    check(logits, 4, 8, 3, bias, sigmoid=True)
    check(logits, 4, 8, 3, bias, sigmoid=False)
