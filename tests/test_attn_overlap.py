"""rope_kv's operands among each other's rows: what one projection or one allocation
leaves beside each other is taken, rows that meet are refused.  On the CPU."""
from __future__ import annotations

import shutil

import pytest

import launch_record
from test_attn_abi import APART, rope
from test_fp8_abi import INVALID, lib, refused

H, KV, D, T = 8, 2, 128, 4  # rope()'s sizes; two bytes an element
Q = APART["q"]
ROW = (H + 2 * KV) * D


def in_place(stride, k, v, t=T, q_head=D, k_stride=None, v_stride=None, **kw):
    """q turned in place at Q; k and v `k` and `v` elements behind it."""
    s = (stride, q_head)
    return dict(q_out=Q, k=Q + 2 * k, v=Q + 2 * v, q_stride=s, q_out_stride=s, k_stride=k_stride or (stride, D), v_stride=v_stride or (stride, D), t=t, **kw)


MEET = {
    "k is q's first heads": in_place(ROW, 0, (H + KV) * D),
    "v is q's first heads": in_place(ROW, H * D, 0),
    "k is q's last heads": in_place(ROW, (H - KV) * D, (H + KV) * D),
    "half a head": in_place(ROW, H * D - 64, (H + KV) * D),
    "q's last heads of the token before": in_place(ROW, ROW - KV * D + 8, H * D),
    "q's rows of the next token": in_place(H * D, H * D, 1 << 20),
    "one token": in_place(0, (H - 1) * D, 1 << 20, t=1),
    "one token for all": in_place(ROW, H * D, (H + KV) * D, k_stride=(0, D)),
    "another step of tokens": in_place(ROW, H * D, (H + KV) * D, k_stride=(2 * ROW, D)),
    "heads in turn, k on q": in_place(3 * H * D, 64, 2 * D, q_head=3 * D, k_stride=(3 * H * D, 3 * D), v_stride=(3 * H * D, 3 * D)),
}
BESIDE = {
    "q, k, v": in_place(ROW, H * D, (H + KV) * D),
    "k, v, q": in_place(ROW, -2 * KV * D, -KV * D),
    "k, q, v": in_place(ROW, -KV * D, H * D),
    "one token of q, k, v": in_place(0, H * D, (H + KV) * D, t=1, k_stride=(0, D), v_stride=(8, D)),
    "a head's q, k and v in turn": in_place(3 * H * D, D, 2 * D, q_head=3 * D, k_stride=(3 * H * D, 3 * D), v_stride=(3 * H * D, 3 * D)),
    "one kv head": in_place((H + 2) * D, H * D, (H + 1) * D, kv_heads=1, k_stride=((H + 2) * D, 0), v_stride=((H + 2) * D, 0)),
    "in memory of their own": in_place(H * D, 1 << 20, 1 << 21, k_stride=(0, D), v_stride=(D, D)),
}


@pytest.mark.parametrize("name", MEET)
def test_q_in_place_over_k_or_v(name):
    refused(lib.r9vx_rope_kv_launch, *rope(**MEET[name]), code=INVALID, text="q_out must not overlap k or v")


CHILD = '''
def rope(st, a):
    a = {n: tuple(v) if isinstance(v, list) else v for n, v in a.items()}
    return L.r9vx_rope_kv_launch(ctypes.byref(ffi.RopeKvStatic(**st)), ctypes.byref(ffi.RopeKvArgs(**a)), None)
'''


def accepted(tmp_path, monkeypatch, cases):
    monkeypatch.setattr(launch_record, "CHILD", launch_record.CHILD.replace("out = []\n", CHILD + "out = []\n", 1))
    calls = []
    for kw in cases.values():
        st, a = ({f: list(v) if hasattr(v := getattr(s, f), "_length_") else v for f, _ in s._fields_} for s in rope(**kw))
        calls.append(("rope", dict(st=st, a=a)))
    out = launch_record.record(launch_record.build(tmp_path), calls)
    assert {n: (rc, msg) for n, (rc, msg, _) in zip(cases, out) if rc} == {}
    assert all(len(ls) == 1 for _, _, ls in out)


RECORDS = pytest.mark.skipif(not launch_record.LIB.exists() or shutil.which("gcc") is None, reason="needs the built libr9vx.so and gcc")


@RECORDS
def test_q_in_place_beside_k_and_v(tmp_path, monkeypatch):
    accepted(tmp_path, monkeypatch, BESIDE)


PAGE, PAGES = 16, 10
TOKEN, WHOLE = KV * D, PAGE * KV * D
K = APART["k_cache"]


def caches(v, k_stride, v_stride=None, **kw):
    """v_cache `v` elements behind k_cache."""
    return dict(v_cache=K + 2 * v, k_cache_stride=k_stride, v_cache_stride=v_stride or k_stride, **kw)


DENSE = (WHOLE, TOKEN, D)
MEETING = {
    "a page on": caches(WHOLE, DENSE),
    "a token on": caches(TOKEN, DENSE),
    "a head on": caches(D, DENSE),
    "half a head on": caches(64, (2 * WHOLE, 2 * TOKEN, 2 * D)),
    "the last page is the first": caches((PAGES - 1) * WHOLE, DENSE),
    "another order in the same pages": caches(D, (2 * WHOLE, 2 * TOKEN, 2 * D), (2 * WHOLE, D, PAGE * D)),
    "half of the second's tokens in the first's": caches(PAGE // 2 * TOKEN, (2 * WHOLE, TOKEN, D)),
    "a page before": caches(-WHOLE, DENSE),
}
APART_CACHES = {
    "one after the other": caches(PAGES * WHOLE, DENSE),
    "pages in turn": caches(WHOLE, (2 * WHOLE, TOKEN, D)),
    "pages in turn, values first": caches(-WHOLE, (2 * WHOLE, TOKEN, D)),
    "tokens in turn": caches(TOKEN, (2 * WHOLE, 2 * TOKEN, D)),
    "heads in turn": caches(D, (2 * WHOLE, 2 * TOKEN, 2 * D)),
    "heads first, then tokens in turn": caches(D, (2 * WHOLE, 2 * D, 2 * PAGE * D)),
    "heads first in halves of a page": caches(PAGE * D, (2 * WHOLE, D, 2 * PAGE * D)),
    "tokens and heads of each in an order of its own, pages in turn": caches(WHOLE, (2 * WHOLE, TOKEN, D), (2 * WHOLE, D, PAGE * D)),
    "one kv head, tokens in turn": caches(D, (2 * PAGE * D, 2 * D, 0), kv_heads=1),
    "one page": caches(TOKEN, (0, 2 * TOKEN, D), pages=1),
    "no page": caches(0, DENSE, pages=0),
}


@pytest.mark.parametrize("name", MEETING)
def test_caches_that_meet(name):
    refused(lib.r9vx_rope_kv_launch, *rope(**MEETING[name]), code=INVALID, text="rows of the cache overlap each other")


@RECORDS
def test_caches_beside_each_other(tmp_path, monkeypatch):
    accepted(tmp_path, monkeypatch, APART_CACHES)
