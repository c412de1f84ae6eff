"""Calls whose rows see six keys of like weight, for tests of what a score goes
through: an error of a probability then shows in the output."""
from __future__ import annotations

import torch

from attn_cases import DT

WINDOW = 6
CASES = [dict(), dict(scale=-0.1), dict(softcap=0.3), dict(softcap=2.0), dict(softcap=20.0), dict(softcap=50.0), dict(softcap=128.0), dict(softcap=129.0),
         dict(softcap=1e4), dict(softcap=1e7), dict(softcap=1e30), dict(slopes=True), dict(softcap=2.0, slopes=True), dict(softcap=1e5, slopes=True)]


def inputs(dim, kind, t, length, heads, kv=1, seed=17):
    """q [t, heads, dim], k and v [length, kv, dim] on the CPU, scores of about 1 at the usual scale."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(t, heads, dim, generator=g)
    k, v = torch.randn(length, kv, dim, generator=g), torch.randn(length, kv, dim, generator=g)
    return q.to(DT[kind]), k.to(DT[kind]), v.to(DT[kind])
