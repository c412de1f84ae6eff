"""Inputs of the attention tests, on the GPU: sequences in shuffled pages of a pool
whose every other place holds NaN."""
from __future__ import annotations

import torch

DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def pool(lengths, page, kv, dim, dtype, seed, layout="pages", spare=2, scale=1.0):
    """(k_cache, v_cache, table): sequence i holds lengths[i] random tokens, NaN behind them and in the spare pages."""
    g = torch.Generator().manual_seed(seed)
    per = [-(-n // page) for n in lengths]
    pages, cols = sum(per) + spare, max(max(per), 1)
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(lengths), cols), -1, dtype=torch.int32)  # a column that nobody needs names no page
    caches = [torch.full((pages, page, kv, dim), float("nan"), dtype=dtype) for _ in range(2)]
    at = 0
    for i, n in enumerate(lengths):
        own = order[at:at + per[i]]
        at += per[i]
        table[i, :per[i]] = own.int()
        for c in caches:
            rows = torch.full((per[i] * page, kv, dim), float("nan"), dtype=dtype)
            rows[:n] = (scale * torch.randn(n, kv, dim, generator=g)).to(dtype)
            c[own] = rows.view(per[i], page, kv, dim)
    k, v = (c.cuda() for c in caches)
    if layout == "heads":  # [pages, kv, page, dim]
        k, v = (c.transpose(1, 2).contiguous().transpose(1, 2) for c in (k, v))
    if layout == "together":  # one allocation
        both = torch.stack((k, v), 1)
        k, v = both[:, 0], both[:, 1]
    return k, v, table.cuda()


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def queries(shape, dtype, seed, strided=False):
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(shape, generator=g).to(dtype)
    if strided:  # a view of wider rows
        wide = torch.full((*shape[:-2], shape[-2] + 3, shape[-1]), float("nan"), dtype=dtype)
        wide[..., 1:1 + shape[-2], :] = q
        return wide.cuda()[..., 1:1 + shape[-2], :]
    return q.cuda()
