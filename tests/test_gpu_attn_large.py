"""Values near the type's largest: attn.decode and attn.prefill against the definition."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import test_gpu_attn_decode as D  # noqa: E402
import test_gpu_attn_prefill as P  # noqa: E402
from attn_cases import DT, ints, pool, queries  # noqa: E402
from r9v_amd import attn  # noqa: E402

pytestmark = pytest.mark.gpu

NAN = float("nan")


def at(table, p, page=16):
    return table[0, p // page].long(), p % page


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("length", [70, 3000])
def test_values_near_the_largest(dim, length):
    """bf16 values of up to 3e38, the scores of later keys above the earlier ones'."""
    k, v, table = pool([length], 16, 1, dim, torch.bfloat16, 185)
    v = (v.float().clamp(-3, 3) * 1e38).to(torch.bfloat16)
    k[..., 0] = torch.where(k[..., 0].isnan(), NAN, 1.0)
    for p in range(length):
        k[at(table, p)[0], at(table, p)[1], 0, 0] = 4.0 * (p // 32) / (length // 32)
    q = queries((2, 4, dim), torch.bfloat16, 186)
    q[..., 0] = 1.0
    scale = dim ** -0.5
    D.check(attn.decode(q[None], k, v, table, ints([length]), scale=scale), q[None], k, v, table, [length], scale=scale)
    P.check(attn.prefill(q, k, v, table, ints([length]), ints([0, 2]), scale=scale), q, k, v, table, [length], [2], scale=scale)
    k[..., 0] *= dim ** 0.5
    for s in (1.0, 2.0):
        D.check(attn.decode(q[None], k, v, table, ints([length]), scale=scale * s), q[None], k, v, table, [length], scale=scale * s)
        P.check(attn.prefill(q, k, v, table, ints([length]), ints([0, 2]), scale=scale * s), q, k, v, table, [length], [2], scale=scale * s)
