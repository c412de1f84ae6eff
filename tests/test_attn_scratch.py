"""The attention kernels take next to no scratch memory, which the runtime allocates for
every lane of the card at a first launch: 390 to 480 MB for a second way that was a
function of its own.  Heads of 256 columns spill some registers of a prompt's."""
from __future__ import annotations

import pytest

from r9v_amd import build as B


@pytest.mark.parametrize("kernel", ["attn_prefill_kernel", "attn_decode_kernel"])
def test_scratch(kernel):
    src = B.CSRC / f"{kernel.rsplit('_', 1)[0]}.hip"
    _, res = B._reuse(src) if B._up_to_date(src) else B._compile(src)
    found = {n: r for n, r in res.items() if kernel in n}
    assert len(found) >= 16
    for name, r in found.items():
        assert r["scratch"] <= (256 if kernel == "attn_prefill_kernel" and "Li256E" in name else 64), (name, r)
