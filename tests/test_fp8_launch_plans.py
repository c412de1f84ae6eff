"""Which e4m3 kernels a call launches and with what grids, recorded on the CPU
(tests/launch_record.py)."""
from __future__ import annotations

import shutil

import pytest

import launch_record

pytestmark = pytest.mark.skipif(not launch_record.LIB.exists() or shutil.which("gcc") is None,
                                reason="needs the built libr9vx.so and gcc")


@pytest.fixture(scope="module")
def runtime(tmp_path_factory):
    return launch_record.build(tmp_path_factory.mktemp("hip"))


GIB = 1 << 30


@pytest.mark.parametrize("kw,least", [
    (dict(m=512, n=1 << 26, k=16, swiglu=True), 128 * GIB), (dict(m=1 << 13, n=1 << 22, k=128, swiglu=True), 128 * GIB),
    (dict(m=1 << 24, n=1 << 11, k=16, swiglu=True), 128 * GIB), (dict(m=960, n=1 << 26, k=16), 240 * GIB),
    (dict(m=1 << 20, n=1 << 16, k=128), 256 * GIB), (dict(m=1 << 20, n=1 << 17, k=128, bf16_out=True, swiglu=True), 256 * GIB),
    (dict(m=1 << 24, n=8, k=1 << 12, bf16_out=True), GIB // 8), (dict(m=8, n=1 << 26, k=16, codes=True), 2 * GIB)])
def test_products_that_fit_the_card_launch(runtime, kw, least):
    """Outputs up to the card's memory in tiles of a few thousand values: a launch
    counts its threads in 32 bits, and one that does not fit them is an error."""
    assert least <= kw["m"] * kw["n"] * (2 if kw.get("bf16_out") else 4) <= 288 * 10 ** 9
    (rc, msg, launches), = launch_record.record(runtime, [("matmul_fp8", kw)])
    assert rc == 0, msg
    assert launches


LAUNCHES = {"quantize_fp8_kernel", "sort_small_kernel", "sort_count_kernel", "sort_scan_kernel", "sort_finish_kernel", "sort_place_kernel",
            "fp8_moe_stream_kernel", "fp8_moe_tile_kernel", "fp8_moe_combine_kernel"}


@pytest.mark.parametrize("kw", [dict(t=1 << 16, e=32, k=32, dm=128, dff=1 << 16), dict(t=1 << 17, e=32, k=32, dm=128, dff=1 << 16, bf16_out=True)])
def test_experts_with_more_tiles_than_a_launch_are_refused(runtime, kw):
    """Not by the runtime, behind launches that are under way; half the tokens fit."""
    (rc, msg, launches), (_, _, fewer) = launch_record.record(runtime, [("moe_fp8", kw), ("moe_fp8", dict(kw, t=kw["t"] // 2))])
    assert rc == -2 and "more tiles than a launch" in msg and not launches
    assert {n.split("<")[0] for n, _, _ in fewer} <= LAUNCHES and fewer[-1][0].startswith("fp8_moe_combine_kernel")


@pytest.mark.parametrize("kw,form", [
    (dict(t=1, e=8, k=2, dm=128, dff=128), "fp8_moe_stream_kernel<1, 2, 4, true>"), (dict(t=64, e=2, k=2, dm=128, dff=128), "fp8_moe_stream_kernel<1, 2, 4, true>"),
    (dict(t=64, e=2, k=2, dm=128, dff=128, bf16_out=True), "fp8_moe_stream_kernel<1, 2, 4, true>"),
    (dict(t=65, e=16, k=2, dm=128, dff=128, bf16_out=True), "fp8_moe_tile_kernel<true, 256, false>"),
    (dict(t=5, t_bucket=65, e=16, k=2, dm=128, dff=128, bf16_out=True), "fp8_moe_tile_kernel<true, 256, false>"),
    (dict(t=256, e=64, k=2, dm=128, dff=128, bf16_out=True), "fp8_moe_stream_kernel<1, 2, 4, true>"),
    (dict(t=257, e=64, k=2, dm=128, dff=128, bf16_out=True), "fp8_moe_tile_kernel<true, 256, false>"),
    (dict(t=128, e=64, k=2, dm=128, dff=128, shared=1, bf16_out=True), "fp8_moe_stream_kernel<1, 2, 4, true>"),
    (dict(t=129, e=64, k=2, dm=128, dff=128, shared=1, bf16_out=True), "fp8_moe_tile_kernel<true, 256, false>"),
    (dict(t=512, e=64, k=2, dm=128, dff=128), "fp8_moe_stream_kernel<1, 2, 4, true>"), (dict(t=513, e=64, k=2, dm=128, dff=128), "fp8_moe_tile_kernel<true, 128, true>"),
    (dict(t=346, e=64, k=2, dm=128, dff=128, shared=1), "fp8_moe_stream_kernel<1, 2, 4, true>"),
    (dict(t=347, e=64, k=2, dm=128, dff=128, shared=1), "fp8_moe_tile_kernel<true, 128, true>")])
def test_the_experts_form(runtime, kw, form):
    """Streaming up to 64 tokens, and up to 8 rows an expert, 16 for f32 outputs, which never run the 8-bit tiles."""
    (rc, msg, launches), = launch_record.record(runtime, [("moe_fp8", kw)])
    assert rc == 0, msg
    assert form in [n for n, _, _ in launches]


def test_long_rows_reach_every_kernel(runtime):
    """The sizes of the tests of long K choose the kernels they are there for."""
    pytest.importorskip("torch")
    from test_gpu_fp8_long_k import CASES

    out = launch_record.record(runtime, [("matmul_fp8", dict(m=m, n=n, k=k, codes=True, bf16_out=not f32, swiglu=gated)) for m, n, k, f32, gated, _ in CASES])
    for case, (rc, msg, launches) in zip(CASES, out):
        assert rc == 0, msg
        assert launches[-1][0] == case[5], case
