"""No memory instruction reads a scalar register before the wait states after the
vector instruction that wrote it: in the assembly of the sources that issue loads
by inline assembly."""
from __future__ import annotations

import concurrent.futures as cf
import subprocess

import pytest

import asm_states
from r9v_amd import build as B

SOURCES = ["attn_prefill.hip", "fp8_gemm.hip", "fp8_moe.hip", "gemm.hip", "moe_gemm.hip"]


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    to = tmp_path_factory.mktemp("asm")

    def compiled(src):
        cmd = [B.HIPCC, *B.FLAGS, "--offload-device-only", "-S", str(B.CSRC / src), "-o", str(to / f"{src}.s")]
        r = subprocess.run(cmd, capture_output=True, text=True)
        assert r.returncode == 0, r.stderr[-2000:]
        return (to / f"{src}.s").read_text()

    with cf.ThreadPoolExecutor(max_workers=len(SOURCES)) as ex:
        return dict(zip(SOURCES, ex.map(compiled, SOURCES)))


@pytest.mark.parametrize("src", SOURCES)
def test_no_base_is_read_too_early(src, assembly):
    functions = asm_states.functions(assembly[src])
    copies = {name: sum(op.startswith("global_load_lds") for op, _ in code) for name, code in functions.items()}
    assert sum(copies.values()) > 0, "no copies into LDS found"
    bad = {name: asm_states.early(code) for name, code in functions.items()}
    assert not any(bad.values()), {name[:80]: (len(b), copies[name], "fewest states", min(s for _, s in b)) for name, b in bad.items() if b}


HEAD = "f:\n\tv_readlane_b32 s4, v0, 3\n\tv_readlane_b32 s5, v1, 3\n"


@pytest.mark.parametrize("body,states", [
    ("\ts_mov_b32 m0, s9\n\ts_and_saveexec_b64 s[6:7], s[2:3]\n\tglobal_load_lds_dwordx4 v2, s[4:5]\n", [2]),
    ("\ts_mov_b32 m0, s9\n\ts_and_saveexec_b64 s[6:7], s[2:3]\n\ts_nop 2\n\tglobal_load_lds_dwordx4 v2, s[4:5]\n", []),
    ("\ts_nop 4\n\tglobal_load_dword v2, v3, s[4:5] offset:16\n", []), ("\ts_nop 3\n\tglobal_load_dword v2, v3, s[4:5] offset:16\n", [4]),
    ("\ts_mov_b64 s[4:5], s[0:1]\n\tglobal_load_dword v2, v3, s[4:5]\n", []),
    ("\ts_cbranch_scc1 .LBB0_2\n\ts_nop 7\n.LBB0_2:\n\tglobal_store_dword v2, v3, s[4:5]\n", [1]),
    (".LBB0_1:\n\ts_nop 7\n\tglobal_load_dword v2, v3, s[4:5]\n\tv_cmp_lt_u32_e64 s[4:5], v0, v1\n\ts_branch .LBB0_1\n", []),
    (".LBB0_1:\n\tbuffer_load_dword v2, v3, s[8:11], s4 offen\n\ts_nop 5\n\tv_readfirstlane_b32 s10, v1\n\ts_cbranch_vccnz .LBB0_1\n", [1])])
def test_the_check_itself(body, states):
    code = asm_states.functions(HEAD + body + "\ts_endpgm\n.Lfunc_end0:\n")["f"]
    assert [n for _, n in asm_states.early(code)] == states
