"""Where the attention kernels read and write (csrc/r9vx_attn_index.h), checked on
the CPU: masks, pages and parts of a sequence's keys, packed tiles, hostile data."""
from __future__ import annotations

import pathlib
import shutil
import subprocess

import pytest

ROOT = pathlib.Path(__file__).resolve().parent.parent


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_index_functions(tmp_path):
    exe = tmp_path / "attn_index"
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{ROOT / 'r9v_amd' / 'csrc'}",
                    str(ROOT / "tests" / "fixtures" / "attn_index.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
