"""Builds and runs tests/native/pages_index_check.cpp: the index arithmetic of the paged
cache's kernels on the host."""
from __future__ import annotations

import subprocess
from pathlib import Path

REPO = Path(__file__).resolve().parent.parent


def test_pages_index(tmp_path):
    exe = tmp_path / "pages_index_check"
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Wextra", "-Werror",
                    f"-I{REPO / 'qwen3-iree_amd' / 'csrc'}",
                    str(REPO / "tests" / "native" / "pages_index_check.cpp"), "-o", str(exe)],
                   check=True)
    out = subprocess.run([str(exe)], stdout=subprocess.PIPE, text=True, timeout=120)
    assert out.returncode == 0, out.stdout
