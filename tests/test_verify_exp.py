"""Builds and runs tests/native/verify_exp_check.cpp: the exp of the drafts' verification
on the host, over temperatures from 1e-45 to infinity and row maxima of every size and sign."""
from __future__ import annotations

import subprocess
from pathlib import Path

REPO = Path(__file__).resolve().parent.parent


def test_verify_exp(tmp_path):
    exe = tmp_path / "verify_exp_check"
    subprocess.run(["g++", "-O2", "-std=c++17", "-ffp-contract=off", "-Wall", "-Wextra", "-Werror",
                    f"-I{REPO / 'qwen3-iree_amd' / 'csrc'}",
                    str(REPO / "tests" / "native" / "verify_exp_check.cpp"), "-o", str(exe)],
                   check=True)
    out = subprocess.run([str(exe)], stdout=subprocess.PIPE, text=True, timeout=120)
    assert out.returncode == 0, out.stdout
