"""Every matrix instruction of the code objects reads VALU results two wait states or
more behind them, what gfx950 asks for between a vector write and an MFMA that reads
it.  The compiler keeps them for its own instructions and knows nothing of a write in
inline assembly."""
from __future__ import annotations

import re
import subprocess

import pytest

OBJECTS = ("q8gemv", "decode", "prefill", "cache")


def registers(operand: str) -> range:
    m = re.match(r"-?\|?v(?:\[(\d+):(\d+)\]|(\d+))", operand)
    if not m:
        return range(0)
    if m[3] is not None:
        return range(int(m[3]), int(m[3]) + 1)
    return range(int(m[1]), int(m[2]) + 1)


def too_close(lines) -> list[str]:
    """The MFMAs of a listing that read a VALU result too early, each with its kernel."""
    found, kernel, at, written = [], "", 0, {}
    for line in lines:
        m = re.match(r"[0-9a-f]+ <(\w+)>:", line)
        if m:
            kernel, at, written = m[1], 0, {}
            continue
        m = re.match(r"\s+([a-z]\w+)\s+([^/]*)", line)
        if not m:
            continue
        op, operands = m[1], [o.strip() for o in m[2].split(",")]
        mfma = op.startswith(("v_mfma", "v_smfma"))
        if mfma:
            for o in operands[1:4]:
                close = [r for r in registers(o) if at - written.get(r, -9) < 2]
                if close:
                    found.append(f"{kernel}: {line.split('//')[0].strip()} reads v{close[0]}")
        at += 1 + (int(operands[0], 0) if op == "s_nop" else 0)
        if op.startswith(("v_", "ds_", "global_", "buffer_", "scratch_")):
            for r in registers(operands[0]):
                if op.startswith("v_") and not mfma and not op.startswith("v_cmp"):
                    written[r] = at
                else:
                    written.pop(r, None)
    return found


def test_the_check_sees_a_missing_wait():
    text = ["0000 <k>:", "\tv_add_f32_e32 v5, v1, v2  // 0", "\ts_nop 0  // 4",
            "\tv_mfma_f32_16x16x32_f16 v[8:11], v[0:3], v[4:7], v[8:11]  // 8"]
    assert len(too_close(text)) == 1 and "reads v5" in too_close(text)[0]
    text[2] = "\ts_nop 1  // 4"
    assert not too_close(text)


@pytest.mark.parametrize("name", OBJECTS)
def test_mfma_sources_have_arrived(Q, name):
    from qwen3_iree_amd import build

    path = build.LIB / f"{name}_gfx950.hsaco"
    out = subprocess.run([str(build.ROCM / "llvm" / "bin" / "llvm-objdump"), "-d", str(path)],
                         check=True, capture_output=True, text=True, timeout=120).stdout
    lines = out.splitlines()
    assert name == "q8gemv" or any("v_mfma" in line for line in lines)
    assert not too_close(lines)
