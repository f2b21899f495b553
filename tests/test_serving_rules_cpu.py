"""Addressing of the serving kernels at the largest sizes that their entry points take,
on the CPU: compiles tests/native/serving_rules.cpp (host side only) against the
library's own headers and runs its checks. A wrong address there would be a read out of
range, which no comparison of outputs shows.
"""
from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

NATIVE = Path(__file__).resolve().parent / "native"


def test_serving_rules():
    sys.path.insert(0, str(NATIVE))
    try:
        import build
    finally:
        sys.path.remove(str(NATIVE))
    library_build = build._library_build()
    # -fwrapv: a sum or product of ints that passes 2^31 wraps, as on the GPU, and is found.
    program, tmp = build.OUT / "serving_rules", build.OUT / "serving_rules.tmp"
    build.OUT.mkdir(parents=True, exist_ok=True)
    build._run([build.HIPCC, "-x", "hip", "--offload-host-only", "-O1", "-std=c++17", "-fwrapv", "-Wno-unused-command-line-argument",
                f"-I{build.ROOT / 'include'}", f"-I{library_build.CSRC}", str(NATIVE / "serving_rules.cpp"), "-o", str(tmp)])
    os.replace(tmp, program)
    result = subprocess.run([str(program)], capture_output=True, text=True, timeout=120)
    assert result.returncode == 0 and "serving rules OK" in result.stdout, result.stdout + result.stderr
