"""The extensions for many continuations of one prompt through the C++ header
(redline::kernels, include/redline_amd/kernels.h) by a compiled program that holds
them against the formulas in 64 bits.  It is built by build() into tests/cpp/bin/."""
import subprocess
from pathlib import Path

import pytest

from tests._util import say

EXE = Path(__file__).resolve().parent / "cpp" / "bin" / "continuations_gpu"


@pytest.mark.gpu
def test_cpp_header_continuations_on_gpu():
    assert EXE.exists(), f"{EXE} is missing: run __graft_entry__.build() first"
    say("C++ header program tests/cpp/bin/continuations_gpu")
    r = subprocess.run([str(EXE)], capture_output=True, text=True, timeout=100)
    print(r.stdout)
    assert r.returncode == 0 and r.stdout.strip().endswith("PASS"), r.stdout + r.stderr
