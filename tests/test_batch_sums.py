"""Running sums of the batch tables where requests are huge: the sums themselves on
the host, and the tables on the GPU against the sequential restatement
(tests/_kv_blocks.py), which adds up unbounded integers."""
import subprocess
from pathlib import Path

import numpy as np
import pytest

from tests._util import say

ROOT = Path(__file__).resolve().parents[1]
HUGE = 2 ** 31 - 1


def test_sums_saturate(tmp_path):
    exe = tmp_path / "sums"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", f"-I{ROOT / 'redline_amd' / 'csrc'}",
                    str(ROOT / "tests" / "cpp" / "sums_main.cpp"), "-o", str(exe)], check=True, capture_output=True)
    assert "PASS" in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout


@pytest.mark.gpu
@pytest.mark.parametrize("S", [6, 70, 600, 3000])  # one wave, two, two a thread, through LDS
@pytest.mark.parametrize("huge", [(1, 2), (1, 2, 3), (0, -2), (2, -3, -2), "half", "all"])
def test_tables_refuse_huge_requests(S, huge):
    """Requests of 2^30 rows and more among small ones: what comes behind them in the
    batch is refused, what comes before keeps its rows and blocks."""
    import torch
    from redline_amd import kernels as K
    from tests.test_batch_tables_gpu import compare
    assert torch.cuda.is_available()
    say(f"tables with huge requests S={S} huge={huge}")
    bs, mb = 16, 3
    rng = np.random.default_rng(S)
    past = rng.integers(0, 17, S)
    new = rng.integers(-1, 4, S)
    at = {"half": range(1, S, 2), "all": range(S)}.get(huge, huge)
    new[list(at)] = rng.choice([HUGE, 2 ** 30, 2 ** 30 + 1, 2 ** 30 - 1], len(at))
    table = np.arange(1, S * mb + 1).reshape(S, mb)
    ring = np.arange(20000, 40000)
    for rows in (64, 5 * S):
        compare(torch, K, past, new, rows, bs, 1, table, ring, 19990, 9000, f"huge, {rows} rows")
