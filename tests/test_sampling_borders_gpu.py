"""Rows whose top-p target lies within a rounding of a bin's end (golden/sampling_borders.npz)."""
from pathlib import Path

import numpy as np
import pytest

from tests._util import say
from tests.test_sampling_gpu import U32, Call, draw, torch  # noqa: F401  (torch: the fixture)

pytestmark = pytest.mark.gpu
GOLDEN = np.load(Path(__file__).resolve().parent / "golden" / "sampling_borders.npz")


@pytest.mark.parametrize("V", [812, 8192, 20011])
def test_target_between_two_sums_of_a_bin(torch, V):  # noqa: F811
    """top_p = 0.5: either side of the border is right (the sums differ by less than the weights'
    precision), each with the log-probability of its own kept mass; a third is not."""
    say("sample borders", V)
    rng = np.random.default_rng(V)
    rows, u = GOLDEN["rows"], np.concatenate([np.linspace(0.001, 0.999, 23), [1 - 2.0 ** -24]]).astype(np.float32)
    x = np.full((len(rows), V), -np.inf, np.float32)
    for r, row in enumerate(rows):
        x[r, rng.permutation(V)[:len(row)]] = row  # (what is left of a golden row is -infinity too)
    args = [(r, a) for r in range(len(rows)) for a in u]
    c = Call(torch, torch.from_numpy(x[[r for r, _ in args]]).cuda(), p=0.5, u=[a for _, a in args])()
    tok, lp = c.tokens.cpu().numpy(), c.lp.cpu().numpy()
    for i, (r, a) in enumerate(args):
        near = [draw(x[r], 1.0, 0, 0.5, 0.0, a, e) for e in ((0, 0, 0), (-1, 0, 0), (1, 0, 0), (-1, 0, -1), (-1, 0, 1),
                                                             (1, 0, -1), (1, 0, 1))]
        assert any(int(tok[i]) == t and abs(float(lp[i]) - q) <= U32 * abs(q) + 2.0 ** -32 for t, q in near), (
            r, int(GOLDEN["heads"][r]), float(a), int(tok[i]), float(lp[i]), near)
