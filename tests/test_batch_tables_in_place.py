"""Batch tables whose lengths take the place of the ones they are made from: the
outputs are what separate arrays give, over as many replays as there are, and any
other overlap with the lengths is refused."""
import ctypes as C

import numpy as np
import pytest

import redline_amd as ra
from redline_amd import _lib
from tests import _kv_blocks as B
from tests._util import say


def call(S=4, rows=8, mb=3, **at):
    """Stand-in addresses far apart, nothing launched unless the check passes."""
    names = ("past", "new", "tab", "q_start", "q_len", "ctx", "pos", "slots", "dt", "ds", "pre", "counts")
    a = {n: 0x10000 * (i + 1) for i, n in enumerate(names)} | at
    p = _lib.BlockPoolView(0x900000, 8, 0x910000, None)
    t = _lib.BatchTables(a["past"], a["new"], S, rows, 16, 1, a["tab"], mb, a["q_start"], a["q_len"], a["ctx"],
                         a["pos"], a["slots"], a["dt"], a["ds"], a["pre"], a["counts"])
    return ra.lib().rlk_build_batch_tables(C.byref(p), C.byref(t), None)


P, N = 0x10000, 0x20000


@pytest.mark.parametrize("at", [
    dict(q_start=P), dict(q_start=N), dict(q_len=P), dict(ctx=N), dict(pre=P), dict(pos=N), dict(slots=P),
    dict(dt=P), dict(ds=N), dict(counts=P), dict(tab=N),
    dict(ctx=P + 4), dict(ctx=P - 12), dict(q_len=N + 12), dict(q_len=N - 4),  # by some elements only
    dict(pos=P - 4 * 7), dict(counts=N + 12), dict(tab=P - 4 * 11),
    dict(ctx=P, q_start=P), dict(q_len=N, pre=N), dict(ctx=P, q_len=P),
])
def test_overlapping_lengths_are_refused(at):
    assert call(**at) == _lib.RLK_EINVAL
    assert b"must not overlap" in ra.lib().rlk_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("scarce", [False, True])  # blocks for all sequences, or for half of them
@pytest.mark.parametrize("S,rows,bs", [(5, 40, 16), (600, 700, 16), (3000, 5000, 32), (8192, 8192, 16)])
def test_lengths_in_place(S, rows, bs, scarce, both):
    """Steps of S sequences, captured once and replayed: each starts from the lengths
    that the one before left.  new_len is written anew between the replays where q_len
    takes its place."""
    import torch
    from redline_amd import kernels as K
    from tests.test_kv_blocks_gpu import dev
    assert torch.cuda.is_available()
    say(f"tables in place S={S} rows={rows} bs={bs} scarce={scarce} both={both}")
    rng = np.random.default_rng(S + rows)
    mb, nb = 6, S // 2 + 2 if scarce else 3 * S
    pool = K.BlockPool.of_blocks(nb)
    ring, head, count = np.arange(1, nb, dtype=np.int32), 0, nb - 1
    table = np.zeros((S, mb), np.int32)
    z = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
    past, new, d_table = z(S), z(S), dev(torch, table)
    t = {"q_start": z(S), "q_len": new if both else z(S), "ctx_len": past, "positions": z(rows),
         "slot_mapping": z(rows), "decode_token": z(rows), "decode_seq": z(rows), "prefill_seq": z(S), "counts": z(4)}
    work = K.batch_tables(pool, past, new, S, rows, bs, 1, d_table, mb, *t.values())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.build_batch_tables(work)
    h_past, refused = np.zeros(S, np.int64), 0
    for step in range(12):
        h_new = np.where(rng.random(S) < 0.5, 1, 0) if step % 3 else rng.integers(-1, 3, S)
        new.copy_(dev(torch, h_new.astype(np.int32)))
        graph.replay()
        torch.cuda.synchronize()
        want = B.tables(h_past, h_new, rows, bs, 1, table, ring, head, count)
        head, count = (int(v) for v in want["state"])
        for n, x in t.items():
            assert np.array_equal(x.cpu().numpy(), want[n]), (step, n)
        assert np.array_equal(d_table.cpu().numpy(), table) and np.array_equal(pool.ring.cpu().numpy(), ring), step
        assert pool.state.tolist() == [head, count, 0]
        h_past = want["ctx_len"].astype(np.int64)
        refused += int(want["counts"][3])
    assert h_past.max() > 3 and (refused > 0 or not scarce)
