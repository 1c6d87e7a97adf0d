"""build_batch_tables against the sequential restatement (tests/_kv_blocks.py)
and against BatchBuilder, and the operators of the block-scaled cache run
together as a serving loop runs them."""
import numpy as np
import pytest

import redline_amd as ra
from tests import _kv_blocks as B
from tests._util import randn_f16, say
from tests.test_attention_blocks_gpu import check
from tests.test_kv_blocks_gpu import dev

pytestmark = pytest.mark.gpu

FIELDS = ("q_start", "q_len", "ctx_len", "positions", "slot_mapping", "decode_token", "decode_seq",
          "prefill_seq", "counts")


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


class Tables:
    """Device buffers of a step of up to S sequences and `rows` token rows."""

    def __init__(self, torch, K, S, rows, bs, thr, mb, pool, past, new, table):
        z = lambda n: torch.full((max(n, 1),), 77, dtype=torch.int32, device="cuda")  # noqa: E731
        self.past, self.new, self.table = dev(torch, past), dev(torch, new), dev(torch, table)
        self.t = {"q_start": z(S), "q_len": z(S), "ctx_len": z(S), "positions": z(rows), "slot_mapping": z(rows),
                  "decode_token": z(rows), "decode_seq": z(rows), "prefill_seq": z(S), "counts": z(4)}
        self.work = K.batch_tables(pool, self.past, self.new, S, rows, bs, thr, self.table, mb, *self.t.values())


def compare(torch, K, past, new, rows, bs, thr, table, ring, head, count, what, in_place=True):
    past, new = np.asarray(past, np.int32), np.asarray(new, np.int32)
    table, ring = np.asarray(table, np.int32), np.asarray(ring, np.int32)
    S, mb = len(past), table.shape[1]
    state = dev(torch, np.array([head, count, 0], np.int32))
    out = None if in_place else dev(torch, np.zeros(2, np.int32))
    d_ring = dev(torch, ring)
    pool = K.BlockPool(d_ring, state, out)
    tb = Tables(torch, K, S, rows, bs, thr, mb, pool, past, new, table)
    for _ in range(1 if in_place else 2):  # a call that keeps the state can be repeated
        K.build_batch_tables(tb.work)
        torch.cuda.synchronize()
    want_table, want_ring = table.copy(), ring.copy()
    want = B.tables(past, new, rows, bs, thr, want_table, want_ring, head, count)
    for n in FIELDS:
        m = {"counts": 4}.get(n, S if n in ("q_start", "q_len", "ctx_len", "prefill_seq") else rows)
        assert np.array_equal(tb.t[n].cpu().numpy()[:m], want[n]), (what, n)
        assert (tb.t[n].cpu().numpy()[m:] == 77).all(), (what, n)
    assert np.array_equal(tb.table.cpu().numpy(), want_table), what
    assert np.array_equal(d_ring.cpu().numpy(), want_ring), what
    got = state.cpu().numpy()
    assert got[2] == 0
    if in_place:
        assert np.array_equal(got[:2], want["state"]), what
    else:
        assert np.array_equal(got[:2], [head, count]) and np.array_equal(out.cpu().numpy(), want["state"]), what


def random_case(rng, S, bs, new_max, past_max, short=0, ended=0.1, idle=0.1):
    past = rng.integers(0, past_max + 1, S)
    new = rng.integers(1, new_max + 1, S)
    new[rng.random(S) < 0.5] = 1
    new[rng.random(S) < ended] = -1
    new[rng.random(S) < idle] = 0
    have = -(-past // bs)
    want = -(-(past + np.maximum(new, 0)) // bs)
    mb = max(1, int(want.max(initial=1)))
    need = int((want - have).sum())
    free = max(0, need - short)
    cap = int(have.sum()) + free + 3
    ids = rng.permutation(np.arange(1, cap + 1))
    table = np.zeros((S, mb), np.int64)
    at = 0
    for s in range(S):
        table[s, :have[s]] = ids[at:at + have[s]]
        at += have[s]
    head = int(rng.integers(0, cap))
    ring = np.zeros(cap, np.int64)
    ring[(head + np.arange(free)) % cap] = ids[at:at + free]
    return past, new, table, ring, head, free


@pytest.mark.parametrize("S,bs,new_max,past_max,short,pad,thr", [
    (1, 16, 1, 0, 0, 0, 1), (1, 16, 40, 100, 0, 3, 1), (7, 16, 5, 50, 0, 0, 4), (33, 32, 100, 900, 4, 2, 1),
    (64, 16, 300, 300, 40, 0, 1), (513, 16, 3, 700, 0, 9, 2), (700, 7, 40, 90, 30, 0, 1), (2050, 16, 20, 2000, 0, 1, 1),
    (8192, 16, 2, 40, 100, 5, 1), (5, 16, 6000, 50, 0, 77, 1), (40, 1, 70, 10, 13, 0, 0),
])
def test_tables(torch, S, bs, new_max, past_max, short, pad, thr):
    from redline_amd import kernels as K
    for seed in range(2):
        say(f"tables S={S} bs={bs} new_max={new_max} short={short} pad={pad} thr={thr} seed={seed}")
        rng = np.random.default_rng(seed * 1000 + S + bs)
        past, new, table, ring, head, free = random_case(rng, S, bs, new_max, past_max, short)
        rows = int(np.maximum(new, 0).sum()) + pad
        compare(torch, K, past, new, rows, bs, thr, table, ring, head, free, "tables", in_place=seed == 0)


def test_tables_refusals(torch):
    """Sequences that do not fit their table row, the token rows or the free
    blocks; a negative past; one without needs behind a refused one; nothing."""
    from redline_amd import kernels as K
    say("tables refusals")
    bs, mb = 16, 4
    table = np.arange(1, 25).reshape(6, mb)
    ring = np.arange(100, 140)
    # want 5 blocks of a row of 4; negative past; 2 blocks; 4 blocks of which 1 is
    # left; no need; rows run out
    compare(torch, K, [60, -1, 0, 0, 17, 3], [6, 2, 30, 60, 5, 40], 130, bs, 1, table, ring, 38, 3, "refused")
    compare(torch, K, [0, 5], [2 ** 31 - 1, 3], 64, bs, 1, table[:2], ring, 0, 40, "huge")
    compare(torch, K, [2 ** 31 - 1, 5], [2 ** 31 - 1, 3], 64, bs, 1, table[:2], ring, 0, 40, "huge past")
    compare(torch, K, [0, 0], [0, 0], 8, bs, 1, table[:2], ring, 5, 7, "idle")
    compare(torch, K, [64, 40], [-1, -1], 4, bs, 1, table[:2], np.zeros(9, int), 7, 0, "all ended")
    compare(torch, K, [20], [1], 0, bs, 1, table[:1], ring, 5, 7, "no rows")
    compare(torch, K, np.zeros(0), np.zeros(0), 6, bs, 1, np.zeros((0, 2)), ring, 5, 7, "no sequences")


def test_tables_match_batch_builder(torch):
    """The same step through BatchBuilder (host) and build_batch_tables."""
    from redline_amd import kernels as K
    say("tables against BatchBuilder")
    rng = np.random.default_rng(5)
    past, new, table, ring, head, free = random_case(rng, 40, 16, 90, 500, ended=0, idle=0)
    rows = int(new.sum())
    want_table = table.copy()
    B.tables(past, new, rows, 16, 2, want_table, ring.copy(), head, free)
    mb = table.shape[1]
    bb = ra.BatchBuilder(rows, 40, 40, mb, 16, 2)
    for s in range(40):
        bb.add(np.zeros(new[s], np.int32), int(past[s]), int(new[s]), None, want_table[s].astype(np.int32))
    meta, shape, lay = bb.write()
    pool = K.BlockPool(dev(torch, ring.astype(np.int32)), dev(torch, np.array([head, free, 0], np.int32)))
    tb = Tables(torch, K, 40, rows, 16, 2, mb, pool, past.astype(np.int32), new.astype(np.int32), table.astype(np.int32))
    K.build_batch_tables(tb.work)
    got = {n: x.cpu().numpy() for n, x in tb.t.items()}
    for n, m, c in (("positions", "positions", rows), ("slot_mapping", "slot_mapping", rows),
                    ("q_start", "seq_q_start", 40), ("q_len", "seq_q_len", 40), ("ctx_len", "seq_ctx_len", 40),
                    ("decode_token", "decode_token", shape.num_decode_items),
                    ("decode_seq", "decode_seq", shape.num_decode_items),
                    ("prefill_seq", "prefill_seq", shape.num_prefill_seqs)):
        assert np.array_equal(got[n][:c], meta[lay[m]:lay[m] + c]), n
    assert np.array_equal(tb.table.cpu().numpy().reshape(-1), meta[lay["block_tables"]:lay["block_tables"] + 40 * mb])
    assert list(got["counts"]) == [rows, shape.num_decode_items, shape.num_prefill_seqs, 0]


@pytest.mark.parametrize("fmt,D,bs,hq,hkv", [(B.INT8, 128, 16, 8, 2), (B.FP8, 64, 32, 6, 2)])
@pytest.mark.parametrize("captured", [False, True])
def test_serving_loop(torch, fmt, D, bs, hq, hkv, captured):
    """Steps of a small server: prompts in chunks, decoding, a sequence that ends
    and one that takes its blocks, as tables -> write -> decode and prefill
    attention on one stream, eager or as one captured step that is replayed with
    new lengths.  The cache equals the restated writes bit for bit; attention is
    float64 attention over it."""
    from redline_amd import kernels as K
    say(f"serving loop fmt={fmt} D={D} bs={bs} captured={captured}")
    rng = np.random.default_rng(12)
    S, mb, rows, nb, max_new = 4, 12, 96, 30, 64
    cache = K.KVBlockCache(1, nb, hkv, D, bs, fmt)
    model = B.Cache(nb, hkv, bs, D, fmt)
    pool = K.BlockPool.of_blocks(nb)
    ring, head, count = np.arange(1, nb, dtype=np.int32), 0, nb - 1
    table = np.zeros((S, mb), np.int32)
    tb = Tables(torch, K, S, rows, bs, 1, mb, pool, np.zeros(S, np.int32), np.zeros(S, np.int32), table)
    cols = (hq + 2 * hkv) * D
    qkv = torch.zeros(rows, cols, dtype=torch.float16, device="cuda")
    out = torch.zeros(rows, hq * D, dtype=torch.float16, device="cuda")
    cos, sin = ra.rope_cos_sin_tables(1e4, D, mb * bs)
    d_cos, d_sin = dev(torch, cos), dev(torch, sin)
    ws = K.DecodeWorkspace(S, hq, 2, D)
    p = K.block_attention_params(qkv, cols, out, hq, 0.06, cache.layer(0), tb.table, mb, tb.t["positions"])
    dw = K.decode_work(tb.t["decode_token"], tb.t["decode_seq"], S, 2, ws)
    pw = K.prefill_work(tb.t["prefill_seq"], tb.t["q_start"], tb.t["q_len"], tb.t["ctx_len"], S, -(-max_new // 32))

    def step():
        K.build_batch_tables(tb.work)
        K.rope_and_write_kv_blocks(qkv, tb.t["positions"], tb.t["slot_mapping"], rows, hq, d_cos, d_sin, cache.layer(0))
        K.paged_attention_decode_blocks(p, dw)
        K.paged_attention_prefill_blocks(p, pw)

    graph = None
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        torch.cuda.synchronize()
    past = np.zeros(S, np.int64)
    steps = [[40, 1, 0, 7], [30, 1, 50, 1], [1, 1, 1, 1], [1, -1, 1, 64], [1, 0, 1, 1], [1, 33, 1, 1], [5, 1, -1, 1],
             [1, 1, 20, 1]]
    for k, new in enumerate(steps):
        new = np.array(new)
        x = randn_f16(rng, (rows, cols)) * np.exp2(rng.integers(-2, 3, (rows, 1))).astype(np.float16)
        qkv.copy_(dev(torch, x))
        tb.past.copy_(dev(torch, past.astype(np.int32)))
        tb.new.copy_(dev(torch, new.astype(np.int32)))
        out.fill_(9.0)
        graph.replay() if captured else step()
        torch.cuda.synchronize()
        want = B.tables(past, new, rows, bs, 1, table, ring, head, count)
        head, count = (int(v) for v in want["state"])
        for n in FIELDS:
            assert np.array_equal(tb.t[n].cpu().numpy()[:len(want[n])], want[n]), (k, n)
        q = B.write(model, x, None, want["positions"], want["slot_mapping"], hq, cos, sin)
        raw = model.raw()
        t = cache.tensors(0)
        for got, w in zip(t[:2], raw):
            assert np.array_equal(got.cpu().numpy().view(np.uint8)[1:], w[1:]), k
        got = out.cpu().numpy().reshape(rows, hq, D)
        for s in range(S):
            n, r0 = int(want["q_len"][s]), int(want["q_start"][s])
            ref, bound = B.attention(model, table[s], q[r0:r0 + n], 0.06, [past[s] + i + 1 for i in range(n)])
            check(got[r0:r0 + n], ref, bound, f"step {k} sequence {s}")
        assert (got[int(want["counts"][0]):] == 9.0).all()
        past = np.where(new < 0, 0, past + want["q_len"])
