"""Decode and prefill attention over the block-scaled cache against float64
attention over the stored values (tests/_kv_blocks.py), within the error that
the kernels' roundings allow (derived there)."""
import numpy as np
import pytest

from tests import _kv_blocks as B
from tests._util import randn_f16, say
from tests.test_kv_blocks_gpu import dev, gpu_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


@pytest.fixture(params=[0, 1], ids=["grid", "range"])
def decode_form(request):
    """The launcher's decode forms, forced where they can serve the call."""
    from redline_amd._lib import tune_knob
    with tune_knob("RLK_TUNE_BLK_DECODE", request.param):
        yield request.param


@pytest.fixture(params=[0, 1, 2], ids=["one", "rows2", "keys2"])
def prefill_split(request):
    """The launcher's three prefill kernels, forced."""
    from redline_amd._lib import tune_knob
    with tune_knob("RLK_TUNE_BLK_PREFILL", request.param):
        yield request.param


def make(rng, hkv, D, bs, fmt, lens, extra=1, lo=-6, hi=-3):
    """A filled cache and tables over distinct blocks; entries past a sequence's
    blocks are 0, and bytes past its context are e4m3 NaNs or 0x80."""
    mb = -(-max(max(lens), 1) // bs) + extra
    nb = 2 + sum(-(-max(n, 0) // bs) for n in lens)
    c = B.Cache(nb, hkv, bs, D, fmt)
    c.fill(rng, lo, hi)
    ids = rng.permutation(np.arange(1, nb))
    tab = np.zeros((len(lens), mb), np.int32)
    at = 0
    for s, n in enumerate(lens):
        k = -(-max(n, 0) // bs)
        tab[s, :k] = ids[at:at + k]
        at += k
        if n > 0 and n % bs:
            for x in c.codes:
                x[tab[s, k - 1], :, n % bs:] = 0xff if fmt == B.FP8 else 0x80
    return c, tab


def check(got, want, bound, what):
    got = got.astype(np.float64)
    assert np.isfinite(got).all(), what
    bad = np.abs(got - want) > bound
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.max(np.abs(got - want) / bound):.2f} of the bound"


def run_decode(torch, K, c, view, tab, q, hq, scale, pos, items, seqs, parts, pad=0, out=None, ws=None):
    T, D = len(q), c.D
    stride = hq * D + pad
    dq = torch.zeros(T, stride, dtype=torch.float16, device="cuda")
    dq[:, :hq * D] = dev(torch, q.reshape(T, -1))
    if out is None:
        out = torch.full((T, hq * D), 9.0, dtype=torch.float16, device="cuda")
    if ws is None and parts > 1:
        ws = K.DecodeWorkspace(len(items), hq, parts, D)
        for x in (ws.out, ws.max, ws.sum):
            x.fill_(float("nan"))
    keep = [dev(torch, np.asarray(a, np.int32)) for a in (tab, pos, items, seqs)]
    p = K.block_attention_params(dq, stride, out, hq, scale, view, keep[0], tab.shape[1], keep[1])
    K.paged_attention_decode_blocks(p, K.decode_work(keep[2], keep[3], len(items), parts, ws))
    torch.cuda.synchronize()
    return out.cpu().numpy().reshape(T, hq, D)


DECODE_CASES = [(hq, hkv, D, bs, fmt, lens) for hq, hkv, D, bs, fmt, lens in [
    (1, 1, 64, 16, B.INT8, [1, 2, 15, 16, 17]), (2, 1, 128, 16, B.FP8, [31, 32, 33, 63, 64, 65]),
    (6, 2, 128, 32, B.INT8, [255, 256, 257, 300]), (8, 2, 64, 32, B.FP8, [511, 512, 513, 1]),
    (5, 1, 128, 16, B.INT8, [700, 90]), (6, 1, 64, 16, B.FP8, [1029, 4]), (14, 2, 128, 32, B.FP8, [777, 1500]),
    (8, 1, 128, 16, B.INT8, [40, 2600]), (8, 1, 128, 16, B.FP8, [130]), (3, 3, 64, 32, B.INT8, [222, 47]),
]]


@pytest.mark.parametrize("scale", ["usual", "large", "negative"])
@pytest.mark.parametrize("hq,hkv,D,bs,fmt,lens", DECODE_CASES)
def test_decode(torch, hq, hkv, D, bs, fmt, lens, scale, decode_form):
    from redline_amd import kernels as K
    say(f"decode_blocks hq={hq} hkv={hkv} D={D} bs={bs} fmt={fmt} lens={lens} scale={scale} form={decode_form}")
    rng = np.random.default_rng(hq * 100 + D + bs)
    c, tab = make(rng, hkv, D, bs, fmt, lens)
    t, view = gpu_cache(torch, K, c)
    n = len(lens)
    q = randn_f16(rng, (n, hq, D))
    sc = {"usual": D ** -0.5 / 4, "large": 1.0, "negative": -D ** -0.5}[scale]
    parts = -(-max(lens) // 256)
    for extra in (0, 3):  # the call's own partitions, and a grid with more
        got = run_decode(torch, K, c, view, tab, q, hq, sc, np.array(lens) - 1, np.arange(n), np.arange(n),
                         parts + extra, pad=8 * extra)
        for s in range(n):
            want, bound = B.attention(c, tab[s], q[s:s + 1], sc, [lens[s]])
            check(got[s:s + 1], want, bound, f"item {s} of {lens[s]} keys")


@pytest.mark.parametrize("fmt", [B.INT8, B.FP8])
def test_decode_scales_far_apart(torch, fmt, decode_form):
    """K and V scales from 2^-24 to 2^10 (e4m3: 2^8), and 0, in one context; V so
    small that the whole output is below fp16's normal range, and mixed."""
    from redline_amd import kernels as K
    say(f"decode_blocks far scales fmt={fmt}")
    rng = np.random.default_rng(1)
    hq, hkv, D, bs, n = 4, 2, 128, 16, 1000
    top = 10 if fmt == B.INT8 else 8
    for lo, hi in ((-24, -20), (-24, top), (-12, -12)):
        c, tab = make(rng, hkv, D, bs, fmt, [n], lo=-6, hi=-3)
        c.scale[1][...] = 2.0 ** rng.integers(lo, hi + 1, c.scale[1].shape)
        lim = B.limit(2.0 ** hi, fmt)
        for h in range(hkv):  # stored values stay fp16 numbers
            v = np.clip(B.values(c.codes[1][:, h], fmt), -lim, lim)
            c.codes[1][:, h] = np.where(np.isnan(v), c.codes[1][:, h], B.bytes_of(np.nan_to_num(v), fmt))
        c.scale[0][tab[0, 3]] = 0
        c.scale[1][tab[0, 5]] = 0
        for which, b in ((0, 3), (1, 5)):
            c.codes[which][tab[0, b]] = 0
        t, view = gpu_cache(torch, K, c)
        q = randn_f16(rng, (1, hq, D))
        got = run_decode(torch, K, c, view, tab, q, hq, 0.02, [n - 1], [0], [0], 4)
        want, bound = B.attention(c, tab[0], q, 0.02, [n])
        check(got, want, bound, f"V scales 2^{lo} .. 2^{hi}")


@pytest.mark.parametrize("fmt", [B.INT8, B.FP8])
def test_decode_skips_empty_rows_and_bad_ids(torch, fmt, decode_form):
    """Items with a negative token write nothing; a negative position gives
    zeros; ids outside the pool are block 0; contexts past the table row or past
    max_partitions end there; several items of one sequence."""
    from redline_amd import kernels as K
    say(f"decode_blocks edges fmt={fmt}")
    rng = np.random.default_rng(2)
    hq, hkv, D, bs = 6, 2, 64, 16
    lens = [40, 600, 320]
    c, tab = make(rng, hkv, D, bs, fmt, lens, extra=0)
    c.codes[0][0], c.codes[1][0] = c.codes[0][1], c.codes[1][1]
    tab[0, 1], tab[1, 7], tab[1, 20] = -3, c.nb, 2 ** 31 - 1
    t, view = gpu_cache(torch, K, c)
    T = 7
    q = randn_f16(rng, (T, hq, D))
    # rows: 0 one item; 1 none; 2 empty; 3, 4 two items of sequence 1; 5 past the table; 6 not an item
    pos = np.array([39, 0, -1, 599, 300, 10 ** 9, 5], np.int32)
    items, seqs = [0, -1, 2, 3, 4, 5, -7], [0, 0, 1, 1, 1, 2, 0]
    got = run_decode(torch, K, c, view, tab, q, hq, 0.05, pos, items, seqs, 3)
    mb = tab.shape[1]
    for row, s, n in ((0, 0, 40), (3, 1, 600), (4, 1, 301), (5, 2, min(mb * bs, 3 * 256))):
        want, bound = B.attention(c, tab[s], q[row:row + 1], 0.05, [n])
        check(got[row:row + 1], want, bound, f"row {row}")
    assert (got[2] == 0).all()
    assert (got[[1, 6]] == 9.0).all()
    short = run_decode(torch, K, c, view, tab, q, hq, 0.05, pos, items, seqs, 1)  # keys past 256 are not read
    want, bound = B.attention(c, tab[1], q[3:4], 0.05, [256])
    check(short[3:4], want, bound, "one partition")


def test_decode_many_items_and_far_blocks(torch):
    """A call large enough for every launch rule (64 items), over a pool of more
    than 2^31 bytes whose last blocks it reads."""
    from redline_amd import kernels as K
    say("decode_blocks far blocks")
    rng = np.random.default_rng(4)
    hq, hkv, D, bs, n = 16, 8, 128, 32, 64
    lens = [int(x) for x in rng.integers(1, 3000, n)]
    c, tab = make(rng, hkv, D, bs, B.INT8, lens)
    t, view = gpu_cache(torch, K, c)
    big = 70000  # 70000 blocks of 8 x 32 x 128 bytes: 2.3 GB each of K and V
    shift = big - c.nb
    g = [torch.zeros((big,) + tuple(x.shape[1:]), dtype=x.dtype, device="cuda") for x in t]
    for x, y in zip(g, t):
        x[shift:] = y
    far = K.kv_block_view(*g, bs, hkv, D, B.INT8)
    q = randn_f16(rng, (n, hq, D))
    a = (np.array(lens) - 1, np.arange(n), np.arange(n), 12)
    near = run_decode(torch, K, c, view, tab, q, hq, 0.02, *a)
    got = run_decode(torch, K, c, far, tab + shift, q, hq, 0.02, *a)
    for s in range(0, n, 5):
        want, bound = B.attention(c, tab[s], q[s:s + 1], 0.02, [lens[s]])
        check(near[s:s + 1], want, bound, f"item {s}")
    assert np.array_equal(near, got)


def run_prefill(torch, K, c, view, tab, q, hq, scale, seq_ids, q_start, q_len, ctx, tiles, pad=0):
    T, D = len(q), c.D
    stride = hq * D + pad
    dq = torch.zeros(T, stride, dtype=torch.float16, device="cuda")
    dq[:, :hq * D] = dev(torch, q.reshape(T, -1))
    out = torch.full((T, hq * D), 9.0, dtype=torch.float16, device="cuda")
    keep = [dev(torch, np.asarray(a, np.int32)) for a in (tab, np.zeros(T), seq_ids, q_start, q_len, ctx)]
    p = K.block_attention_params(dq, stride, out, hq, scale, view, keep[0], tab.shape[1], keep[1])
    K.paged_attention_prefill_blocks(p, K.prefill_work(*keep[2:], len(seq_ids), tiles))
    torch.cuda.synchronize()
    return out.cpu().numpy().reshape(T, hq, D)


PREFILL_CASES = [
    (1, 1, 64, 16, B.INT8, [(0, 1), (0, 16), (0, 17), (5, 3)]),
    (2, 1, 128, 16, B.FP8, [(0, 33), (63, 2), (64, 64), (0, 65)]),
    (6, 2, 128, 32, B.INT8, [(100, 50), (0, 130)]),
    (7, 1, 64, 32, B.FP8, [(31, 40), (0, 129), (200, 1)]),
    (8, 8, 128, 16, B.FP8, [(17, 31)]),
    (8, 1, 128, 16, B.INT8, [(300, 37), (0, 5)]),
    (5, 1, 64, 16, B.INT8, [(0, 150), (511, 20)]),
    (3, 1, 128, 32, B.FP8, [(250, 100)]),
]


@pytest.mark.parametrize("scale", ["usual", "large", "negative"])
@pytest.mark.parametrize("hq,hkv,D,bs,fmt,segs", PREFILL_CASES)
def test_prefill(torch, hq, hkv, D, bs, fmt, segs, scale, prefill_split):
    from redline_amd import kernels as K
    say(f"prefill_blocks hq={hq} hkv={hkv} D={D} bs={bs} fmt={fmt} segs={segs} scale={scale} split={prefill_split}")
    rng = np.random.default_rng(hq * 100 + D + bs)
    lens = [p + n for p, n in segs]
    c, tab = make(rng, hkv, D, bs, fmt, lens)
    t, view = gpu_cache(torch, K, c)
    new = np.array([n for _, n in segs])
    start = np.cumsum(new) - new + 1  # one row before and two behind belong to nobody
    T = int(new.sum()) + 3
    q = randn_f16(rng, (T, hq, D))
    sc = {"usual": D ** -0.5 / 4, "large": 1.0, "negative": -D ** -0.5}[scale]
    order = rng.permutation(len(segs))
    got = run_prefill(torch, K, c, view, tab, q, hq, sc, order, start, new, lens, -(-max(new) // 32) + 1, pad=16)
    for s, (past, n) in enumerate(segs):
        r = slice(start[s], start[s] + n)
        want, bound = B.attention(c, tab[s], q[r], sc, [past + i + 1 for i in range(n)])
        check(got[r], want, bound, f"sequence {s}")
    assert (got[[0, -2, -1]] == 9.0).all()


@pytest.mark.parametrize("fmt", [B.INT8, B.FP8])
def test_prefill_edges(torch, fmt, prefill_split):
    """Skipped and idle sequences, rows before the context's start (zeros), ids
    outside the pool, a context that ends at its table row."""
    from redline_amd import kernels as K
    say(f"prefill_blocks edges fmt={fmt}")
    rng = np.random.default_rng(8)
    hq, hkv, D, bs = 4, 2, 64, 16
    lens = [60, 10, 96]
    c, tab = make(rng, hkv, D, bs, fmt, lens, extra=0)
    c.codes[0][0], c.codes[1][0] = c.codes[0][1], c.codes[1][1]
    tab[0, 1], tab[2, 2] = -1, c.nb + 5
    t, view = gpu_cache(torch, K, c)
    # 0: 20 of 60; 1: 30 rows but a context of 10 (20 rows see nothing); 2: 40 rows
    # up to position 109, its table row holds 96 keys; 3: idle
    start, new, ctx = [0, 20, 50, 90], [20, 30, 40, 0], [60, 10, 110, 5]
    q = randn_f16(rng, (95, hq, D))
    tab = np.concatenate([tab, tab[:1]])
    got = run_prefill(torch, K, c, view, tab, q, hq, 0.05, [2, -1, 0, 3, 1], start, new, ctx, 2)
    for s in range(3):
        r = slice(start[s], start[s] + new[s])
        past = ctx[s] - new[s]
        want, bound = B.attention(c, tab[s], q[r], 0.05, [past + i + 1 for i in range(new[s])])
        check(got[r], want, bound, f"sequence {s}")
    assert (got[20:40] == 0).all() and (got[90:] == 9.0).all()


@pytest.mark.parametrize("fmt", [B.INT8, B.FP8])
@pytest.mark.parametrize("gap", [10.5, 14.0])
def test_many_small_probabilities(torch, fmt, gap, decode_form, prefill_split):
    """One key ahead of thousands of equal ones by `gap` (natural log): each of
    those is near or below the smallest normal fp16 number relative to it, all of
    them together are not small (gap 10.5: 0.14 of the sum)."""
    from redline_amd import kernels as K
    say(f"small probabilities fmt={fmt} gap={gap}")
    rng = np.random.default_rng(13)
    hq, hkv, D, bs, n = 2, 1, 128, 16, 5200
    c, tab = make(rng, hkv, D, bs, fmt, [n])
    c.codes[0][...] = 0
    c.scale[0][...] = 1.0
    one = B.bytes_of(np.array([1.0]), fmt)[0]
    c.codes[0][tab[0, 100], 0, 5, 0] = one  # key 1605 has 1 in dim 0, the others 0
    q = np.zeros((1, hq, D), np.float16)
    q[:, :, 0] = gap
    t, view = gpu_cache(torch, K, c)
    want, bound = B.attention(c, tab[0], q, 1.0, [n])
    got = run_decode(torch, K, c, view, tab, q, hq, 1.0, [n - 1], [0], [0], 21)
    check(got, want, bound, "decode")
    got = run_prefill(torch, K, c, view, tab, q, hq, 1.0, [0], [0], [1], [n], 1)
    check(got, want, bound, "prefill")


def test_attention_in_graphs_sharing_a_workspace(torch):
    """Decode and prefill captured, two decode graphs over one workspace,
    replayed in turn on one stream with eager work between: every replay equals
    the eager call."""
    from redline_amd import kernels as K
    say("attention_blocks graphs")
    rng = np.random.default_rng(11)
    hq, hkv, D, bs = 8, 2, 128, 16
    lens = [900, 40, 333]
    c, tab = make(rng, hkv, D, bs, B.FP8, lens)
    t, view = gpu_cache(torch, K, c)
    d_tab, d_pos, ids = dev(torch, tab), dev(torch, np.array(lens, np.int32) - 1), dev(torch, np.arange(3, dtype=np.int32))
    ws = K.DecodeWorkspace(3, hq, 4, D)
    qs = [dev(torch, randn_f16(rng, (3, hq * D))) for _ in range(2)]
    outs = [torch.zeros(3, hq * D, dtype=torch.float16, device="cuda") for _ in range(2)]
    calls = [(K.block_attention_params(q, hq * D, o, hq, 0.05, view, d_tab, tab.shape[1], d_pos),
              K.decode_work(ids, ids, 3, 4, ws)) for q, o in zip(qs, outs)]
    want = []
    for call, o in zip(calls, outs):
        K.paged_attention_decode_blocks(*call)
        torch.cuda.synchronize()
        want.append(o.clone())
    graphs = []
    for call in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            K.paged_attention_decode_blocks(*call)
        graphs.append(g)
    for _ in range(3):
        for g, o, w in zip(graphs, outs, want):
            o.zero_()
            g.replay()
            ws.sum.mul_(1.0)  # eager work on the same buffers between the replays
            torch.cuda.synchronize()
            assert torch.equal(o, w)
