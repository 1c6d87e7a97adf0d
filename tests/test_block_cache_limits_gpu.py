"""The block-scaled cache's kernels at the limits of what they take: scales from 2^-24
to the largest and 0 in prefill, pools whose offsets pass 32 bits in write, read and
prefill, and the sizes at which the launch rules change."""
import numpy as np
import pytest

import redline_amd as ra
from tests import _kv_blocks as B
from tests._util import randn_f16, say
from tests.test_attention_blocks_gpu import check, make, run_prefill
from tests.test_batch_tables_gpu import compare, random_case
from tests.test_kv_blocks_gpu import dev, gpu_cache, segments

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


@pytest.fixture(params=[0, 2], ids=["large", "keys2"])
def prefill_split(request):
    """The two prefill kernels of a head dim, forced."""
    from redline_amd._lib import tune_knob
    with tune_knob("RLK_TUNE_BLK_PREFILL", request.param):
        yield request.param


def set_scales(c, which, scales):
    """New scales, with codes whose values are fp16 numbers under them (as all stored
    values are): inside the scale's limit, and multiples of 2^-24."""
    c.scale[which][...] = scales
    s = np.broadcast_to(scales[:, :, None, None], c.codes[which].shape)
    v = B.values(c.codes[which], c.fmt)
    keep = np.isnan(v) | (c.codes[which] == 0x80)  # bytes behind a context
    lim = np.where(s >= 1024, 63.0, 127.0) if c.fmt == B.INT8 else np.where(s >= 256, 240.0, 448.0)
    grid = np.where(s > 0, 2.0 ** -24 / np.where(s > 0, s, 1.0), 1.0)
    v = np.clip(np.rint(np.nan_to_num(v) / grid) * grid, -lim, lim) * (s > 0)
    c.codes[which][...] = np.where(keep, c.codes[which], B.bytes_of(v, c.fmt))


@pytest.mark.parametrize("fmt", [B.INT8, B.FP8])
@pytest.mark.parametrize("D,bs,hq,hkv", [(128, 16, 4, 2), (64, 32, 3, 1)])
@pytest.mark.parametrize("lo,hi", [(-24, -20), (-24, 10), (-12, -12), (10, 10)])
def test_prefill_scales(torch, fmt, D, bs, hq, hkv, lo, hi, prefill_split):
    from redline_amd import kernels as K
    hi, lo = (hi, lo) if fmt == B.INT8 else (min(hi, 8), min(lo, 8))
    say(f"prefill_blocks scales 2^{lo} .. 2^{hi} D={D} bs={bs} fmt={fmt} split={prefill_split}")
    rng = np.random.default_rng(lo + 2 * hi + D)
    segs = [(300, 45), (0, 70)]
    lens = [p + n for p, n in segs]
    c, tab = make(rng, hkv, D, bs, fmt, lens)
    for which in range(2):
        scales = 2.0 ** rng.integers(lo, hi + 1, (c.nb, hkv))
        scales[tab[0, 3 + which]] = 0
        set_scales(c, which, scales)
    t, view = gpu_cache(torch, K, c)
    q = randn_f16(rng, (115, hq, D))
    top = max(np.abs(c.stored(0, b)[:, :1 if b == tab[s, (n - 1) // bs] else bs]).max()
              for s, n in enumerate(lens) for b in tab[s, :-(-n // bs)])
    sc = 1 / (top * D ** 0.5)  # scores of a few units
    got = run_prefill(torch, K, c, view, tab, q, hq, sc, [0, 1], [0, 45], [45, 70], lens, 3)
    for s, (past, n) in enumerate(segs):
        r = slice(45 * s, 45 * s + n)
        want, bound = B.attention(c, tab[s], q[r], sc, [past + i + 1 for i in range(n)])
        check(got[r], want, bound, f"sequence {s}")


def test_prefill_of_many_sequences(torch):
    """Calls on either side of the launch rule (two workgroups of 128 rows a compute
    unit), chosen by the rule itself."""
    from redline_amd import kernels as K
    hkv = 8
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    for D, bs, G, fmt in ((128, 16, 4, B.INT8), (128, 32, 2, B.FP8), (64, 16, 4, B.FP8), (64, 32, 3, B.INT8)):
        tiles = 4
        per = -(-tiles * 32 * G // 128) * hkv
        for seqs in (2 * cus // per, 2 * cus // per + 1):
            say(f"prefill_blocks of {seqs} sequences D={D} G={G} fmt={fmt}")
            rng = np.random.default_rng(D + seqs)
            segs = [(int(rng.integers(0, 90)), int(rng.integers(1, 129))) for _ in range(seqs)]
            lens = [p + n for p, n in segs]
            c, tab = make(rng, hkv, D, bs, fmt, lens)
            t, view = gpu_cache(torch, K, c)
            new = np.array([n for _, n in segs])
            start = np.cumsum(new) - new
            q = randn_f16(rng, (int(new.sum()), G * hkv, D))
            sc = D ** -0.5 / 4
            got = run_prefill(torch, K, c, view, tab, q, G * hkv, sc, np.arange(seqs), start, new, lens, tiles)
            for s in range(0, seqs, 5):
                r = slice(start[s], start[s] + new[s])
                want, bound = B.attention(c, tab[s], q[r], sc, [segs[s][0] + i + 1 for i in range(new[s])])
                check(got[r], want, bound, f"sequence {s}")


@pytest.mark.parametrize("fmt", [B.INT8, B.FP8])
def test_far_blocks(torch, fmt):
    """Write, read back and prefill over the last blocks of a pool of more than 2^32
    bytes each of K and V: the same bits as in a small one."""
    from redline_amd import kernels as K
    say(f"far blocks fmt={fmt}")
    rng = np.random.default_rng(14)
    hq, hkv, D, bs, big = 16, 8, 128, 32, 140000  # 140000 x 8 x 32 x 128 bytes: 4.6 GB
    segs = [(0, 300), (31, 2), (64, 1), (90, 80)]
    lens = [p + n for p, n in segs]
    c, tab = make(rng, hkv, D, bs, fmt, lens)
    shift = big - c.nb
    pos = np.concatenate([np.arange(p, p + n) for p, n in segs]).astype(np.int32)
    seq = np.repeat(np.arange(len(segs)), [n for _, n in segs])
    slots = (tab[seq, pos // bs].astype(np.int64) * bs + pos % bs).astype(np.int32)
    T = len(pos)
    cos, sin = ra.rope_cos_sin_tables(1e4, D, 512)
    x = randn_f16(rng, (T, (hq + 2 * hkv) * D))
    new = np.array([n for _, n in segs])
    start = np.cumsum(new) - new
    got = []
    for far in (False, True):
        t, view = gpu_cache(torch, K, c)
        if far:
            g = [torch.zeros((big,) + tuple(u.shape[1:]), dtype=u.dtype, device="cuda") for u in t]
            for u, w in zip(g, t):
                u[shift:] = w
            t, view = g, K.kv_block_view(*g, bs, hkv, D, fmt)
        at = shift if far else 0
        qkv = dev(torch, x)
        d_slots = dev(torch, slots + at * bs)
        K.rope_and_write_kv_blocks(qkv, dev(torch, pos), d_slots, T, hq, dev(torch, cos), dev(torch, sin), view)
        k, v = (torch.zeros(T, hkv * D, dtype=torch.float16, device="cuda") for _ in "kv")
        K.read_kv_blocks(view, d_slots, T, k, v)
        q = qkv.cpu().numpy().reshape(T, -1, D)[:, :hq]
        o = run_prefill(torch, K, c, view, tab + at, q, hq, 0.05, np.arange(len(segs)), start, new, lens, 10)
        got.append([u[at:].cpu().numpy() for u in t] + [k.cpu().numpy(), v.cpu().numpy(), q, o])
        assert far is False or all(not u[1:shift].any().item() for u in t)
    for a, b in zip(*got):
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
    B.write(c, x, None, pos, slots, hq, cos, sin)
    for a, w in zip(got[1][:2], c.raw()):
        assert np.array_equal(a.view(np.uint8), w)


@pytest.mark.parametrize("S", [512, 513, 2560, 2561])
def test_tables_at_the_rules(torch, S):
    """As many sequences as a launch form takes, and one more."""
    from redline_amd import kernels as K
    say(f"tables of {S} sequences")
    rng = np.random.default_rng(S)
    past, new, table, ring, head, free = random_case(rng, S, 16, 3, 300, 7)
    compare(torch, K, past, new, int(np.maximum(new, 0).sum()), 16, 1, table, ring, head, free, "tables")


def test_write_at_the_rule(torch):
    """1024 rows and one more: the two forms of the write, chosen by the rule."""
    from redline_amd import kernels as K
    from tests.test_kv_blocks_gpu import run_write
    for T in (1024, 1025):
        say(f"write_blocks of {T} rows")
        rng = np.random.default_rng(T)
        segs = [(5, T - 40)] + [(i, 1) for i in range(40)]
        nb = 2 + sum((p + n - 1) // 16 - p // 16 + 2 for p, n in segs)
        c = B.Cache(nb, 2, 16, 64, B.INT8)
        c.fill(rng, -5, 0)
        t, view = gpu_cache(torch, K, c)
        cos, sin = ra.rope_cos_sin_tables(1e4, 64, 2048)
        pos, slots = segments(rng, segs, 16, nb)
        run_write(torch, K, c, t, view, randn_f16(rng, (T, 8 * 64)), None, pos, slots, 4, cos, sin, f"{T} rows")
