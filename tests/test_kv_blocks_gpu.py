"""The block-scaled cache's write and read back against the numpy restatement
(tests/_kv_blocks.py).  The rotation is fixed to the bit and the scales are
powers of two, so q, every byte of the cache and every scale are compared
exactly."""
import numpy as np
import pytest

import redline_amd as ra
from tests import _kv_blocks as B
from tests._util import assert_bits_equal, randn_f16, say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


def dev(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def gpu_cache(torch, K, c):
    """The numpy cache's contents as (tensors, view)."""
    k, v = c.raw()
    dt = np.int8 if c.fmt == B.INT8 else np.uint8
    t = [dev(torch, k.view(dt)), dev(torch, v.view(dt)), dev(torch, c.scale[0].astype(np.float32)),
         dev(torch, c.scale[1].astype(np.float32))]
    return t, K.kv_block_view(*t, c.bs, c.hkv, c.D, c.fmt)


def check_cache(t, c, what):
    for got, want, n in zip(t, (*c.raw(), c.scale[0].astype(np.float32), c.scale[1].astype(np.float32)),
                            ("k", "v", "k_scale", "v_scale")):
        assert_bits_equal(got.cpu().numpy().view(want.dtype), want, f"{what}: {n}")


def segments(rng, segs, bs, nb):
    """Positions and slots of packed sequences (past, new) over distinct blocks."""
    ids = rng.permutation(np.arange(1, nb))
    pos, slots, at = [], [], 0
    for past, new in segs:
        first = past // bs
        n = (past + new - 1) // bs - first + 1
        tab = {first + i: ids[at + i] for i in range(n)}
        at += n
        for p in range(past, past + new):
            pos.append(p)
            slots.append(tab[p // bs] * bs + p % bs)
    return np.array(pos, np.int32), np.array(slots, np.int32)


def run_write(torch, K, c, t, view, qkv, bias, pos, slots, hq, cos, sin, what):
    d = dev(torch, qkv)
    K.rope_and_write_kv_blocks(d, dev(torch, pos), dev(torch, slots), len(pos), hq, dev(torch, cos),
                               dev(torch, sin), view, None if bias is None else dev(torch, bias))
    torch.cuda.synchronize()
    q = B.write(c, qkv, bias, pos, slots, hq, cos, sin)
    got = d.cpu().numpy().reshape(len(pos), -1, c.D)
    want = qkv.reshape(len(pos), -1, c.D).copy()
    want[:, :hq] = q
    assert_bits_equal(got, want, f"{what}: qkv")
    check_cache(t, c, what)


WRITE_CASES = [
    # hq, hkv, D, bs, fmt, bias, segments
    (4, 2, 128, 16, B.INT8, False, [(0, 1)]),
    (4, 2, 128, 16, B.FP8, False, [(15, 1), (16, 1), (31, 1), (0, 16), (7, 9), (3, 30)]),
    (6, 3, 64, 16, B.INT8, True, [(5, 40), (0, 17), (14, 3), (33, 1)]),
    (7, 1, 64, 32, B.FP8, True, [(31, 34), (0, 32), (1, 1), (40, 7)]),
    (2, 2, 128, 32, B.INT8, True, [(30, 5), (0, 64), (63, 1), (17, 50)]),
    (5, 5, 128, 32, B.FP8, False, [(0, 100), (18, 3)]),
    (3, 1, 128, 16, B.INT8, False, [(i % 23, 1) for i in range(70)]),
    # more than 1024 rows: waves that look at 16 rows
    (4, 2, 64, 16, B.INT8, False, [(3, 500), (0, 41), (9, 700)] + [(i % 40, 1 + i % 3) for i in range(40)]),
    (2, 1, 128, 32, B.FP8, True, [(29, 900), (0, 1), (5, 333)]),
]


@pytest.fixture(params=[None, 4, 16], ids=["rule", "rows4", "rows16"])
def write_rows(request):
    """Rows that a wave looks at: the launcher's choice, and each forced."""
    from redline_amd._lib import tune_knob
    with tune_knob("RLK_TUNE_BLK_WRITE", request.param):
        yield request.param


@pytest.mark.parametrize("hq,hkv,D,bs,fmt,bias,segs", WRITE_CASES)
def test_write_matches_definition(torch, hq, hkv, D, bs, fmt, bias, segs, write_rows):
    """Two steps, the second continuing blocks with larger and smaller rows, so
    scales grow and stay; bytes outside the runs are untouched."""
    from redline_amd import kernels as K
    say(f"write_blocks hq={hq} hkv={hkv} D={D} bs={bs} fmt={fmt} bias={bias} seqs={len(segs)} rows={write_rows}")
    rng = np.random.default_rng(len(segs) * 7 + D + bs)
    nb = 2 + sum((p + n - 1) // bs - p // bs + 2 for p, n in segs)
    c = B.Cache(nb, hkv, bs, D, fmt)
    c.fill(rng, -5, 0)
    t, view = gpu_cache(torch, K, c)
    cos, sin = ra.rope_cos_sin_tables(1e4, D, 2048)
    pos, slots = segments(rng, segs, bs, nb)
    for step in range(2):
        T = len(pos)
        rows = randn_f16(rng, (T, (hq + 2 * hkv) * D)) * np.exp2(rng.integers(-4, 5, (T, 1))).astype(np.float16)
        b = randn_f16(rng, (hq + 2 * hkv) * D) if bias else None
        run_write(torch, K, c, t, view, rows, b, pos, slots, hq, cos, sin, f"step {step}")


@pytest.mark.parametrize("fmt", [B.INT8, B.FP8])
@pytest.mark.parametrize("D,bs", [(64, 16), (128, 32)])
def test_write_token_by_token_and_skips(torch, fmt, D, bs):
    """One token a call through two blocks; then a call whose rows hold slots
    that are negative or past the pool between valid ones."""
    from redline_amd import kernels as K
    say(f"write_blocks token by token fmt={fmt} D={D} bs={bs}")
    rng = np.random.default_rng(3)
    hq, hkv, nb = 2, 2, 6
    c = B.Cache(nb, hkv, bs, D, fmt)
    t, view = gpu_cache(torch, K, c)
    cos, sin = ra.rope_cos_sin_tables(1e4, D, 256)
    for p in range(bs + 3):
        x = randn_f16(rng, (1, (hq + 2 * hkv) * D)) * np.float16(2.0 ** (p % 7 - 3))
        if p == 1:
            x[:] = 0
        run_write(torch, K, c, t, view, x, None, np.array([p], np.int32),
                  np.array([(3 if p < bs else 4) * bs + p % bs], np.int32), hq, cos, sin, f"token {p}")
    slots = np.array([-1, 2 * bs, 2 * bs + 1, -5, 2 * bs + 2, nb * bs, nb * bs + 1, 5 * bs, 2 ** 31 - 1, 5 * bs + 1,
                      5 * bs + 2, -1], np.int32)
    # (the runs at 2 * bs + 2 and 5 * bs + 1 continue a block that an earlier run of
    # the call started: two calls, so that no two runs of one share a block)
    first = slots.copy()
    first[[4, 9, 10]] = -1
    second = np.full_like(slots, -1)
    second[[4, 9, 10]] = slots[[4, 9, 10]]
    x = randn_f16(rng, (len(slots), (hq + 2 * hkv) * D), 3.0)
    for s in (first, second):
        run_write(torch, K, c, t, view, x, None, np.arange(len(slots), dtype=np.int32), s, hq, cos, sin, "skips")


@pytest.mark.parametrize("fmt", [B.INT8, B.FP8])
def test_write_extreme_values(torch, fmt):
    """Zeros, fp16's smallest and largest numbers and infinities in V, and scale
    borders: amax exactly at and one step above the largest code times 2^e."""
    from redline_amd import kernels as K
    say(f"write_blocks extremes fmt={fmt}")
    D, bs, hq, hkv = 64, 16, 1, 1
    top = int(B.QMAX[fmt])
    mags = [0.0, 2.0 ** -24, 3 * 2.0 ** -24, 2.0 ** -14, top / 64, np.nextafter(np.float16(top / 64), np.float16(np.inf)),
            1.0, 65504.0, 65024.0, 32768.0, np.inf]
    c = B.Cache(len(mags) + 1, hkv, bs, D, fmt)
    t, view = gpu_cache(torch, K, c)
    cos, sin = ra.rope_cos_sin_tables(1e4, D, 16)
    rng = np.random.default_rng(9)
    for i, mag in enumerate(mags):
        x = np.zeros((bs, (hq + 2 * hkv) * D), np.float16)
        u = rng.uniform(-1, 1, (bs, D))
        with np.errstate(over="ignore", invalid="ignore"):
            x[:, -D:] = np.where(np.isinf(mag), 60000.0 * u, mag * u).astype(np.float16)
        x[3, -5], x[7, -D] = mag, -mag
        run_write(torch, K, c, t, view, x, None, np.zeros(bs, np.int32),
                  ((i + 1) * bs + np.arange(bs)).astype(np.int32), hq, cos, sin, f"magnitude {mag}")
        got = torch.zeros(bs, D, dtype=torch.float16, device="cuda")
        K.read_kv_blocks(view, dev(torch, ((i + 1) * bs + np.arange(bs)).astype(np.int32)), bs, None, got)
        got = got.cpu().numpy().astype(np.float64)
        assert np.isfinite(got).all()
        # half a step: 2^-4 of an e4m3 value (its subnormal spacing 2^-9 s), half a
        # scale for INT8; at the largest scale up to the saturated code
        want = np.clip(x[:, -D:].astype(np.float64), -65504, 65504)
        s = c.scale[1][i + 1, 0]
        half = np.maximum(np.abs(want) * 2.0 ** -4, s * 2.0 ** -10) if fmt == B.FP8 else s / 2
        sat = np.abs(want) > B.limit(s, fmt) * s
        assert (np.abs(got - want) <= np.where(sat, 65504 - B.limit(s, fmt) * s, half)).all()


@pytest.mark.parametrize("fmt", [B.INT8, B.FP8])
@pytest.mark.parametrize("hkv,D,bs", [(1, 64, 16), (3, 128, 16), (2, 64, 32), (8, 128, 32)])
def test_read_back(torch, fmt, hkv, D, bs):
    """Rows in any order, repeated, aligned quads and not; skipped rows stay."""
    from redline_amd import kernels as K
    say(f"read_blocks fmt={fmt} hkv={hkv} D={D} bs={bs}")
    rng = np.random.default_rng(5)
    c = B.Cache(7, hkv, bs, D, fmt)
    c.fill(rng, -8, 4)
    t, view = gpu_cache(torch, K, c)
    slots = np.concatenate([np.arange(4 * bs), rng.integers(0, 7 * bs, 37), [-1, 7 * bs, 2 ** 31 - 1, 5, 5, 5]]).astype(np.int32)
    for n in (len(slots), 1, 4, 5):
        outs = [torch.full((len(slots), hkv * D), 7.0, dtype=torch.float16, device="cuda") for _ in "kv"]
        K.read_kv_blocks(view, dev(torch, slots), n, *outs)
        for which, o in enumerate(outs):
            want = np.full((len(slots), hkv, D), 7.0)
            for i in range(n):
                if 0 <= slots[i] < 7 * bs:
                    want[i] = c.stored(which, slots[i] // bs)[:, slots[i] % bs]
            assert_bits_equal(o.cpu().numpy(), want.astype(np.float16).reshape(len(slots), -1), f"read {n}")
    only = torch.zeros((4 * bs, hkv * D), dtype=torch.float16, device="cuda")
    K.read_kv_blocks(view, dev(torch, slots), 4 * bs, only, None)
    want = np.stack([c.stored(0, p // bs)[:, p % bs] for p in range(4 * bs)])
    assert_bits_equal(only.cpu().numpy(), want.astype(np.float16).reshape(4 * bs, -1), "k alone")


def test_write_on_another_stream_and_in_a_graph(torch):
    """The call follows the stream it is given; a captured call replayed gives
    what the eager one does."""
    from redline_amd import kernels as K
    say("write_blocks stream and graph")
    rng = np.random.default_rng(6)
    hq, hkv, D, bs, nb = 4, 2, 128, 16, 40
    cos, sin = (dev(torch, a) for a in ra.rope_cos_sin_tables(1e4, D, 256))
    pos, slots = segments(rng, [(0, 30), (5, 1), (12, 20)], bs, nb)
    x = dev(torch, randn_f16(rng, (len(pos), (hq + 2 * hkv) * D)))
    d_pos, d_slots = dev(torch, pos), dev(torch, slots)

    def fresh():
        c = B.Cache(nb, hkv, bs, D, B.INT8)
        return gpu_cache(torch, K, c)

    t0, v0 = fresh()
    x0 = x.clone()
    K.rope_and_write_kv_blocks(x0, d_pos, d_slots, len(pos), hq, cos, sin, v0)
    side = torch.cuda.Stream()
    t1, v1 = fresh()
    x1 = x.clone()
    side.wait_stream(torch.cuda.current_stream())
    K.rope_and_write_kv_blocks(x1, d_pos, d_slots, len(pos), hq, cos, sin, v1, stream=side)
    side.synchronize()
    t2, v2 = fresh()
    x2 = x.clone()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        K.rope_and_write_kv_blocks(x2, d_pos, d_slots, len(pos), hq, cos, sin, v2)
    for _ in range(3):
        x2.copy_(x)
        for u in t2:
            u.zero_()
        g.replay()
        torch.cuda.synchronize()
        for a, b, c in zip((x0, *t0), (x1, *t1), (x2, *t2)):
            assert torch.equal(a, b) and torch.equal(a, c)


def test_launches_refuse_another_device(torch):
    """A launch goes to the current device: tensors of another are refused (the
    views carry their device, which this test changes)."""
    from redline_amd import kernels as K
    cache = K.KVBlockCache(1, 4, 2, 64)
    kv = cache.layer(0)
    i = torch.zeros(4, dtype=torch.int32, device="cuda")
    x = torch.zeros(4, 8 * 64, dtype=torch.float16, device="cuda")
    p = K.block_attention_params(x, 512, x.clone(), 4, 0.1, kv, i, 1, i)
    pool = K.BlockPool.of_blocks(4)
    tb = K.batch_tables(pool, i, i, 1, 1, 16, 1, i, 1, *[torch.zeros(4, dtype=torch.int32, device="cuda") for _ in range(9)])
    K.read_kv_blocks(kv, i, 4, x[:, :128].contiguous(), None)
    kv.device, p.device, pool.device = 1, 1, 1
    f = torch.zeros(16, 32, device="cuda")
    for call in (lambda: K.read_kv_blocks(kv, i, 4, x, None), lambda: K.paged_attention_decode_blocks(p, K.decode_work(i, i, 1, 1)),
                 lambda: K.paged_attention_prefill_blocks(p, K.prefill_work(i, i, i, i, 1, 1)),
                 lambda: K.build_batch_tables(tb),
                 lambda: K.rope_and_write_kv_blocks(x, i, i, 4, 4, f, f, kv)):
        with pytest.raises(ra.Error, match="device"):
            call()
