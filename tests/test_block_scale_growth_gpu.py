"""Blocks of the block-scaled cache whose scale grows to the largest one: the codes
of the earlier tokens saturate where the new scale's own codes do, so that every
stored value stays a finite fp16 number."""
import numpy as np
import pytest

import redline_amd as ra
from tests import _kv_blocks as B
from tests._util import assert_bits_equal, say
from tests.test_attention_blocks_gpu import check, run_decode, run_prefill
from tests.test_kv_blocks_gpu import check_cache, dev, gpu_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


@pytest.fixture(params=[4, 16])
def write_rows(request):
    from redline_amd._lib import tune_knob
    with tune_knob("RLK_TUNE_BLK_WRITE", request.param):
        yield request.param


def write_clamped(c, rows, blk, off):
    """Cache.write_run, with the earlier codes held inside the new scale's limit
    (it lets an INT8 code of 127 become 64 at 2^10, which is 65536)."""
    c.write_run(rows, blk, off)
    for which in range(2):
        for h in range(c.hkv):
            lim = B.limit(c.scale[which][blk, h], c.fmt)
            old = c.codes[which][blk, h, :off]
            c.codes[which][blk, h, :off] = B.bytes_of(np.clip(B.values(old, c.fmt), -lim, lim), c.fmt)


@pytest.mark.parametrize("fmt", [B.INT8, B.FP8])
@pytest.mark.parametrize("D,bs", [(64, 16), (128, 32)])
@pytest.mark.parametrize("off", [1, 2, 5, 8, 15, 21, 31])  # inside the first quad, behind whole ones, the second tile
@pytest.mark.parametrize("first", [65024.0, 64768.0, 57344.0, 32512.0, 3.0])
def test_growth_to_the_largest_scale(torch, fmt, D, bs, off, first, write_rows):
    from redline_amd import kernels as K
    say(f"block growth fmt={fmt} D={D} bs={bs} off={off} first={first} rows={write_rows}")
    off = min(off, bs - 1)
    rng = np.random.default_rng(off)
    hq, hkv, nb = 2, 2, 3
    cols = (hq + 2 * hkv) * D
    c = B.Cache(nb, hkv, bs, D, fmt)
    t, view = gpu_cache(torch, K, c)
    cos, sin = np.ones((1, D // 2), np.float32), np.zeros((1, D // 2), np.float32)
    d_cos, d_sin = dev(torch, cos), dev(torch, sin)

    def write(x, at):
        n = len(x)
        K.rope_and_write_kv_blocks(dev(torch, x), dev(torch, np.zeros(n, np.int32)),
                                   dev(torch, (bs + at + np.arange(n)).astype(np.int32)), n, hq, d_cos, d_sin, view)
        torch.cuda.synchronize()
        y = x.astype(np.float64).reshape(n, -1, D)
        write_clamped(c, (y[:, hq:hq + hkv], y[:, hq + hkv:]), 1, at)
        check_cache(t, c, f"rows at {at}")

    # every token has the block's largest magnitude, in either sign, and smaller ones
    x = (rng.uniform(-1, 1, (off, cols)) * first).astype(np.float16)
    x[:, ::7], x[:, 1::7] = first, -first
    write(x, 0)
    last = (rng.uniform(-1, 1, (1, cols)) * 60000).astype(np.float16)
    last[:, ::5], last[:, 1::5] = 65504.0, -65504.0
    write(last, off)
    n = off + 1
    assert (c.scale[0][1] == (1024 if fmt == B.INT8 else 256)).all()
    k, v = (torch.zeros(n, hkv * D, dtype=torch.float16, device="cuda") for _ in "kv")
    K.read_kv_blocks(view, dev(torch, (bs + np.arange(n)).astype(np.int32)), n, k, v)
    for which, got in enumerate((k, v)):
        want = c.stored(which, 1)[:, :n].transpose(1, 0, 2).reshape(n, -1)
        assert np.abs(want).max() <= 65504
        assert_bits_equal(got.cpu().numpy(), want.astype(np.float16), "read back")
    # rows of the earlier tokens see none of the last one, and all are finite
    tab, sc = np.array([[1]], np.int32), 2.0 ** -24
    q = (rng.standard_normal((n, hq, D))).astype(np.float16)
    want, bound = B.attention(c, tab[0], q, sc, list(range(1, n + 1)))
    got = run_prefill(torch, K, c, view, tab, q, hq, sc, [0], [0], [n], [n], 1)
    check(got, want, bound, "prefill")
    got = run_decode(torch, K, c, view, tab, q, hq, sc, np.arange(n), np.arange(n), np.zeros(n), 1)
    check(got, want, bound, "decode")
