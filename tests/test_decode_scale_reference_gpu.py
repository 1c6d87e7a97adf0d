"""Decode attention where blocks with large V scales have next to no probability: the
attended values keep their bits however much smaller their scale is."""
import numpy as np
import pytest

from tests import _kv_blocks as B
from tests._util import say
from tests.test_attention_blocks_gpu import check, make, run_decode, run_prefill
from tests.test_kv_blocks_gpu import gpu_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


@pytest.fixture(params=[0, 1], ids=["grid", "range"])
def decode_form(request):
    from redline_amd._lib import tune_knob
    with tune_knob("RLK_TUNE_BLK_DECODE", request.param):
        yield request.param


def attention(c, table, q, scale, n):
    """float64 attention of one row q [hq, D] over n keys: (out, bound of decode, bound
    of prefill), by the roundings of each:
      fp16 output         2^-11 |o| and half its subnormal spacing, 2^-25
      fp32 scores         as in _kv_blocks.attention
      fp16 operand        2^-11 sum p|v|, and below fp16's normal range 2^-25 a key,
                          relative to the row's largest operand or less.  Decode's
                          operand is p s (s the key's V scale, 2^-24 where it is 0) and
                          multiplies a code; prefill's is p, multiplies the value, and
                          loses no more than the key's p where that is less.
    """
    hq, D = q.shape
    G = hq // c.hkv
    ids = table[:-(-n // c.bs)]
    k = np.concatenate([c.stored(0, b) for b in ids], 1)[:, :n]
    v = np.concatenate([c.stored(1, b) for b in ids], 1)[:, :n]
    vs = np.maximum(np.repeat(c.scale[1][ids].T, c.bs, 1)[:, :n], 2.0 ** -24)
    out, dec, pre = (np.zeros((hq, D)) for _ in range(3))
    for h in range(hq):
        kk, vv, s = k[h // G], v[h // G], vs[h // G]
        x = q[h].astype(np.float64)
        z = kk @ x * scale
        p = np.exp(z - z.max())
        L = p.sum()
        out[h] = p @ vv / L
        a = p @ np.abs(vv) / L
        dev = 2 * (D + 8) * 2.0 ** -24 * abs(scale) * np.max(np.abs(kk) @ np.abs(x))
        both = 2.0 ** -25 + 2.0 ** -11 * np.abs(out[h]) + (2.0 ** -11 + 2 * dev + 2.0 ** -18) * a
        dec[h] = both + n * 2.0 ** -25 * np.max(p * s) * B.QMAX[c.fmt] / L
        pre[h] = both + np.minimum(p, 2.0 ** -25) @ np.abs(vv) / L
    return out, dec, pre


@pytest.mark.parametrize("gap", [40.0, 18.0])  # e^-18 2^26 is about 1: both sides weigh alike
@pytest.mark.parametrize("fmt", [B.INT8, B.FP8])
@pytest.mark.parametrize("D,bs,n", [(128, 16, 40), (128, 16, 1000), (64, 32, 3000), (64, 16, 700)])
@pytest.mark.parametrize("loud", ["first", "last", "every third", "all but one"])
def test_loud_blocks_without_weight(torch, D, bs, n, fmt, loud, gap, decode_form):
    from redline_amd import kernels as K
    say(f"decode_blocks loud blocks D={D} bs={bs} n={n} fmt={fmt} loud={loud} gap={gap} form={decode_form}")
    rng = np.random.default_rng(D + n)
    hq, hkv = 6, 2
    c, tab = make(rng, hkv, D, bs, fmt, [n])
    blocks = tab[0, :-(-n // bs)]
    top = 10 if fmt == B.INT8 else 8
    pick = {"first": blocks[:1], "last": blocks[-1:], "every third": blocks[1::3],
            "all but one": np.delete(blocks, len(blocks) // 2)}[loud]
    c.codes[0][...] = 0
    c.scale[0][...] = 1.0
    c.codes[0][pick, :, :, 0] = B.bytes_of(np.array([1.0]), fmt)[0]  # loud keys have 1 in dim 0, the others 0
    c.scale[1][blocks] = 2.0 ** (top - 26)
    c.scale[1][pick] = 2.0 ** top
    lim = B.limit(2.0 ** top, fmt)
    for b in blocks:  # stored values stay fp16 numbers, and bytes behind the context as they are
        used = slice(0, n - bs * int(np.flatnonzero(blocks == b)[0]))
        vals = B.values(c.codes[1][b][:, used], fmt)
        c.codes[1][b][:, used] = B.bytes_of(np.clip(vals, -lim, lim), fmt)
    t, view = gpu_cache(torch, K, c)
    q = np.zeros((1, hq, D), np.float16)
    q[:, :, 0] = -gap
    want, dec, pre = attention(c, tab[0], q[0], 1.0, n)
    assert np.abs(want).max() > 64 * 2.0 ** -25  # not all below fp16's spacing
    parts = -(-n // 256)
    got = run_decode(torch, K, c, view, tab, q, hq, 1.0, [n - 1], [0], [0], parts)
    check(got[0], want, dec, "decode")
    got = run_prefill(torch, K, c, view, tab, q, hq, 1.0, [0], [0], [1], [n], 1)
    check(got[0], want, pre, "prefill")
