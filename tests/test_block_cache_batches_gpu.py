"""Whole batches over the block-scaled cache: BatchBuilder metadata padded to a
graph's size, and two calls at once on two streams."""
import numpy as np
import pytest

import redline_amd as ra
from tests import _kv_blocks as B
from tests._util import randn_f16, say
from tests.test_attention_blocks_gpu import check, make
from tests.test_kv_blocks_gpu import dev, gpu_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


@pytest.mark.parametrize("fmt", [B.INT8, B.FP8])
def test_padded_decode_batch(torch, fmt):
    """Five sequences padded to a batch of 40: the padding rows all write and read the
    scratch block, and the others get what they get without it, to the bit."""
    from redline_amd import kernels as K
    say(f"padded batch fmt={fmt}")
    rng = np.random.default_rng(21)
    hq, hkv, D, bs, S = 8, 2, 128, 16, 5
    past = [0, 15, 16, 700, 333]
    c, tab = make(rng, hkv, D, bs, fmt, [n + 1 for n in past])
    mb, cols = tab.shape[1], (hq + 2 * hkv) * D
    x = randn_f16(rng, (40, cols))
    cos, sin = ra.rope_cos_sin_tables(1e4, D, mb * bs)
    got = []
    for rows in (S, 40):
        bb = ra.BatchBuilder(40, 40, 40, mb, bs, 1)
        for s in range(S):
            bb.add(np.zeros(1, np.int32), past[s], 1, None, tab[s])
        bb.pad_decode_to(rows)
        meta, shape, lay = bb.write()
        assert shape.num_tokens == rows and shape.num_decode_items == rows
        d_meta = dev(torch, meta)
        t, view = gpu_cache(torch, K, c)
        qkv = dev(torch, x[:rows])
        out = torch.full((rows, hq * D), 9.0, dtype=torch.float16, device="cuda")
        K.rope_and_write_kv_blocks(qkv, d_meta[lay["positions"]:], d_meta[lay["slot_mapping"]:], rows, hq,
                                   dev(torch, cos), dev(torch, sin), view)
        ws = K.DecodeWorkspace(rows, hq, 3, D)
        K.paged_attention_decode_blocks(
            K.block_attention_params(qkv, cols, out, hq, 0.08, view, d_meta[lay["block_tables"]:], mb,
                                     d_meta[lay["positions"]:]),
            K.decode_work(d_meta[lay["decode_token"]:], d_meta[lay["decode_seq"]:], rows, 3, ws))
        torch.cuda.synchronize()
        got.append(([a.cpu().numpy()[1:] for a in t], out.cpu().numpy()[:S]))
    for a, b in zip(got[0][0], got[1][0]):
        assert np.array_equal(a, b)
    pos = np.array(past, np.int32)
    slots = np.array([tab[s, n // bs] * bs + n % bs for s, n in enumerate(past)], np.int32)
    q = B.write(c, x[:S], None, pos, slots, hq, cos, sin)
    for _, out in got:
        for s, n in enumerate(past):
            ref, bound = B.attention(c, tab[s], q[s:s + 1], 0.08, [n + 1])
            check(out[s:s + 1].reshape(1, hq, D), ref, bound, f"sequence {s}")


def test_two_streams_at_once(torch):
    """The same steps on two streams at once, each with its own cache, pool and workspace:
    every result is what the calls give one after the other."""
    from redline_amd import kernels as K
    say("two streams")
    rng = np.random.default_rng(22)
    hq, hkv, D, bs, rows, S, mb = 8, 4, 64, 32, 700, 6, 16
    cos, sin = (dev(torch, a) for a in ra.rope_cos_sin_tables(1e4, D, mb * bs))
    x = [dev(torch, randn_f16(rng, (rows, (hq + 2 * hkv) * D))) for _ in range(2)]
    new = [dev(torch, np.array(n, np.int32)) for n in ([300, 1, 90, 1, 200, 64], [1, 1, 400, 1, 1, 260])]

    class Side:
        def __init__(self, k):
            z = lambda *n: torch.zeros(*n, dtype=torch.int32, device="cuda")  # noqa: E731
            self.cache, self.pool = K.KVBlockCache(1, 60, hkv, D, bs, k % 2), K.BlockPool.of_blocks(60)
            self.t = [z(S * mb), z(S), z(S), z(S), z(rows), z(rows), z(rows), z(rows), z(S), z(4)]
            bt, q_start, q_len, ctx, pos, self.slots, tok, seq, pre, _ = self.t
            self.work = K.batch_tables(self.pool, z(S), new[k], S, rows, bs, 1, bt, mb, *self.t[1:])
            self.qkv, self.pos, self.src = torch.empty_like(x[k]), pos, x[k]
            self.out = torch.zeros(rows, hq * D, dtype=torch.float16, device="cuda")
            self.k, self.v = (torch.zeros(rows, hkv * D, dtype=torch.float16, device="cuda") for _ in range(2))
            self.p = K.block_attention_params(self.qkv, self.qkv.shape[1], self.out, hq, 0.1, self.cache.layer(0),
                                              bt, mb, pos)
            self.ws = K.DecodeWorkspace(S, hq, 2, D)
            self.dw, self.pw = K.decode_work(tok, seq, S, 2, self.ws), K.prefill_work(pre, q_start, q_len, ctx, S, 13)

        def step(self):
            self.qkv.copy_(self.src)
            K.build_batch_tables(self.work)
            K.rope_and_write_kv_blocks(self.qkv, self.pos, self.slots, rows, hq, cos, sin, self.cache.layer(0))
            K.paged_attention_decode_blocks(self.p, self.dw)
            K.paged_attention_prefill_blocks(self.p, self.pw)
            K.read_kv_blocks(self.cache.layer(0), self.slots, rows, self.k, self.v)

        def results(self):
            return [a.cpu().numpy() for a in (self.out, self.k, self.v, *self.t, *self.cache.tensors(0))]

    want = []
    for k in range(2):
        s = Side(k)
        s.step()
        torch.cuda.synchronize()
        want.append(s.results())
        assert want[k][12].tolist()[3] == 0
    for _ in range(3):
        sides, streams = [Side(k) for k in range(2)], [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        for side, stream in zip(sides, streams):
            with torch.cuda.stream(stream):
                side.step()
        torch.cuda.synchronize()
        for side, w in zip(sides, want):
            for a, b in zip(side.results(), w):
                assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
