"""The work descriptions of the attention launchers: they keep the tensors whose
pointers they hold, and lists or workspaces that are too small or on another
device are refused before anything is launched."""
import gc
import weakref

import pytest

import redline_amd as ra

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


def ints(torch, n):
    return torch.zeros(n, dtype=torch.int32, device="cuda")


def test_work_lists_are_kept(torch):
    from redline_amd import kernels as K
    made = [ints(torch, 4) for _ in range(6)]
    ws = K.DecodeWorkspace(4, 2, 2, 64)
    refs = [weakref.ref(t) for t in (*made, ws.out, ws.max, ws.sum)]
    work = K.decode_work(*made[:2], 4, 2, ws), K.prefill_work(*made[2:], 4, 1)
    del made, ws
    gc.collect()
    assert all(r() is not None for r in refs)
    del work
    gc.collect()
    assert all(r() is None for r in refs)


def test_short_lists_and_workspaces_are_refused(torch):
    from redline_amd import kernels as K
    i = ints(torch, 4)
    for kw in (dict(item_token=i[:3], item_seq=i), dict(item_token=i, item_seq=i[:2])):
        with pytest.raises(ra.Error, match="holds"):
            K.decode_work(**kw, num_items=4, max_partitions=1)
    with pytest.raises(ra.Error, match="seq_ids holds"):
        K.prefill_work(i[:1], i, i, i, 2, 1)
    K.prefill_work(i[:1], i, i, i, 2, 0)  # nothing to do, whatever the lists hold
    cache = K.KVBlockCache(1, 4, 2, 64)
    x = torch.zeros(4, 4 * 64, dtype=torch.float16, device="cuda")
    p = K.block_attention_params(x, 256, torch.zeros_like(x), 4, 0.1, cache.layer(0), ints(torch, 8), 2, i)
    for what, cut in (("out", 1), ("max", 1), ("sum", 1)):
        ws = K.DecodeWorkspace(4, 4, 2, 64)
        setattr(ws, what, getattr(ws, what)[:-cut])
        with pytest.raises(ra.Error, match="the workspace holds"):
            K.paged_attention_decode_blocks(p, K.decode_work(i, i, 4, 2, ws))
    K.paged_attention_decode_blocks(p, K.decode_work(i, i, 4, 2, K.DecodeWorkspace(4, 4, 2, 64)))
    torch.cuda.synchronize()


def test_work_lists_of_another_device_are_refused(torch):
    """(The descriptions carry their device, which this test changes.)"""
    from redline_amd import kernels as K
    cache = K.KVBlockCache(1, 4, 2, 64)
    i = ints(torch, 4)
    x = torch.zeros(4, 4 * 64, dtype=torch.float16, device="cuda")
    p = K.block_attention_params(x, 256, torch.zeros_like(x), 4, 0.1, cache.layer(0), ints(torch, 8), 2, i)
    d, f = K.decode_work(i, i, 4, 1), K.prefill_work(i, i, i, i, 1, 1)
    d.device = f.device = 1
    for call in (lambda: K.paged_attention_decode_blocks(p, d), lambda: K.paged_attention_prefill_blocks(p, f)):
        with pytest.raises(ra.Error, match="another device"):
            call()
