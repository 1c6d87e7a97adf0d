"""Refusals of the shared-prefix decode attention, before anything is launched (no GPU)."""
import ctypes as C

import pytest

import redline_amd as ra
from redline_amd import _lib

P = 16  # a non-null, 16-byte aligned stand-in: nothing is launched
EINVAL, EUNSUP = _lib.RLK_EINVAL, _lib.RLK_EUNSUPPORTED


def call(kv=(), p=(), w=(), sd=0):
    f = dict(k=P, v=P, k_scale=P, v_scale=P, block_size=16, num_kv_heads=2, head_dim=64, dtype=_lib.RLK_KV_INT8)
    view = _lib.KVLayerView(*(f | dict(kv)).values())
    f = dict(q=P, q_stride=512, out=P, num_heads=4, scale=0.1, kv=view, tables=P, max_blocks=4, positions=P)
    params = _lib.AttentionParams(*(f | dict(p)).values())
    f = dict(token=P, seq=P, items=2, start=P, prefix=P, groups=1, max_items=2, prefix_parts=1, parts=1, o=P, m=P, s=P)
    work = _lib.SharedPrefixWork(*(f | dict(w)).values())
    return ra.lib().rlk_paged_attention_decode_shared(C.byref(params), C.byref(work),
                                                      C.byref(_lib.AttentionOptions(sd)), None)


@pytest.mark.parametrize("kw,status,text", [
    (dict(kv=dict(head_dim=96)), EUNSUP, b"head_dim 96"), (dict(kv=dict(dtype=2)), EINVAL, b"dtype 2"),
    (dict(kv=dict(block_size=0)), EINVAL, b"block size"), (dict(kv=dict(num_kv_heads=0)), EINVAL, b"head count"),
    (dict(kv=dict(k=None)), EINVAL, b"null"), (dict(kv=dict(k_scale=None)), EINVAL, b"null"),
    (dict(kv=dict(v=24)), EINVAL, b"16-byte"), (dict(sd=3), EINVAL, b"scale dtype"),
    (dict(p=dict(num_heads=5)), EINVAL, b"multiple"), (dict(p=dict(num_heads=18)), EUNSUP, b"group size 9"),
    (dict(p=dict(num_heads=0)), EINVAL, b"multiple"), (dict(p=dict(q=None)), EINVAL, b"null"),
    (dict(p=dict(q=8)), EINVAL, b"16-byte"), (dict(p=dict(q_stride=516)), EINVAL, b"q_stride 516"),
    (dict(p=dict(out=40)), EINVAL, b"16-byte"), (dict(p=dict(max_blocks=0)), EINVAL, b"table width"),
    (dict(p=dict(max_blocks=2 ** 31 - 1)), EINVAL, b"table width"), (dict(p=dict(positions=None)), EINVAL, b"null"),
    (dict(w=dict(groups=-1)), EINVAL, b"group counts"), (dict(w=dict(max_items=-1)), EINVAL, b"group counts"),
    (dict(w=dict(parts=0)), EINVAL, b"partition"), (dict(w=dict(prefix_parts=-1)), EINVAL, b"partition"),
    (dict(w=dict(prefix_parts=2 ** 30)), EINVAL, b"partition"), (dict(w=dict(start=None)), EINVAL, b"null"),
    (dict(w=dict(token=None)), EINVAL, b"null"), (dict(w=dict(m=None)), EINVAL, b"workspace"),
    (dict(w=dict(items=2 ** 31 - 1)), EINVAL, b"split"), (dict(w=dict(groups=2 ** 31 - 1)), EINVAL, b"split")])
def test_refusals(kw, status, text):
    assert call(**kw) == status, ra.lib().rlk_last_error()
    assert text in ra.lib().rlk_last_error()


def test_nothing_to_do():
    assert call(w=dict(items=0)) == 0 and call(w=dict(items=-1, token=None)) == 0
    assert ra.lib().rlk_paged_attention_decode_shared(None, None, None, None) == EINVAL


def test_scales_that_are_no_number():
    for bad in (float("nan"), float("inf"), -float("inf")):
        assert call(p=dict(scale=bad)) == EINVAL and b"finite" in ra.lib().rlk_last_error()


def test_the_workspace_is_one():
    from redline_amd import kernels as K
    for bad in (None, 5, "x"):
        with pytest.raises(ra.Error, match="DecodeWorkspace"):
            K.shared_prefix_work(None, None, 1, None, None, 0, 0, 0, 1, bad)


def test_more_units_than_a_launch_takes():
    for w in (dict(), dict(groups=0)):
        assert call(kv=dict(num_kv_heads=32), p=dict(num_heads=32), w=dict(items=1 << 20) | w) == EINVAL
        assert b"split the call" in ra.lib().rlk_last_error()
