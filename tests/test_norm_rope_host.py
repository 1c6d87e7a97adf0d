"""Refusals of the normed cache write and of the row read, before anything is launched
(no GPU)."""
import ctypes as C

import pytest

import redline_amd as ra
from redline_amd import _lib

P = 16  # a non-null, 16-byte aligned stand-in: nothing is launched
EINVAL, EUNSUP = _lib.RLK_EINVAL, _lib.RLK_EUNSUPPORTED


def view(**kw):
    f = dict(k=P, v=P, k_scale=P, v_scale=P, block_size=16, num_kv_heads=2, head_dim=64, dtype=_lib.RLK_KV_INT8)
    return _lib.KVLayerView(*(f | kw).values())


def options(**kw):
    f = dict(q_norm=P, k_norm=P, eps=1e-6, qkv_bias=None, scale_dtype=0, num_axes=0,
             sections=(C.c_int * 4)(*kw.pop("sections", ())), interleaved=0)
    return _lib.NormRopeOptions(*(f | kw).values())


def write(kv=None, opt=None, n=3, **kw):
    f = dict(qkv=P, pos=P, slots=P, n=n, heads=4, cos=P, sin=P) | kw
    return ra.lib().rlk_rope_and_write_kv_norm(*f.values(), C.byref(kv or view()), C.byref(opt or options()), None)


def read(kv=None, n=3, slots=P, k=P, v=P, sd=0):
    return ra.lib().rlk_read_kv(C.byref(kv or view()), slots, n, k, v, sd, None)


@pytest.mark.parametrize("kw,status,text", [
    (dict(head_dim=96), EUNSUP, b"head_dim 96"), (dict(dtype=3), EINVAL, b"dtype 3"), (dict(k=None), EINVAL, b"null"),
    (dict(v_scale=None), EINVAL, b"null"), (dict(v=24), EINVAL, b"16-byte"), (dict(block_size=0), EINVAL, b"block size"),
    (dict(num_kv_heads=0), EINVAL, b"head count")])
def test_bad_views(kw, status, text):
    for call in (write, read):
        assert call(view(**kw)) == status and text in ra.lib().rlk_last_error()


@pytest.mark.parametrize("kw,text", [
    (dict(num_axes=5), b"5 position axes"), (dict(num_axes=-1), b"position axes"),
    (dict(num_axes=2, sections=(16, 15)), b"31 pairs of 32"), (dict(num_axes=2, sections=(40, -8)), b"negative section"),
    (dict(num_axes=3, sections=(2, 30, 0), interleaved=1), b"do not fit"), (dict(eps=-1.0), b"eps"),
    (dict(eps=float("nan")), b"eps"), (dict(scale_dtype=2), b"scale dtype"), (dict(q_norm=8), b"16-byte"),
    (dict(qkv_bias=24), b"16-byte"), (dict(num_axes=2, sections=(2 ** 31 - 1, 2 ** 31 - 1)), b"pairs")])
def test_bad_options(kw, text):
    assert write(opt=options(**kw)) == EINVAL and text in ra.lib().rlk_last_error()


def test_bad_arguments():
    err = ra.lib().rlk_last_error
    for kw, text in ((dict(qkv=None), b"null"), (dict(pos=None), b"null"), (dict(sin=None), b"null"),
                     (dict(qkv=8), b"16-byte"), (dict(cos=20), b"16-byte"), (dict(heads=-1), b"head count"),
                     (dict(heads=2 ** 31 - 1), b"heads")):
        assert write(**kw) == EINVAL and text in err()
    assert ra.lib().rlk_rope_and_write_kv_norm(P, P, P, 1, 4, P, P, None, None, None) == EINVAL
    for kw, text in ((dict(slots=None), b"null"), (dict(k=8), b"16-byte"), (dict(sd=2), b"scale dtype"),
                     (dict(n=2 ** 31 - 1), b"split")):
        assert read(**kw) == EINVAL and text in err()


def test_nothing_to_do():
    assert write(n=0) == 0 and write(n=-1, qkv=None) == 0 and read(n=0, slots=None) == 0
    assert read(k=None, v=None) == 0


def test_more_tokens_than_a_launch_takes():
    assert write(n=2 ** 31 - 1, heads=40) == EINVAL and b"split the call" in ra.lib().rlk_last_error()
