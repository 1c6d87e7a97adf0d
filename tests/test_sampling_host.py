"""Refusals of the sampling entry points, before anything is launched (no GPU)."""
import ctypes as C

import pytest

import redline_amd as ra
from redline_amd import _lib

P = 256  # a non-null, aligned stand-in: nothing is launched
EINVAL, EUNSUP = _lib.RLK_EINVAL, _lib.RLK_EUNSUPPORTED


def call(**kw):
    f = dict(logits=P, fp32=1, stride=1000, rows=3, vocab=1000, param_row=None, temperature=P, top_k=P, top_p=P, min_p=None,
             uniform=P, tokens=P, logprobs=None, workspace=P, bytes=1 << 30)
    return ra.lib().rlk_sample_tokens(C.byref(_lib.SamplingWork(*(f | kw).values())), None)


@pytest.mark.parametrize("kw,status,text", [
    (dict(vocab=0), EUNSUP, b"vocabulary of 0"), (dict(vocab=(1 << 20) + 1, stride=1 << 21), EUNSUP, b"vocabulary"),
    (dict(vocab=-1), EUNSUP, b"vocabulary"), (dict(logits=None), EINVAL, b"null"), (dict(tokens=None), EINVAL, b"null"),
    (dict(temperature=None), EINVAL, b"null"), (dict(top_k=None), EINVAL, b"null"), (dict(top_p=None), EINVAL, b"null"),
    (dict(uniform=None), EINVAL, b"null"), (dict(workspace=None), EINVAL, b"null"), (dict(stride=999), EINVAL, b"overlap"),
    (dict(stride=-1000), EINVAL, b"overlap"), (dict(logits=258), EINVAL, b"aligned"),
    (dict(logits=257, fp32=0), EINVAL, b"aligned"), (dict(workspace=128), EINVAL, b"256-byte"),
    (dict(bytes=100), EINVAL, b"needs"), (dict(rows=2 ** 31 - 1), EINVAL, b"needs")])
def test_refusals(kw, status, text):
    assert call(**kw) == status, ra.lib().rlk_last_error()
    assert text in ra.lib().rlk_last_error()


def test_workspace_and_nothing_to_do():
    size = ra.lib().rlk_sampling_workspace_bytes
    assert size(0, 5) == size(5, 0) == size(5, (1 << 20) + 1) == size(-1, 5) == 0
    assert 0 < size(1, 1) <= size(2, 1) <= size(2, 5000) and size(2 ** 31 - 1, 1 << 20) > 1 << 40
    n = size(3, 1000)
    assert call(bytes=n - 1) == EINVAL and call(rows=0) == 0 and call(rows=-1, logits=None) == 0
    assert ra.lib().rlk_sample_tokens(None, None) == EINVAL


def test_the_workspace_is_one():
    from redline_amd import kernels as K
    for bad in (None, 5, "x"):
        with pytest.raises(ra.Error, match="SamplingWorkspace"):
            K.sampling_work(None, 1, 10, None, None, None, None, None, bad)


def test_more_rows_than_a_launch_takes():
    for rows, vocab in ((1 << 23, 1000), (1 << 17, 1 << 20)):
        assert call(rows=rows, vocab=vocab, stride=vocab, bytes=1 << 62) == EINVAL
        assert b"split the call" in ra.lib().rlk_last_error()
