"""Refusals of the block-scaled cache's and the batch tables' entry points,
before anything is launched (no GPU)."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

import redline_amd as ra
from redline_amd import _lib
from tests import _kv_blocks as B

ROOT = Path(__file__).resolve().parents[1]
D16 = 16  # a non-null, 16-byte aligned stand-in: nothing is launched
EINVAL, EUNSUP = _lib.RLK_EINVAL, _lib.RLK_EUNSUPPORTED


def view(**kw):
    f = dict(k=D16, v=D16, k_scale=D16, v_scale=D16, num_blocks=8, block_size=16, num_kv_heads=2, head_dim=64, format=0)
    return _lib.KVBlockView(*(f | kw).values())


BAD_VIEWS = [(dict(head_dim=96), EUNSUP, b"head_dim 96"), (dict(block_size=8), EUNSUP, b"block size 8"),
             (dict(block_size=0), EUNSUP, b"block size"), (dict(format=2), EINVAL, b"format 2"),
             (dict(num_blocks=0), EINVAL, b"block count"), (dict(num_kv_heads=0), EINVAL, b"kv heads"),
             (dict(num_blocks=1 << 28, block_size=16), EINVAL, b"32-bit"), (dict(k=None), EINVAL, b"null pointer"),
             (dict(v_scale=None), EINVAL, b"null pointer"), (dict(v=24), EINVAL, b"16-byte aligned")]


def params(kv, **kw):
    f = dict(q=D16, q_stride=512, out=D16, num_heads=4, scale=0.1, kv=kv, block_tables=D16, max_blocks=4, positions=D16)
    return _lib.BlockAttentionParams(*(f | kw).values())


def decode(p, **kw):
    f = dict(t=D16, s=D16, n=2, parts=1, o=None, m=None, u=None)
    w = _lib.DecodeAttentionWork(*(f | kw).values())
    return ra.lib().rlk_paged_attention_decode_blocks(C.byref(p), C.byref(w), None)


def prefill(p, **kw):
    f = dict(i=D16, s=D16, n=D16, c=D16, num=2, tiles=1)
    w = _lib.PrefillAttentionWork(*(f | kw).values())
    return ra.lib().rlk_paged_attention_prefill_blocks(C.byref(p), C.byref(w), None)


def write(kv, n=3, **kw):
    f = dict(qkv=D16, pos=D16, slots=D16, n=n, heads=4, cos=D16, sin=D16, kv=C.byref(kv) if kv is not None else None,
             bias=None)
    return ra.lib().rlk_rope_and_write_kv_blocks(*(f | kw).values(), None)


def read(kv, n=3, slots=D16, k=D16, v=D16):
    return ra.lib().rlk_read_kv_blocks(C.byref(kv) if kv is not None else None, slots, n, k, v, None)


@pytest.mark.parametrize("kw,status,text", BAD_VIEWS)
def test_bad_views_are_refused(kw, status, text):
    kv = view(**kw)
    for call in (lambda: write(kv), lambda: read(kv), lambda: decode(params(kv)), lambda: prefill(params(kv))):
        assert call() == status
        assert text in ra.lib().rlk_last_error()


def test_bad_arguments_are_refused():
    L, kv = ra.lib(), view()

    def refused(status, code, text):
        assert status == code and text in L.rlk_last_error(), (status, L.rlk_last_error())

    for bad in (dict(qkv=None), dict(pos=None), dict(slots=None), dict(cos=None), dict(sin=None)):
        refused(write(kv, **bad), EINVAL, b"null pointer")
    for bad in (dict(qkv=24), dict(bias=8), dict(cos=4), dict(sin=8)):
        refused(write(kv, **bad), EINVAL, b"16-byte aligned")
    refused(write(kv, heads=-1), EINVAL, b"head count")
    refused(write(None), EINVAL, b"null KV block view")
    refused(read(kv, slots=None), EINVAL, b"null pointer")
    refused(read(kv, k=8), EINVAL, b"16-byte aligned")
    assert read(kv, k=None, v=None) == 0
    for call in (decode, prefill):
        refused(call(params(kv, num_heads=3)), EINVAL, b"multiple of num_kv_heads")
        refused(call(params(kv, num_heads=18)), EUNSUP, b"group size 9")
        refused(call(params(kv, max_blocks=0)), EINVAL, b"table width")
        for bad in (dict(q=None), dict(out=None), dict(block_tables=None), dict(positions=None)):
            refused(call(params(kv, **bad)), EINVAL, b"null pointer")
        refused(call(params(kv, q_stride=516)), EINVAL, b"16-byte aligned")
        refused(call(params(kv, out=8)), EINVAL, b"16-byte aligned")
    refused(decode(params(kv), t=None), EINVAL, b"null pointer")
    refused(decode(params(kv), parts=0), EINVAL, b"max_partitions")
    refused(decode(params(kv), parts=5000, o=D16, m=D16, u=D16), EUNSUP, b"exceeds")
    refused(decode(params(kv), parts=2), EINVAL, b"workspace")
    refused(decode(params(kv), n=70000), EINVAL, b"split the call")
    refused(prefill(params(kv), c=None), EINVAL, b"null pointer")
    refused(prefill(params(kv), num=70000), EINVAL, b"split the call")
    refused(prefill(params(kv), tiles=1 << 28), EINVAL, b"split the call")


def test_empty_calls_are_noops():
    bad = view(head_dim=96)
    assert write(bad, n=0) == 0 and read(bad, n=0) == 0
    assert decode(params(bad), n=0) == 0 and prefill(params(bad), num=0) == 0 and prefill(params(bad), tiles=0) == 0


def table_call(pool_kw={}, **kw):
    pf = dict(ring=D16, capacity=8, state=D16, state_out=None) | pool_kw
    f = dict(past=D16, new=D16, S=2, rows=4, bs=16, thr=1, tab=D16, mb=4, q_start=D16, q_len=D16, ctx=D16, pos=D16,
             slots=D16, dt=D16, ds=D16, pre=D16, counts=D16) | kw
    p, t = _lib.BlockPoolView(*pf.values()), _lib.BatchTables(*f.values())
    return ra.lib().rlk_build_batch_tables(C.byref(p), C.byref(t), None)


def test_batch_tables_refusals():
    L = ra.lib()
    assert L.rlk_build_batch_tables(None, None, None) == EINVAL
    assert table_call(S=0, rows=0) == 0
    for kw, code, text in ((dict(S=-1), EINVAL, b"sequence count"), (dict(rows=-2), EINVAL, b"row count"),
                           (dict(S=8193), EUNSUP, b"split the batch"), (dict(bs=0), EINVAL, b"block size"),
                           (dict(mb=0), EINVAL, b"table width"), (dict(thr=-1), EINVAL, b"threshold"),
                           (dict(bs=1 << 20, mb=1 << 20), EINVAL, b"32-bit"), (dict(past=None), EINVAL, b"null pointer"),
                           (dict(tab=None), EINVAL, b"null pointer"), (dict(slots=None), EINVAL, b"null pointer"),
                           (dict(counts=None), EINVAL, b"null pointer"),
                           (dict(pool_kw=dict(capacity=0)), EINVAL, b"ring capacity"),
                           (dict(pool_kw=dict(ring=None)), EINVAL, b"null pointer"),
                           (dict(pool_kw=dict(state=None)), EINVAL, b"null pointer")):
        assert table_call(**kw) == code and text in L.rlk_last_error(), (kw, L.rlk_last_error())


def test_python_launchers_check_their_tensors():
    torch = pytest.importorskip("torch")
    from redline_amd import kernels as K
    z = torch.zeros(8, 2, 16 * 64, dtype=torch.int8)
    s = torch.zeros(8, 2)
    with pytest.raises(ra.Error, match="GPU tensor"):
        K.kv_block_view(z, z, s, s, 16, 2, 64, K.KVBlockFormat.kINT8)
    with pytest.raises(ra.Error, match="torch.uint8"):
        K.kv_block_view(z, z, s, s, 16, 2, 64, K.KVBlockFormat.kFP8)
    with pytest.raises(ra.Error, match="whole blocks"):
        K.kv_block_view(z.view(-1)[:-1], z, s, s, 16, 2, 64, K.KVBlockFormat.kINT8)
    with pytest.raises(ra.Error, match="k_scale holds"):
        K.kv_block_view(z, z, s[:4], s, 16, 2, 64, K.KVBlockFormat.kINT8)
    i = torch.zeros(8, dtype=torch.int32)
    with pytest.raises(ra.Error, match="state holds"):
        K.BlockPool(i, i[:2])
    with pytest.raises(ra.Error, match="positions holds"):
        K.batch_tables(None, i, i, 2, 20, 16, 1, i, 4, i, i, i, i, i, i, i, i, i)
    with pytest.raises(ra.Error, match="bad KV cache"):
        K.KVBlockCache(1, 1, 2, 64)


def test_cpp_header_wraps_the_entry_points(tmp_path):
    """The C++ launchers compile, throw redline::Error on bad arguments and are
    no-ops for empty calls."""
    exe = tmp_path / "blocks"
    subprocess.run(["/opt/rocm/bin/hipcc", "-std=c++17", f"-I{ROOT / 'include'}",
                    str(ROOT / "tests" / "cpp" / "blocks_main.cpp"), "-o", str(exe), f"-L{ROOT / 'redline_amd'}",
                    "-lrlk", f"-Wl,-rpath,{ROOT / 'redline_amd'}"], check=True, capture_output=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    assert "PASS" in out, out


def test_restated_layout_and_codes():
    """The restatement the GPU tests compare with: its layout covers every byte
    once, and its codes agree with torch's e4m3 conversion."""
    for bs, D in ((16, 64), (32, 128)):
        for p in B.places(bs, D):
            assert np.array_equal(np.sort(p.reshape(-1)), np.arange(bs * D))
    torch = pytest.importorskip("torch")
    x = np.concatenate([np.linspace(-448, 448, 4001), 2.0 ** np.arange(-12, 9), B.E4M3[:127],
                        (B.E4M3[:126] + B.E4M3[1:127]) / 2])
    want = torch.from_numpy(x).float().to(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(B.nearest(x, B.FP8), want)
    assert np.array_equal(B.values(B.bytes_of(want, B.FP8), B.FP8), want)
