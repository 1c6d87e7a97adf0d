"""Python launch interface over the C ABI, mirroring redline::kernels.

Names, parameter order and meaning follow the reference's launchers
(src/cuda/kernels/kernels.h:64-88 in Neil456/Redline).  Arguments are torch
tensors on the GPU (device memory and streams come from PyTorch; the compute
is the HIP code in librlk.so).  Errors raise redline_amd.Error before anything
is launched, as the reference's RL_CHECK throws.  Every launcher is
asynchronous on `stream` (default: torch's current stream).
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import KVBlockView, KVLayerView, check, lib

__all__ = [
    "embedding_lookup", "embedding_rmsnorm", "fused_add_rmsnorm", "silu_and_mul", "silu_and_mul_interleaved",
    "gather_rows", "resolve_input_ids", "rope_and_write_kv", "rope_and_write_kv_ex", "KVDType",
    "KVCache", "SCALE_F32", "SCALE_F16", "paged_attention_decode", "paged_attention_decode_ex",
    "attention_params",
    "decode_work", "prefill_work", "paged_attention_prefill", "paged_attention_prefill_ex",
    "DecodeWorkspace", "kDecodePartitionSize", "gemv_w8a16", "gemv_w4a16", "gemv_w4a16_swiglu",
    "kGemvW4MaxM", "KVBlockFormat", "KVBlockCache", "kv_block_view", "rope_and_write_kv_blocks",
    "read_kv_blocks", "block_attention_params", "paged_attention_decode_blocks",
    "paged_attention_prefill_blocks", "BlockPool", "batch_tables", "build_batch_tables",
    "kRopeMaxAxes", "kv_layer_view", "rope_and_write_kv_norm", "read_kv", "shared_prefix_work",
    "paged_attention_decode_shared", "SamplingWorkspace", "sampling_work", "sample_tokens",
]

kDecodePartitionSize = _lib.RLK_DECODE_PARTITION_SIZE
kGemvW4MaxM = _lib.RLK_GEMV_W4_MAX_M
kRopeMaxAxes = _lib.RLK_ROPE_MAX_AXES

SCALE_F32 = _lib.RLK_SCALE_F32
SCALE_F16 = _lib.RLK_SCALE_F16


class KVDType:
    kFP16 = _lib.RLK_KV_FP16
    kINT8 = _lib.RLK_KV_INT8


def _stream(stream) -> int:
    if stream is None:  # the current stream's handle, without a Stream object (2.6 us less a call)
        return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())
    if isinstance(stream, torch.cuda.Stream):
        return stream.cuda_stream
    return int(stream)


def _ptr(t, dtype, what, allow_none=False):
    if t is None:
        if allow_none:
            return None
        raise _lib.Error(_lib.RLK_EINVAL, f"{what} must not be None")
    if not isinstance(t, torch.Tensor):
        raise _lib.Error(_lib.RLK_EINVAL, f"{what} must be a torch.Tensor")
    if t.dtype != dtype:
        raise _lib.Error(_lib.RLK_EINVAL, f"{what} must be {dtype}, got {t.dtype}")
    if not t.is_cuda:
        raise _lib.Error(_lib.RLK_EINVAL, f"{what} must be a GPU tensor")
    if not t.is_contiguous():
        raise _lib.Error(_lib.RLK_EINVAL, f"{what} must be contiguous")
    return t.data_ptr()


def _need(t, n, what):
    if t is not None and t.numel() < n:
        raise _lib.Error(_lib.RLK_EINVAL, f"{what} holds {t.numel()} elements, needs {n}")


def embedding_lookup(ids, table, n, hidden, out, stream=None):
    """out[t, :] = table[ids[t], :] for t < n (kernels::embedding_lookup)."""
    if n > 0:
        _need(ids, n, "ids"); _need(out, n * hidden, "out")
    check(lib().rlk_embedding_lookup(_ptr(ids, torch.int32, "ids"), _ptr(table, torch.float16, "table"),
                                     n, hidden, _ptr(out, torch.float16, "out"), _stream(stream)))


def fused_add_rmsnorm(residual, delta, weight, rows, hidden, eps, out, stream=None):
    """residual += delta (unless None); out = rmsnorm(residual) * weight."""
    if rows > 0:
        for t, w in ((residual, "residual"), (delta, "delta"), (out, "out")):
            _need(t, rows * hidden, w)
        _need(weight, hidden, "weight")
    check(lib().rlk_fused_add_rmsnorm(
        _ptr(residual, torch.float16, "residual"), _ptr(delta, torch.float16, "delta", True),
        _ptr(weight, torch.float16, "weight"), rows, hidden, float(eps),
        _ptr(out, torch.float16, "out"), _stream(stream)))


def embedding_rmsnorm(ids, table, n, hidden, weight, eps, residual, out, stream=None):
    """Extension: residual[t, :] = table[ids[t], :]; out = rmsnorm(residual) *
    weight, in one launch -- the reference's embedding_lookup followed by
    fused_add_rmsnorm(delta=None) (llama.cpp:79-80), same results."""
    if n > 0:
        _need(ids, n, "ids"); _need(residual, n * hidden, "residual"); _need(out, n * hidden, "out")
        _need(weight, hidden, "weight")
    check(lib().rlk_embedding_rmsnorm(
        _ptr(ids, torch.int32, "ids"), _ptr(table, torch.float16, "table"), n, hidden,
        _ptr(weight, torch.float16, "weight"), float(eps), _ptr(residual, torch.float16, "residual"),
        _ptr(out, torch.float16, "out"), _stream(stream)))


def silu_and_mul(gate_up, rows, inter, out, stream=None):
    """out[r, i] = silu(gate_up[r, i]) * gate_up[r, inter + i]."""
    if rows > 0:
        _need(gate_up, rows * 2 * inter, "gate_up"); _need(out, rows * inter, "out")
    check(lib().rlk_silu_and_mul(_ptr(gate_up, torch.float16, "gate_up"), rows, inter,
                                 _ptr(out, torch.float16, "out"), _stream(stream)))


def silu_and_mul_interleaved(gate_up, rows, inter, out, stream=None):
    """Same with (gate_i, up_i) interleaved columns."""
    if rows > 0:
        _need(gate_up, rows * 2 * inter, "gate_up"); _need(out, rows * inter, "out")
    check(lib().rlk_silu_and_mul_interleaved(_ptr(gate_up, torch.float16, "gate_up"), rows, inter,
                                             _ptr(out, torch.float16, "out"), _stream(stream)))


def gemv_w8a16(x, m, w, scales, bias, n, k, y, y_fp32=False, stream=None):
    """y[m, n] = (x[m, k] . w^T) * scales (+ bias): INT8 weight [n, k] with one
    fp16 scale per row; y fp16, or fp32 with y_fp32."""
    if m > 0 and n > 0 and k > 0:
        _need(x, m * k, "x"); _need(w, n * k, "w"); _need(scales, n, "scales"); _need(y, m * n, "y")
        if bias is not None:
            _need(bias, n, "bias")
    check(lib().rlk_gemv_w8a16(
        _ptr(x, torch.float16, "x"), m, _ptr(w, torch.int8, "w"), _ptr(scales, torch.float16, "scales"),
        _ptr(bias, torch.float16, "bias", True), n, k,
        _ptr(y, torch.float32 if y_fp32 else torch.float16, "y"), int(bool(y_fp32)), _stream(stream)))


def _gemv_w4_need(x, m, w, scales, offsets, group_size, n, k):
    if m > 0 and k > 0 and group_size > 0 and k % group_size == 0:
        _need(x, m * k, "x"); _need(w, n * k // 2, "w")
        _need(scales, n * (k // group_size), "scales"); _need(offsets, n * (k // group_size), "offsets")


def gemv_w4a16(x, m, w, scales, offsets, group_size, bias, n, k, y, y_fp32=False, stream=None):
    """y[m, n] = x[m, k] . dequant(w)^T (+ bias): INT4 weight [n, k/2] uint8 with
    fp16 scales/offsets [n, k/group_size]; y fp16, or fp32 with y_fp32."""
    _gemv_w4_need(x, m, w, scales, offsets, group_size, n, k)
    if m > 0:
        _need(y, m * n, "y")
    check(lib().rlk_gemv_w4a16(
        _ptr(x, torch.float16, "x"), m, _ptr(w, torch.uint8, "w"),
        _ptr(scales, torch.float16, "scales"), _ptr(offsets, torch.float16, "offsets"), group_size,
        _ptr(bias, torch.float16, "bias", True), n, k,
        _ptr(y, torch.float32 if y_fp32 else torch.float16, "y"), int(bool(y_fp32)),
        _stream(stream)))


def gemv_w4a16_swiglu(x, m, w, scales, offsets, group_size, n, k, y, stream=None):
    """y[m, n/2] = silu(gate) * up from an INT4 weight whose rows are interleaved
    (gate_i, up_i), in the GEMV epilogue."""
    _gemv_w4_need(x, m, w, scales, offsets, group_size, n, k)
    if m > 0:
        _need(y, m * (n // 2), "y")
    check(lib().rlk_gemv_w4a16_swiglu(
        _ptr(x, torch.float16, "x"), m, _ptr(w, torch.uint8, "w"),
        _ptr(scales, torch.float16, "scales"), _ptr(offsets, torch.float16, "offsets"), group_size,
        n, k, _ptr(y, torch.float16, "y"), _stream(stream)))


def gather_rows(src, idx, n, cols, dst, stream=None):
    """dst[i, :] = src[idx[i], :] (idx None: dst[i, :] = src[i, :])."""
    if n > 0:
        if idx is not None:
            _need(idx, n, "idx")
        _need(dst, n * cols, "dst")
    check(lib().rlk_gather_rows(_ptr(src, torch.float16, "src"), _ptr(idx, torch.int32, "idx", True), n, cols,
                                _ptr(dst, torch.float16, "dst"), _stream(stream)))


def resolve_input_ids(input_ids, src, prev_sampled, n, stream=None):
    """input_ids[i] = prev_sampled[src[i]] where src[i] >= 0."""
    if n > 0:
        _need(input_ids, n, "input_ids"); _need(src, n, "src")
    check(lib().rlk_resolve_input_ids(_ptr(input_ids, torch.int32, "input_ids"),
                                      _ptr(src, torch.int32, "src"),
                                      _ptr(prev_sampled, torch.int32, "prev_sampled"), n,
                                      _stream(stream)))


def rope_and_write_kv(qkv, positions, slot_mapping, num_tokens, num_heads, cos_table, sin_table,
                      kv: KVLayerView, stream=None):
    """RoPE on q/k heads (q in place) and paged KV write at slot_mapping[t]."""
    if num_tokens > 0:
        _need(positions, num_tokens, "positions"); _need(slot_mapping, num_tokens, "slot_mapping")
        _need(qkv, num_tokens * (num_heads + 2 * kv.num_kv_heads) * kv.head_dim, "qkv")
    check(lib().rlk_rope_and_write_kv(
        _ptr(qkv, torch.float16, "qkv"), _ptr(positions, torch.int32, "positions"),
        _ptr(slot_mapping, torch.int32, "slot_mapping"), num_tokens, num_heads,
        _ptr(cos_table, torch.float32, "cos_table"), _ptr(sin_table, torch.float32, "sin_table"),
        C.byref(kv), _stream(stream)))


def rope_and_write_kv_ex(qkv, positions, slot_mapping, num_tokens, num_heads, cos_table, sin_table,
                         kv: KVLayerView, qkv_bias=None, scale_dtype=SCALE_F32, stream=None):
    """Extension: optional QKV bias added before RoPE, optional fp16 INT8 scales."""
    if num_tokens > 0:
        _need(positions, num_tokens, "positions"); _need(slot_mapping, num_tokens, "slot_mapping")
        _need(qkv, num_tokens * (num_heads + 2 * kv.num_kv_heads) * kv.head_dim, "qkv")
        _need(qkv_bias, (num_heads + 2 * kv.num_kv_heads) * kv.head_dim, "qkv_bias")
    opt = _lib.RopeKVOptions(_ptr(qkv_bias, torch.float16, "qkv_bias", True), scale_dtype)
    check(lib().rlk_rope_and_write_kv_ex(
        _ptr(qkv, torch.float16, "qkv"), _ptr(positions, torch.int32, "positions"),
        _ptr(slot_mapping, torch.int32, "slot_mapping"), num_tokens, num_heads,
        _ptr(cos_table, torch.float32, "cos_table"), _ptr(sin_table, torch.float32, "sin_table"),
        C.byref(kv), C.byref(opt), _stream(stream)))


def attention_params(q, q_stride, out, num_heads, scale, kv: KVLayerView, block_tables,
                     max_blocks_per_seq, positions) -> _lib.AttentionParams:
    """kernels::AttentionParams from torch tensors (q may be a view into qkv).
    The struct keeps its tensors."""
    params = _lib.AttentionParams(
        _ptr(q, torch.float16, "q"), q_stride, _ptr(out, torch.float16, "out"), num_heads,
        float(scale), kv, _ptr(block_tables, torch.int32, "block_tables"), max_blocks_per_seq,
        _ptr(positions, torch.int32, "positions"))
    params.device, params.tensors = kv.device, (kv, q, out, block_tables, positions)
    return params


def decode_work(item_token, item_seq, num_items, max_partitions, workspace=None):
    """kernels::DecodeAttentionWork; `workspace` is a DecodeWorkspace (needed
    when max_partitions > 1).  The struct keeps its tensors."""
    ws = workspace
    work = _lib.DecodeAttentionWork(
        _ptr(item_token, torch.int32, "item_token"), _ptr(item_seq, torch.int32, "item_seq"),
        num_items, max_partitions,
        None if ws is None else ws.out.data_ptr(), None if ws is None else ws.max.data_ptr(),
        None if ws is None else ws.sum.data_ptr())
    _need(item_token, num_items, "item_token"); _need(item_seq, num_items, "item_seq")
    if ws is not None and max_partitions > 1:  # (item, head) rows that the workspace holds, elements of ws.out
        work.room = min(ws.max.numel(), ws.sum.numel()) // max_partitions, ws.out.numel() // max_partitions
    return _keep(work, item_token, item_seq, *(() if ws is None else (ws.out, ws.max, ws.sum)))


def _keep(work, *tensors):
    """`work` with the tensors whose pointers it holds, and their device."""
    work.device, work.tensors = tensors[0].get_device(), tensors
    _one_device(work.device, *tensors)
    return work


def prefill_work(seq_ids, q_start, q_len, ctx_len, num_seqs, max_q_tiles):
    """kernels::PrefillAttentionWork (max_q_tiles in 32-row tiles, as BatchBuilder writes it).
    The struct keeps its tensors."""
    work = _lib.PrefillAttentionWork(
        _ptr(seq_ids, torch.int32, "seq_ids"), _ptr(q_start, torch.int32, "q_start"),
        _ptr(q_len, torch.int32, "q_len"), _ptr(ctx_len, torch.int32, "ctx_len"), num_seqs,
        max_q_tiles)
    if max_q_tiles > 0:
        _need(seq_ids, num_seqs, "seq_ids")
    return _keep(work, seq_ids, q_start, q_len, ctx_len)


def paged_attention_prefill(params: _lib.AttentionParams, work: _lib.PrefillAttentionWork,
                            stream=None):
    """Causal paged prefill attention (kernels::paged_attention_prefill)."""
    check(lib().rlk_paged_attention_prefill(C.byref(params), C.byref(work), _stream(stream)))


def paged_attention_prefill_ex(params: _lib.AttentionParams, work: _lib.PrefillAttentionWork,
                               scale_dtype=SCALE_F32, stream=None):
    """Extension: prefill attention over an INT8 cache with fp16 scales."""
    opt = _lib.AttentionOptions(scale_dtype)
    check(lib().rlk_paged_attention_prefill_ex(C.byref(params), C.byref(work), C.byref(opt),
                                               _stream(stream)))


class DecodeWorkspace:
    """Split-K partials of the decode attention, sized like the reference
    model's workspace (src/cuda/model/llama.cpp:37-40)."""

    def __init__(self, max_items, num_heads, max_partitions, head_dim, device="cuda"):
        rows = max_items * num_heads * max_partitions
        self.out = torch.empty(rows * head_dim, dtype=torch.float32, device=device)
        self.max = torch.empty(rows, dtype=torch.float32, device=device)
        self.sum = torch.empty(rows, dtype=torch.float32, device=device)


def paged_attention_decode(params: _lib.AttentionParams, work: _lib.DecodeAttentionWork,
                           stream=None):
    """Flash-decoding paged attention (kernels::paged_attention_decode)."""
    check(lib().rlk_paged_attention_decode(C.byref(params), C.byref(work), _stream(stream)))


def paged_attention_decode_ex(params: _lib.AttentionParams, work: _lib.DecodeAttentionWork,
                              scale_dtype=SCALE_F32, stream=None):
    """Extension: decode attention over an INT8 cache with fp16 scales
    (written by rope_and_write_kv_ex with SCALE_F16)."""
    opt = _lib.AttentionOptions(scale_dtype)
    check(lib().rlk_paged_attention_decode_ex(C.byref(params), C.byref(work), C.byref(opt),
                                              _stream(stream)))


class KVCache:
    """Paged KV cache in one zeroed device allocation, laid out per layer as
    K, V (then k_scale, v_scale for INT8), each [num_blocks, Hkv, bs, D]
    (scales [num_blocks, Hkv, bs] fp32) — the layout of the reference's
    KVCache (src/cuda/model/kv_cache.cpp:25-52).  Block 0 is the scratch block
    that padded rows write into."""

    def __init__(self, num_layers, num_blocks, num_kv_heads, head_dim, block_size=16,
                 dtype=KVDType.kFP16, device="cuda", scale_dtype=SCALE_F32):
        if num_blocks <= 1 or block_size <= 0 or num_layers <= 0:
            raise _lib.Error(_lib.RLK_EINVAL, "bad KV cache config")
        self.num_layers, self.num_blocks = num_layers, num_blocks
        self.num_kv_heads, self.head_dim, self.block_size, self.dtype = (
            num_kv_heads, head_dim, block_size, dtype)
        cells = num_blocks * num_kv_heads * block_size
        elem = 2 if dtype == KVDType.kFP16 else 1
        sbytes = 2 if scale_dtype == SCALE_F16 else 4
        sdt = torch.float16 if scale_dtype == SCALE_F16 else torch.float32
        per_layer = 2 * cells * head_dim * elem + (2 * cells * sbytes if dtype == KVDType.kINT8 else 0)
        self.storage = torch.zeros(per_layer * num_layers, dtype=torch.uint8, device=device)
        self._views, self._tensors = [], []
        shape = (num_blocks, num_kv_heads, block_size, head_dim)
        tdt = torch.float16 if dtype == KVDType.kFP16 else torch.int8
        off = 0
        for _ in range(num_layers):
            kb = cells * head_dim * elem
            k = self.storage[off:off + kb].view(tdt).view(shape); off += kb
            v = self.storage[off:off + kb].view(tdt).view(shape); off += kb
            ks = vs = None
            if dtype == KVDType.kINT8:
                ks = self.storage[off:off + cells * sbytes].view(sdt).view(shape[:3]); off += cells * sbytes
                vs = self.storage[off:off + cells * sbytes].view(sdt).view(shape[:3]); off += cells * sbytes
            view = KVLayerView(k.data_ptr(), v.data_ptr(), ks.data_ptr() if ks is not None else None,
                               vs.data_ptr() if vs is not None else None, block_size, num_kv_heads,
                               head_dim, dtype)
            view.device, view.tensors = self.storage.get_device(), (k, v, ks, vs)
            view.scale_dtype = scale_dtype if dtype == KVDType.kINT8 else None
            self._views.append(view)
            self._tensors.append((k, v, ks, vs))

    def layer(self, i) -> KVLayerView:
        return self._views[i]

    def tensors(self, i):
        """(k, v, k_scale, v_scale) torch views of layer i (scales None for FP16)."""
        return self._tensors[i]


# ------------------------------------------------- block-scaled 8-bit KV cache

def _one_device(dev, *tensors):
    if dev is None:  # a struct filled in by hand
        return
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise _lib.Error(_lib.RLK_EINVAL, f"tensors are on different devices (cuda:{dev} and {t.device})")


def _arg(t, dtype, what, n, dev):
    """_ptr of a tensor of at least n elements on device dev, with the checks in one call."""
    try:  # (dev -1, of a cache on the CPU, ends at _stream_on)
        if (t.dtype is dtype and (t.get_device() == dev or dev is None and t.is_cuda) and t.is_contiguous()
                and t.numel() >= n):
            return t.data_ptr()
    except AttributeError:
        pass
    p = _ptr(t, dtype, what)  # says which check fails
    _need(t, n, what)
    _one_device(dev, t)
    return p


def _stream_on(dev, stream):
    """_stream, for tensors of device dev: a launch goes to the current device, which must
    be theirs and the stream's."""
    if dev is not None:
        if dev < 0:  # before the driver is asked, which a machine without a GPU answers with an error of its own
            raise _lib.Error(_lib.RLK_EINVAL, "the cache and the tensors beside it must be GPU tensors")
        cur = torch._C._cuda_getDevice()
        if cur != dev:
            raise _lib.Error(_lib.RLK_EINVAL, f"tensors are on cuda:{dev}, the current device is cuda:{cur}")
        if stream is None:
            return torch._C._cuda_getCurrentRawStream(dev)
        if isinstance(stream, torch.cuda.Stream) and stream.device_index != dev:
            raise _lib.Error(_lib.RLK_EINVAL, f"tensors are on cuda:{dev}, the stream on cuda:{stream.device_index}")
    return _stream(stream)


class KVBlockFormat:
    kINT8 = _lib.RLK_KV_BLOCK_INT8
    kFP8 = _lib.RLK_KV_BLOCK_FP8  # e4m3, finite values only


def kv_block_view(k, v, k_scale, v_scale, block_size, num_kv_heads, head_dim, fmt) -> KVBlockView:
    """One layer of a block-scaled cache (extension): k, v [num_blocks, Hkv,
    block_size * D] int8 (INT8) or uint8 (FP8) codes in the tile layout of rlk.h,
    k_scale, v_scale fp32 [num_blocks, Hkv]."""
    dt = torch.int8 if fmt == KVBlockFormat.kINT8 else torch.uint8
    per = num_kv_heads * block_size * head_dim
    if not isinstance(k, torch.Tensor) or per <= 0 or k.numel() % per != 0:
        raise _lib.Error(_lib.RLK_EINVAL, "k must hold whole blocks")
    nb = k.numel() // per
    _need(v, nb * per, "v")
    for t, w in ((k_scale, "k_scale"), (v_scale, "v_scale")):
        _need(t, nb * num_kv_heads, w)
    view = KVBlockView(_ptr(k, dt, "k"), _ptr(v, dt, "v"), _ptr(k_scale, torch.float32, "k_scale"),
                       _ptr(v_scale, torch.float32, "v_scale"), nb, block_size, num_kv_heads,
                       head_dim, fmt)
    view.device, view.tensors = k.get_device(), (k, v, k_scale, v_scale)  # kept with their pointers
    _one_device(view.device, v, k_scale, v_scale)
    return view


class KVBlockCache:
    """Paged block-scaled cache (extension), zeroed: per layer K and V codes and
    one fp32 scale per (block, kv head) of each.  Block 0 is the scratch block,
    as in KVCache."""

    def __init__(self, num_layers, num_blocks, num_kv_heads, head_dim, block_size=16,
                 fmt=KVBlockFormat.kINT8, device="cuda"):
        if num_blocks <= 1 or block_size <= 0 or num_layers <= 0:
            raise _lib.Error(_lib.RLK_EINVAL, "bad KV cache config")
        self.num_layers, self.num_blocks, self.block_size = num_layers, num_blocks, block_size
        self.num_kv_heads, self.head_dim, self.fmt = num_kv_heads, head_dim, fmt
        dt = torch.int8 if fmt == KVBlockFormat.kINT8 else torch.uint8
        self._tensors = [tuple(torch.zeros((num_blocks, num_kv_heads, block_size * head_dim), dtype=dt,
                                           device=device) for _ in range(2)) +
                         tuple(torch.zeros((num_blocks, num_kv_heads), dtype=torch.float32, device=device)
                               for _ in range(2)) for _ in range(num_layers)]
        self._views = [kv_block_view(*t, block_size, num_kv_heads, head_dim, fmt) for t in self._tensors]

    def layer(self, i) -> KVBlockView:
        return self._views[i]

    def tensors(self, i):
        """(k, v, k_scale, v_scale) torch tensors of layer i (codes in the tile layout)."""
        return self._tensors[i]


def rope_and_write_kv_blocks(qkv, positions, slot_mapping, num_tokens, num_heads, cos_table, sin_table,
                             kv: KVBlockView, qkv_bias=None, stream=None):
    """Extension: RoPE on q/k heads (q in place) and the write of k/v into a
    block-scaled cache; rows of a block come consecutively, at rising offsets."""
    n, dev = max(num_tokens, 0), kv.device
    cols = (num_heads + 2 * kv.num_kv_heads) * kv.head_dim if n > 0 else 0
    check(lib().rlk_rope_and_write_kv_blocks(
        _arg(qkv, torch.float16, "qkv", n * cols, dev), _arg(positions, torch.int32, "positions", n, dev),
        _arg(slot_mapping, torch.int32, "slot_mapping", n, dev), num_tokens, num_heads,
        _arg(cos_table, torch.float32, "cos_table", 0, dev), _arg(sin_table, torch.float32, "sin_table", 0, dev),
        C.byref(kv), None if qkv_bias is None else _arg(qkv_bias, torch.float16, "qkv_bias", cols, dev),
        _stream_on(dev, stream)))


def read_kv_blocks(kv: KVBlockView, slots, n, k_out=None, v_out=None, stream=None):
    """Extension: the stored rows of `slots` as fp16 [n, Hkv * D] (code * scale);
    a slot outside the pool leaves its rows as they were."""
    dev, size = kv.device, max(n, 0) * kv.num_kv_heads * kv.head_dim
    check(lib().rlk_read_kv_blocks(
        C.byref(kv), _arg(slots, torch.int32, "slots", n, dev), n,
        None if k_out is None else _arg(k_out, torch.float16, "k_out", size, dev),
        None if v_out is None else _arg(v_out, torch.float16, "v_out", size, dev), _stream_on(dev, stream)))


def block_attention_params(q, q_stride, out, num_heads, scale, kv: KVBlockView, block_tables,
                           max_blocks_per_seq, positions) -> _lib.BlockAttentionParams:
    """Parameters of the attention over a block-scaled cache (q may be a view
    into qkv)."""
    params = _lib.BlockAttentionParams(
        _ptr(q, torch.float16, "q"), q_stride, _ptr(out, torch.float16, "out"), num_heads,
        float(scale), kv, _ptr(block_tables, torch.int32, "block_tables"), max_blocks_per_seq,
        _ptr(positions, torch.int32, "positions"))
    params.device, params.tensors = kv.device, (kv, q, out, block_tables, positions)
    _one_device(kv.device, q, out, block_tables, positions)
    return params


def _same_device(params, work):
    if params.device is not None and work.device is not None and params.device != work.device:
        raise _lib.Error(_lib.RLK_EINVAL, f"the work lists are on cuda:{work.device}, the tensors on another "
                                          f"device (cuda:{params.device})")


def paged_attention_decode_blocks(params: _lib.BlockAttentionParams, work: _lib.DecodeAttentionWork,
                                  stream=None):
    """Extension: flash-decoding attention over a block-scaled cache; items with
    a negative token are skipped."""
    if work.device != params.device:
        _same_device(params, work)
    if work.room is not None:
        rows = work.num_items * params.num_heads
        if rows > work.room[0] or rows * params.kv.head_dim > work.room[1]:
            raise _lib.Error(_lib.RLK_EINVAL, f"the workspace holds {work.room[0]} (item, head) rows and "
                                              f"{work.room[1]} elements a partition, needs {rows} of "
                                              f"{params.kv.head_dim}")
    check(lib().rlk_paged_attention_decode_blocks(C.byref(params), C.byref(work),
                                                    _stream_on(params.device, stream)))


def paged_attention_prefill_blocks(params: _lib.BlockAttentionParams, work: _lib.PrefillAttentionWork,
                                   stream=None):
    """Extension: causal prefill attention over a block-scaled cache; negative
    sequence ids are skipped."""
    if work.device != params.device:
        _same_device(params, work)
    check(lib().rlk_paged_attention_prefill_blocks(C.byref(params), C.byref(work),
                                                     _stream_on(params.device, stream)))


# ------------------------------------------------------- block tables on the GPU

class BlockPool:
    """Free blocks of a paged cache in device memory (extension): `ring` int32
    [capacity] block ids, `state` int32 [3] {head, count, 0} with the count free
    ones from head on; with `state_out` int32 [2] a call leaves `state` as it was
    and writes the new {head, count} there."""

    def __init__(self, ring, state, state_out=None):
        _need(state, 3, "state"); _need(state_out, 2, "state_out")
        self.ring, self.state, self.state_out = ring, state, state_out
        self.view = _lib.BlockPoolView(_ptr(ring, torch.int32, "ring"), ring.numel(),
                                       _ptr(state, torch.int32, "state"),
                                       _ptr(state_out, torch.int32, "state_out", True))
        self.device = ring.get_device()
        _one_device(self.device, state, state_out)

    @classmethod
    def of_blocks(cls, num_blocks, device="cuda"):
        """All blocks of a cache of num_blocks but the scratch block 0, free."""
        ring = torch.arange(1, num_blocks, dtype=torch.int32, device=device)
        return cls(ring, torch.tensor([0, num_blocks - 1, 0], dtype=torch.int32, device=device))


def batch_tables(pool: BlockPool, past_len, new_len, num_seqs, num_rows, block_size,
                 decode_query_threshold, block_tables, max_blocks_per_seq, q_start, q_len, ctx_len,
                 positions, slot_mapping, decode_token, decode_seq, prefill_seq, counts):
    """What build_batch_tables reads and writes (rlk_batch_tables); all int32."""
    for t, n, w in ((past_len, num_seqs, "past_len"), (new_len, num_seqs, "new_len"),
                    (block_tables, num_seqs * max_blocks_per_seq, "block_tables"),
                    (q_start, num_seqs, "q_start"), (q_len, num_seqs, "q_len"),
                    (ctx_len, num_seqs, "ctx_len"), (prefill_seq, num_seqs, "prefill_seq"),
                    (positions, num_rows, "positions"), (slot_mapping, num_rows, "slot_mapping"),
                    (decode_token, num_rows, "decode_token"), (decode_seq, num_rows, "decode_seq"),
                    (counts, 4, "counts")):
        _need(t, n, w)
    i = lambda t, w: _ptr(t, torch.int32, w)  # noqa: E731
    work = _lib.BatchTables(
        i(past_len, "past_len"), i(new_len, "new_len"), num_seqs, num_rows, block_size,
        decode_query_threshold, i(block_tables, "block_tables"), max_blocks_per_seq,
        i(q_start, "q_start"), i(q_len, "q_len"), i(ctx_len, "ctx_len"), i(positions, "positions"),
        i(slot_mapping, "slot_mapping"), i(decode_token, "decode_token"),
        i(decode_seq, "decode_seq"), i(prefill_seq, "prefill_seq"), i(counts, "counts"))
    work.tensors = (past_len, new_len, block_tables, q_start, q_len, ctx_len, positions, slot_mapping,
                    decode_token, decode_seq, prefill_seq, counts)
    _one_device(pool.device, *work.tensors)
    return pool, work


def build_batch_tables(tables, stream=None):
    """Extension: positions, slots, work lists and block tables of a step from
    its request lengths, with blocks from the pool; `tables` from batch_tables()."""
    pool, work = tables
    check(lib().rlk_build_batch_tables(C.byref(pool.view), C.byref(work), _stream_on(pool.device, stream)))


# ------------------------- normed heads, several position axes, rows read back

def kv_layer_view(k, v, k_scale=None, v_scale=None) -> KVLayerView:
    """One layer of a paged cache from tensors of its own: k, v [num_blocks, Hkv,
    block_size, D] fp16, or int8 with k_scale, v_scale [num_blocks, Hkv, block_size]
    fp32 or fp16.  The view keeps its tensors."""
    kp = _ptr(k, torch.int8 if k_scale is not None else torch.float16, "k")
    vp = _ptr(v, k.dtype, "v")
    if k.dim() != 4 or v.shape != k.shape:
        raise _lib.Error(_lib.RLK_EINVAL, "k and v must have one shape [num_blocks, Hkv, block_size, D]")
    _, hkv, bs, dim = k.shape
    ksp = vsp = sd = None
    if k_scale is not None:
        sdt = torch.float16 if isinstance(k_scale, torch.Tensor) and k_scale.dtype == torch.float16 else torch.float32
        sd = SCALE_F16 if sdt == torch.float16 else SCALE_F32
        ksp, vsp = _ptr(k_scale, sdt, "k_scale"), _ptr(v_scale, sdt, "v_scale")
        _need(k_scale, k.numel() // max(dim, 1), "k_scale"); _need(v_scale, k.numel() // max(dim, 1), "v_scale")
    elif v_scale is not None:
        raise _lib.Error(_lib.RLK_EINVAL, "v_scale without k_scale")
    view = KVLayerView(kp, vp, ksp, vsp, bs, hkv, dim, KVDType.kFP16 if ksp is None else KVDType.kINT8)
    view.device, view.tensors, view.scale_dtype = k.get_device(), (k, v, k_scale, v_scale), sd
    _one_device(view.device, v, k_scale, v_scale)
    return view


def _scales(kv: KVLayerView, scale_dtype):
    if kv.scale_dtype is not None and scale_dtype != kv.scale_dtype:
        raise _lib.Error(_lib.RLK_EINVAL, f"scale dtype {scale_dtype}, the cache's scales have {kv.scale_dtype}")


def rope_and_write_kv_norm(qkv, positions, slot_mapping, num_tokens, num_heads, cos_table, sin_table,
                           kv: KVLayerView, q_norm=None, k_norm=None, eps=1e-6, qkv_bias=None,
                           scale_dtype=SCALE_F32, sections=None, interleaved=False, stream=None):
    """Extension: rope_and_write_kv_ex with an RMS norm of each query and key head
    (q_norm, k_norm fp16 [D] or None) before the rotation, and a rotation by several
    position axes: `sections` are the pairs of each (D/2 in all), positions then
    [len(sections), num_tokens]."""
    n, dev, f16, i32, f32 = max(num_tokens, 0), kv.device, torch.float16, torch.int32, torch.float32
    if scale_dtype != kv.scale_dtype:
        _scales(kv, scale_dtype)
    dim = kv.head_dim if n > 0 else 0
    cols = (num_heads + 2 * kv.num_kv_heads) * dim
    opt = _lib.NormRopeOptions(None if q_norm is None else _arg(q_norm, f16, "q_norm", dim, dev),
                               None if k_norm is None else _arg(k_norm, f16, "k_norm", dim, dev), eps,
                               None if qkv_bias is None else _arg(qkv_bias, f16, "qkv_bias", cols, dev), scale_dtype)
    axes = len(sections) if sections else 0
    if axes:
        if axes > kRopeMaxAxes:
            raise _lib.Error(_lib.RLK_EINVAL, f"{axes} position axes (at most {kRopeMaxAxes})")
        opt.num_axes, opt.sections, opt.interleaved = axes, tuple(sections), bool(interleaved)
    check(lib().rlk_rope_and_write_kv_norm(
        _arg(qkv, f16, "qkv", n * cols, dev), _arg(positions, i32, "positions", n * max(1, axes), dev),
        _arg(slot_mapping, i32, "slot_mapping", n, dev), num_tokens, num_heads,
        _arg(cos_table, f32, "cos_table", 0, dev), _arg(sin_table, f32, "sin_table", 0, dev),
        C.byref(kv), C.byref(opt), _stream_on(dev, stream)))


def read_kv(kv: KVLayerView, slots, n, k_out=None, v_out=None, scale_dtype=SCALE_F32, stream=None):
    """Extension: the stored rows of `slots` as fp16 [n, Hkv * D] (INT8: code * scale);
    a negative slot leaves its rows as they were."""
    dev, size = kv.device, max(n, 0) * kv.num_kv_heads * kv.head_dim
    if scale_dtype != kv.scale_dtype:
        _scales(kv, scale_dtype)
    check(lib().rlk_read_kv(
        C.byref(kv), _arg(slots, torch.int32, "slots", n, dev), n,
        None if k_out is None else _arg(k_out, torch.float16, "k_out", size, dev),
        None if v_out is None else _arg(v_out, torch.float16, "v_out", size, dev), scale_dtype,
        _stream_on(dev, stream)))


# ------------------------------------------- decode attention over a shared prefix

def shared_prefix_work(item_token, item_seq, num_items, group_start, group_prefix, num_groups, max_group_items,
                       max_prefix_partitions, max_partitions, workspace):
    """What paged_attention_decode_shared works on (rlk_shared_prefix_work); `workspace`
    is a DecodeWorkspace of max_prefix_partitions + max_partitions partitions.  The
    struct keeps its tensors."""
    if not isinstance(workspace, DecodeWorkspace):
        raise _lib.Error(_lib.RLK_EINVAL, "workspace must be a DecodeWorkspace")
    i = lambda t, n, w: _arg(t, torch.int32, w, n, None)  # noqa: E731
    ws, groups = workspace, num_groups > 0
    work = _lib.SharedPrefixWork(
        i(item_token, num_items, "item_token"), i(item_seq, num_items, "item_seq"), num_items,
        i(group_start, num_groups + 1, "group_start") if groups else None,
        i(group_prefix, num_groups, "group_prefix") if groups else None, num_groups, max_group_items,
        max_prefix_partitions, max_partitions, ws.out.data_ptr(), ws.max.data_ptr(), ws.sum.data_ptr())
    parts = max(1, max_prefix_partitions + max_partitions)
    work.room = min(ws.max.numel(), ws.sum.numel()) // parts, ws.out.numel() // parts
    return _keep(work, item_token, item_seq, *((group_start, group_prefix) if groups else ()), ws.out, ws.max, ws.sum)


def paged_attention_decode_shared(params: _lib.AttentionParams, work: _lib.SharedPrefixWork,
                                  scale_dtype=SCALE_F32, stream=None):
    """Extension: decode attention for groups of items that share their first tokens in
    the cache; a group's prefix is read once for all its items.  Items with a negative
    token are skipped."""
    if work.device != params.device:
        _same_device(params, work)
    if params.tensors is not None:
        _scales(params.tensors[0], scale_dtype)
        _one_device(params.device, *params.tensors[1:])
    if work.room is not None:
        rows = work.num_items * params.num_heads
        if rows > work.room[0] or rows * params.kv.head_dim > work.room[1]:
            raise _lib.Error(_lib.RLK_EINVAL, f"the workspace holds {work.room[0]} (item, head) rows and "
                                              f"{work.room[1]} elements a partition, needs {rows} of "
                                              f"{params.kv.head_dim}")
    opt = _lib.AttentionOptions(scale_dtype)
    check(lib().rlk_paged_attention_decode_shared(C.byref(params), C.byref(work), C.byref(opt),
                                                  _stream_on(params.device, stream)))


# --------------------------------------------------------------------- sampling

class SamplingWorkspace:
    """Memory of sample_tokens calls of up to max_rows rows of up to max_vocab tokens;
    calls that may run at the same time need one each."""

    def __init__(self, max_rows, max_vocab, device="cuda"):
        size = lib().rlk_sampling_workspace_bytes(max_rows, max_vocab)
        if size == 0:
            raise _lib.Error(_lib.RLK_EINVAL, f"no sampling workspace of {max_rows} rows of {max_vocab} tokens")
        self.memory = torch.empty(size, dtype=torch.uint8, device=device)


def sampling_work(logits, num_rows, vocab, temperature, top_k, top_p, uniform, tokens, workspace, min_p=None,
                  param_row=None, logprobs=None):
    """What sample_tokens reads and writes (rlk_sampling_work): logits fp16 or fp32
    [num_rows, >= vocab], rows contiguous; without param_row, row r has the settings
    temperature[r], ...  Values of param_row must lie in the settings.  The struct keeps
    its tensors."""
    if not isinstance(workspace, SamplingWorkspace):
        raise _lib.Error(_lib.RLK_EINVAL, "workspace must be a SamplingWorkspace")
    if not isinstance(logits, torch.Tensor) or logits.dtype not in (torch.float16, torch.float32):
        raise _lib.Error(_lib.RLK_EINVAL, "logits must be a tensor of torch.float16 or torch.float32")
    if not logits.is_cuda:
        raise _lib.Error(_lib.RLK_EINVAL, "logits must be a GPU tensor")
    n = max(num_rows, 0)
    if logits.dim() != 2 or logits.shape[0] < n or (n > 0 and logits.shape[1] < vocab):
        raise _lib.Error(_lib.RLK_EINVAL, f"logits must hold {n} rows of {vocab}, has {tuple(logits.shape)}")
    if logits.shape[1] > 1 and logits.stride(1) != 1:
        raise _lib.Error(_lib.RLK_EINVAL, "rows of logits must be contiguous")
    dev = logits.get_device()
    rows = n if param_row is None else min(n, 1)  # settings that are there for certain
    f, i = torch.float32, torch.int32
    work = _lib.SamplingWork(
        logits.data_ptr(), logits.dtype == f, logits.stride(0) if n > 1 else vocab, num_rows, vocab,
        None if param_row is None else _arg(param_row, i, "param_row", n, dev),
        _arg(temperature, f, "temperature", rows, dev), _arg(top_k, i, "top_k", rows, dev),
        _arg(top_p, f, "top_p", rows, dev), None if min_p is None else _arg(min_p, f, "min_p", rows, dev),
        _arg(uniform, f, "uniform", n, dev), _arg(tokens, i, "tokens", n, dev),
        None if logprobs is None else _arg(logprobs, f, "logprobs", n, dev),
        _arg(workspace.memory, torch.uint8, "workspace", 0, dev), workspace.memory.numel())
    return _keep(work, logits, *(t for t in (param_row, temperature, top_k, top_p, min_p, uniform, tokens, logprobs,
                                             workspace.memory) if t is not None))


def sample_tokens(work: _lib.SamplingWork, stream=None):
    """Extension: the next token of each row of logits by temperature, top-k, top-p and
    min-p, from one given random number a row; `work` from sampling_work()."""
    check(lib().rlk_sample_tokens(C.byref(work), _stream_on(work.device, stream)))
