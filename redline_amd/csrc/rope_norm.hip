// RMS norm of each query and key head, rotary embedding over one to four
// position axes and the paged KV-cache write in one pass; and the stored rows
// of a paged cache read back.  gfx950.
//
// Per token and head, x = the head's D elements (bias added first, if any):
//   n_i = x_i / sqrt(sum(x^2) / D + eps) * w_i        (q and k heads)
//   y_i = n_i c - n_{i+D/2} s,  y_{i+D/2} = n_{i+D/2} c + n_i s,   i < D/2
// with c, s the table row of the position that pair i's axis has.  n and y are
// held in fp32 and rounded to fp16 once, at the end; the sum of squares is in fp32.
//
// The mapping is that of the plain RoPE kernel: a lane owns 8 pairs, a head is
// D/16 lanes, so the sum of squares is 16 products in the lane and 2 or 3 DPP
// steps; one token per workgroup, its heads spread over the waves.  With one axis a
// lane loads its 8 cos and sin as vectors.  With several, an axis of a pair is two bits
// of the launch arguments, and the first D/2 threads gather a cos and a sin each into
// LDS for all heads (every lane for itself, 16 gathers: 19.4 us against 15.2 for 5024
// tokens of 40 heads of 64).
// Bound: HBM, as the plain kernel (11470 tokens of 48 heads of 128, FP16, write and read
// back: 67.2 us, 5.7 TB/s; 16384 tokens of 36 heads, INT8: 70.3 us, 4.9 TB/s); at a decode step's
// size the launch (5.0 us).
#include <hip/hip_runtime.h>

#include <cstdint>

#include "device.hpp"
#include "kv_cell.hpp"
#include "redline_amd/rlk.h"
#include "status.hpp"

namespace rlk {
namespace {

// How the pairs' axes lie: one for all, one for every lane's 8 pairs, or in any order.
enum Axes { kOne, kPerLane, kPerPair };

struct NormRopeArgs {
  _Float16* qkv;
  const int32_t* positions;  // [num_axes, num_tokens]
  const int32_t* slots;
  const float* cos_t;
  const float* sin_t;
  CellPlanes kv;
  const _Float16* bias;    // [heads * D] or null
  const _Float16* q_norm;  // [D] or null
  const _Float16* k_norm;
  float eps;
  int num_tokens, hq, hkv, block_size, num_axes;
  uint32_t axis[4];  // two bits a pair
};

template <int D, bool kInt8, int kAxes>
__global__ __launch_bounds__(512, kInt8 ? 1 : 8) void norm_rope_kv_kernel(NormRopeArgs a) {
#pragma clang fp contract(off)  // without norms the bits of the plain kernel
  constexpr bool NT = true;
  constexpr int kHalf = D / 2, kLPH = kHalf / 8, kHeadsPerWave = kWave / kLPH;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int step = kHeadsPerWave * (blockDim.x / kWave);
  const int hg = wave * kHeadsPerWave + lane / kLPH, part = lane % kLPH, p0 = part * 8;
  const int heads = a.hq + 2 * a.hkv;
  const int64_t t = blockIdx.x;
  _Float16* row = a.qkv + t * heads * D;
  u32x4 v0, v1;
  if (hg < heads) {
    v0 = ld16<NT>(reinterpret_cast<const u32x4*>(row + hg * D + p0));
    v1 = ld16<NT>(reinterpret_cast<const u32x4*>(row + hg * D + kHalf + p0));
  }
  const int slot = a.slots[t];
  f32x8 c, s;
  // the token's positions are uniform: scalar loads, selected by axis
  int pos[kAxes == kOne ? 1 : RLK_ROPE_MAX_AXES];
  pos[0] = a.positions[t];
  if constexpr (kAxes != kOne) {
#pragma unroll
    for (int x = 1; x < RLK_ROPE_MAX_AXES; ++x)
      pos[x] = a.positions[static_cast<int64_t>(min(x, a.num_axes - 1)) * a.num_tokens + t];
  }
  auto position_of = [&](int pair) -> int64_t {
    if constexpr (kAxes == kOne) return pos[0];
    else {
      uint32_t bits = a.axis[0];
#pragma unroll
      for (int w = 1; w < D / 32; ++w) bits = pair / 16 == w ? a.axis[w] : bits;
      const uint32_t x = bits >> (2 * (pair % 16)) & 3;
      const int lo = x & 1 ? pos[1] : pos[0], hi = x & 1 ? pos[3] : pos[2];
      return x & 2 ? hi : lo;
    }
  };
  if constexpr (kAxes == kPerPair) {
    __shared__ f32x4 turn[2][kHalf / 4];
    for (int i = threadIdx.x; i < kHalf; i += blockDim.x) {
      const int64_t at = position_of(i) * kHalf + i;
      reinterpret_cast<float*>(turn[0])[i] = a.cos_t[at];
      reinterpret_cast<float*>(turn[1])[i] = a.sin_t[at];
    }
    __syncthreads();
    c = __builtin_shufflevector(turn[0][2 * part], turn[0][2 * part + 1], 0, 1, 2, 3, 4, 5, 6, 7);
    s = __builtin_shufflevector(turn[1][2 * part], turn[1][2 * part + 1], 0, 1, 2, 3, 4, 5, 6, 7);
  } else {
    const int64_t at = position_of(p0) * kHalf + p0;
    const f32x4* cp = reinterpret_cast<const f32x4*>(a.cos_t + at);
    const f32x4* sp = reinterpret_cast<const f32x4*>(a.sin_t + at);
    c = __builtin_shufflevector(cp[0], cp[1], 0, 1, 2, 3, 4, 5, 6, 7);
    s = __builtin_shufflevector(sp[0], sp[1], 0, 1, 2, 3, 4, 5, 6, 7);
  }
  for (int h = hg; h < heads; h += step) {
    _Float16* hp = row + h * D;
    if (h != hg) {
      v0 = ld16<NT>(reinterpret_cast<const u32x4*>(hp + p0));
      v1 = ld16<NT>(reinterpret_cast<const u32x4*>(hp + kHalf + p0));
    }
    if (a.bias != nullptr) {  // fp16(x + b), as the plain kernel adds it
      const _Float16* b = a.bias + h * D + p0;
      v0 = __builtin_bit_cast(u32x4, __builtin_bit_cast(f16x8, v0) + *reinterpret_cast<const f16x8*>(b));
      v1 = __builtin_bit_cast(u32x4, __builtin_bit_cast(f16x8, v1) + *reinterpret_cast<const f16x8*>(b + kHalf));
    }
    f32x8 x0 = unpack8(v0), x1 = unpack8(v1);
    const bool is_q = h < a.hq, is_v = h >= a.hq + a.hkv;
    if (!is_v) {
      const _Float16* w = is_q ? a.q_norm : a.k_norm;
      if (w != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += x0[j] * x0[j] + x1[j] * x1[j];
        const float inv = 1.f / __builtin_sqrtf(group_sum<kLPH>(ss) / D + a.eps);
        x0 = x0 * inv * unpack8(load16(w + p0));
        x1 = x1 * inv * unpack8(load16(w + kHalf + p0));
      }
      const f32x8 y0 = x0 * c - x1 * s, y1 = x1 * c + x0 * s;
      x0 = y0;
      x1 = y1;
    }
    if (is_q) {
      st16<NT>(reinterpret_cast<u32x4*>(hp + p0), pack8(x0));
      st16<NT>(reinterpret_cast<u32x4*>(hp + kHalf + p0), pack8(x1));
      continue;
    }
    if (slot < 0) continue;
    const int blk = slot / a.block_size, off = slot - blk * a.block_size;
    const int kvh = h - a.hq - (is_v ? a.hkv : 0);
    store_cell<D, kInt8>(a.kv, is_v, (static_cast<int64_t>(blk) * a.hkv + kvh) * a.block_size + off, p0,
                         round_f16(x0), round_f16(x1));
  }
}

template <int D, bool kInt8>
void launch_axes(const NormRopeArgs& a, Axes axes, int waves, hipStream_t stream) {
  const dim3 grid(a.num_tokens), block(waves * kWave);
  switch (axes) {
    case kOne: norm_rope_kv_kernel<D, kInt8, kOne><<<grid, block, 0, stream>>>(a); break;
    case kPerLane: norm_rope_kv_kernel<D, kInt8, kPerLane><<<grid, block, 0, stream>>>(a); break;
    default: norm_rope_kv_kernel<D, kInt8, kPerPair><<<grid, block, 0, stream>>>(a); break;
  }
}

// The axis of each of the `half` pairs into `bits`, two bits a pair; RLK_OK or a
// failure status.
int axes_of_pairs(const rlk_norm_rope_options& o, int half, uint32_t (&bits)[4], Axes* axes, const char* what) {
  for (uint32_t& b : bits) b = 0;
  *axes = kOne;
  if (o.num_axes < 0 || o.num_axes > RLK_ROPE_MAX_AXES)
    return fail(RLK_EINVAL, "%s: %d position axes (at most %d)", what, o.num_axes, RLK_ROPE_MAX_AXES);
  if (o.num_axes <= 1) return RLK_OK;
  const int n = o.num_axes;
  int64_t sum = 0;
  for (int x = 0; x < n; ++x) {
    if (o.sections[x] < 0) return fail(RLK_EINVAL, "%s: negative section %d", what, o.sections[x]);
    sum += o.sections[x];
  }
  if (sum != half) return fail(RLK_EINVAL, "%s: the sections hold %lld pairs of %d", what, static_cast<long long>(sum), half);
  int of[64];
  if (o.interleaved) {
    for (int x = 1; x < n; ++x)
      if (o.sections[x] > 0 && n * (o.sections[x] - 1) + x >= half)
        return fail(RLK_EINVAL, "%s: %d pairs of axis %d do not fit %d turns", what, o.sections[x], x, half / n);
    for (int i = 0; i < half; ++i) of[i] = i / n < o.sections[i % n] ? i % n : 0;
  } else {
    int at = 0;
    for (int x = 0; x < n; ++x)
      for (int i = 0; i < o.sections[x]; ++i) of[at++] = x;
  }
  *axes = kPerLane;
  for (int i = 0; i < half; ++i) {
    bits[i / 16] |= static_cast<uint32_t>(of[i]) << (2 * (i % 16));
    if (of[i] != of[i / 8 * 8]) *axes = kPerPair;
  }
  return RLK_OK;
}

// ---- rows read back

struct ReadArgs {
  CellPlanes kv;
  const int32_t* slots;
  u32x4* k_out;
  u32x4* v_out;
  int64_t vecs;  // 8-element vectors of one output
  int hkv, block_size;
};

// One 16-byte vector of K and of V per lane.
template <int D, bool kInt8>
__global__ __launch_bounds__(256) void read_kv_kernel(ReadArgs a) {
  constexpr int kPer = D / 8;
  const int64_t g = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (g >= a.vecs) return;
  const int64_t hr = g / kPer;
  const int e = static_cast<int>(g % kPer), kvh = static_cast<int>(hr % a.hkv);
  const int slot = a.slots[hr / a.hkv];
  if (slot < 0) return;
  const int blk = slot / a.block_size, off = slot - blk * a.block_size;
  const int64_t cell = (static_cast<int64_t>(blk) * a.hkv + kvh) * a.block_size + off;
  auto row = [&](const void* base, const void* scales) -> u32x4 {
    if constexpr (!kInt8) {
      return ld16<true>(reinterpret_cast<const u32x4*>(static_cast<const _Float16*>(base) + cell * D) + e);
    } else {
      const i8x8 q = __builtin_bit_cast(i8x8, *(reinterpret_cast<const u32x2*>(static_cast<const int8_t*>(base) + cell * D) + e));
      const float s = a.kv.scale16 ? static_cast<float>(static_cast<const _Float16*>(scales)[cell])
                                   : static_cast<const float*>(scales)[cell];
      return pack8(__builtin_convertvector(q, f32x8) * s);
    }
  };
  u32x4 k, v;
  if (a.k_out != nullptr) k = row(a.kv.k, a.kv.k_scale);
  if (a.v_out != nullptr) v = row(a.kv.v, a.kv.v_scale);
  if (a.k_out != nullptr) st16<true>(a.k_out + g, k);
  if (a.v_out != nullptr) st16<true>(a.v_out + g, v);
}

// Checks of a layer view that both entry points share.
int check_layer_view(const rlk_kv_layer_view* kv, int scale_dtype, const char* what) {
  if (kv == nullptr) return fail(RLK_EINVAL, "%s: null KV layer view", what);
  if (kv->head_dim != 64 && kv->head_dim != 128)
    return fail(RLK_EUNSUPPORTED, "%s: unsupported head_dim %d (supported: 64, 128)", what, kv->head_dim);
  if (kv->dtype != RLK_KV_FP16 && kv->dtype != RLK_KV_INT8)
    return fail(RLK_EINVAL, "%s: unknown KV dtype %d", what, kv->dtype);
  if (scale_dtype != RLK_SCALE_F32 && scale_dtype != RLK_SCALE_F16)
    return fail(RLK_EINVAL, "%s: unknown scale dtype %d", what, scale_dtype);
  if (kv->num_kv_heads <= 0 || kv->block_size <= 0)
    return fail(RLK_EINVAL, "%s: bad kv head count %d or block size %d", what, kv->num_kv_heads, kv->block_size);
  if (kv->k == nullptr || kv->v == nullptr ||
      (kv->dtype == RLK_KV_INT8 && (kv->k_scale == nullptr || kv->v_scale == nullptr)))
    return fail(RLK_EINVAL, "%s: null pointer argument", what);
  if (((reinterpret_cast<uintptr_t>(kv->k) | reinterpret_cast<uintptr_t>(kv->v)) & 15) != 0)
    return fail(RLK_EINVAL, "%s: the cache planes must be 16-byte aligned", what);
  return RLK_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace rlk

using namespace rlk;

extern "C" int rlk_rope_and_write_kv_norm(uint16_t* qkv, const int32_t* positions, const int32_t* slot_mapping,
                                          int num_tokens, int num_heads, const float* cos_table,
                                          const float* sin_table, const rlk_kv_layer_view* kv,
                                          const rlk_norm_rope_options* options, hipStream_t stream) {
  const char* what = "rope_and_write_kv_norm";
  if (num_tokens <= 0) return RLK_OK;
  const rlk_norm_rope_options none = {};
  const rlk_norm_rope_options& o = options != nullptr ? *options : none;
  if (const int st = check_layer_view(kv, o.scale_dtype, what); st != RLK_OK) return st;
  if (num_heads < 0) return fail(RLK_EINVAL, "%s: bad head count %d", what, num_heads);
  const int64_t heads = static_cast<int64_t>(num_heads) + 2 * static_cast<int64_t>(kv->num_kv_heads);
  if (heads * kv->head_dim > (1 << 30)) return fail(RLK_EINVAL, "%s: a row of %lld heads", what, static_cast<long long>(heads));
  if (qkv == nullptr || positions == nullptr || slot_mapping == nullptr || cos_table == nullptr || sin_table == nullptr)
    return fail(RLK_EINVAL, "%s: null pointer argument", what);
  if (!aligned16(qkv) || !aligned16(cos_table) || !aligned16(sin_table) || !aligned16(o.qkv_bias) ||
      !aligned16(o.q_norm) || !aligned16(o.k_norm))
    return fail(RLK_EINVAL, "%s: qkv, tables, bias and norm weights must be 16-byte aligned", what);
  if ((o.q_norm != nullptr || o.k_norm != nullptr) && !(o.eps >= 0.f))
    return fail(RLK_EINVAL, "%s: bad eps", what);
  NormRopeArgs a;
  Axes axes;
  if (const int st = axes_of_pairs(o, kv->head_dim / 2, a.axis, &axes, what); st != RLK_OK) return st;
  a.qkv = reinterpret_cast<_Float16*>(qkv);
  a.positions = positions;
  a.slots = slot_mapping;
  a.cos_t = cos_table;
  a.sin_t = sin_table;
  a.kv = {kv->k, kv->v, kv->k_scale, kv->v_scale, o.scale_dtype == RLK_SCALE_F16};
  a.bias = reinterpret_cast<const _Float16*>(o.qkv_bias);
  a.q_norm = reinterpret_cast<const _Float16*>(o.q_norm);
  a.k_norm = reinterpret_cast<const _Float16*>(o.k_norm);
  a.eps = o.eps;
  a.num_tokens = num_tokens;
  a.hq = num_heads;
  a.hkv = kv->num_kv_heads;
  a.block_size = kv->block_size;
  a.num_axes = o.num_axes;
  const int per_wave = kWave / (kv->head_dim / 16);
  const int waves = static_cast<int>(heads + per_wave - 1) / per_wave;
  const int w = waves > 8 ? 8 : waves;
  if (static_cast<int64_t>(num_tokens) * w * kWave > UINT32_MAX)
    return fail(RLK_EINVAL, "%s: %d tokens exceed one launch; split the call", what, num_tokens);
  const bool int8 = kv->dtype == RLK_KV_INT8;
  if (kv->head_dim == 128)
    int8 ? launch_axes<128, true>(a, axes, w, stream) : launch_axes<128, false>(a, axes, w, stream);
  else
    int8 ? launch_axes<64, true>(a, axes, w, stream) : launch_axes<64, false>(a, axes, w, stream);
  return launch_status(what);
}

extern "C" int rlk_read_kv(const rlk_kv_layer_view* kv, const int32_t* slots, int n, uint16_t* k_out, uint16_t* v_out,
                           int scale_dtype, hipStream_t stream) {
  const char* what = "read_kv";
  if (n <= 0) return RLK_OK;
  if (const int st = check_layer_view(kv, scale_dtype, what); st != RLK_OK) return st;
  if (slots == nullptr) return fail(RLK_EINVAL, "%s: null pointer argument", what);
  if (!aligned16(k_out) || !aligned16(v_out))
    return fail(RLK_EINVAL, "%s: outputs must be 16-byte aligned", what);
  if (k_out == nullptr && v_out == nullptr) return RLK_OK;
  ReadArgs a;
  a.kv = {kv->k, kv->v, kv->k_scale, kv->v_scale, scale_dtype == RLK_SCALE_F16};
  a.slots = slots;
  a.k_out = reinterpret_cast<u32x4*>(k_out);
  a.v_out = reinterpret_cast<u32x4*>(v_out);
  a.vecs = static_cast<int64_t>(n) * kv->num_kv_heads * (kv->head_dim / 8);
  a.hkv = kv->num_kv_heads;
  a.block_size = kv->block_size;
  if (a.vecs > (int64_t{1} << 31)) return fail(RLK_EINVAL, "%s: %d rows exceed one launch; split the call", what, n);
  const uint32_t grid = static_cast<uint32_t>((a.vecs + 255) / 256);
  const bool int8 = kv->dtype == RLK_KV_INT8;
  if (kv->head_dim == 128)
    int8 ? read_kv_kernel<128, true><<<grid, 256, 0, stream>>>(a) : read_kv_kernel<128, false><<<grid, 256, 0, stream>>>(a);
  else
    int8 ? read_kv_kernel<64, true><<<grid, 256, 0, stream>>>(a) : read_kv_kernel<64, false><<<grid, 256, 0, stream>>>(a);
  return launch_status(what);
}
