// Paged decode attention over the block-scaled 8-bit cache, for gfx950.
//
// Flash-decoding: o = sum_k p_k v_k / sum_k p_k with p_k = exp(scale q.k - m),
// split over the keys and joined by the rule of the running maximum.  One wave
// takes a contiguous range of keys of one (item, kv head) and all G query heads
// of the group, so every code is read once; the 4 waves of a workgroup take
// neighbouring ranges and meet in LDS once, at the end; workgroups of one item
// meet in a second kernel through the caller's workspace.
//
// The cache's byte order (rlk.h) is the matrix cores' operand order, so a wave
// step of 32 keys (two tiles of 16) moves whole contiguous kilobytes and no
// element changes its lane:
//   q.k  v_mfma_f32_16x16x32_f16, A = K (row r = token), B = q (column c = query
//        head): lane (rho, r) takes the 16 bytes of piece 4x + rho, token r, two
//        8-dim operands;
//   P.V  A = V (row m), B = P: lane (rho, m) takes the bytes of tokens
//        4 rho .. 4 rho + 3, and the scores of those tokens are what the first
//        product left in the lane.
// Codes become fp16 exactly; the K scale multiplies the fp32 scores (with the
// softmax scale), the V scale the fp32 probabilities, relative to the largest V
// scale that the wave has met (a power of two, so the ratio is exact and the
// fp16 operand keeps its 11 bits however small V is).  m, l and the output stay
// in fp32.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cstdint>

#include "kv_blocks.hpp"

namespace rlk {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kPart = RLK_DECODE_PARTITION_SIZE;
constexpr int kStepTokens = 32;
constexpr int kMaxSlots = 4096;  // workspace slots that the merge joins

struct DecodeArgs {
  rlk_block_attention_params p;
  rlk_decode_attention_work w;
  int wave_tokens;  // keys of a wave: a multiple of 64
};

// Keys that an item attends to: its context, inside its table row and the
// partitions of the call.
__device__ __forceinline__ int keys_of(const DecodeArgs& a, int token) {
  const int64_t most = min(static_cast<int64_t>(a.p.max_blocks_per_seq) * a.p.kv.block_size,
                           static_cast<int64_t>(a.w.max_partitions) * kPart);
  return static_cast<int>(min(static_cast<int64_t>(a.p.positions[token]) + 1, most));
}

// The codes of one wave step in flight: two tiles.
template <int D>
struct StepCodes {
  u32x4 r[2][D / 64];
};

template <int D>
__device__ __forceinline__ void issue(StepCodes<D>& s, const uint8_t* t0, const uint8_t* t1, int lane) {
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int x = 0; x < D / 64; ++x) {
    s.r[0][x] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(t0 + x * 1024) + lane);
    s.r[1][x] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(t1 + x * 1024) + lane);
  }
  __builtin_amdgcn_sched_barrier(0);
}

template <int D, int G>
struct DecodeLds {
  float o[kWaves][G][D];
  float m[kWaves][G], l[kWaves][G];
};

template <int D, int G, bool kFp8>
__global__ __launch_bounds__(kThreads, 4) void decode_blocks_kernel(DecodeArgs a) {
  constexpr int E = D / 16, kX = D / 64;
  constexpr float kLog2e = 1.4426950408889634f;
  __shared__ DecodeLds<D, G> s;
  const rlk_block_attention_params& p = a.p;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int rho = lane / 16, c = lane % 16;
  const int slot = blockIdx.x, kvh = blockIdx.y, item = blockIdx.z;
  const int token = a.w.item_token[item];
  if (token < 0) return;
  const int n = keys_of(a, token);
  const int group_tokens = kWaves * a.wave_tokens;
  _Float16* out = reinterpret_cast<_Float16*>(p.out) + (static_cast<int64_t>(token) * p.num_heads + kvh * G) * D;
  if (slot * group_tokens >= n) {
    if (slot == 0)  // nothing to attend to
      for (int i = tid; i < G * D; i += kThreads) out[i] = static_cast<_Float16>(0.f);
    return;
  }
  const int seq = a.w.item_seq[item];
  const int first = slot * group_tokens + wave * a.wave_tokens;
  const int count = min(a.wave_tokens, n - first);  // <= 0: a wave without keys

  f32x4 o[E];
#pragma unroll
  for (int d = 0; d < E; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -FLT_MAX, l = 0.f, vref = 0.f;
  if (count > 0) {
    const int bs = p.kv.block_size, tpb = bs / kTileTokens, hkv = p.kv.num_kv_heads;
    const int tiles = (count + kTileTokens - 1) / kTileTokens, tile0 = first / kTileTokens;
    // lane t < tiles: the block of the wave's tile t (a wave has at most 64)
    const int bt = (tile0 + min(lane, tiles - 1)) / tpb;
    int blk = p.block_tables[static_cast<int64_t>(seq) * p.max_blocks_per_seq + bt];
    blk = static_cast<uint32_t>(blk) < static_cast<uint32_t>(p.kv.num_blocks) ? blk : 0;
    const uint8_t* kbase = static_cast<const uint8_t*>(p.kv.k);
    const uint8_t* vbase = static_cast<const uint8_t*>(p.kv.v);
    auto cell_of = [&](int t) {  // uniform; tiles past the last repeat it
      return static_cast<int64_t>(__builtin_amdgcn_readlane(blk, min(t, tiles - 1))) * hkv + kvh;
    };
    auto tile_at = [&](const uint8_t* base, int t) {
      return base + (cell_of(t) * tpb + (tile0 + min(t, tiles - 1)) % tpb) * (kTileTokens * D);
    };
    StepCodes<D> kc, vc;
    issue<D>(kc, tile_at(kbase, 0), tile_at(kbase, 1), lane);
    issue<D>(vc, tile_at(vbase, 0), tile_at(vbase, 1), lane);
    // q: column c = head c, zero past the group
    const _Float16* q = reinterpret_cast<const _Float16*>(p.q) + static_cast<int64_t>(token) * p.q_stride +
                        (kvh * G + min(c, G - 1)) * D;
    f16x8 qb[kX][2];
#pragma unroll
    for (int x = 0; x < kX; ++x)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x4 v = load16(q + h * (D / 2) + 8 * (4 * x + rho));
        qb[x][h] = __builtin_bit_cast(f16x8, c < G ? v : u32x4{0, 0, 0, 0});
      }
    const float qscale = p.scale * kLog2e;
    const int steps = (tiles + 1) / 2;
    for (int st = 0; st < steps; ++st) {
      const int64_t c0 = cell_of(2 * st), c1 = cell_of(2 * st + 1);
      const float ks[2] = {p.kv.k_scale[c0] * qscale, p.kv.k_scale[c1] * qscale};
      const float vs[2] = {p.kv.v_scale[c0], p.kv.v_scale[c1]};
      f32x4 acc[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < kX; ++x)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const f16x4 lo = codes_to_f16<kFp8>(kc.r[t][x][2 * h]), hi = codes_to_f16<kFp8>(kc.r[t][x][2 * h + 1]);
            const f16x8 av = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, qb[x][h], acc[t], 0, 0, 0);
          }
      }
      issue<D>(kc, tile_at(kbase, 2 * st + 2), tile_at(kbase, 2 * st + 3), lane);
      // this lane: tokens 4 rho + i of both tiles, head c
      const int left = count - st * kStepTokens;  // keys of this step (may pass 32)
      float e[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) e[t][i] = acc[t][i] * ks[t];
      if (left < kStepTokens) {  // uniform: only a wave's last step
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (16 * t + 4 * rho + i >= left) e[t][i] = -FLT_MAX;
        // bytes of tokens past the context may be anything (an e4m3 NaN too)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int keep = min(max(left - 16 * t - 4 * rho, 0), 4);
          const uint32_t mask = keep == 0 ? 0u : 0xffffffffu >> (32 - 8 * keep);
#pragma unroll
          for (int x = 0; x < kX; ++x) vc.r[t][x] &= u32x4{mask, mask, mask, mask};
        }
      }
      float mx = fmaxf(fmaxf(fmaxf(e[0][0], e[0][1]), fmaxf(e[0][2], e[0][3])),
                       fmaxf(fmaxf(e[1][0], e[1][1]), fmaxf(e[1][2], e[1][3])));
      mx = rows_max<true>(rows_max<false>(mx));
      const float mn = fmaxf(m, mx), vn = fmaxf(vref, fmaxf(vs[0], vs[1]));
      if (__any(mn != m) || vn != vref) {  // the output so far moves to the new references
        const float f = __builtin_amdgcn_exp2f(m - mn);
        l *= f;
        const float fo = f * vref * inv_scale(vn);
#pragma unroll
        for (int d = 0; d < E; ++d) o[d] *= fo;
        m = mn;
        vref = vn;
      }
      const float vi = inv_scale(vref);
      const float w[2] = {vs[0] * vi, vs[1] * vi};
      f16x8 b;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float pr = __builtin_amdgcn_exp2f(e[t][i] - m);
          l += pr;
          b[4 * t + i] = static_cast<_Float16>(pr * w[t]);
        }
#pragma unroll
      for (int x = 0; x < kX; ++x)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f16x4 lo = codes_to_f16<kFp8>(vc.r[0][x][j]), hi = codes_to_f16<kFp8>(vc.r[1][x][j]);
          const f16x8 av = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
          o[4 * x + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, b, o[4 * x + j], 0, 0, 0);
        }
      issue<D>(vc, tile_at(vbase, 2 * st + 2), tile_at(vbase, 2 * st + 3), lane);
    }
    l = rows_sum<true>(rows_sum<false>(l));
  }
  if (c < G) {
#pragma unroll
    for (int d = 0; d < E; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) s.o[wave][c][E * (4 * rho + i) + d] = o[d][i] * vref;
    if (rho == 0) {
      s.m[wave][c] = m;
      s.l[wave][c] = l;
    }
  }
  __syncthreads();
  const bool whole = n <= group_tokens;  // the item's only workgroup
  for (int i = tid; i < G * D; i += kThreads) {
    const int g = i / D, d = i % D;
    float M = s.m[0][g];
#pragma unroll
    for (int v = 1; v < kWaves; ++v) M = fmaxf(M, s.m[v][g]);
    float L = 0.f, acc = 0.f;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      const float f = __builtin_amdgcn_exp2f(s.m[v][g] - M);  // 0 for a wave without keys
      L += f * s.l[v][g];
      acc += f * s.o[v][g][d];
    }
    if (whole) {
      out[i] = static_cast<_Float16>(acc / L);
    } else {
      const int64_t row = (static_cast<int64_t>(item) * p.num_heads + kvh * G + g) * a.w.max_partitions + slot;
      a.w.ws_out[row * D + d] = acc;
      if (d == 0) {
        a.w.ws_max[row] = M;
        a.w.ws_sum[row] = L;
      }
    }
  }
}

// Joins the partials of one (item, head): lane d takes dim d.
template <int D>
__global__ __launch_bounds__(D) void merge_blocks_kernel(DecodeArgs a) {
  const int item = blockIdx.x, h = blockIdx.y, d = threadIdx.x;
  const int token = a.w.item_token[item];
  if (token < 0) return;
  const int n = keys_of(a, token), group_tokens = kWaves * a.wave_tokens;
  if (n <= group_tokens) return;
  const int slots = (n + group_tokens - 1) / group_tokens;
  const int64_t row = (static_cast<int64_t>(item) * a.p.num_heads + h) * a.w.max_partitions;
  float M = -FLT_MAX, L = 0.f, o = 0.f;
  for (int s = 0; s < slots; ++s) M = fmaxf(M, a.w.ws_max[row + s]);
  for (int s = 0; s < slots; ++s) {
    const float f = __builtin_amdgcn_exp2f(a.w.ws_max[row + s] - M);
    L += f * a.w.ws_sum[row + s];
    o += f * a.w.ws_out[(row + s) * D + d];
  }
  reinterpret_cast<_Float16*>(a.p.out)[(static_cast<int64_t>(token) * a.p.num_heads + h) * D + d] =
      static_cast<_Float16>(o / L);
}

template <int D, int G, bool kFp8>
void launch_g(const DecodeArgs& a, hipStream_t stream) {
  const int group_tokens = kWaves * a.wave_tokens;
  const int slots = (a.w.max_partitions * kPart + group_tokens - 1) / group_tokens;
  const dim3 grid(slots, a.p.kv.num_kv_heads, a.w.num_items);
  decode_blocks_kernel<D, G, kFp8><<<grid, kThreads, 0, stream>>>(a);
  if (slots > 1) merge_blocks_kernel<D><<<dim3(a.w.num_items, a.p.num_heads), D, 0, stream>>>(a);
}

template <int D, bool kFp8>
bool launch_d(const DecodeArgs& a, int G, hipStream_t stream) {
  switch (G) {
    case 1: launch_g<D, 1, kFp8>(a, stream); return true;
    case 2: launch_g<D, 2, kFp8>(a, stream); return true;
    case 3: launch_g<D, 3, kFp8>(a, stream); return true;
    case 4: launch_g<D, 4, kFp8>(a, stream); return true;
    case 5: launch_g<D, 5, kFp8>(a, stream); return true;
    case 6: launch_g<D, 6, kFp8>(a, stream); return true;
    case 7: launch_g<D, 7, kFp8>(a, stream); return true;
    case 8: launch_g<D, 8, kFp8>(a, stream); return true;
    default: return false;
  }
}

}  // namespace

// Checks that the attention entry points share; RLK_OK or a failure status.
int check_block_params(const rlk_block_attention_params* p, const char* what) {
  if (const int st = check_block_view(&p->kv, what); st != RLK_OK) return st;
  if (p->num_heads <= 0 || p->num_heads % p->kv.num_kv_heads != 0)
    return fail(RLK_EINVAL, "%s: num_heads must be a multiple of num_kv_heads (%d, %d)", what,
                p->num_heads, p->kv.num_kv_heads);
  if (p->num_heads / p->kv.num_kv_heads > 8)
    return fail(RLK_EUNSUPPORTED, "%s: unsupported GQA group size %d", what,
                p->num_heads / p->kv.num_kv_heads);
  if (p->max_blocks_per_seq <= 0)
    return fail(RLK_EINVAL, "%s: bad table width %d", what, p->max_blocks_per_seq);
  if (p->q == nullptr || p->out == nullptr || p->block_tables == nullptr || p->positions == nullptr)
    return fail(RLK_EINVAL, "%s: null pointer argument", what);
  if (p->q_stride % 8 != 0 || ((reinterpret_cast<uintptr_t>(p->q) | reinterpret_cast<uintptr_t>(p->out)) & 15) != 0)
    return fail(RLK_EINVAL, "%s: q and out rows must be 16-byte aligned (q_stride %d)", what,
                p->q_stride);
  return RLK_OK;
}

}  // namespace rlk

using namespace rlk;

extern "C" int rlk_paged_attention_decode_blocks(const rlk_block_attention_params* p,
                                                 const rlk_decode_attention_work* w,
                                                 hipStream_t stream) {
  const char* what = "paged_attention_decode_blocks";
  if (p == nullptr || w == nullptr) return fail(RLK_EINVAL, "%s: null params or work", what);
  if (w->num_items <= 0) return RLK_OK;
  if (const int st = check_block_params(p, what); st != RLK_OK) return st;
  if (w->num_items > 65535 || p->kv.num_kv_heads > 65535 || p->num_heads > 65535)
    return fail(RLK_EINVAL, "%s: %d items exceed one launch; split the call", what, w->num_items);
  if (w->max_partitions < 1)
    return fail(RLK_EINVAL, "%s: bad max_partitions %d", what, w->max_partitions);
  if (w->max_partitions > kMaxSlots)
    return fail(RLK_EUNSUPPORTED, "%s: max_partitions %d exceeds %d", what, w->max_partitions, kMaxSlots);
  if (w->item_token == nullptr || w->item_seq == nullptr)
    return fail(RLK_EINVAL, "%s: null pointer argument", what);
  if (w->max_partitions > 1 && (w->ws_out == nullptr || w->ws_max == nullptr || w->ws_sum == nullptr))
    return fail(RLK_EINVAL, "%s: split-K workspace is required when max_partitions > 1", what);
  DecodeArgs a = {*p, *w, 64};
  const int64_t units = static_cast<int64_t>(w->num_items) * p->kv.num_kv_heads * w->max_partitions;
  if (units > 4096) a.wave_tokens = 128;
  const int G = p->num_heads / p->kv.num_kv_heads;
  const bool fp8 = p->kv.format == RLK_KV_BLOCK_FP8;
  const bool ok = p->kv.head_dim == 128
                      ? (fp8 ? launch_d<128, true>(a, G, stream) : launch_d<128, false>(a, G, stream))
                      : (fp8 ? launch_d<64, true>(a, G, stream) : launch_d<64, false>(a, G, stream));
  if (!ok) return fail(RLK_EUNSUPPORTED, "%s: unsupported GQA group size %d", what, G);
  return launch_status(what);
}
