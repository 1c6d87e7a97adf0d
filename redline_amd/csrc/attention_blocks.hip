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
// softmax scale), the V scale s_k the fp32 probabilities.  The running reference m
// is the maximum of scale q.k + log s_k, not of scale q.k alone: the fp16 operand
// p_k s_k then has its 11 bits for the keys that weigh most in the output, however
// small their V is and whatever V the keys without weight have (scales lie in
// 2^-24 .. 2^10, so p_k and its sum stay far inside fp32's range).  m, l and the
// output stay in fp32.
// Bound: HBM reads for full batches, which stream at 6.1 TB/s between a start of
// about 4 us (lengths, table entries, scales: dependent reads) and the merge's 4-5:
// 32 items to 8191 keys (INT8, 8 kv heads of 128, 257 MB) 52 us in all, 4.9 TB/s;
// 12 items to 40000 (e4m3, 4 kv heads, 332 MB) 65 us, 5.1 TB/s.  Small calls by two
// launches and those reads: one item of 2000 keys 5 + 3 us.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cstdint>
#include <type_traits>

#include "kv_blocks.hpp"

namespace rlk {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kPart = RLK_DECODE_PARTITION_SIZE;
constexpr int kStep = 32;        // keys of a wave step
constexpr int kMaxSlots = 4096;  // workspace slots that the merge joins
constexpr int kMaxItemsLds = 1024;
constexpr int kMinRange = 512 / kStep, kMaxRange = 1024 / kStep;  // steps of a wave's range
// Steps in flight and ranges per CU of the range form.  Two waves of a SIMD with 3
// steps of 8 KB each in flight; measured at 32 items to 8191 keys (8 kv heads of
// 128, INT8) / 12 items to 40000 (4 kv heads, e4m3) / 32 items of 8000-8191, us:
// 3 steps and 2 waves 48.4 / 60.4 / 91.6, 4 and 2 48.9 / 59.7 / 91.3, 2 and 3
// 46.3 / 63.8 / 92.4, 2 and 4 (spills) 63.6 / 81.5 / 115.7; at D = 64 all within 5%.
constexpr int kDepth = 3, kWavesPerCu = 8;
constexpr float kLog2e = 1.4426950408889634f;

struct DecodeArgs {
  rlk_block_attention_params p;
  rlk_decode_attention_work w;
  int group_tokens;  // grid form: keys of a workgroup
  int ranges;        // range form: ranges that the call is split into, at least
};

// Keys that an item attends to: its context, inside its table row and the
// partitions of the call.
__device__ __forceinline__ int keys_of(const DecodeArgs& a, int token) {
  const int64_t most = min(static_cast<int64_t>(a.p.max_blocks_per_seq) * a.p.kv.block_size,
                           static_cast<int64_t>(a.w.max_partitions) * kPart);
  return static_cast<int>(max(min(static_cast<int64_t>(a.p.positions[token]) + 1, most), static_cast<int64_t>(0)));
}

// The codes of one wave step in flight: two tiles of K and of V.
template <int D>
struct StepCodes {
  u32x4 k[2][D / 64], v[2][D / 64];
};

__device__ __forceinline__ float lane_value(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// What a wave has of its keys: column c = lane % 16 (head), rows 4 (lane / 16) + i
// of output tile d; m and l per head, the same in the 4 row groups after finish().
template <int D>
struct WaveState {
  f32x4 o[D / 16];
  float m = -FLT_MAX, l = 0.f;

  __device__ __forceinline__ WaveState() {
#pragma unroll
    for (int d = 0; d < D / 16; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  __device__ __forceinline__ void finish() { l = rows_sum<true>(rows_sum<false>(l)); }
  // element i of output tile d: dim
  __device__ __forceinline__ static int dim(int d, int i) {
    return (D / 16) * (4 * (static_cast<int>(threadIdx.x) % kWave / 16) + i) + d;
  }
};

// Block of tile tile0 + lane in each lane; entries past the table row repeat its
// last one.
__device__ __forceinline__ int table_entries(const DecodeArgs& a, int seq, int tile0) {
  const int t = tile0 + static_cast<int>(threadIdx.x) % kWave;
  const int b = min(a.p.kv.block_size == 32 ? t / 2 : t, a.p.max_blocks_per_seq - 1);
  return a.p.block_tables[static_cast<int64_t>(seq) * a.p.max_blocks_per_seq + b];
}

// One wave over `count` keys (at most 1024) from tile tile0 of one (item, kv
// head); blk: table_entries(tile0).  kDepth steps are in flight: each step's
// codes are requested kDepth steps ahead into the registers that it frees.
template <int D, int G, bool kFp8, int kDepth>
__device__ __forceinline__ void attend(const DecodeArgs& a, WaveState<D>& w, int token, int kvh, int tile0,
                                       int count, int blk) {
  constexpr int E = D / 16, kX = D / 64;
  const rlk_block_attention_params& p = a.p;
  const int lane = threadIdx.x % kWave, rho = lane / 16, c = lane % 16;
  const int tiles = (count + kTileTokens - 1) / kTileTokens, steps = (tiles + 1) / 2;
  const int tsh = p.kv.block_size == 32 ? 1 : 0;  // log2 tiles of a block
  blk = static_cast<uint32_t>(blk) < static_cast<uint32_t>(p.kv.num_blocks) ? blk : 0;
  const uint32_t cell = static_cast<uint32_t>(blk) * p.kv.num_kv_heads + kvh;
  const uint32_t tile = (cell << tsh) + ((tile0 + lane) & tsh);  // layout tile of the pool
  const uint8_t* kbase = static_cast<const uint8_t*>(p.kv.k);
  const uint8_t* vbase = static_cast<const uint8_t*>(p.kv.v);
  StepCodes<D> codes[kDepth];
  // steps past the last repeat its last tile, so that every request is unconditional
  auto issue = [&](StepCodes<D>& s, int st) {
    __builtin_amdgcn_sched_barrier(0);
    uint64_t at[2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
      at[t] = static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(
                  static_cast<int>(tile), min(2 * st + t, tiles - 1)))) * (kTileTokens * D);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int x = 0; x < kX; ++x)
        s.k[t][x] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kbase + at[t] + x * 1024) + lane);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int x = 0; x < kX; ++x)
        s.v[t][x] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(vbase + at[t] + x * 1024) + lane);
    __builtin_amdgcn_sched_barrier(0);
  };
  // lane t: the scales of tile t, and the V scale's logarithm (0 counts as 2^-24)
  float ksl = p.kv.k_scale[cell];
  const float vsl = p.kv.v_scale[cell];
  const float vll = static_cast<float>(max(static_cast<int>(__builtin_bit_cast(uint32_t, vsl) >> 23) - 127, -24));
  // q: column c = head c, zero past the group
  const _Float16* q = reinterpret_cast<const _Float16*>(p.q) + static_cast<int64_t>(token) * p.q_stride +
                      (kvh * G + min(c, G - 1)) * D;
  f16x8 qb[kX][2];
#pragma unroll
  for (int x = 0; x < kX; ++x)
#pragma unroll
    for (int h = 0; h < 2; ++h) qb[x][h] = __builtin_bit_cast(f16x8, load16(q + h * (D / 2) + 8 * (4 * x + rho)));
#pragma unroll
  for (int b = 0; b < kDepth; ++b) issue(codes[b], b);
#pragma unroll
  for (int x = 0; x < kX; ++x)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (c >= G) qb[x][h] = f16x8{0, 0, 0, 0, 0, 0, 0, 0};
  ksl *= p.scale * kLog2e;
  auto step = [&](StepCodes<D>& s, int st, bool tail) {
    f32x4 acc[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < kX; ++x)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f16x4 lo = codes_to_f16<kFp8>(s.k[t][x][2 * h]), hi = codes_to_f16<kFp8>(s.k[t][x][2 * h + 1]);
          const f16x8 av = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
          acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, qb[x][h], acc[t], 0, 0, 0);
        }
    }
    // this lane: tokens 4 rho + i of both tiles, head c
    const int t1 = min(2 * st + 1, tiles - 1);
    const float ks[2] = {lane_value(ksl, 2 * st), lane_value(ksl, t1)};
    const float vs[2] = {lane_value(vsl, 2 * st), lane_value(vsl, t1)};
    const float vl[2] = {lane_value(vll, 2 * st), lane_value(vll, t1)};
    float e[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) e[t][i] = acc[t][i] * ks[t];
    if (tail) {  // uniform
      const int left = count - st * kStep;  // keys of this step
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (16 * t + 4 * rho + i >= left) e[t][i] = -FLT_MAX;
        // bytes of tokens past the context may be anything (an e4m3 NaN too)
        const int keep = min(max(left - 16 * t - 4 * rho, 0), 4);
        const uint32_t mask = keep == 0 ? 0u : 0xffffffffu >> (32 - 8 * keep);
#pragma unroll
        for (int x = 0; x < kX; ++x) s.v[t][x] &= u32x4{mask, mask, mask, mask};
      }
    }
    float mx = fmaxf(fmaxf(fmaxf(e[0][0], e[0][1]), fmaxf(e[0][2], e[0][3])) + vl[0],
                     fmaxf(fmaxf(e[1][0], e[1][1]), fmaxf(e[1][2], e[1][3])) + vl[1]);
    mx = rows_max<true>(rows_max<false>(mx));
    // m is a reference within 2^8 of the maximum: moving it costs a pass over the
    // output, and p s up to 2^8 fits fp16 as well as p s up to 1 does
    if (__any(mx > w.m + 8.f)) {
      const float mn = fmaxf(w.m, mx), f = __builtin_amdgcn_exp2f(w.m - mn);
      w.l *= f;
#pragma unroll
      for (int d = 0; d < E; ++d) w.o[d] *= f;
      w.m = mn;
    }
    f16x8 b;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float pr = __builtin_amdgcn_exp2f(e[t][i] - w.m);
        w.l += pr;
        b[4 * t + i] = static_cast<_Float16>(pr * vs[t]);
      }
#pragma unroll
    for (int x = 0; x < kX; ++x)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f16x4 lo = codes_to_f16<kFp8>(s.v[0][x][j]), hi = codes_to_f16<kFp8>(s.v[1][x][j]);
        const f16x8 av = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        w.o[4 * x + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, b, w.o[4 * x + j], 0, 0, 0);
      }
  };
  int st = 0;
  for (; st + kDepth < steps; st += kDepth) {
#pragma unroll
    for (int b = 0; b < kDepth; ++b) {
      step(codes[b], st + b, false);
      issue(codes[b], st + b + kDepth);
    }
  }
#pragma unroll
  for (int b = 0; b < kDepth; ++b)
    if (st + b < steps) step(codes[b], st + b, (st + b + 1) * kStep > count);
}

// An item's output row of one head, or its partial in a slot of the workspace.
// The last slot of an item is followed by the sum -1, which no sum of
// exponentials takes; the rows of an item written whole have it in slot 0.
__device__ __forceinline__ int64_t slot_row(const DecodeArgs& a, int item, int head) {
  return (static_cast<int64_t>(item) * a.p.num_heads + head) * a.w.max_partitions;
}
__device__ __forceinline__ _Float16* out_row(const DecodeArgs& a, int token, int head, int D) {
  return reinterpret_cast<_Float16*>(a.p.out) + (static_cast<int64_t>(token) * a.p.num_heads + head) * D;
}
__device__ __forceinline__ void mark_whole(const DecodeArgs& a, int item, int head) {
  if (a.w.max_partitions > 1) a.w.ws_sum[slot_row(a, item, head)] = -1.f;
}

// The rows of an item that attends to nothing, for one kv head.
template <int D, int G>
__device__ __forceinline__ void attend_nothing(const DecodeArgs& a, int item, int token, int kvh) {
  for (int i = threadIdx.x; i < G * D; i += blockDim.x) {
    out_row(a, token, kvh * G, D)[i] = static_cast<_Float16>(0.f);
    if (i % D == 0) mark_whole(a, item, kvh * G + i / D);
  }
}

// Grid form: one workgroup per (group_tokens keys, kv head, item), whose waves
// split the keys and meet in LDS.
template <int D, int G, bool kFp8>
__global__ __launch_bounds__(kThreads, 2) void decode_blocks_grid_kernel(DecodeArgs a) {
  struct Lds {
    float o[kWaves][G][D + 4];  // padded: heads of one dim in different banks
    float m[kWaves][G], l[kWaves][G];
  };
  __shared__ alignas(16) Lds s;
  const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int slot = blockIdx.x, kvh = blockIdx.y, item = blockIdx.z;
  const int token = a.w.item_token[item];
  if (token < 0) return;
  const int wave_tokens = a.group_tokens / kWaves, first = slot * a.group_tokens + wave * wave_tokens;
  const int blk = table_entries(a, a.w.item_seq[item], first / kTileTokens);
  const int n = keys_of(a, token);
  if (slot * a.group_tokens >= n) {
    if (slot == 0) attend_nothing<D, G>(a, item, token, kvh);
    return;
  }
  WaveState<D> w;
  if (first < n) attend<D, G, kFp8, 2>(a, w, token, kvh, first / kTileTokens, min(wave_tokens, n - first), blk);
  w.finish();
  const int c = lane % 16;
  if (c < G) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = 0; d < D / 16; d += 4)
        *reinterpret_cast<f32x4*>(&s.o[wave][c][w.dim(d, i)]) =
            f32x4{w.o[d][i], w.o[d + 1][i], w.o[d + 2][i], w.o[d + 3][i]};
    if (lane < 16) {
      s.m[wave][c] = w.m;
      s.l[wave][c] = w.l;
    }
  }
  __syncthreads();
  const bool whole = n <= a.group_tokens, last = (slot + 1) * a.group_tokens >= n;
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
      out_row(a, token, kvh * G, D)[i] = static_cast<_Float16>(acc / L);
      if (d == 0) mark_whole(a, item, kvh * G + g);
    } else {
      const int64_t row = slot_row(a, item, kvh * G + g) + slot;
      a.w.ws_out[row * D + d] = acc;
      if (d == 0) {
        a.w.ws_max[row] = M;
        a.w.ws_sum[row] = L;
        if (last && slot + 1 < a.w.max_partitions) a.w.ws_sum[row + 1] = -1.f;
      }
    }
  }
}

// Range form: the steps of all (item, kv head) pairs in one row, cut into equal
// ranges, one a wave, each with its own partial: no wave waits for another and
// none has more to do, whatever the contexts are.  Every workgroup sums the
// items' steps itself.
template <int D, int G, bool kFp8>
__global__ __launch_bounds__(kThreads, 2) void decode_blocks_range_kernel(DecodeArgs a) {
  __shared__ int it_token[kMaxItemsLds], it_seq[kMaxItemsLds], it_keys[kMaxItemsLds];
  __shared__ int it_before[kMaxItemsLds + 1];  // steps before item i, of one kv head
  __shared__ int wave_tot[kWaves];
  const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int items = a.w.num_items, hkv = a.p.kv.num_kv_heads;
  const int per = (items + kThreads - 1) / kThreads;
  const int i0 = min(tid * per, items), i1 = min(i0 + per, items);
  int sum = 0;
  for (int i = i0; i < i1; ++i) {
    const int token = a.w.item_token[i];
    it_seq[i] = a.w.item_seq[i];
    const int n = token < 0 ? 0 : keys_of(a, token);
    it_token[i] = token;
    it_keys[i] = n;
    sum += (n + kStep - 1) / kStep;
  }
  int incl = sum;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int v = __shfl_up(incl, o, kWave);
    if (lane >= o) incl += v;
  }
  if (lane == kWave - 1) wave_tot[wave] = incl;
  __syncthreads();
  int before = incl - sum;
  for (int v = 0; v < wave; ++v) before += wave_tot[v];
  for (int i = i0; i < i1; ++i) {
    it_before[i] = before;
    before += (it_keys[i] + kStep - 1) / kStep;
  }
  if (tid == kThreads - 1) it_before[items] = before;
  __syncthreads();
  for (int i = blockIdx.x; i < items; i += gridDim.x) {  // (uniform: rarely anything to do)
    if (it_keys[i] > 0) continue;
    const int token = it_token[i];
    if (token >= 0)
      for (int h = 0; h < hkv; ++h) attend_nothing<D, G>(a, i, token, h);
  }
  // (steps fit 31 bits: the launch rule sees to that)
  const int total = __builtin_amdgcn_readfirstlane(it_before[items]) * hkv;
  const int range = min(max((total + a.ranges - 1) / a.ranges, kMinRange), kMaxRange);
  const int r = blockIdx.x * kWaves + wave;
  if (r > total / range) return;
  int u = r * range;
  const int end = min(u + range, total);
  if (u >= end) return;
  int lo = 0, hi = items - 1;  // the last item that starts at or before u (the others there are empty)
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (it_before[mid] * hkv <= u) lo = mid; else hi = mid - 1;
  }
  int item = __builtin_amdgcn_readfirstlane(lo);
  while (u < end) {
    const int n = __builtin_amdgcn_readfirstlane(it_keys[item]), steps = (n + kStep - 1) / kStep;
    if (steps == 0) {
      ++item;
      continue;
    }
    const int item0 = __builtin_amdgcn_readfirstlane(it_before[item]) * hkv;
    const int kvh = (u - item0) / steps;
    const int seg = item0 + kvh * steps;  // where this (item, kv head) starts
    const int at = u - seg, todo = min(end - u, steps - at);
    const int token = __builtin_amdgcn_readfirstlane(it_token[item]), tile0 = 2 * at;
    WaveState<D> w;
    attend<D, G, kFp8, kDepth>(a, w, token, kvh, tile0, min(todo * kStep, n - at * kStep),
                          table_entries(a, __builtin_amdgcn_readfirstlane(it_seq[item]), tile0));
    w.finish();
    const int c = lane % 16;
    if (c < G) {
      const int head = kvh * G + c;
      if (todo == steps) {
        const float inv = 1.f / w.l;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          _Float16* o = out_row(a, token, head, D) + w.dim(0, i);
#pragma unroll
          for (int d = 0; d < D / 16; ++d) o[d] = static_cast<_Float16>(w.o[d][i] * inv);
        }
        if (lane < 16) mark_whole(a, item, head);
      } else {
        const int slot = r - seg / range;
        const int64_t row = slot_row(a, item, head) + slot;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float* o = a.w.ws_out + row * D + w.dim(0, i);
#pragma unroll
          for (int d = 0; d < D / 16; d += 4)
            *reinterpret_cast<f32x4*>(o + d) = f32x4{w.o[d][i], w.o[d + 1][i], w.o[d + 2][i], w.o[d + 3][i]};
        }
        if (lane < 16) {
          a.w.ws_max[row] = w.m;
          a.w.ws_sum[row] = w.l;
          if (at + todo == steps && slot + 1 < a.w.max_partitions) a.w.ws_sum[row + 1] = -1.f;
        }
      }
    }
    u += todo;
    if (at + todo == steps && kvh == hkv - 1) ++item;
  }
}

// Joins the partials of one (item, head): lane d of the workgroup takes dim d.
// Each wave holds the weights of 64 slots, one a lane, and hands them to the
// rows' sums.
template <int D>
__global__ __launch_bounds__(D) void merge_blocks_kernel(DecodeArgs a) {
  constexpr int kUnroll = 16;
  const int item = blockIdx.x, h = blockIdx.y, d = threadIdx.x, lane = d % kWave;
  const int mp = a.w.max_partitions;
  const int64_t row = slot_row(a, item, h);
  const float* src = a.w.ws_out + row * D + d;
  const int token = a.w.item_token[item];
  float M = -FLT_MAX, L = 0.f, o = 0.f;
  for (int s0 = 0; s0 < mp; s0 += kWave) {
    const int at = min(s0 + lane, mp - 1);
    const float ls = a.w.ws_sum[row + at], m0 = a.w.ws_max[row + at];
    // the first rows are requested before the number of slots is known (slots
    // that are not the item's hold anything and are not used)
    float v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) v[u] = src[static_cast<int64_t>(min(s0 + u, mp - 1)) * D];
    // slots up to the one marked -1 (or all)
    const uint64_t stop = __ballot(s0 + lane >= mp || ls < 0.f);
    const int here = stop != 0 ? __builtin_ctzll(stop) : kWave;
    if (token < 0 || (here == 0 && s0 == 0)) return;  // skipped, or written whole
    if (here == 0) break;
    const float ms = lane < here ? m0 : -FLT_MAX;
    const float mn = fmaxf(M, rows_max<true>(rows_max<false>(group_max<16>(ms))));
    const float f0 = __builtin_amdgcn_exp2f(M - mn), f = __builtin_amdgcn_exp2f(ms - mn);
    L = L * f0 + wave_sum(lane < here ? f * ls : 0.f);
    o *= f0;
    M = mn;
    for (int s = 0; s < here; s += kUnroll) {
      float next[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        next[u] = src[static_cast<int64_t>(s0 + min(s + kUnroll + u, here - 1)) * D];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (s + u < here) o += lane_value(f, s + u) * v[u];
        v[u] = next[u];
      }
    }
    if (here < kWave) break;
  }
  out_row(a, token, h, D)[d] = static_cast<_Float16>(o / L);
}

template <int D, int G, bool kFp8>
void launch_g(DecodeArgs a, hipStream_t stream) {
  const int mp = a.w.max_partitions;
  const int64_t units = static_cast<int64_t>(a.w.num_items) * a.p.kv.num_kv_heads * mp;
  const int cus = compute_units();
  bool merge;
  // RLK_TUNE_BLK_DECODE forces a form where it can serve the call (0 grid, 1
  // range; tests and tuning runs)
  // Equal ranges pay where contexts are several ranges long and fill the chip;
  // they cost a longer start, and more where a range holds several short contexts.
  // us, grid / range (8 kv heads of 128, contexts from 0 to the named one): 8 items
  // to 8191 20.1 / 20.0, 16 35.5 / 27.7, 32 59 / 49; 32 to 4000 33.1 / 27.0; 32 to
  // 2000 19.7 / 24.0, 64 31.6 / 30.5; 128 to 1000 29.7 / 36.2; 256 to 500 27.4 / 44.5
  // (the merge's 5-7 us, which the grid form does without there, come on top).
  const bool range = mp >= 8 && units > static_cast<int64_t>(cus) * 8;
  if (tune_knob(kBlkDecode, range) != 0 && a.w.num_items <= kMaxItemsLds && mp > 1 &&
      units * (kPart / kStep) < (1 << 30)) {
    a.ranges = kWavesPerCu * cus;
    const int64_t most = std::max<int64_t>(a.ranges, (units * (kPart / kStep) + kMaxRange - 1) / kMaxRange);
    decode_blocks_range_kernel<D, G, kFp8>
        <<<static_cast<uint32_t>((most + kWaves - 1) / kWaves), kThreads, 0, stream>>>(a);
    merge = true;
  } else {
    // as many slots as fill the chip with 4 workgroups a CU, of at most 4096 keys
    const int64_t pairs = static_cast<int64_t>(a.w.num_items) * a.p.kv.num_kv_heads;
    const int want = static_cast<int>(std::min<int64_t>(mp, (cus * 4 + pairs - 1) / pairs));
    constexpr int kUnit = kWaves * kStep;
    a.group_tokens = std::min((mp * kPart / want + kUnit - 1) / kUnit * kUnit, 1024 * kWaves);
    const int slots = (mp * kPart + a.group_tokens - 1) / a.group_tokens;
    const dim3 grid(slots, a.p.kv.num_kv_heads, a.w.num_items);
    decode_blocks_grid_kernel<D, G, kFp8><<<grid, kThreads, 0, stream>>>(a);
    merge = slots > 1;
  }
  if (merge) merge_blocks_kernel<D><<<dim3(a.w.num_items, a.p.num_heads), D, 0, stream>>>(a);
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
  const DecodeArgs a = {*p, *w, 0, 0};
  const int G = p->num_heads / p->kv.num_kv_heads;
  const bool fp8 = p->kv.format == RLK_KV_BLOCK_FP8;
  const bool ok = p->kv.head_dim == 128
                      ? (fp8 ? launch_d<128, true>(a, G, stream) : launch_d<128, false>(a, G, stream))
                      : (fp8 ? launch_d<64, true>(a, G, stream) : launch_d<64, false>(a, G, stream));
  if (!ok) return fail(RLK_EUNSUPPORTED, "%s: unsupported GQA group size %d", what, G);
  return launch_status(what);
}
