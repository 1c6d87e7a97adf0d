// Paged prefill attention over the block-scaled 8-bit cache, for gfx950.
//
// Causal attention of a sequence's new tokens over its cached and new keys.
// Rows are (token, query head) pairs of one kv head, head fastest, so K and V
// are read and converted once for the G heads of the group; a wave takes 32
// rows and walks the keys in tiles of 64.
//   * Codes go to registers a tile ahead, become fp16 (exactly) and are written
//     to LDS images in the operand order of v_mfma_f32_32x32x16_f16: K as
//     16-byte chunks [piece][half][key], V as [16-key tile][lane half][dim], each
//     chunk the 8 keys of a lane's own scores; both are read as whole contiguous
//     rows (no bank conflicts), and neither operand is transposed or exchanged
//     anywhere.
//   * S^T = K Q^T leaves one query row per lane (its keys split over the two lane
//     halves), so the running maximum and sum are lane-local, and the scores are
//     the B operand of O^T = V^T P^T as they stand.
//   * A tile is two phases, a matrix phase X (P.V of the tile before, K.Q of this
//     one, then the conversion of K) and a vector phase Y (softmax, conversion of V; at
//     D = 64 V is converted in X too).  At D = 128 X takes some 1400 + 260 clocks and Y
//     1800; with all conversion in Y it was 1350 and 2060, 4 x 4096 tokens 1390 us
//     against 1313.  A workgroup has one or two groups of 4 waves; two groups are half a
//     tile apart, so that of the two waves of a SIMD one has the matrix cores while the
//     other has the vector ALU.  The groups take
//       kRows2   256 rows, the same tiles (one image for both): large calls, D = 128;
//       kOne     one group, three workgroups to a CU: large calls, D = 64;
//       kKeys2   the same 128 rows, even and odd tiles (an image each), and join
//                their partials at the end: calls that do not fill the chip.
// m, l and the output accumulate in fp32; P is rounded to fp16 (at most 2^8), and
// l sums the rounded values, so that numerator and denominator agree.
// Bound: long prompts by X and Y in turn at the clock that the chip holds under them
// (about 1.8 GHz of 2.4): 4 x 4096 tokens at depths to 4096, 32 / 8 heads of 128, take
// 1275-1330 us INT8 (by run) and 1275 e4m3, 1.0-1.05 PFLOP/s or 83-86% of a large library
// product; 4 x 4096 at D = 64 699 us.  Short ones by the longest workgroup's chain of tiles: 2 chunks of
// 512 tokens at depths 0 and 1585 41 us, 24 ragged prompts at D = 64 92 us (560 TFLOP/s).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cstdint>
#include <type_traits>

#include "kv_blocks.hpp"

namespace rlk {

int check_block_params(const rlk_block_attention_params* p, const char* what);

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kGroupThreads = 256;  // a group: 4 waves, one per SIMD
constexpr int kWaveRows = 32;       // (token, head) rows of a wave
constexpr int kTileKeys = 64;

struct PrefillArgs {
  rlk_block_attention_params p;
  rlk_prefill_attention_work w;
  int group;  // query heads per kv head
};

// What no kernel writes while this one reads it, for scalar loads at uniform
// addresses.
template <class T>
using ScalarPtr = const __attribute__((address_space(4))) T*;
template <class T>
__device__ __forceinline__ ScalarPtr<T> scalar(const T* p) {
  return (ScalarPtr<T>)(p);
}

// Four codes as fp16, exactly: e4m3 times the scale (the conversion takes it),
// INT8 V times the scale, INT8 K as it is (its scale multiplies the scores).
__device__ __forceinline__ u32x2 fp8_scaled_f16(uint32_t w, float s) {
  const f16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, false);
  const f16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, true);
  return u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
}
__device__ __forceinline__ u32x2 int8_scaled_f16(uint32_t w, _Float16 s) {
  return __builtin_bit_cast(u32x2, codes_to_f16<false>(w) * s);
}

// Two images of K and of V, used in turn, and the score scale of each 16-key tile
// of the last 4 key tiles (INT8).
template <int D>
struct PrefillLds {
  u32x4 k[2][D / 16][2][kTileKeys];  // chunk (piece, half, key): 8 dims
  u32x4 v[2][4][2][D];               // chunk (16-key tile, lane half, dim index): 8 keys
  f32x4 ks[4];
};

enum Split { kOne, kRows2, kKeys2 };

// Phases, with t the key tile (kKeys2: the group's t-th) and S its scores; group 1
// is one phase behind.  kRows2:
//   group 0   X(t) at 2t, converts its half of K(t + 1)      Y(t) at 2t + 1, of V(t)
//   group 1   X(t) at 2t + 1, converts its half of K(t + 1)  Y(t) at 2t + 2, of V(t + 1)
// X(t) reads K(t) and V(t - 1).  So K(t) is written in the phases 2t - 2 and
// 2t - 1 and read in 2t and 2t + 1, V(t) is written in 2t and 2t + 1 and read in
// 2t + 2 and 2t + 3, and neither meets the image of tile t - 2 in the same buffer.
// Alone or with its own image a group does as group 0, with whole tiles.
template <int D, bool kFp8, Split kSplit>
__global__ __launch_bounds__(kGroupThreads * (kSplit == kOne ? 1 : 2), 2) void prefill_blocks_kernel(PrefillArgs a) {
  constexpr int kGroups = kSplit == kRows2 ? 2 : 1;  // that share a tile's image
  constexpr bool kKeys = kSplit == kKeys2;
  // where V is converted: beside K in X, or (at D = 128) in Y, for phases of one length
  constexpr bool kVInX = D == 64;
  constexpr int E = D / 16, kRows = 4 * kWaveRows * kGroups;
  constexpr int kPerTile = D;                                  // 16-byte pieces of a layout tile
  constexpr int kItems = 2 * 4 * kPerTile / kGroups / kGroupThreads;  // K and V pieces of a thread and tile
  constexpr float kLog2e = 1.4426950408889634f;
  extern __shared__ u32x4 lds_raw[];
  const rlk_block_attention_params& p = a.p;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int tid = threadIdx.x % kGroupThreads, grp = wave / 4;
  const int rgrp = kKeys ? 0 : grp, kgrp = kKeys ? grp : 0;  // the group's part of the rows, of the tiles
  PrefillLds<D>& lds = reinterpret_cast<PrefillLds<D>*>(lds_raw)[kgrp];
  const int half = lane / 32, col = lane % 32;
  const int kvh = blockIdx.x, G = a.group;
  const int seq = a.w.seq_ids[blockIdx.z];
  if (seq < 0) return;
  const int q_len = a.w.q_len[seq], rows = q_len * G;
  // the rows with the most keys first
  const int row0 = (gridDim.y - 1 - blockIdx.y) * kRows;
  if (row0 >= rows) return;
  const int past = a.w.ctx_len[seq] - q_len, q_start = a.w.q_start[seq];
  const int tsh = p.kv.block_size == 32 ? 1 : 0, hkv = p.kv.num_kv_heads;  // log2 tiles of a block
  const int most = static_cast<int>(min(static_cast<int64_t>(p.max_blocks_per_seq) * p.kv.block_size,
                                        static_cast<int64_t>(1 << 30)));
  // keys of the workgroup's last row; those of each lane's row
  const int last_row = min(row0 + kRows, rows) - 1;
  const int keys = min(past + last_row / G + 1, most);
  const int wrow = row0 + (rgrp * 4 + wave % 4) * kWaveRows;  // the wave's first row
  const int row = min(wrow + col, rows - 1);  // rows past the end repeat the last one
  const int tok = row / G, head = kvh * G + row - tok * G;
  const int row_keys = min(past + tok + 1, most);
  const int full = min(past + min(wrow, rows - 1) / G + 1, most);  // keys that every row of the wave sees

  const _Float16* q = reinterpret_cast<const _Float16*>(p.q) + static_cast<int64_t>(q_start + tok) * p.q_stride + head * D;
  f16x8 qb[E];
#pragma unroll
  for (int pc = 0; pc < E; ++pc) {
    qb[pc] = __builtin_bit_cast(f16x8, load16(q + half * (D / 2) + 8 * pc));
    if (p.scale < 0.f) qb[pc] = -qb[pc];  // the maximum is taken before the scale
  }

  // Item j of a thread: 16-byte piece (tid + 256 j') of its group's part of a K or
  // V tile, the K pieces first; all lanes of a wave are in one layout tile, so that
  // its block, scale and address are scalar.  Tiles past the last repeat its last
  // 16 keys.
  static_assert(kItems % 2 == 0, "an item is K or V for the whole group");
  constexpr int kHalf = kItems * kGroupThreads / 2;  // K pieces of a group's part
  static_assert(kPerTile % kWave == 0, "a wave's pieces lie in one layout tile");
  struct Item {
    u32x4 codes;
    float scale;
  };
  Item item[kItems];
  int id[kItems];
  const int wave0 = wave % 4 * kWave;  // tid of the wave's first lane
  const ScalarPtr<int32_t> table = scalar(p.block_tables + static_cast<int64_t>(seq) * p.max_blocks_per_seq);
  // tiles of a group (kKeys2: its last may lie behind the keys; all of it is masked)
  const int all_tiles = (keys + kTileKeys - 1) / kTileKeys, tiles = kKeys ? (all_tiles + 1) / 2 : all_tiles;
  auto real = [&](int t) { return kKeys ? 2 * t + kgrp : t; };
  const int last16 = (max(keys, 1) - 1) / kTileTokens;
  auto is_v = [&](int j) { return j >= kItems / 2; };
  // first piece of the wave in the group's part; this lane's in its layout tile
  auto wave_piece = [&](int j) { return (j * kGroupThreads + wave0) % kHalf; };
  auto piece = [&](int j) { return wave_piece(j) % kPerTile + lane; };
  auto part16 = [&](int j) { return rgrp * (4 / kGroups) + wave_piece(j) / kPerTile; };  // 16-key tile of the key tile
  auto layout_tile = [&](int j, int t) { return min(4 * real(t) + part16(j), last16); };
  // block of item j for conversion c (K of tile c + 1, V of tile c)
  auto entry = [&](int j, int c) { return table[layout_tile(j, is_v(j) ? c : c + 1) >> tsh]; };
  // cell (block, head) of item j for conversion c, from its block id[j]; its codes
  auto cell_of = [&](int j) __attribute__((always_inline)) {
    const int b = static_cast<uint32_t>(id[j]) < static_cast<uint32_t>(p.kv.num_blocks) ? id[j] : 0;
    return static_cast<uint32_t>(b) * hkv + kvh;
  };
  auto fetch = [&](int j, int c, uint32_t cell) __attribute__((always_inline)) {
    const uint32_t tile = (cell << tsh) + (layout_tile(j, is_v(j) ? c : c + 1) & tsh);
    const uint8_t* base = static_cast<const uint8_t*>(is_v(j) ? p.kv.v : p.kv.k) +
                          static_cast<uint64_t>(tile) * (kTileTokens * D) + wave_piece(j) % kPerTile * 16;
    item[j].codes = reinterpret_cast<const u32x4*>(base)[lane];
  };
  auto scale_of = [&](int j, uint32_t cell) { return scalar(is_v(j) ? p.kv.v_scale : p.kv.k_scale)[cell]; };
  const float cs = __builtin_fabsf(p.scale) * kLog2e;
  // Conversion c of item j: the codes as fp16, and their way to the image.
  struct Halves {
    u32x2 x[4];
  };
  auto convert = [&](int j, int c) __attribute__((always_inline)) {
    Halves h;
    u32x4 w = item[j].codes;
    if (!is_v(j)) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        h.x[e] = kFp8 ? fp8_scaled_f16(w[e], item[j].scale) : __builtin_bit_cast(u32x2, codes_to_f16<kFp8>(w[e]));
    } else {
      if ((real(c) + 1) * kTileKeys > keys) {  // uniform: bytes past the keys may be anything
        const int keep = min(max(keys - real(c) * kTileKeys - 16 * part16(j) - 4 * (piece(j) / 16 % 4), 0), 4);
        const uint32_t mask = keep == 0 ? 0u : 0xffffffffu >> (32 - 8 * keep);
        w &= u32x4{mask, mask, mask, mask};
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        h.x[e] = kFp8 ? fp8_scaled_f16(w[e], item[j].scale)
                      : int8_scaled_f16(w[e], static_cast<_Float16>(item[j].scale));
    }
    return h;
  };
  auto store = [&](int j, int c, const Halves& h) __attribute__((always_inline)) {
    const int t16 = part16(j), pc = piece(j);
    if (!is_v(j)) {
      const int buf = (c + 1) & 1, kp = pc / 16, key = 16 * t16 + pc % 16;
      lds.k[buf][kp][0][key] = u32x4{h.x[0][0], h.x[0][1], h.x[1][0], h.x[1][1]};
      lds.k[buf][kp][1][key] = u32x4{h.x[2][0], h.x[2][1], h.x[3][0], h.x[3][1]};
      // (the same word and value from each lane)
      if (!kFp8) reinterpret_cast<float*>(&lds.ks[(c + 1) & 3])[t16] = item[j].scale * cs;
    } else {
      const int g = pc / 64, rho = pc / 16 % 4, m = pc % 16;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        reinterpret_cast<u32x2*>(&lds.v[c & 1][t16][rho % 2][(4 * g + e) * 16 + m])[rho / 2] = h.x[e];
    }
  };

  f32x16 o[D / 32], s[2];
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  f16x8 pb[4];
  // (below every score of fp16 rows, and far above a masked one)
  float m = -1e30f, l = 0.f;

  // Operands come from LDS kAhead fragments before their product; the schedule is
  // pinned, because the compiler by itself waits for each pair of reads.
  // After the products come K's part of conversion t, the request of the next codes, and
  // the cells of the next scales.
  uint32_t cell[kItems];
  auto convert_x = [&](int t) __attribute__((always_inline)) {
    constexpr int kEnd = kVInX ? kItems : kItems / 2;
    Halves h[kEnd];
#pragma unroll
    for (int j = 0; j < kEnd; ++j) {
      h[j] = convert(j, t);
      cell[j] = cell_of(j);
      fetch(j, t + 1, cell[j]);
    }
#pragma unroll
    for (int j = 0; j < kEnd; ++j) store(j, t, h[j]);
#pragma unroll
    for (int j = kEnd; j < kItems; ++j) cell[j] = cell_of(j);
    __builtin_amdgcn_sched_barrier(0);
  };
  // V's part of conversion c
  auto convert_v = [&](int c) __attribute__((always_inline)) {
#pragma unroll
    for (int j = kItems / 2; j < kItems; ++j) {
      const Halves h = convert(j, c);
      fetch(j, c + 1, cell[j]);
      store(j, c, h);
    }
  };
  auto phase_x = [&](int t, auto pv, auto qk) __attribute__((always_inline)) {
    constexpr int kPv = decltype(pv)::value ? 4 * (D / 32) : 0, kQk = decltype(qk)::value ? 2 * E : 0;
    constexpr int kAll = kPv + kQk, kAhead = kAll < 8 ? kAll : 8;
    __builtin_amdgcn_sched_barrier(0);
    const u32x4* vp = &lds.v[(t + 1) & 1][0][half][col];  // V of tile t - 1
    const u32x4* kp = &lds.k[t & 1][0][half][col];
    auto fragment = [&](int i) {
      return i < kPv ? vp[(i / (D / 32)) * 2 * D + 32 * (i % (D / 32))]
                     : kp[((i - kPv) / 2) * 2 * kTileKeys + 32 * ((i - kPv) % 2)];
    };
    u32x4 f[kAll];
#pragma unroll
    for (int i = 0; i < kAll; ++i) f[i] = fragment(i);
    if constexpr (kQk > 0) {
#pragma unroll
      for (int kh = 0; kh < 2; ++kh)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kh][i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < kAll; ++i) {
      const f16x8 x = __builtin_bit_cast(f16x8, f[i]);
      if (i < kPv) {
        const int d = i % (D / 32);
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, pb[i / (D / 32)], o[d], 0, 0, 0);
      } else {
        const int kh = (i - kPv) % 2;
        s[kh] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, qb[(i - kPv) / 2], s[kh], 0, 0, 0);
      }
    }
    __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);  // LDS reads
#pragma unroll
    for (int i = 0; i < kAll - kAhead; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);  // a product
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, kAhead, 0);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (kQk > 0) convert_x(t);
  };
  auto softmax = [&](int t) __attribute__((always_inline)) {
    // element i of half kh: key 64 real(t) + 32 kh + 8 (i / 4) + 4 half + i % 4
    f32x4 c4 = kFp8 ? f32x4{cs, cs, cs, cs} : lds.ks[t & 3];  // score scale of each 16 keys
    float mx;
    const int first_key = real(t) * kTileKeys;
    if (first_key + kTileKeys > full) {  // uniform over the wave: scaled, then masked
#pragma unroll
      for (int kh = 0; kh < 2; ++kh)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float v = s[kh][i] * c4[2 * kh + i / 8];
          s[kh][i] = first_key + 32 * kh + 8 * (i / 4) + 4 * half + i % 4 < row_keys ? v : -FLT_MAX;
        }
      c4 = f32x4{1.f, 1.f, 1.f, 1.f};
    }
    // (the scales are not negative, so the largest score of 16 keys is scaled once)
    mx = -FLT_MAX;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      float y = -FLT_MAX;
#pragma unroll
      for (int i = 0; i < 8; ++i) y = fmaxf(y, s[x / 2][8 * (x % 2) + i]);
      mx = fmaxf(mx, y * c4[x]);
    }
    mx = rows_max<true>(mx);
    // m is a reference within 2^8 of the maximum: moving it costs a pass over the
    // output, and p up to 2^8 fits fp16 as well as p up to 1 does
    if (__any(mx > m + 8.f)) {
      const float mn = fmaxf(m, mx), f = __builtin_amdgcn_exp2f(m - mn);
      l *= f;
#pragma unroll
      for (int d = 0; d < D / 32; ++d) o[d] *= f;
      m = mn;
    }
    // scalar loads for the next conversions, waited for at the end of the phase
    float next_scale[kItems];
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      next_scale[j] = scale_of(j, cell[j]);
      id[j] = entry(j, (is_v(j) ? t + rgrp : t) + 2);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (!kVInX) convert_v(t + rgrp);
#pragma unroll
    for (int j = 0; j < kItems; ++j) item[j].scale = next_scale[j];
    float ls[4] = {l, 0.f, 0.f, 0.f};
    const f16x2 ones = {static_cast<_Float16>(1), static_cast<_Float16>(1)};
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float e0 = __builtin_amdgcn_exp2f(fmaf(s[x / 2][8 * (x % 2) + i], c4[x], -m));
        const float e1 = __builtin_amdgcn_exp2f(fmaf(s[x / 2][8 * (x % 2) + i + 1], c4[x], -m));
        const f16x2 e = {static_cast<_Float16>(e0), static_cast<_Float16>(e1)};
        pb[x][i] = e[0];
        pb[x][i + 1] = e[1];
        ls[x] = __builtin_amdgcn_fdot2(e, ones, ls[x], false);
      }
    l = (ls[0] + ls[1]) + (ls[2] + ls[3]);
  };

  if (tiles > 0) {
    // conversion -1 has K(0) only: there is no V tile -1
    auto read = [&](int j, int c) __attribute__((always_inline)) {
      id[j] = entry(j, c);
      cell[j] = cell_of(j);
      fetch(j, c, cell[j]);
      item[j].scale = scale_of(j, cell[j]);
    };
#pragma unroll
    for (int j = 0; j < kItems; ++j)
      if (!is_v(j) || rgrp == 1) read(j, is_v(j) ? 0 : -1);
#pragma unroll
    for (int j = 0; j < kItems; ++j)
      if (!is_v(j) || rgrp == 1) store(j, is_v(j) ? 0 : -1, convert(j, is_v(j) ? 0 : -1));
#pragma unroll
    for (int j = 0; j < kItems; ++j) read(j, is_v(j) ? rgrp : 0);
#pragma unroll
    for (int j = 0; j < kItems; ++j) id[j] = entry(j, (is_v(j) ? rgrp : 0) + 1);
  }
  __syncthreads();
  if (grp == 1) __syncthreads();  // one phase behind
  auto phase_y = [&](int t) __attribute__((always_inline)) {
    __syncthreads();
    softmax(t);
    __syncthreads();
  };
  if (tiles > 0) {
    phase_x(0, std::false_type{}, std::true_type{});
    phase_y(0);
    for (int t = 1; t < tiles; ++t) {
      phase_x(t, std::true_type{}, std::true_type{});
      phase_y(t);
    }
    phase_x(tiles, std::true_type{}, std::false_type{});
  }
  if (kSplit != kOne && grp == 0) __syncthreads();  // as many barriers as group 1
  l = rows_sum<true>(l);
  if constexpr (kKeys) {  // group 1's partial joins group 0's through LDS
    __syncthreads();      // the images have been read
    struct Partial {
      float o[D / 2][kGroupThreads], m[kGroupThreads], l[kGroupThreads];
    };
    static_assert(sizeof(Partial) <= 2 * sizeof(PrefillLds<D>), "fits where the images were");
    Partial& part = *reinterpret_cast<Partial*>(lds_raw);
    if (grp == 1) {
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) part.o[16 * d + i][tid] = o[d][i];
      part.m[tid] = m;
      part.l[tid] = l;
    }
    __syncthreads();
    if (grp == 1) return;
    const float m1 = part.m[tid], mn = fmaxf(m, m1);
    const float f0 = __builtin_amdgcn_exp2f(m - mn), f1 = __builtin_amdgcn_exp2f(m1 - mn);
    l = l * f0 + part.l[tid] * f1;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = o[d][i] * f0 + part.o[16 * d + i][tid] * f1;
  }
  if (wrow + col >= rows) return;  // no barrier follows
  const float inv = l > 0.f ? 1.f / l : 0.f;
  _Float16* out = reinterpret_cast<_Float16*>(p.out) + (static_cast<int64_t>(q_start + tok) * p.num_heads + head) * D;
  // element i of tile d: dim index 32 d + 8 (i / 4) + 4 half + i % 4 = 16 dt + mm, i.e. dim E mm + dt
#pragma unroll
  for (int j = 0; j < 8; ++j) {  // mm = 8 (j / 4) + 4 half + j % 4
    _Float16 y[E];
#pragma unroll
    for (int dt = 0; dt < E; ++dt) y[dt] = static_cast<_Float16>(o[dt / 2][8 * (dt % 2) + j] * inv);
    const int mm = 8 * (j / 4) + 4 * half + j % 4;
    if constexpr (E == 8) {
      store16(out + 8 * mm, __builtin_bit_cast(u32x4, f16x8{y[0], y[1], y[2], y[3], y[4], y[5], y[6], y[7]}));
    } else {
      *reinterpret_cast<u32x2*>(out + 4 * mm) = __builtin_bit_cast(u32x2, f16x4{y[0], y[1], y[2], y[3]});
    }
  }
}

template <int D, bool kFp8, Split kSplit>
hipError_t launch_s(const PrefillArgs& a, int64_t rows, hipStream_t stream) {
  constexpr int per = kSplit == kRows2 ? 256 : 128;
  const size_t bytes = sizeof(PrefillLds<D>) * (kSplit == kKeys2 ? 2 : 1);
  if (bytes > 64 * 1024) {
    const hipError_t e = grant_dynamic_lds(
        reinterpret_cast<const void*>(prefill_blocks_kernel<D, kFp8, kSplit>), bytes);
    if (e != hipSuccess) return e;
  }
  const dim3 grid(a.p.kv.num_kv_heads, static_cast<uint32_t>((rows + per - 1) / per), a.w.num_seqs);
  prefill_blocks_kernel<D, kFp8, kSplit>
      <<<grid, kGroupThreads * (kSplit == kOne ? 1 : 2), bytes, stream>>>(a);
  return hipSuccess;
}

template <int D, bool kFp8>
hipError_t launch(const PrefillArgs& a, int64_t rows, hipStream_t stream) {
  // Workgroups of 128 rows (of the grid: ragged prompts leave some of them empty).
  // Up to two per CU, splitting the keys beats more rows; past that, at D = 128,
  // 256 rows to an image beat 128, at D = 64 they do not (the slower one is not built).
  // us, kOne / kRows2 / kKeys2: 2 chunks of 512, 8 kv heads of 128, e4m3 60 / 61 / 45;
  // of 1024 87 / 80 / 69; of 2048 174 / 157 / 188; 4 x 4096 INT8 1525 / 1319 / 1547;
  // D = 64, kOne / kKeys2: 2 chunks of 512 44 / 31, 24 ragged prompts 111 / 154, 4 x 4096
  // 699 / 815.  (Between one and two per CU it depends on what the host does not know: even,
  // deep contexts lose by kKeys2, 1 x 2048 INT8 at 3986 217 / 239, uneven or short ones
  // gain, 8 x 100-256 62 / 46.)  RLK_TUNE_BLK_PREFILL forces a split (tests and tuning runs).
  const int64_t groups = (rows + 127) / 128 * a.p.kv.num_kv_heads * a.w.num_seqs;
  constexpr Split kLarge = D == 64 ? kOne : kRows2;
  const Split rule = groups <= 2 * compute_units() ? kKeys2 : kLarge;
  if (tune_knob(kBlkPrefill, rule) == kKeys2) return launch_s<D, kFp8, kKeys2>(a, rows, stream);
  return launch_s<D, kFp8, kLarge>(a, rows, stream);
}

}  // namespace
}  // namespace rlk

using namespace rlk;

extern "C" int rlk_paged_attention_prefill_blocks(const rlk_block_attention_params* p,
                                                  const rlk_prefill_attention_work* w,
                                                  hipStream_t stream) {
  const char* what = "paged_attention_prefill_blocks";
  if (p == nullptr || w == nullptr) return fail(RLK_EINVAL, "%s: null params or work", what);
  if (w->num_seqs <= 0 || w->max_q_tiles <= 0) return RLK_OK;
  if (const int st = check_block_params(p, what); st != RLK_OK) return st;
  if (w->seq_ids == nullptr || w->q_start == nullptr || w->q_len == nullptr || w->ctx_len == nullptr)
    return fail(RLK_EINVAL, "%s: null pointer argument", what);
  const int G = p->num_heads / p->kv.num_kv_heads;
  const int64_t rows = static_cast<int64_t>(w->max_q_tiles) * RLK_PREFILL_TILE_Q * G;
  if (w->num_seqs > 65535 || (rows + 127) / 128 > 65535)
    return fail(RLK_EINVAL, "%s: %d sequences of %d query tiles exceed one launch; split the call",
                what, w->num_seqs, w->max_q_tiles);
  const PrefillArgs a = {*p, *w, G};
  const bool fp8 = p->kv.format == RLK_KV_BLOCK_FP8;
  const hipError_t e = p->kv.head_dim == 128
                           ? (fp8 ? launch<128, true>(a, rows, stream) : launch<128, false>(a, rows, stream))
                           : (fp8 ? launch<64, true>(a, rows, stream) : launch<64, false>(a, rows, stream));
  if (e != hipSuccess) return fail(static_cast<int>(e), "%s: %s", what, hipGetErrorString(e));
  return launch_status(what);
}
