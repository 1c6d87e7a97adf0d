// Paged decode attention for groups of items that share a prefix, for gfx950.
//
// Flash-decoding: o = sum_k p_k v_k / sum_k p_k, p_k = exp(scale q.k - m), with the
// keys in two parts that are joined by the rule of the running maximum:
//   prefix  a unit is (group, kv head, 128 rows, range of keys), a row being one
//           (item, query head of the kv head) pair: every K and V byte of the range is
//           read once for all rows;
//   suffix  a unit is (item, kv head, range of keys) with the item's G rows.
// Both run in one launch; a second kernel joins a row's partials (o, m, l in fp32)
// through the caller's workspace.
//
// Prefix: tiles of 32 keys go through registers into LDS stages (INT8 codes become
// fp16 on the way), the loads of the next three or four in flight while one is used, the
// scores computed one tile ahead of the softmax.  A wave owns 32 rows:
//   S^T = K Q^T    v_mfma_f32_32x32x16_f16, K rows from LDS, q in registers: a lane
//                  gets one row (its column) and 16 of the tile's 32 keys, so the
//                  softmax is per lane with one exchange between the lane halves;
//   O^T = V^T P^T  the probabilities a lane holds are its B operand, the keys taken in
//                  the order in which S^T hands them over; V^T by transposing LDS reads.
// LDS chunks of 16 bytes are XOR-ed with the row so that neither read has bank conflicts.
//
// Suffix, and prefixes of groups of few rows, by tiles of 16 rows: each of the four waves
// owns a range of keys, without barriers until they are joined.  Tiles of 32 keys, the rows
// of two in flight, as v_mfma_f32_16x16x32_f16: K as A (16 keys x 32 dims), loaded as
// whole rows and laid out through a part of LDS that the wave alone uses, up to 16 rows
// as B.  The lanes of key group g get the scores of keys 4 g + i of both halves of the
// tile, which is their share of the B operand of O^T = V^T P^T; as A a lane loads those 8
// keys' dims E m .. E m + E - 1 (E = D / 16, m = lane % 16), and tile dt of the output
// takes dim E m + dt: 8 x E values to be transposed inside the lane, a byte permute per
// register.
//
// INT8: K scales multiply the scores, V scales the probabilities before they are rounded,
// so that codes stay exact and a value is rounded once, as in an FP16 cache; the reference of
// the exponentials is that of the products (kNoValue).
//
// A probability (INT8: with its V scale) goes to fp16 for the second product: 2.5-2.7e-4 from 64
// bits in the 2-norm, where outputs that are rounded alone are off by 2.1e-4; a second term
// would double that product's instructions.
//
// Bound (D = 128; clock stamps, caches warm - cold):
//   64 items x 7 heads a kv head over 32 k and up to 2 k of their own: 72.6 us, 425 TFLOP/s.  A
//   prefix unit's 64 tiles at 0.88 - 0.99 us each (a wave's chain LDS -> product -> exponential ->
//   product; one prefix wave a SIMD, whose products take 512 of some 2000 clocks),
//   3 us to the merge, which takes 6.
//   32 items x 4 over 8 k: 30.3 us.  Units end at 22 - 30: 2.3 - 3.3 until the first loads, 8
//   prefix tiles at 1.4 - 2.1 beside the suffix's loads; 3.4 to the merge and 5.6 in it, of 17 MB
//   of partials.
//   118 items of 7 groups, INT8: 70.5 us, 3.3 TB/s.  512 of 1160 units are resident; prefix units
//   (26 tiles at 1.2 us) hold their places to 37 - 54 us, the last of the long suffix units, of 15 -
//   18 us, start at 40 - 46.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cstdint>

#include "device.hpp"
#include "redline_amd/rlk.h"
#include "status.hpp"

namespace rlk {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kTile = 32;               // keys
constexpr int kWaveRows = 32;
constexpr int kRows = kThreads / kWave * kWaveRows;  // of a workgroup
constexpr int kPart = RLK_DECODE_PARTITION_SIZE;
constexpr int kMaxGroup = 8;            // query heads of a kv head
constexpr int kFewRows = 16;            // of units without shared tiles
constexpr int64_t kMaxBlocks = (int64_t{1} << 32) / kThreads - 1;  // (a grid has 32 bits of threads)
constexpr float kLog2e = 1.4426950408889634f;

enum Format { kF16, kI8, kI8Half };  // FP16 cells; INT8 with fp32, with fp16 scales

struct SharedArgs {
  rlk_attention_params p;
  rlk_shared_prefix_work w;
  int grp;                 // query heads of a kv head
  int prefix_keys, suffix_keys;      // keys of a unit, whole tiles
  int prefix_splits, suffix_splits;  // units of the longest prefix, of the longest rest
  int row_tiles;
  int few_rows;  // units of at most so many rows go by tiles of 16
  uint32_t prefix_blocks;
  // key / block_size = key >> lbs where magic is 0, else umulhi(key, magic) >> lbs
  uint32_t magic;
  int lbs;
};

// The table's block that a key is in.
__device__ __forceinline__ int block_of(const SharedArgs& a, int key) {
  const uint32_t q = a.magic != 0 ? __umulhi(static_cast<uint32_t>(key), a.magic) : static_cast<uint32_t>(key);
  return static_cast<int>(q >> a.lbs);
}

// Keys that an item attends to, those inside its table row.
__device__ __forceinline__ int keys_of(const SharedArgs& a, int token) {
  const int64_t most = static_cast<int64_t>(a.p.max_blocks_per_seq) * a.p.kv.block_size;
  return static_cast<int>(max(min(static_cast<int64_t>(a.p.positions[token]) + 1, most), static_cast<int64_t>(0)));
}
// The part of group g's prefix that its units read.
__device__ __forceinline__ int prefix_of(const SharedArgs& a, int g) {
  const int64_t most = min(static_cast<int64_t>(a.p.max_blocks_per_seq) * a.p.kv.block_size,
                           static_cast<int64_t>(a.w.max_prefix_partitions) * kPart);
  return static_cast<int>(max(min(static_cast<int64_t>(a.w.group_prefix[g]), most), static_cast<int64_t>(0)));
}
// The prefix that an item shares, 0 outside the groups; by a whole wave.
__device__ __forceinline__ int shared_prefix(const SharedArgs& a, int item) {
  const int lane = threadIdx.x % kWave;
  int found = 0;  // of the last group that starts at or before the item
  for (int g0 = 0; g0 < a.w.num_groups; g0 += kWave) {
    const int g = min(g0 + lane, a.w.num_groups - 1), first = a.w.group_start[g], last = a.w.group_start[g + 1];
    const int prefix = prefix_of(a, g);
    const bool in = first >= 0 && item < last && item - first < a.w.max_group_items;
    const uint64_t before = __ballot(g0 + lane < a.w.num_groups && first <= item);
    if (before != 0) found = __builtin_amdgcn_readlane(in ? prefix : 0, 63 - __builtin_clzll(before));
    if (before != ~0ull) break;
  }
  return found;
}

__device__ __forceinline__ int64_t slot_row(const SharedArgs& a, int item, int head) {
  return (static_cast<int64_t>(item) * a.p.num_heads + head) * (a.w.max_prefix_partitions + a.w.max_partitions);
}

// Scores enter the exponential as q.k c - m: c > 0, the sign of the scale in q, so that the
// largest product is the largest score (and not 0, which a masked score must not meet).
__device__ __forceinline__ float score_factor(float scale) {
  return fmaxf(__builtin_fabsf(scale) * kLog2e, 0x1p-126f);
}
__device__ __forceinline__ f16x8 signed_by(float scale, u32x4 q) {
  return __builtin_bit_cast(f16x8, q ^ (scale < 0.f ? 0x80008000u : 0u));
}
// (fmaxf would first pass each operand through an instruction of its own; NaN stays)
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// LDS image of a tile row: 16-byte chunk c of row r stands at chunk c ^ swizzle(r).
template <int D>
__device__ __forceinline__ int k_swizzle(int r) { return D == 128 ? r & 15 : (r >> 1) & 7; }
template <int D>
__device__ __forceinline__ int v_swizzle(int r) { return D == 128 ? (r & 3) << 2 : ((r >> 1) & 1) << 2; }

// INT8: the reference m of the exponentials is the maximum of score + log2(V scale) of the same
// key, since p vs is what is rounded: keys of a large V scale that have no weight, or that are
// masked, take no bits from the others.  A row of zeros (whose scale is 1) gives nothing and is
// not to set it either; its scale counts as 0, whose logarithm is held at kNoValue: where the
// scores of such keys lie further above all others, the output is below fp16, and their
// exponentials stay in fp32.
constexpr float kNoValue = -64.f;
__device__ __forceinline__ float log2_scale(float vs) {
  return __builtin_amdgcn_logf(fmaxf(vs, 0x1p-64f));
}
template <int CTRL>
__device__ __forceinline__ uint32_t or_dpp(uint32_t v) {
  return v | static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), CTRL, 0xF, 0xF, true));
}
// Bits of v of aligned groups of 4 or 8 lanes.
template <int N>
__device__ __forceinline__ uint32_t group_or(uint32_t v) {
  static_assert(N == 4 || N == 8);
  v = or_dpp<0x4E>(or_dpp<0xB1>(v));
  if constexpr (N == 8) v = or_dpp<0x141>(v);
  return v;
}

// The rows of one key that a lane of the suffix loads: E = D / 16 dims of V, 8 of K.
template <int kBytes> struct RawOf;
template <> struct RawOf<16> { using Type = u32x4; };
template <> struct RawOf<8> { using Type = u32x2; };
template <> struct RawOf<4> { using Type = uint32_t; };

// One wave's part of a unit of up to 16 rows: keys [begin, end) of the table row, for row lane % 16
// those below `last`.  In: q as B operands; kbuf: 32 rows of K in LDS, scales: of 32 keys, this wave's
// own.  Out: m, l and o[dt][i] = dim E (4 (lane / 16) + i) + dt of row lane % 16.
template <int D, int kFmt>
__device__ __forceinline__ void attend_alone(const SharedArgs& a, const int32_t* table, int kvh, int begin, int end, int last,
                                             const f16x8 (&q)[D / 32], unsigned char* kbuf, float (*scales)[32], float& m, float& l,
                                             f32x4 (&o)[D / 16]) {
  constexpr bool kInt8 = kFmt != kF16;
  constexpr int E = D / 16, kElem = kInt8 ? 1 : 2, kAhead = 2, kKeys = 32;
  constexpr int kAheadV = kInt8 ? 2 : 1;  // (FP16: with two tiles the registers do not suffice)
  // K: whole rows by consecutive lanes.  Loaded as the operands want them, a row a lane, the address
  // unit took the lanes of an instruction one by one (64 items over 32 k: 87 us against 73).
  constexpr int kRow = D * kElem, kChunks = kRow / 16, kRowsAtOnce = kWave / kChunks, kLoads = kKeys / kRowsAtOnce;
  using VRaw = typename RawOf<E * kElem>::Type;
  const rlk_kv_layer_view& kv = a.p.kv;
  const int lane = threadIdx.x % kWave, col = lane % 16, kg = lane / 16, hkv = kv.num_kv_heads, bs = kv.block_size;
  const float c = score_factor(a.p.scale);
  m = -FLT_MAX;
  l = 0.f;
#pragma unroll
  for (int d = 0; d < E; ++d) o[d] = f32x4{0, 0, 0, 0};
  if (begin >= end) return;
  int whole = last;  // every row has the keys up to this one
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) whole = min(whole, __shfl_xor(whole, o, kWave));
  whole = __builtin_amdgcn_readfirstlane(min(whole, end));

  struct Cell { int id, off; };
  auto find = [&](int k0) -> Cell {  // of key lane % 32 of a tile
    const int pos = min(k0 + lane % kKeys, end - 1), b = block_of(a, pos);
    return {table[b], pos - b * bs};
  };
  u32x4 kr[kAhead][kLoads];
  VRaw vr[kAheadV][8];
  uint32_t cell[kAhead];
  float ks[kAhead], vs[kAhead];
  auto request_k = [&](int u, Cell at) {
    cell[u] = (static_cast<uint32_t>(at.id) * hkv + kvh) * bs + at.off;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const uint32_t from = __shfl(cell[u], j * kRowsAtOnce + lane / kChunks, kWave);
      kr[u][j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(
          static_cast<const unsigned char*>(kv.k) + static_cast<int64_t>(from) * kRow + lane % kChunks * 16));
    }
    if constexpr (kFmt == kI8) {
      ks[u] = kv.k_scale[cell[u]];
      vs[u] = kv.v_scale[cell[u]];
    } else if constexpr (kFmt == kI8Half) {
      ks[u] = static_cast<float>(reinterpret_cast<const _Float16*>(kv.k_scale)[cell[u]]);
      vs[u] = static_cast<float>(reinterpret_cast<const _Float16*>(kv.v_scale)[cell[u]]);
    }
  };
  auto request_v = [&](int u) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t at = __shfl(cell[u], 16 * (j / 4) + 4 * kg + j % 4, kWave);
      vr[u % kAheadV][j] = __builtin_nontemporal_load(reinterpret_cast<const VRaw*>(
          static_cast<const unsigned char*>(kv.v) + static_cast<int64_t>(at) * (D * kElem) + col * (E * kElem)));
    }
    asm volatile("" ::: "memory");  // else the compiler moves these loads to where they are used
  };
  // One tile from slot u; the slot's rows are requested for the tile kAhead on, past the range its last
  // key again.  Loads complete in order: a table entry is requested before the rows beside it.
  Cell cells[kAhead];
  // 16-byte chunk c of row r of kbuf stands at chunk c ^ swizzle(r): no bank conflicts either way
  auto swizzle = [](int r) { return kChunks == 16 ? r & 15 : (kChunks == 8 ? (r >> 1) & 7 : (r >> 2) & 3); };
  auto step = [&](int k0, int u) {
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {  // (a wave's LDS accesses complete in order)
      const int r = j * kRowsAtOnce + lane / kChunks;
      store16(kbuf + r * kRow + ((lane % kChunks ^ swizzle(r)) << 4), kr[u][j]);
    }
    if constexpr (kInt8) {
      scales[0][lane % kKeys] = ks[u];
      scales[1][lane % kKeys] = vs[u];
      scales[2][lane % kKeys] = log2_scale(vs[u]);
    }
    f32x4 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int x = 0; x < D / 32; ++x) {
        const unsigned char* row = kbuf + (16 * t + col) * kRow;
        f16x8 kf;
        if constexpr (kInt8) kf = int8x8_to_f16(*reinterpret_cast<const u32x2*>(row + ((2 * x + kg / 2) ^ swizzle(col)) * 16 + kg % 2 * 8));
        else kf = *reinterpret_cast<const f16x8*>(row + (((4 * x + kg) ^ swizzle(col)) << 4));
        s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q[x], s[t], 0, 0, 0);
      }
    }
    // s[t][i]: key k0 + 16 t + 4 kg + i
    f32x4 vscale[2], vlog[2];
    if constexpr (kInt8) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int key = 16 * t + 4 * kg;
        const f32x4 f = *reinterpret_cast<const f32x4*>(&scales[0][key]);
        vscale[t] = *reinterpret_cast<const f32x4*>(&scales[1][key]);
        vlog[t] = *reinterpret_cast<const f32x4*>(&scales[2][key]);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[t][i] *= f[i];
      }
    }
    const Cell next = find(k0 + 2 * kAhead * kKeys);
    request_k(u, cells[u]);
    cells[u] = next;
    __builtin_amdgcn_sched_barrier(0);
    if (k0 + kKeys > whole) {
      const int left = min(last, end) - k0 - 4 * kg;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (16 * t + i >= left) s[t][i] = -INFINITY;
    }
    auto largest = [&] {
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float x = s[i / 4][i % 4];
        if constexpr (kInt8) x = __builtin_fmaf(x, c, vlog[i / 4][i % 4]);
        mx = larger(mx, x);
      }
      mx = rows_max<true>(rows_max<false>(mx));
      return kInt8 ? mx : mx * c;
    };
    float mx = largest();
    if (__any(mx > m + 8.f)) {  // as in the prefix
      if constexpr (kInt8) {  // rows of zeros are looked for only where m would move
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t any = 0;
          if constexpr (E == 8) any = vr[u][j][0] | vr[u][j][1];
          else any = vr[u][j];
          const uint64_t rows = __ballot(any != 0) >> (16 * kg);  // (the 16 lanes of a group hold a row)
          const bool value = (rows & 0xffff) != 0;
          vscale[j / 4][j % 4] = value ? vscale[j / 4][j % 4] : 0.f;
          vlog[j / 4][j % 4] = value ? vlog[j / 4][j % 4] : kNoValue;
        }
        mx = largest();
      }
      const float mn = fmaxf(m, mx), f = __builtin_amdgcn_exp2f(m - mn);
      l *= f;
#pragma unroll
      for (int d = 0; d < E; ++d) o[d] *= f;
      m = mn;
    }
    f16x8 p;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i / 4][i % 4], c, -m));
      l += e;
      if constexpr (kInt8) e *= vscale[i / 4][i % 4];
      p[i] = static_cast<_Float16>(e);
    }
    // operands: element dt of the 8 rows; those past the range are cleared, since 0 times an
    // infinity is no 0
    VRaw row[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) row[j] = vr[u % kAheadV][j];
    if (k0 + kKeys > end) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k0 + 16 * (j / 4) + 4 * kg + j % 4 >= end) row[j] = VRaw{};
    }
    u32x4 vt[E];
    if constexpr (kInt8) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (E == 8) {
          f16x2 pair[8];
          int8x8_pairs_to_f16x2(row[2 * j], row[2 * j + 1], pair);
#pragma unroll
          for (int d = 0; d < 8; ++d) vt[d][j] = __builtin_bit_cast(uint32_t, pair[d]);
        } else {
          const uint32_t x = row[2 * j] ^ 0x80808080u, y = row[2 * j + 1] ^ 0x80808080u;
          const uint32_t lo = __builtin_amdgcn_perm(y, x, 0x05010400u), hi = __builtin_amdgcn_perm(y, x, 0x07030602u);
          const uint32_t w[4] = {__builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u),
                                 __builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u)};
#pragma unroll
          for (int d = 0; d < 4; ++d)
            vt[d][j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, w[d]) - static_cast<_Float16>(1152));
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int d = 0; d < E; d += 2) {
          vt[d][j] = __builtin_amdgcn_perm(row[2 * j + 1][d / 2], row[2 * j][d / 2], 0x05040100u);
          vt[d + 1][j] = __builtin_amdgcn_perm(row[2 * j + 1][d / 2], row[2 * j][d / 2], 0x07060302u);
        }
    }
    request_v((u + kAheadV) % kAhead);
#pragma unroll
    for (int d = 0; d < E; ++d)
      o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, vt[d]), p, o[d], 0, 0, 0);
  };
#pragma unroll
  for (int u = 0; u < kAhead; ++u) cells[u] = find(begin + u * kKeys);
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    const Cell next = find(begin + (kAhead + u) * kKeys);
    request_k(u, cells[u]);
    cells[u] = next;
    __builtin_amdgcn_sched_barrier(0);
    if (u < kAheadV) request_v(u);
  }
#pragma unroll 1
  for (int k0 = begin; k0 < end; k0 += kAhead * kKeys)
#pragma unroll
    for (int u = 0; u < kAhead; ++u) step(k0 + u * kKeys, u);  // (a tile past the range has no part in the sums)
  l = rows_sum<true>(rows_sum<false>(l));
}

template <int D, int kFmt>
__global__ __launch_bounds__(kThreads, 2) void shared_attention_kernel(SharedArgs a) {
  constexpr bool kInt8 = kFmt != kF16;
  constexpr int kPitch = 2 * D, kQ = D / 16, kO = D / 32;
  constexpr int kChunks = D / (kInt8 ? 16 : 8);             // loads of a row
  constexpr int kRowStep = kThreads / kChunks;              // rows between a thread's loads
  constexpr int kItems = (kTile + kRowStep - 1) / kRowStep; // loads of a thread and tile, of K and of V
  constexpr int kAhead = kItems > 1 ? 3 : 4;                // tiles in flight, LDS stages
  struct Stages {
    unsigned char k[kAhead][kTile * kPitch], v[kAhead][kTile * kPitch];
    float ks[kAhead][kTile], vs[kAhead][kTile], vlog[kAhead][kTile];
  };
  struct Suffix {
    unsigned char k[kThreads / kWave][32 * D * (kInt8 ? 1 : 2)];
    float scales[kThreads / kWave][3][32];  // of K, of V and their logarithms
    // of each wave, to be joined
    float o[kThreads / kWave][kFewRows][D + 4], m[kThreads / kWave][16], l[kThreads / kWave][16];
    int token[16];
  };
  __shared__ alignas(1024) union { Stages st; Suffix suffix; } shared;
  Stages& lds = shared.st;
  const rlk_attention_params& p = a.p;
  const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int col = lane % 32, half = lane / 32;
  const int hkv = p.kv.num_kv_heads, bs = p.kv.block_size, G = a.grp;

  // the unit
  int kvh, first, rows, row0 = 0, begin, end, slot;
  if (blockIdx.x < a.prefix_blocks) {
    // the row tiles of a range stand 8 blocks apart: on one XCD, whose L2 has the range
    const int b = blockIdx.x / 8, rt = b % a.row_tiles, u = b / a.row_tiles * 8 + blockIdx.x % 8;
    const int split = u % a.prefix_splits, gk = u / a.prefix_splits, g = gk / hkv;
    kvh = gk - g * hkv;
    if (g >= a.w.num_groups) return;
    first = a.w.group_start[g];
    const int n = min(min(a.w.group_start[g + 1], a.w.num_items) - first, a.w.max_group_items);
    rows = n * G;
    row0 = rt * (rows <= a.few_rows ? kFewRows : kRows);
    if (first < 0 || rows <= row0) return;
    begin = split * a.prefix_keys;
    end = min(prefix_of(a, g), begin + a.prefix_keys);
    slot = split;
  } else {
    const int u = static_cast<int>(blockIdx.x - a.prefix_blocks);
    const int split = u % a.suffix_splits, ik = u / a.suffix_splits;
    first = ik / hkv;
    kvh = ik - first * hkv;
    const int token = a.w.item_token[first];
    if (token < 0) return;
    rows = G;
    const int prefix = shared_prefix(a, first);
    const int64_t keys = min(static_cast<int64_t>(keys_of(a, token)),
                             prefix + static_cast<int64_t>(a.w.max_partitions) * kPart);
    const int64_t at = prefix + static_cast<int64_t>(split) * a.suffix_keys;
    if (at >= keys) return;
    begin = static_cast<int>(at);
    end = static_cast<int>(min(keys, at + a.suffix_keys));
    slot = a.w.max_prefix_partitions + split;
  }
  if (begin >= end) return;
  const int32_t* table = p.block_tables + static_cast<int64_t>(a.w.item_seq[first]) * p.max_blocks_per_seq;

  if (rows <= a.few_rows) {
    // the tile's rows; a wave's keys, whole tiles but for the last
    const int here = min(rows - row0, kFewRows);
    constexpr int kWaves = kThreads / kWave;
    const int per = ((end - begin + kWaves - 1) / kWaves + 31) / 32 * 32;
    const int b0 = min(begin + wave * per, end), b1 = min(b0 + per, end);
    const int r = lane % 16, item = first + (row0 + r) / G, token = r < here ? a.w.item_token[item] : -1;
    int last = end;
    f16x8 q[D / 32];
#pragma unroll
    for (int x = 0; x < D / 32; ++x) q[x] = f16x8{0, 0, 0, 0, 0, 0, 0, 0};
    if (token >= 0) {
      last = keys_of(a, token);
      const _Float16* qp = reinterpret_cast<const _Float16*>(p.q) + static_cast<int64_t>(token) * p.q_stride + (kvh * G + (row0 + r) % G) * D + 8 * (lane / 16);
#pragma unroll
      for (int x = 0; x < D / 32; ++x) q[x] = signed_by(p.scale, load16(qp + 32 * x));
    }
    float m, l;
    f32x4 o[D / 16];
    attend_alone<D, kFmt>(a, table, kvh, b0, b1, last, q, shared.suffix.k[wave], shared.suffix.scales[wave], m, l, o);
    // the waves joined
    Suffix& j = shared.suffix;
    if (lane < 16) {
      j.m[wave][lane] = m;
      j.l[wave][lane] = l;
      j.token[lane] = token;
    }
    if (r < here) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < D / 16; d += 4)
          *reinterpret_cast<f32x4*>(&j.o[wave][r][D / 16 * (4 * (lane / 16) + i) + d]) =
              f32x4{o[d][i], o[d + 1][i], o[d + 2][i], o[d + 3][i]};
    }
    __syncthreads();
    for (int e = tid; e < here * D; e += kThreads) {
      const int x = e / D, d = e % D;
      if (j.token[x] < 0) continue;
      float M = j.m[0][x], L = 0.f, sum = 0.f;
#pragma unroll
      for (int w = 1; w < kWaves; ++w) M = fmaxf(M, j.m[w][x]);
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = __builtin_amdgcn_exp2f(j.m[w][x] - M);
        L += f * j.l[w][x];
        sum += f * j.o[w][x][d];
      }
      const int64_t to = slot_row(a, first + (row0 + x) / G, kvh * G + (row0 + x) % G) + slot;
      a.w.ws_out[to * D + d] = sum;
      if (d == 0) {
        a.w.ws_max[to] = M;
        a.w.ws_sum[to] = L;
      }
    }
    return;
  }

  // the lane's row
  const bool busy = row0 + wave * kWaveRows < rows;  // the wave has rows
  const int r = row0 + wave * kWaveRows + col, item = first + r / G, head = kvh * G + r % G;
  const int token = r < rows ? a.w.item_token[item] : -1;
  int last = end;  // keys of the row, up to this one
  f16x8 q[kQ];
#pragma unroll
  for (int s = 0; s < kQ; ++s) q[s] = f16x8{0, 0, 0, 0, 0, 0, 0, 0};
  if (token >= 0) {
    last = min(end, keys_of(a, token));
    const _Float16* qp = reinterpret_cast<const _Float16*>(p.q) + static_cast<int64_t>(token) * p.q_stride + head * D + 8 * half;
#pragma unroll
    for (int s = 0; s < kQ; ++s) q[s] = signed_by(p.scale, load16(qp + 16 * s));
  }
  int whole = last;  // every row of the wave has the keys up to this one
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) whole = min(whole, __shfl_xor(whole, o, kWave));
  whole = __builtin_amdgcn_readfirstlane(whole);

  // this thread's part of a tile; lane k finds the cell of key k % 32
  const int ch = tid % kChunks, tr = tid / kChunks;
  u32x4 kraw[kAhead][kItems], vraw[kAhead][kItems];
  float ksc[kAhead], vsc[kAhead];  // INT8: wave 0 has the K scales, every thread that of its V row
  static_assert(!kInt8 || kItems == 1);
  struct Cell { int id, off; };
  auto find = [&](int k0) -> Cell {
    const int pos = min(k0 + lane % kTile, end - 1), b = block_of(a, pos);
    return {table[b], pos - b * bs};
  };
  auto request = [&](int u, Cell at) {
    const uint32_t cell = (static_cast<uint32_t>(at.id) * hkv + kvh) * bs + at.off;
    uint32_t row;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      row = __shfl(cell, (tr + i * kRowStep) % kTile, kWave);
      const uint64_t from = static_cast<uint64_t>(row) * (kInt8 ? D : 2 * D) + ch * 16;
      kraw[u][i] = load16(static_cast<const unsigned char*>(p.kv.k) + from);
      vraw[u][i] = load16(static_cast<const unsigned char*>(p.kv.v) + from);
    }
    if constexpr (kInt8) {
      auto scale = [](const float* of, uint32_t at) {
        return kFmt == kI8 ? of[at] : static_cast<float>(reinterpret_cast<const _Float16*>(of)[at]);
      };
      vsc[u] = scale(p.kv.v_scale, row);
      if (wave == 0) ksc[u] = scale(p.kv.k_scale, cell);
    }
  };
  auto put = [&](int k0, int u) {
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int row = tr + i * kRowStep;
      if (kRowStep * kItems > kTile && row >= kTile) break;
      // rows past the range hold its last key; their V is cleared, since 0 times an infinity is no 0
      unsigned char* kd = lds.k[u] + row * kPitch;
      unsigned char* vd = lds.v[u] + row * kPitch;
      const u32x4 kr = kraw[u][i], vr = k0 + row < end ? vraw[u][i] : u32x4{0, 0, 0, 0};
      if constexpr (kInt8) {
        const float f = group_or<kChunks>(vr[0] | vr[1] | vr[2] | vr[3]) != 0 ? vsc[u] : 0.f;
        if (ch == 0) {
          lds.vs[u][row] = f;
          lds.vlog[u][row] = log2_scale(f);
        }
      }
      if constexpr (!kInt8) {
        store16(kd + ((ch ^ k_swizzle<D>(row)) << 4), kr);
        store16(vd + ((ch ^ v_swizzle<D>(row)) << 4), vr);
      } else {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const u32x2 kc = {kr[2 * x], kr[2 * x + 1]}, vc = {vr[2 * x], vr[2 * x + 1]};
          store16(kd + (((2 * ch + x) ^ k_swizzle<D>(row)) << 4), __builtin_bit_cast(u32x4, int8x8_to_f16(kc)));
          store16(vd + (((2 * ch + x) ^ v_swizzle<D>(row)) << 4), __builtin_bit_cast(u32x4, int8x8_to_f16(vc)));
        }
      }
    }
    if constexpr (kInt8) {
      if (wave == 0 && lane < kTile) lds.ks[u][lane] = ksc[u];
    }
  };

  const float c = score_factor(p.scale);
  f32x16 o[kO];
#pragma unroll
  for (int d = 0; d < kO; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  float m = -FLT_MAX, l = 0.f;
  // V^T reads: lane (g, tk, tm) of 16 lanes takes 4 dims of key 4 half + tk
  const int tk = lane % 16 / 4, tm = lane % 4;
  const int vrow = (4 * half + tk) * kPitch, vsw = v_swizzle<D>(tk);
  int vat[kO];
#pragma unroll
  for (int d = 0; d < kO; ++d)
    vat[d] = vrow + (((4 * d + 2 * (lane / 16 % 2) + tm / 2) ^ vsw) << 4) + (tm & 1) * 8;

  // element i of a tile's scores: key k0 + 8 (i / 4) + 4 half + i % 4
  auto scores = [&](int u) {
    f32x16 s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
    const unsigned char* kr = lds.k[u] + col * kPitch;
#pragma unroll
    for (int x = 0; x < kQ; ++x) {
      const f16x8 kf = *reinterpret_cast<const f16x8*>(kr + (((2 * x + half) ^ k_swizzle<D>(col)) << 4));
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, q[x], s, 0, 0, 0);
    }
    return s;
  };
  // The tile at k0 from stage u, whose scores are there; returns those of stage v.
  auto attend = [&](f32x16 s, int k0, int u, int v) {
    if constexpr (kInt8) {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const f32x4 f = *reinterpret_cast<const f32x4*>(&lds.ks[u][8 * b + 4 * half]);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[4 * b + i] *= f[i];
      }
    }
    if (k0 + kTile > whole) {
      const int left = last - k0 - 4 * half;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (8 * (i / 4) + i % 4 >= left) s[i] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      f32x4 f;
      if constexpr (kInt8) f = *reinterpret_cast<const f32x4*>(&lds.vlog[u][8 * b + 4 * half]);
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = larger(mx, kInt8 ? __builtin_fmaf(s[4 * b + i], c, f[i]) : s[4 * b + i]);
    }
    mx = rows_max<true>(mx);
    if constexpr (!kInt8) mx *= c;
    // m is a reference within 2^8 of the maximum: moving it costs a pass over the
    // output, and probabilities (INT8: with their V scale) up to 2^8 have the same 11 bits in fp16
    if (__any(mx > m + 8.f)) {
      const float mn = fmaxf(m, mx), f = __builtin_amdgcn_exp2f(m - mn);
      l *= f;
#pragma unroll
      for (int d = 0; d < kO; ++d) o[d] *= f;
      m = mn;
    }
    // the next tile's scores run on the matrix cores beside this one's exponentials
    const f32x16 next = scores(v);
    f16x8 pb[2];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      f32x4 f;
      if constexpr (kInt8) f = *reinterpret_cast<const f32x4*>(&lds.vs[u][8 * b + 4 * half]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * b + i], c, -m));
        l += e;
        if constexpr (kInt8) e *= f[i];
        pb[b / 2][b % 2 * 4 + i] = static_cast<_Float16>(e);
      }
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      unsigned char* vt = lds.v[u] + 16 * x * kPitch;
#pragma unroll
      for (int d = 0; d < kO; ++d) {
        typedef __attribute__((address_space(3))) s16x4* LdsPtr;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(vt + vat[d]));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(vt + vat[d] + 8 * kPitch));
        const f16x8 vf = __builtin_bit_cast(f16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pb[x], o[d], 0, 0, 0);
      }
    }
    return next;
  };

  Cell cells[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) cells[u] = find(begin + u * kTile);
  // Loads complete in order: a table entry that is waited for takes everything before it along.  So
  // entries are requested as far ahead of their use as tiles are.
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    request(u, cells[u]);
    cells[u] = find(begin + (kAhead + u) * kTile);
    __builtin_amdgcn_sched_barrier(0);
  }
  auto stage = [&](int k0, int u) {  // the tile at k0 into stage u, its registers to the one kAhead tiles on
    put(k0, u);
    request(u, cells[u]);  // past the range its last key again
    cells[u] = find(k0 + 2 * kAhead * kTile);
    __builtin_amdgcn_sched_barrier(0);
  };
  stage(begin, 0);
  __syncthreads();
  f32x16 s = scores(0);
#pragma unroll 1
  for (int k0 = begin; k0 < end; k0 += kAhead * kTile) {  // (no exit inside: the loads in flight are then known)
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int at = k0 + u * kTile, v = (u + 1) % kAhead;
      stage(at + kTile, v);
      __syncthreads();  // stage v was last read before the barrier of the step before
      if (busy && at < end) s = attend(s, at, u, v);
    }
  }
  if (token < 0) return;
  l += __shfl_xor(l, 32, kWave);
  const int64_t at = slot_row(a, item, head) + slot;
  float* dst = a.w.ws_out + at * D + 4 * half;
#pragma unroll
  for (int d = 0; d < kO; ++d)
#pragma unroll
    for (int b = 0; b < 4; ++b)
      *reinterpret_cast<f32x4*>(dst + 32 * d + 8 * b) = f32x4{o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]};
  if (half == 0) {
    a.w.ws_max[at] = m;
    a.w.ws_sum[at] = l;
  }
}

// Joins the partials of one (item, head): lane d of the workgroup takes dim d; each
// wave holds the weights of 64 slots, one a lane.  The statistics of the first 64 are
// requested before it is known which of them were written.
template <int D>
__global__ __launch_bounds__(D) void shared_merge_kernel(SharedArgs a) {
  constexpr int kUnroll = 8;
  const int item = blockIdx.x, head = blockIdx.y, d = threadIdx.x, lane = d % kWave;
  const int total = a.w.max_prefix_partitions + a.w.max_partitions;
  const int64_t row = slot_row(a, item, head);
  float ms = a.w.ws_max[row + min(lane, total - 1)], ls = a.w.ws_sum[row + min(lane, total - 1)];
  const int token = a.w.item_token[item], prefix = shared_prefix(a, item);
  if (token < 0) return;
  const int keys = keys_of(a, token);
  const int np = (prefix + a.prefix_keys - 1) / max(a.prefix_keys, 1);
  const int rest = min(max(keys - prefix, 0), a.w.max_partitions * kPart);
  const int ns = (rest + a.suffix_keys - 1) / a.suffix_keys;
  float M = -FLT_MAX, L = 0.f, o = 0.f;
  for (int j0 = 0; j0 < total; j0 += kWave) {
    const int j = j0 + lane;
    const bool there = j < np || (j >= a.w.max_prefix_partitions && j - a.w.max_prefix_partitions < ns);
    uint64_t left = __ballot(there);
    if (left == 0) continue;
    if (j0 > 0) {
      ms = a.w.ws_max[row + min(j, total - 1)];
      ls = a.w.ws_sum[row + min(j, total - 1)];
    }
    const float mine = there ? ms : -FLT_MAX;
    const float mn = fmaxf(M, rows_max<true>(rows_max<false>(group_max<16>(mine))));
    const float f0 = __builtin_amdgcn_exp2f(M - mn), f = there ? __builtin_amdgcn_exp2f(mine - mn) : 0.f;
    L = L * f0 + wave_sum(there ? f * ls : 0.f);
    o *= f0;
    M = mn;
    while (left != 0) {
      float v[kUnroll], w[kUnroll];
      int at = 0;
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {  // past the last one its row again, with no weight
        const bool more = left != 0;
        at = more ? __builtin_ctzll(left) : at;
        left &= left - 1;
        const float x = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), at));
        w[u] = more ? x : 0.f;
        v[u] = a.w.ws_out[(row + j0 + at) * D + d];
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) o += w[u] != 0.f ? w[u] * v[u] : 0.f;
    }
  }
  reinterpret_cast<_Float16*>(a.p.out)[(static_cast<int64_t>(token) * a.p.num_heads + head) * D + d] =
      static_cast<_Float16>(keys > 0 ? o / L : 0.f);
}

template <int D, int kFmt>
int launch(SharedArgs a, const char* what, hipStream_t stream) {
  const int64_t cus = compute_units(), hkv = a.p.kv.num_kv_heads;
  const int pp = a.w.num_groups > 0 && a.w.max_group_items > 0 ? a.w.max_prefix_partitions : 0;
  // Ranges of at least 256 keys (a workspace slot each) that give `want` units in all.  With a prefix
  // its units come first, one a CU, and leave room for one of the suffix beside each: the ones compute
  // where the others load.
  const int64_t want_each = pp > 0 ? cus : 2 * cus;
  auto keys_of_unit = [&](int partitions, int64_t units) {
    const int64_t keys = static_cast<int64_t>(partitions) * kPart, want = std::max<int64_t>(1, (want_each + units - 1) / units);
    return static_cast<int>(std::max<int64_t>((keys + want - 1) / want + kTile - 1, kPart) / kTile * kTile);
  };
  // Up to 48 rows a group: tiles of 16 rows whose waves split the keys; four waves of keys outweigh
  // reading a range up to three times, from L2 (24 rows over 24 k, D = 64, INT8: 25.7 us against 35.3).  In a call
  // with larger groups too only groups of one such tile.
  const int most_rows = std::min(a.w.max_group_items, a.w.num_items) * a.grp;
  a.few_rows = most_rows <= 3 * kFewRows ? 3 * kFewRows : kFewRows;
  const int tile_rows = most_rows <= a.few_rows ? kFewRows : kRows;
  a.row_tiles = (most_rows + tile_rows - 1) / tile_rows;
  int64_t blocks = 0;
  if (pp > 0) {
    const int64_t tiles = std::min<int64_t>(static_cast<int64_t>(a.w.num_groups) * a.row_tiles,
                                            static_cast<int64_t>(a.w.num_items) * a.grp / tile_rows + a.w.num_groups);
    a.prefix_keys = keys_of_unit(pp, tiles * hkv);
    a.prefix_splits = (pp * kPart + a.prefix_keys - 1) / a.prefix_keys;
    const int64_t ranges = a.w.num_groups * hkv * a.prefix_splits;
    if (ranges > kMaxBlocks) return fail(RLK_EINVAL, "%s: %d groups exceed one launch; split the call", what, a.w.num_groups);
    blocks = (ranges + 7) / 8 * 8 * a.row_tiles;
  } else {
    a.prefix_keys = kPart;
    a.w.num_groups = 0;
  }
  a.suffix_keys = keys_of_unit(a.w.max_partitions, a.w.num_items * hkv);
  a.suffix_splits = (a.w.max_partitions * kPart + a.suffix_keys - 1) / a.suffix_keys;
  a.prefix_blocks = static_cast<uint32_t>(blocks <= kMaxBlocks ? blocks : 0);
  blocks += a.w.num_items * hkv * a.suffix_splits;
  if (blocks > kMaxBlocks) return fail(RLK_EINVAL, "%s: %d items exceed one launch; split the call", what, a.w.num_items);
  shared_attention_kernel<D, kFmt><<<static_cast<uint32_t>(blocks), kThreads, 0, stream>>>(a);
  shared_merge_kernel<D><<<dim3(a.w.num_items, a.p.num_heads), D, 0, stream>>>(a);
  return launch_status(what);
}

}  // namespace
}  // namespace rlk

using namespace rlk;

extern "C" int rlk_paged_attention_decode_shared(const rlk_attention_params* p, const rlk_shared_prefix_work* w,
                                                 const rlk_attention_options* options, hipStream_t stream) {
  const char* what = "paged_attention_decode_shared";
  if (p == nullptr || w == nullptr) return fail(RLK_EINVAL, "%s: null params or work", what);
  if (w->num_items <= 0) return RLK_OK;
  const int scale_dtype = options != nullptr ? options->scale_dtype : RLK_SCALE_F32;
  const rlk_kv_layer_view& kv = p->kv;
  if (scale_dtype != RLK_SCALE_F32 && scale_dtype != RLK_SCALE_F16)
    return fail(RLK_EINVAL, "%s: unknown scale dtype %d", what, scale_dtype);
  if (kv.head_dim != 64 && kv.head_dim != 128)
    return fail(RLK_EUNSUPPORTED, "%s: unsupported head_dim %d (supported: 64, 128)", what, kv.head_dim);
  if (kv.dtype != RLK_KV_FP16 && kv.dtype != RLK_KV_INT8)
    return fail(RLK_EINVAL, "%s: unknown KV dtype %d", what, kv.dtype);
  if (kv.num_kv_heads <= 0 || kv.block_size <= 0)
    return fail(RLK_EINVAL, "%s: bad kv head count %d or block size %d", what, kv.num_kv_heads, kv.block_size);
  if (p->num_heads <= 0 || p->num_heads % kv.num_kv_heads != 0)
    return fail(RLK_EINVAL, "%s: num_heads must be a multiple of num_kv_heads (%d, %d)", what, p->num_heads, kv.num_kv_heads);
  const int G = p->num_heads / kv.num_kv_heads;
  if (G > kMaxGroup) return fail(RLK_EUNSUPPORTED, "%s: unsupported GQA group size %d", what, G);
  if (p->max_blocks_per_seq <= 0 || static_cast<int64_t>(p->max_blocks_per_seq) * kv.block_size > (1 << 30))
    return fail(RLK_EINVAL, "%s: bad table width %d", what, p->max_blocks_per_seq);
  if (w->num_groups < 0 || w->max_group_items < 0)
    return fail(RLK_EINVAL, "%s: bad group counts (%d, %d)", what, w->num_groups, w->max_group_items);
  if (w->max_partitions < 1 || w->max_prefix_partitions < 0 || w->max_partitions > (1 << 20) ||
      w->max_prefix_partitions > (1 << 20))
    return fail(RLK_EINVAL, "%s: bad partition counts (%d, %d)", what, w->max_prefix_partitions, w->max_partitions);
  if (p->num_heads > 65535 || w->num_items > (1 << 20) || w->num_groups > (1 << 20))
    return fail(RLK_EINVAL, "%s: %d items in %d groups exceed one launch; split the call", what, w->num_items, w->num_groups);
  if (!(p->scale - p->scale == 0.f)) return fail(RLK_EINVAL, "%s: the scale is no finite number", what);
  if (p->q == nullptr || p->out == nullptr || p->block_tables == nullptr || p->positions == nullptr ||
      kv.k == nullptr || kv.v == nullptr || (kv.dtype == RLK_KV_INT8 && (kv.k_scale == nullptr || kv.v_scale == nullptr)) ||
      w->item_token == nullptr || w->item_seq == nullptr ||
      (w->num_groups > 0 && (w->group_start == nullptr || w->group_prefix == nullptr)))
    return fail(RLK_EINVAL, "%s: null pointer argument", what);
  if (w->ws_out == nullptr || w->ws_max == nullptr || w->ws_sum == nullptr)
    return fail(RLK_EINVAL, "%s: the workspace is required", what);
  if (p->q_stride % 8 != 0 || ((reinterpret_cast<uintptr_t>(p->q) | reinterpret_cast<uintptr_t>(p->out) |
                                reinterpret_cast<uintptr_t>(kv.k) | reinterpret_cast<uintptr_t>(kv.v) |
                                reinterpret_cast<uintptr_t>(w->ws_out)) & 15) != 0)
    return fail(RLK_EINVAL, "%s: q and out rows, cache planes and workspace must be 16-byte aligned (q_stride %d)", what,
                p->q_stride);
  SharedArgs a = {};
  a.p = *p;
  a.w = *w;
  while ((int64_t{1} << a.lbs) < kv.block_size) ++a.lbs;
  if ((int64_t{1} << a.lbs) != kv.block_size) {  // exact for keys below 2^31
    a.magic = static_cast<uint32_t>((int64_t{1} << (31 + a.lbs)) / kv.block_size + 1);
    --a.lbs;
  }
  a.grp = G;
  const int fmt = kv.dtype == RLK_KV_FP16 ? kF16 : (scale_dtype == RLK_SCALE_F16 ? kI8Half : kI8);
  if (kv.head_dim == 128) {
    if (fmt == kF16) return launch<128, kF16>(a, what, stream);
    return fmt == kI8 ? launch<128, kI8>(a, what, stream) : launch<128, kI8Half>(a, what, stream);
  }
  if (fmt == kF16) return launch<64, kF16>(a, what, stream);
  return fmt == kI8 ? launch<64, kI8>(a, what, stream) : launch<64, kI8Half>(a, what, stream);
}
