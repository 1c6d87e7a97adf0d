// The next token of each row of logits: temperature, top-k, top-p, min-p and the
// draw from one given random number, for gfx950.
//
// With the tokens in order of falling logit (ties: rising index) and w_j =
// exp((l_j - l_max) / T), what the three limits keep is always the first n of them,
// and the draw is the first whose running weight passes u times the kept weight.  So
// nothing is sorted: a histogram over bins of the value, with the count and the weight
// of each, leads to the one bin that a limit or the draw falls into, and only among
// that bin's tokens is the place sought.
//
//   bins      p = l c, c = 8 log2(e) / T in fp64; bin floor(p): an eighth of an octave of
//             weight.  A chunk of the row keeps the 384 bins (48 octaves) below its own
//             largest logit; chunks meet by their bins' whole-number distance.
//   weights   2^((p - floor(p) - 1/2) / 8) in fp64 by a polynomial of degree 5
//             (interpolated at the Chebyshev nodes, error 2^-41), as a whole number of
//             2^-34: sums of whole numbers do not depend on their order, so atomics give
//             the same bits at every call.  Count (15 bits) and weight (49) share one
//             64-bit LDS atomic.  fp32 exponentials would move a border of the running sum
//             by up to 1e-7 of the whole, and of rows with 10^5 tokens to draw from some
//             would change theirs.
//   kernel 1  one chunk of 8192 a workgroup: the logits are read once, and the places of
//             its tokens go out in the order of their bins, without those that top-k, or
//             min-p as the only limit, leaves out for certain.
//   kernel 2  one row a workgroup: chunks' bins summed and scanned, then for each limit
//             and the draw the bin and its tokens from the chunks' lists; narrowed to at most
//             128 by histograms of their keys (value, then index); of those every pair is
//             compared.
//   A row of at most one chunk is done by one workgroup, its list in LDS.
//
// Bound: kernel 1 by memory and by the vector and LDS operations of a token about equally
// (152064 fp32 logits x 256 rows: 56 us, 156 MB read and up to 100 MB written; with lists of a
// quarter of a chunk 45 us, but a row whose bin lies behind them takes 100 us from its
// logits); kernel 2 by its chain of scans and gathers, 13 us for one row of 32000, 28 for
// those 256.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>
#include <type_traits>

#include "device.hpp"
#include "redline_amd/rlk.h"
#include "status.hpp"

namespace rlk {
namespace {

typedef unsigned long long u64;

constexpr int kBins = 384;        // of a chunk and of a row: 48 octaves
constexpr int kPer = 16;          // logits of a thread
constexpr int kThreads = 512;
constexpr int kWaves = kThreads / kWave;
constexpr int kChunk = kThreads * kPer;
constexpr int kMaxVocab = 1 << 20;
constexpr int kMaxChunks = kMaxVocab / kChunk;
constexpr int kCountShift = 49;   // count above, weight in 2^-34 below
constexpr u64 kCountOne = u64{1} << kCountShift, kWeightMask = kCountOne - 1, kWeightOne = u64{1} << 34;
constexpr double kBinsPerNat = 11.541560327111707;  // 8 log2(e)
constexpr double kFarBins = 2251799813685248.0;     // 2^51: |l c| from here on is not binned

struct ChunkTop {
  float max;
  int index;  // the lowest with it, where the temperature asks for the largest
};

struct SampleArgs {
  rlk_sampling_work w;
  u64* hist;       // [rows, chunks, kBins]
  ChunkTop* top;   // [rows, chunks]
  uint16_t* start; // [rows, chunks, kBins] tokens before the bin
  uint16_t* list;  // [rows, chunks, kChunk] places in the chunk of its tokens, by bins
  int chunks;
};

// Order-preserving whole number of a logit; NaN as -infinity, -0 as +0.
__device__ __forceinline__ float clean(float l) { return l != l ? -INFINITY : l + 0.f; }
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t b = __builtin_bit_cast(uint32_t, l);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// Value and index as one number: larger for a larger value, then for a lower index.
__device__ __forceinline__ u64 rank_key(float l, int index) {
  return static_cast<u64>(key_of(clean(l))) << 32 | (0xffffffffu - static_cast<uint32_t>(index));
}
__device__ __forceinline__ float key_value(u64 k) { return value_of(static_cast<uint32_t>(k >> 32)); }
__device__ __forceinline__ int key_index(u64 k) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(k)); }

// Where a row's bins are: p = l c; far: |l_max c| is too large to bin (a tiny
// temperature or an infinite logit), only logits equal to the largest have weight.
struct Scale {
  double c;
  __device__ explicit Scale(float temperature) : c(kBinsPerNat / static_cast<double>(temperature)) {}
  __device__ bool far(float l) const { return !(__builtin_fabs(static_cast<double>(l) * c) < kFarBins); }
  __device__ double bin(float l) const { return __builtin_floor(static_cast<double>(l) * c); }
  // the weight of l over that of its bin's middle in 2^-34, below 2^52 in the bits of 2^52 + weight;
  // all weights carry one factor of 1 + 2.6e-11, with which the constant is a whole number
  __device__ u64 weight_bits(float l, double bin) const {
    const double f = __builtin_fma(static_cast<double>(l), c, -bin);
    // (kept in scalar registers: as literals each would be moved into a vector register per use)
    double c5 = 699.1093111382294, c4 = 38597.3698262215, c3 = 1783466.322640276, c2 = 61751342.16030201;
    double c1 = 1425413776.8902755, c0 = 4503599627370496.0 + 16451499093.0;
    asm("" : "+s"(c5), "+s"(c4), "+s"(c3), "+s"(c2), "+s"(c1), "+s"(c0));
    double y = __builtin_fma(f, c5, c4);
    y = __builtin_fma(y, f, c3);
    y = __builtin_fma(y, f, c2);
    y = __builtin_fma(y, f, c1);
    return __builtin_bit_cast(u64, __builtin_fma(y, f, c0));
  }
  static constexpr u64 kBits = 0x4330000000000000ull;  // 2^52
  __device__ u64 weight(float l, double bin) const { return weight_bits(l, bin) - kBits; }
};

template <bool kF32>
__device__ __forceinline__ const void* row_of(const SampleArgs& a, int row) {
  return static_cast<const char*>(a.w.logits) + static_cast<int64_t>(row) * a.w.row_stride * (kF32 ? 4 : 2);
}
template <bool kF32>
__device__ __forceinline__ float logit(const void* row, int i) {
  if constexpr (kF32) return static_cast<const float*>(row)[i];
  else return static_cast<float>(static_cast<const _Float16*>(row)[i]);
}

// kPer logits a thread from `base` on: element j of the thread stands at
// index_of(base, tid, j), those at `stop` and behind are -infinity.
template <bool kF32>
struct ChunkLoad {
  static constexpr int kVec = kF32 ? 4 : 8;
  bool vec;
  __device__ ChunkLoad(const void* row) : vec((reinterpret_cast<uintptr_t>(row) & 15) == 0) {}
  __device__ int index_of(int base, int tid, int j) const {
    return vec ? base + (j / kVec * kThreads + tid) * kVec + j % kVec : base + j * kThreads + tid;
  }
  // index_of from element and thread as one number, element * kThreads + thread
  __device__ int index_of(int base, int place) const { return index_of(base, place % kThreads, place / kThreads); }
  __device__ void load(const void* row, int base, int tid, int stop, float (&l)[kPer]) const {
    if (vec) {
#pragma unroll
      for (int b = 0; b < kPer / kVec; ++b) {
        const int i = base + (b * kThreads + tid) * kVec;
        if (i + kVec <= stop) {
          if constexpr (kF32) {
            const f32x4 v = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(static_cast<const float*>(row) + i));
#pragma unroll
            for (int j = 0; j < 4; ++j) l[4 * b + j] = v[j];
          } else {
            const f32x8 v = unpack8(ld16<true>(reinterpret_cast<const u32x4*>(static_cast<const _Float16*>(row) + i)));
#pragma unroll
            for (int j = 0; j < 8; ++j) l[8 * b + j] = v[j];
          }
        } else {
#pragma unroll
          for (int j = 0; j < kVec; ++j) l[b * kVec + j] = i + j < stop ? logit<kF32>(row, i + j) : -INFINITY;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int i = base + j * kThreads + tid;
        l[j] = i < stop ? logit<kF32>(row, i) : -INFINITY;
      }
    }
  }
};

__device__ __forceinline__ float wave_max(float v) { return rows_max<true>(rows_max<false>(group_max<16>(v))); }

// Sum of v over the lanes before this one.
template <class T>
__device__ __forceinline__ T lanes_before(T v) {
  T incl = v;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const T y = __shfl_up(incl, o, kWave);
    if (static_cast<int>(threadIdx.x % kWave) >= o) incl += y;
  }
  return incl - v;
}

struct ChunkLds {
  u64 hist[kBins + kWave];  // (one a lane for what has no bin, so that no lane branches)
  float max[kWaves];
  int index[kWaves];
};

// A token's bin below the chunk's largest (kBins and above: none) and its place among those
// of the bin, in any order: the count that its atomic found.
struct Place {
  uint32_t bits;
  __device__ void set(int bin, u64 found) { bits = static_cast<uint32_t>(found >> kCountShift) << 16 | static_cast<uint32_t>(bin); }
  __device__ int bin() const { return static_cast<int>(bits & 0xffffu); }
  __device__ int place() const { return static_cast<int>(bits >> 16); }
};

// The logits of a chunk in registers, their places and the chunk's histogram.  False: no bins
// are asked for.
template <bool kF32>
__device__ __forceinline__ bool bin_chunk(const void* src, int base, int vocab, float T, ChunkLds& s,
                                          float (&l)[kPer], Place (&d)[kPer], ChunkTop* top) {
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const ChunkLoad<kF32> ld(src);
  ld.load(src, base, tid, vocab, l);
  for (int i = tid; i < kBins; i += kThreads) s.hist[i] = 0;
  float mx = -INFINITY;
#pragma unroll
  for (int j = 0; j < kPer; ++j) mx = fmaxf(mx, l[j]);  // (passes NaN by)
  mx = wave_max(mx);
  if (lane == 0) s.max[wave] = mx;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < kWaves; ++v) mx = fmaxf(mx, s.max[v]);
  *top = {mx, base};
  if (mx == -INFINITY) return false;
  if (!(T > 0.f)) {
    int at = INT_MAX;
#pragma unroll
    for (int j = 0; j < kPer; ++j) at = l[j] == mx ? min(at, ld.index_of(base, tid, j)) : at;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) at = min(at, __shfl_xor(at, o, kWave));
    if (lane == 0) s.index[wave] = at;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < kWaves; ++v) at = min(at, s.index[v]);
    top->index = at;
    return false;
  }
  const Scale sc(T);
  if (sc.far(mx)) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int bin = l[j] == mx ? 0 : kBins + lane;
      d[j].set(bin, atomicAdd(&s.hist[bin], kCountOne + kWeightOne));
    }
  } else {
    const double first = sc.bin(mx);
    constexpr int kAtOnce = 4;  // weights outside the branches, so that their chains overlap
#pragma unroll
    for (int j0 = 0; j0 < kPer; j0 += kAtOnce) {
      u64 w[kAtOnce], found[kAtOnce];
      int bin[kAtOnce];
#pragma unroll
      for (int x = 0; x < kAtOnce; ++x) {
        const double b = sc.bin(l[j0 + x]), below = first - b;
        bin[x] = below < kBins ? static_cast<int>(below) : kBins + lane;  // (none for NaN)
        w[x] = sc.weight_bits(l[j0 + x], b) + (kCountOne - Scale::kBits);
      }
#pragma unroll
      for (int x = 0; x < kAtOnce; ++x) found[x] = atomicAdd(&s.hist[bin[x]], w[x]);
#pragma unroll
      for (int x = 0; x < kAtOnce; ++x) d[j0 + x].set(bin[x], found[x]);
    }
  }
  __syncthreads();
  return true;
}

template <bool kF32>
__global__ __launch_bounds__(kThreads) void sample_chunks_kernel(SampleArgs a) {
  constexpr int kScan = kBins / 2;  // threads that scan, two bins each
  __shared__ ChunkLds s;
  __shared__ alignas(16) uint16_t list[kChunk];
  __shared__ int first[kBins];  // tokens before the bin
  __shared__ int wave_sum[kScan / kWave];
  __shared__ int listed[2];  // bins and tokens of the list
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks, base = chunk * kChunk;
  const void* src = row_of<kF32>(a, row);
  const int pr = a.w.param_row != nullptr ? a.w.param_row[row] : row;
  const float T = a.w.temperature[pr], least = a.w.min_p != nullptr ? fminf(a.w.min_p[pr], 1.f) : 0.f;
  // Bins behind top_k of the chunk's tokens are not listed; nor, where min_p is the only limit,
  // those of less than min_p of the chunk's largest (two more: one for the largest's place in its
  // own bin, one for the logarithm's error).
  const int k = a.w.top_k[pr], most = k > 0 ? k : kChunk;
  const bool cut = least > 0.f && k <= 0 && !(a.w.top_p[pr] < 1.f);
  const int bins = cut ? static_cast<int>(fminf(-8.f * __log2f(least), 1e4f)) + 3 : kBins;
  const int64_t rec = static_cast<int64_t>(row) * a.chunks + chunk;
  float l[kPer];
  Place d[kPer];
  ChunkTop top;
  if (tid == 0) listed[0] = min(bins, kBins);
  const bool binned = bin_chunk<kF32>(src, base, a.w.vocab, T, s, l, d, &top);
  if (tid == 0) a.top[rec] = top;
  if (!binned) return;
  int c0 = 0, c1 = 0, before = 0;
  if (tid < kScan) {
    const u64 h0 = s.hist[2 * tid], h1 = s.hist[2 * tid + 1];
    a.hist[rec * kBins + 2 * tid] = h0;
    a.hist[rec * kBins + 2 * tid + 1] = h1;
    c0 = static_cast<int>(h0 >> kCountShift);
    c1 = static_cast<int>(h1 >> kCountShift);
    before = lanes_before(c0 + c1);
    if (lane == kWave - 1) wave_sum[wave] = before + c0 + c1;
  }
  __syncthreads();
  if (tid < kScan) {
#pragma unroll
    for (int v = 0; v < kScan / kWave; ++v) before += v < wave ? wave_sum[v] : 0;
    const int mid = before + c0, end = mid + c1;
    first[2 * tid] = before;
    first[2 * tid + 1] = mid;
    reinterpret_cast<uint32_t*>(a.start + rec * kBins)[tid] = static_cast<uint32_t>(before) | static_cast<uint32_t>(mid) << 16;
    // the first bin that is not listed: `most` tokens stand before it
    if (before < most && end >= most) atomicMin(&listed[0], mid >= most ? 2 * tid + 1 : 2 * tid + 2);
  }
  __syncthreads();
  const int nb = listed[0];
  if (tid == (nb - 1) / 2) listed[1] = before + c0 + ((nb & 1) != 0 ? 0 : c1);
#pragma unroll
  for (int j = 0; j < kPer; ++j)
    if (d[j].bin() < nb) list[first[d[j].bin()] + d[j].place()] = static_cast<uint16_t>(j * kThreads + tid);
  __syncthreads();
  const int nt = listed[1];
  u32x4* dst = reinterpret_cast<u32x4*>(a.list + rec * kChunk);
  for (int i = tid; 8 * i < nt; i += kThreads) dst[i] = reinterpret_cast<const u32x4*>(list)[i];
}

// ---- the rows

constexpr int kList = 1024;   // tokens of a bin that are kept in LDS
constexpr int kDigitBits = 10, kDigits = 1 << kDigitBits;  // classes of a narrowing
constexpr int kFew = 128;     // tokens of which all pairs are compared
constexpr int kGroup = 16;    // lanes that read a chunk's list

struct RowLds {
  ChunkLds chunk;              // kOne: of the row
  uint16_t place[kChunk];      // kOne: the row's tokens in the order of their bins
  u64 key[kList + kFew], weight[kList + kFew];  // the tokens of one bin; from kList on what is left of a bin
  u64 few_upto[kFew];
  int few_place[kFew], few_bin[kFew];
  u64 digit_weight[kDigits];
  int digit_count[kDigits];
  double mass[kBins + 1];      // weight before bin j
  int count[kBins + 1];        // tokens before bin j
  double bin_scale[kBins];     // of whole-number weights
  int shift[kMaxChunks];       // of a chunk's bins; kBins: none
  int n;
  u64 top[kWaves];
  u64 wave_u64[kWaves];
  double wave_f64[kWaves];
  int wave_int[kWaves];
  int wave_bin[2][kWaves];
  u64 found_key, found_weight;
  int found, found_count;
};

// What is looked for: the first token whose place (from 1) is `most` or whose running mass
// passes the target (reaches it, if not strict); or, with least > 0, all tokens whose weight
// is at least that of the largest.
struct Goal {
  int most;
  double target;
  bool strict;
  double least;
  __device__ bool met(int place, double mass) const {
    return place >= most || (strict ? mass > target : mass >= target);
  }
};

template <bool kF32, bool kOne>
struct RowSampler {
  RowLds& s;
  const SampleArgs& a;
  const void* src;
  int row, tid, lane, wave;
  Scale sc;
  double per_bin;    // 1 / sc.c
  bool far;
  float mx;
  double first;      // bin of mx
  int cached = -1;   // the bin in s.key
  int turn = 0;      // of find_bin

  __device__ u64 weight(float v) const { return far ? kWeightOne : sc.weight(v, sc.bin(v)); }

  // Every token of the bin (kAll: of all bins up to it) to f(key); by all threads.
  template <bool kAll = false, class F>
  __device__ void each(int bin, F f) {
    const ChunkLoad<kF32> ld(src);
    if constexpr (kOne) {
      for (int i = (kAll ? 0 : s.count[bin]) + tid; i < s.count[bin + 1]; i += kThreads) {
        const int at = ld.index_of(0, s.place[i]);
        f(rank_key(logit<kF32>(src, at), at));
      }
    } else {
      for (int c = tid / kGroup; c < a.chunks; c += kThreads / kGroup) {
        const int b = bin - s.shift[c];
        if (b < 0) continue;  // (no bins: shift kBins)
        const int64_t rec = static_cast<int64_t>(row) * a.chunks + c;
        const int n = static_cast<int>(a.hist[rec * kBins + b] >> kCountShift), at = a.start[rec * kBins + b];
        const uint16_t* list = a.list + rec * kChunk;
        constexpr int kUnroll = 4;
        for (int i0 = (kAll ? 0 : at) + tid % kGroup; i0 < at + n; i0 += kUnroll * kGroup) {
          int index[kUnroll];
          float v[kUnroll];
#pragma unroll
          for (int x = 0; x < kUnroll; ++x) index[x] = ld.index_of(c * kChunk, list[min(i0 + x * kGroup, at + n - 1)]);
#pragma unroll
          for (int x = 0; x < kUnroll; ++x) v[x] = logit<kF32>(src, index[x]);
#pragma unroll
          for (int x = 0; x < kUnroll; ++x)
            if (i0 + x * kGroup < at + n) f(rank_key(v[x], index[x]));
        }
      }
    }
  }

  // Sums of v and c before this thread's, over the workgroup.
  __device__ void scan(u64& v, int& c) {
    const u64 vb = lanes_before(v);
    const int cb = lanes_before(c);
    __syncthreads();
    if (lane == kWave - 1) {
      s.wave_u64[wave] = vb + v;
      s.wave_int[wave] = cb + c;
    }
    __syncthreads();
    v = vb;
    c = cb;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      v += w < wave ? s.wave_u64[w] : 0;
      c += w < wave ? s.wave_int[w] : 0;
    }
  }

  // Of each of n <= kFew tokens in s.key from at0 on its place among them and the weight up to and
  // with it (kBinned: of its bin's), in s.few_place and s.few_upto; the threads share a token's pairs.
  template <bool kBinned>
  __device__ void compare(int at0, int n) {
    __syncthreads();
    if (tid < kFew) {
      s.few_upto[tid] = 0;
      s.few_place[tid] = 0;
    }
    __syncthreads();
    const int span = n <= kWave ? kWave : kFew, i = tid % span;
    const int parts = kThreads / span, per = (n + parts - 1) / parts;
    if (i < n) {
      const int j0 = tid / span * per, j1 = min(j0 + per, n), bin = kBinned ? s.few_bin[i] : 0;
      const u64 mine = s.key[at0 + i];
      u64 w = 0;
      int c = 0;
      for (int j = j0; j < j1; ++j) {
        const bool in = s.key[at0 + j] >= mine;
        w += in && (!kBinned || s.few_bin[j] == bin) ? s.weight[at0 + j] : 0;
        c += in;
      }
      if (c != 0) {
        atomicAdd(&s.few_upto[i], w);
        atomicAdd(&s.few_place[i], c);
      }
    }
    __syncthreads();
  }

  // The limits from `step` on and the draw, of `kept` tokens of weight Z, where the tokens up to the bin are
  // few: by one wave, two tokens a lane.
  __device__ void finish_few(int step, int bin, int k, float top_p, float least, float u, int kept, double Z) {
    __syncthreads();
    if (tid == 0) s.n = 0;
    __syncthreads();
    each<true>(bin, [&](u64 key) {
      const int at = atomicAdd(&s.n, 1);
      if (at < kFew) {
        const float v = key_value(key);
        s.key[at] = key;
        s.weight[at] = weight(v);
        s.few_bin[at] = far ? 0 : static_cast<int>(first - sc.bin(v));
      }
    });
    const int n = s.count[bin + 1];
    compare<true>(0, n);
    if (wave != 0) return;
    int place[2];
    double upto[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int t = min(lane + e * kWave, n - 1), b = s.few_bin[t];
      place[e] = lane + e * kWave < n ? s.few_place[t] : INT_MAX;
      upto[e] = s.mass[b] + static_cast<double>(s.few_upto[t]) * s.bin_scale[b];
    }
    auto lane_of = [&](int c, int* e) {  // of the token with this place
      const uint64_t b0 = __ballot(place[0] == c), b1 = __ballot(place[1] == c);
      *e = b0 == 0;
      return b0 != 0 ? __builtin_ctzll(b0) : (b1 != 0 ? __builtin_ctzll(b1) : 0);
    };
    auto mass_to = [&](int c) {
      int e;
      const int at = lane_of(c, &e);
      return __shfl(e == 0 ? upto[0] : upto[1], at, kWave);
    };
    // The least place of which f holds, the last if of none, as in select: find_bin went by the scan's
    // mass up to the bin's end, which may lie a rounding above what its tokens add up to here.
    auto first_that = [&](auto f) {
      int c = min(f(place[0], upto[0]) ? place[0] : INT_MAX, f(place[1], upto[1]) ? place[1] : INT_MAX);
#pragma unroll
      for (int o = 1; o < kWave; o <<= 1) c = min(c, __shfl_xor(c, o, kWave));
      return min(c, n);
    };
    if (step == 0) {
      kept = k;
      Z = mass_to(kept);
    }
    if (step <= 1 && top_p < 1.f) {
      const double target = static_cast<double>(top_p) * Z;
      kept = first_that([&](int c, double m) { return c >= kept || m >= target; });
      Z = mass_to(kept);
    }
    if (least > 0.f && !far) {
      int c = 0;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float v = key_value(s.key[min(lane + e * kWave, n - 1)]);
        c += __popcll(__ballot(place[e] <= kept && place[e] != INT_MAX &&
                               exp2((static_cast<double>(v) - mx) * sc.c * 0.125) >= static_cast<double>(least)));
      }
      if (c < kept) {
        kept = c;
        Z = mass_to(kept);
      }
    }
    const double target = static_cast<double>(u) * Z;
    int e;
    const int at = lane_of(first_that([&](int c, double m) { return c >= kept || m > target; }), &e);
    write(s.key[at + e * kWave], s.few_bin[at + e * kWave], Z);
  }

  // The row's results: the token drawn of `bin`, of tokens of weight Z.
  __device__ void write(u64 key, int bin, double Z) {
    if (tid != 0) return;
    a.w.tokens[row] = key_index(key);
    if (a.w.logprobs != nullptr) {
      // ln(own / Z) by the rest, which is exact where one token is left
      const double own = static_cast<double>(weight(key_value(key))) * s.bin_scale[bin];
      a.w.logprobs[row] = static_cast<float>(-log1p(fmax(Z - own, 0.0) / own));
    }
  }

  // The token of the bin that the goal (of places in the bin) is met by, the last if by none:
  // its place in *place, the mass up to and with it in *upto; its key by return.
  __device__ u64 select(int bin, const Goal& goal, int* place, double* upto) {
    enum { kCount, kSum, kKeep };
    const double scale = s.bin_scale[bin], before_bin = s.mass[bin];
    auto met = [&](int c, u64 w) { return goal.met(c, before_bin + static_cast<double>(w) * scale); };
    const int all = s.count[bin + 1] - s.count[bin];
    int n = all, skipped = 0;  // tokens that are left, those before them
    u64 skipped_w = 0;
    bool listed = cached == bin;  // they are in s.key
    int held = all, at0 = 0;      // tokens in s.key, the first that is left
    // keys of the values whose product with c lies in the bin, with a rounding's room
    u64 lo = 0, hi = ~u64{0};
    if (far) {
      lo = static_cast<u64>(key_of(mx)) << 32;
      hi = lo | 0xffffffffu;
    } else if (sc.c > 0.0) {  // (T infinite: all keys)
      const double v0 = (first - bin) * per_bin, v1 = (first - bin + 1.0) * per_bin;
      lo = static_cast<u64>(key_of(clean(static_cast<float>(v0 - __builtin_fabs(v0) * 0x1p-22 - 0x1p-140)))) << 32;
      hi = static_cast<u64>(key_of(clean(static_cast<float>(v1 + __builtin_fabs(v1) * 0x1p-22 + 0x1p-140)))) << 32 | 0xffffffffu;
    }
#pragma unroll 1
    for (int pass = 0; pass < 10; ++pass) {  // (64 bits, 10 a narrowing)
      const bool sums = goal.least > 0.0;
      if (listed && n == held && n <= kFew && !sums) break;
      const int mode = sums ? kSum : (n > (listed ? kFew : kList) ? kCount : kKeep);
      const int bits = 64 - __builtin_clzll((hi - lo) | 1), low = max(bits - kDigitBits, 0);
      const int keep = listed ? kList : 0, room = listed ? kFew : kList;
      __syncthreads();
      if (mode == kCount) {
        for (int i = tid; i < kDigits; i += kThreads) {
          s.digit_weight[i] = 0;
          s.digit_count[i] = 0;
        }
      }
      if (tid == 0) {
        s.n = 0;
        s.found_weight = 0;
        s.found_count = 0;
      }
      __syncthreads();
      u64 wsum = 0;
      int csum = 0;
      auto take = [&](u64 k, u64 w) {
        if (k < lo || k > hi) return;
        if (mode == kCount) {
          const int x = static_cast<int>((hi - k) >> low);  // falling keys
          atomicAdd(&s.digit_weight[x], w);
          atomicAdd(&s.digit_count[x], 1);
        } else if (mode == kKeep) {
          const int at = atomicAdd(&s.n, 1);
          if (at < room) {
            s.key[keep + at] = k;
            s.weight[keep + at] = w;
          }
        } else if (exp2((static_cast<double>(key_value(k)) - mx) * sc.c * 0.125) >= goal.least) {
          wsum += w;
          ++csum;
        }
      };
      if (listed) {
        for (int i = tid; i < held; i += kThreads) take(s.key[i], s.weight[i]);
      } else {
        each(bin, [&](u64 k) { take(k, weight(key_value(k))); });
      }
      if (mode == kSum) {
        if (csum != 0) {
          atomicAdd(&s.found_weight, wsum);
          atomicAdd(&s.found_count, csum);
        }
        __syncthreads();
        *place = s.found_count;
        *upto = before_bin + static_cast<double>(s.found_weight) * scale;
        return 0;
      }
      __syncthreads();
      if (mode == kKeep) {
        if (listed) {
          at0 = kList;
          break;
        }
        listed = true;
        held = n;
        cached = n == all ? bin : -1;
        continue;
      }
      constexpr int kEach = kDigits / kThreads;
      int cb = 0;
      u64 wb = 0;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        wb += s.digit_weight[tid * kEach + e];
        cb += s.digit_count[tid * kEach + e];
      }
      scan(wb, cb);
      wb += skipped_w;
      cb += skipped;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int x = tid * kEach + e, cn = s.digit_count[x];
        const u64 wn = s.digit_weight[x];
        if (cn != 0 && !(cb > 0 && met(cb, wb)) && (met(cb + cn, wb + wn) || cb + cn == skipped + n)) {
          s.found = x;
          s.found_weight = wb;
          s.found_count = cb;
          s.n = cn;
        }
        cb += cn;
        wb += wn;
      }
      __syncthreads();
      hi -= static_cast<u64>(s.found) << low;
      if (const u64 end = hi - ((u64{1} << low) - 1); end > lo && end <= hi) lo = end;
      skipped = s.found_count;
      skipped_w = s.found_weight;
      n = s.n;
    }
    n = min(n, kFew);
    compare<false>(at0, n);
    if (tid < n) {
      const int at = skipped + s.few_place[tid];
      const u64 w = skipped_w + s.few_upto[tid];
      if ((met(at, w) || at == skipped + n) && !(at > 1 && met(at - 1, w - s.weight[at0 + tid]))) {
        s.found = at;
        s.found_weight = w;
        s.found_key = s.key[at0 + tid];
      }
    }
    __syncthreads();
    *place = s.found;
    *upto = before_bin + static_cast<double>(s.found_weight) * scale;
    return s.found_key;
  }

  // The first bin that has tokens and meets the goal (of places in the row), the last if none.
  __device__ int find_bin(const Goal& goal) {
    uint64_t hit = 0;
    if (tid < kBins) {
      const int c0 = s.count[tid], c1 = s.count[tid + 1];
      hit = __ballot(c1 > c0 && (goal.met(c1, s.mass[tid + 1]) || c1 == s.count[kBins]));
    }
    int* out = s.wave_bin[turn];  // (the call before the last has been read by all)
    turn ^= 1;
    if (lane == 0) out[wave] = hit != 0 ? wave * kWave + __builtin_ctzll(hit) : kBins - 1;
    __syncthreads();
    int b = kBins - 1;
#pragma unroll
    for (int w = 0; w < kBins / kWave; ++w) b = min(b, out[w]);
    return b;
  }
};

template <bool kF32, bool kOne>
__global__ __launch_bounds__(kThreads) void sample_rows_kernel(SampleArgs a) {
  __shared__ RowLds s;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, row = blockIdx.x;
  const int pr = a.w.param_row != nullptr ? a.w.param_row[row] : row;
  const float T = a.w.temperature[pr];
  const int k = a.w.top_k[pr];
  const float top_p = a.w.top_p[pr], least = a.w.min_p != nullptr ? fminf(a.w.min_p[pr], 1.f) : 0.f;
  float u = a.w.uniform[row];
  u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;  // (NaN: 0)
  float l[kPer];
  Place d[kPer];
  float mx;
  int top_index;
  if constexpr (kOne) {
    ChunkTop t;
    bin_chunk<kF32>(row_of<kF32>(a, row), 0, a.w.vocab, T, s.chunk, l, d, &t);
    mx = t.max;
    top_index = t.index;
  } else {
    u64 top = 0;
    if (tid < a.chunks) {
      const ChunkTop t = a.top[static_cast<int64_t>(row) * a.chunks + tid];
      top = rank_key(t.max, t.index);
      s.shift[tid] = __builtin_bit_cast(int, t.max);
    }
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) top = max(top, static_cast<u64>(__shfl_xor(top, o, kWave)));
    if (lane == 0) s.top[wave] = top;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < kWaves; ++v) top = max(top, s.top[v]);
    mx = key_value(top);
    top_index = key_index(top);
  }
  if (!(T > 0.f) || mx == -INFINITY) {
    if (tid == 0) {
      a.w.tokens[row] = top_index;
      if (a.w.logprobs != nullptr) a.w.logprobs[row] = 0.f;
    }
    return;
  }
  const Scale sc(T);
  const bool far = sc.far(mx);
  const double first = far ? 0.0 : sc.bin(mx);
  u64 w = 0;
  int n = 0;
  if constexpr (kOne) {
    if (tid < kBins) {
      w = s.chunk.hist[tid] & kWeightMask;
      n = static_cast<int>(s.chunk.hist[tid] >> kCountShift);
    }
  } else {
    if (tid < a.chunks) {
      const float m = __builtin_bit_cast(float, s.shift[tid]);
      int shift = kBins;
      if (far) {
        shift = m == mx ? 0 : kBins;
      } else if (m != -INFINITY && !sc.far(m)) {  // (a chunk too low to bin is far below the row's largest)
        const double x = first - sc.bin(m);
        shift = x < kBins ? static_cast<int>(x) : kBins;
      }
      s.shift[tid] = shift;
    }
    __syncthreads();
    if (tid < kBins) {
      const u64* h = a.hist + static_cast<int64_t>(row) * a.chunks * kBins;
      constexpr int kUnroll = 16;
      for (int c0 = 0; c0 < a.chunks; c0 += kUnroll) {
        u64 v[kUnroll];
#pragma unroll
        for (int x = 0; x < kUnroll; ++x) {
          // (a chunk without bins has no histogram; its place in the workspace is read all the same)
          const int c = min(c0 + x, a.chunks - 1);
          v[x] = h[c * kBins + max(tid - s.shift[c], 0)];
        }
#pragma unroll
        for (int x = 0; x < kUnroll; ++x) {
          const int c = min(c0 + x, a.chunks - 1);
          if (c0 + x < a.chunks && tid >= s.shift[c]) {
            w += v[x] & kWeightMask;
            n += static_cast<int>(v[x] >> kCountShift);
          }
        }
      }
    }
  }
  // running counts and masses; the order of the sums is fixed
  double scale = 0.0;
  if (tid < kBins) {
    scale = ((tid & 1 ? 0.91700404320467123 : 1.0) * (tid & 2 ? 0.84089641525371454 : 1.0)) * (tid & 4 ? 0.70710678118654752 : 1.0);
    scale = ldexp(scale, -(tid >> 3) - 34);
    s.bin_scale[tid] = scale;
  }
  double mass = static_cast<double>(w) * scale;
  int count = n;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const double y = __shfl_up(mass, o, kWave);
    const int z = __shfl_up(count, o, kWave);
    if (lane >= o) {
      mass += y;
      count += z;
    }
  }
  if (lane == kWave - 1) {
    s.wave_f64[wave] = mass;
    s.wave_int[wave] = count;
  }
  __syncthreads();
  double before = 0.0;
  int cbefore = 0;
  for (int v = 0; v < wave; ++v) {
    before += s.wave_f64[v];
    cbefore += s.wave_int[v];
  }
  if (tid < kBins) {
    s.mass[tid + 1] = before + mass;
    s.count[tid + 1] = cbefore + count;
  }
  if (tid == 0) {
    s.mass[0] = 0.0;
    s.count[0] = 0;
  }
  __syncthreads();
  if constexpr (kOne) {  // all places in the order of the bins
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (d[j].bin() < kBins) s.place[s.count[d[j].bin()] + d[j].place()] = static_cast<uint16_t>(j * kThreads + tid);
    __syncthreads();
  }

  RowSampler<kF32, kOne> rs{s, a, row_of<kF32>(a, row), row, tid, lane, wave, sc, T / kBinsPerNat, far, mx, first};
  int kept = s.count[kBins], bin = 0;
  double Z = s.mass[kBins];
  u64 key = 0;
  // the limits in turn, then the draw: one loop, since the code is fetched for every row anew
#pragma unroll 1
  for (int step = 0; step < 4; ++step) {
    Goal goal = {INT_MAX, 0.0, true, 0.0};
    if (step == 0) {
      if (k <= 0 || k >= kept) continue;
      goal.most = k;
      goal.target = __builtin_inf();
    } else if (step == 1) {
      if (!(top_p < 1.f)) continue;
      goal = {kept, static_cast<double>(top_p) * Z, false, 0.0};
    } else if (step == 2) {
      if (!(least > 0.f) || far) continue;
      // the bin that the least weight falls into
      const double x = first - __builtin_floor(__builtin_fma(static_cast<double>(mx), sc.c, 8.0 * log2(static_cast<double>(least))));
      if (!(x < kBins) || s.count[static_cast<int>(x)] >= kept) continue;
      bin = static_cast<int>(x);
      goal.least = least;
    } else {
      goal = {kept, static_cast<double>(u) * Z, true, 0.0};
    }
    if (step != 2) bin = rs.find_bin(goal);
    if (step < 3 && s.count[bin + 1] <= kFew) {
      rs.finish_few(step, bin, k, top_p, least, u, kept, Z);
      return;
    }
    const int base = s.count[bin];
    if (step == 0 && s.count[bin + 1] == k) {
      kept = k;
      Z = s.mass[bin + 1];
      continue;
    }
    goal.most = min(goal.most, s.count[bin + 1]) - base;
    int place;
    double upto;
    key = rs.select(bin, goal, &place, &upto);
    if (step < 3 && base + place <= kept) {
      kept = base + place;
      Z = upto;
    }
  }
  rs.write(key, bin, Z);
}

int chunks_of(int vocab) { return (vocab + kChunk - 1) / kChunk; }

// Where a call's records stand in its workspace; its size.
size_t layout(int64_t rows, int vocab, SampleArgs* a) {
  const size_t recs = static_cast<size_t>(rows) * chunks_of(vocab);
  size_t n = 0;
  auto take = [&](auto*& p, size_t count) {
    if (a != nullptr) p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(static_cast<char*>(a->w.workspace) + n);
    n += (count * sizeof(*p) + 255) / 256 * 256;
  };
  SampleArgs none;
  SampleArgs& to = a != nullptr ? *a : none;
  take(to.hist, recs * kBins);
  take(to.top, recs);
  take(to.start, recs * kBins);
  take(to.list, recs * kChunk);
  return n;
}

template <bool kF32>
void launch(const SampleArgs& a, hipStream_t stream) {
  if (a.chunks == 1) {
    sample_rows_kernel<kF32, true><<<a.w.num_rows, kThreads, 0, stream>>>(a);
    return;
  }
  sample_chunks_kernel<kF32><<<static_cast<uint32_t>(a.w.num_rows) * a.chunks, kThreads, 0, stream>>>(a);
  sample_rows_kernel<kF32, false><<<a.w.num_rows, kThreads, 0, stream>>>(a);
}

}  // namespace
}  // namespace rlk

using namespace rlk;

extern "C" size_t rlk_sampling_workspace_bytes(int max_rows, int max_vocab) {
  if (max_rows <= 0 || max_vocab <= 0 || max_vocab > kMaxVocab) return 0;
  return layout(max_rows, max_vocab, nullptr);
}

extern "C" int rlk_sample_tokens(const rlk_sampling_work* w, hipStream_t stream) {
  const char* what = "sample_tokens";
  if (w == nullptr) return fail(RLK_EINVAL, "%s: null work", what);
  if (w->num_rows <= 0) return RLK_OK;
  if (w->vocab <= 0 || w->vocab > kMaxVocab)
    return fail(RLK_EUNSUPPORTED, "%s: unsupported vocabulary of %d (1 .. %d)", what, w->vocab, kMaxVocab);
  if (w->logits == nullptr || w->temperature == nullptr || w->top_k == nullptr || w->top_p == nullptr ||
      w->uniform == nullptr || w->tokens == nullptr || w->workspace == nullptr)
    return fail(RLK_EINVAL, "%s: null pointer argument", what);
  if (w->row_stride < w->vocab && w->num_rows > 1)
    return fail(RLK_EINVAL, "%s: rows of %d logits overlap at a stride of %lld", what, w->vocab, static_cast<long long>(w->row_stride));
  if ((reinterpret_cast<uintptr_t>(w->logits) & (w->logits_fp32 ? 3 : 1)) != 0)
    return fail(RLK_EINVAL, "%s: logits must be aligned to their elements", what);
  if ((reinterpret_cast<uintptr_t>(w->workspace) & 255) != 0)
    return fail(RLK_EINVAL, "%s: the workspace must be 256-byte aligned", what);
  const size_t need = layout(w->num_rows, w->vocab, nullptr);
  if (w->workspace_bytes < need)
    return fail(RLK_EINVAL, "%s: a workspace of %zu bytes, needs %zu", what, w->workspace_bytes, need);
  SampleArgs a;
  a.w = *w;
  a.chunks = chunks_of(w->vocab);
  if (static_cast<int64_t>(w->num_rows) * a.chunks * kThreads > UINT32_MAX)
    return fail(RLK_EINVAL, "%s: %d rows exceed one launch; split the call", what, w->num_rows);
  layout(w->num_rows, w->vocab, &a);
  w->logits_fp32 ? launch<true>(a, stream) : launch<false>(a, stream);
  return launch_status(what);
}
