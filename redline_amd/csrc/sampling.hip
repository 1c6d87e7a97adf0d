// The next token of each row of logits: temperature, top-k, top-p, min-p and the
// draw from one given random number, for gfx950.
//
// With the tokens in order of falling logit (ties: rising index) and w_j =
// exp((l_j - l_max) / T), what the three limits keep is always the first n of them,
// and the draw is the first whose running weight passes u times the kept weight.  So
// nothing is sorted: a histogram over bins of the value, with the count and the weight
// of each, leads to the one bin that a limit or the draw falls into, and only that
// bin's tokens are put in order.
//
//   bins      p = l c, c = 8 log2(e) / T in fp64; bin floor(p): an eighth of an octave of
//             weight.  A chunk of the row keeps the 384 bins (48 octaves) below its own
//             largest logit; chunks meet by their bins' whole-number distance.
//   weights   2^((p - floor(p) - 1/2) / 8) in fp64 by a polynomial of degree 6 (|x| <
//             0.0434, error 6e-14), then rounded to a whole number of 2^-34: sums of whole
//             numbers do not depend on their order, so atomics give the same bits at
//             every call.  Count (15 bits) and weight (49) share one 64-bit LDS atomic.
//             fp32 exponentials would move a border of the running sum by up to 1e-7 of the
//             whole, and of rows with 10^5 tokens to draw from some would change theirs.
//   kernel 1  one chunk a workgroup: the logits are read once.
//   kernel 2  one row a workgroup: chunks' bins summed and scanned, then for each limit
//             and the draw the bin, its tokens gathered from the chunks that have some,
//             sorted in LDS (bitonic on value and index) and scanned.  A bin of more
//             than 2048 tokens is narrowed first, by digits of the value's bits.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "device.hpp"
#include "redline_amd/rlk.h"
#include "status.hpp"

namespace rlk {
namespace {

typedef unsigned long long u64;

constexpr int kBins = 384;        // of a chunk and of a row: 48 octaves
constexpr int kPer = 16;          // logits of a thread of kernel 1
constexpr int kSmallChunk = 256 * kPer, kLargeChunk = 1024 * kPer;
constexpr int kMaxVocab = 1 << 20;
constexpr int kMaxChunks = kMaxVocab / kSmallChunk;
constexpr int kCountShift = 49;   // count above, weight in 2^-34 below
constexpr u64 kWeightMask = (u64{1} << kCountShift) - 1;
constexpr double kOne = 17179869184.0;  // 2^34
constexpr double kBinsPerNat = 11.541560327111707;  // 8 log2(e)
constexpr double kFarBins = 2251799813685248.0;     // 2^51: |l c| from here on is not binned

struct ChunkTop {
  float max;
  int index;  // the lowest with it
};

struct SampleArgs {
  rlk_sampling_work w;
  ChunkTop* top;  // [rows, chunks]
  u64* hist;      // [rows, chunks, kBins]
  int chunk, chunks;
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

// Where a row's bins are: p = l c; far: |l_max c| is too large to bin (a tiny
// temperature or an infinite logit), only logits equal to the largest have weight.
struct Scale {
  double c;
  __device__ explicit Scale(float temperature) : c(kBinsPerNat / static_cast<double>(temperature)) {}
  __device__ bool far(float l) const { return !(__builtin_fabs(static_cast<double>(l) * c) < kFarBins); }
  __device__ double bin(float l) const { return __builtin_floor(static_cast<double>(l) * c); }
  // the weight of l over that of its bin's middle, in 2^-34
  __device__ u64 weight(float l, double bin) const {
    const double f = __builtin_fma(static_cast<double>(l), c, -(bin + 0.5));
    constexpr double a = 0.08664339756999316;  // ln(2) / 8
    double y = a * a * a * a * a * a / 720.0;
    y = __builtin_fma(y, f, a * a * a * a * a / 120.0);
    y = __builtin_fma(y, f, a * a * a * a / 24.0);
    y = __builtin_fma(y, f, a * a * a / 6.0);
    y = __builtin_fma(y, f, a * a / 2.0);
    y = __builtin_fma(y, f, a);
    y = __builtin_fma(y, f, 1.0);
    // adding 2^52 leaves the rounded whole number in the low bits
    return __builtin_bit_cast(u64, __builtin_fma(y, kOne, 4503599627370496.0)) - 0x4330000000000000ull;
  }
};

template <bool kF32>
__device__ __forceinline__ const void* row_of(const SampleArgs& a, int row) {
  return static_cast<const char*>(a.w.logits) + static_cast<int64_t>(row) * a.w.row_stride * (kF32 ? 4 : 2);
}
template <bool kF32>
__device__ __forceinline__ float logit(const void* row, int i) {
  if constexpr (kF32) return clean(static_cast<const float*>(row)[i]);
  else return clean(static_cast<float>(static_cast<const _Float16*>(row)[i]));
}

// The kPer logits of thread tid of a chunk that starts at `base`: element j of the
// thread stands at index_of(base, tid, j), tokens past the vocabulary are -infinity.
template <bool kF32, int kThreads>
struct ChunkLoad {
  static constexpr int kVec = kF32 ? 4 : 8;
  bool vec;
  __device__ ChunkLoad(const void* row) : vec((reinterpret_cast<uintptr_t>(row) & 15) == 0) {}
  __device__ int index_of(int base, int tid, int j) const {
    return vec ? base + (j / kVec * kThreads + tid) * kVec + j % kVec : base + j * kThreads + tid;
  }
  __device__ void load(const void* row, int base, int tid, int vocab, float (&l)[kPer]) const {
    if (vec) {
#pragma unroll
      for (int b = 0; b < kPer / kVec; ++b) {
        const int i = base + (b * kThreads + tid) * kVec;
        if (i + kVec <= vocab) {
          if constexpr (kF32) {
            const f32x4 v = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(static_cast<const float*>(row) + i));
#pragma unroll
            for (int j = 0; j < 4; ++j) l[4 * b + j] = clean(v[j]);
          } else {
            const f32x8 v = unpack8(__builtin_nontemporal_load(reinterpret_cast<const u32x4*>(static_cast<const _Float16*>(row) + i)));
#pragma unroll
            for (int j = 0; j < 8; ++j) l[8 * b + j] = clean(v[j]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < kVec; ++j) l[b * kVec + j] = i + j < vocab ? logit<kF32>(row, i + j) : -INFINITY;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int i = base + j * kThreads + tid;
        l[j] = i < vocab ? logit<kF32>(row, i) : -INFINITY;
      }
    }
  }
};

__device__ __forceinline__ u64 wave_max(u64 v) {
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) v = max(v, static_cast<u64>(__shfl_xor(v, o, kWave)));
  return v;
}
// Value and index as one number: larger for a larger value, then for a lower index.
__device__ __forceinline__ u64 rank_key(float l, int index) {
  return static_cast<u64>(key_of(l)) << 32 | (0xffffffffu - static_cast<uint32_t>(index));
}

template <bool kF32, int kThreads>
__global__ __launch_bounds__(kThreads) void sample_chunks_kernel(SampleArgs a) {
  constexpr int kWaves = kThreads / kWave;
  __shared__ u64 hist[kBins];
  __shared__ u64 tops[kWaves];
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks, base = chunk * kThreads * kPer;
  const void* src = row_of<kF32>(a, row);
  const ChunkLoad<kF32, kThreads> ld(src);
  float l[kPer];
  ld.load(src, base, tid, a.w.vocab, l);
  const float T = a.w.temperature[a.w.param_row != nullptr ? a.w.param_row[row] : row];
  for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
  u64 top = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) top = max(top, rank_key(l[j], ld.index_of(base, tid, j)));
  top = wave_max(top);
  if (lane == 0) tops[wave] = top;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < kWaves; ++v) top = max(top, tops[v]);
  const float mx = value_of(static_cast<uint32_t>(top >> 32));
  const int64_t rec = static_cast<int64_t>(row) * a.chunks + chunk;
  if (tid == 0) a.top[rec] = {mx, static_cast<int>(0xffffffffu - static_cast<uint32_t>(top))};
  if (!(T > 0.f) || mx == -INFINITY) return;  // no bins are asked for
  const Scale sc(T);
  if (sc.far(mx)) {
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (l[j] == mx) atomicAdd(&hist[0], (u64{1} << kCountShift) + (u64{1} << 34));
  } else {
    const double first = sc.bin(mx);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const double b = sc.bin(l[j]), d = first - b;
      if (d < kBins) atomicAdd(&hist[static_cast<int>(d)], sc.weight(l[j], b) + (u64{1} << kCountShift));
    }
  }
  __syncthreads();
  for (int i = tid; i < kBins; i += kThreads) a.hist[rec * kBins + i] = hist[i];
}

// ---- kernel 2

constexpr int kRowThreads = 512;
constexpr int kRowWaves = kRowThreads / kWave;
constexpr int kSort = 2048;   // tokens that are sorted in LDS
constexpr int kDigits = 2048;
constexpr int kSub = 1024;    // tokens of a stretch that one wave counts

struct RowLds {
  union {
    struct {
      u64 key[kSort];   // in order once sorted
      u64 upto[kSort];  // running weight
    } list;
    struct {
      u64 weight[kDigits];
      uint32_t count[kDigits];
    } digit;
    uint32_t ties[kMaxVocab / kSub];
  };
  double mass[kBins + 1];      // weight before bin j
  int count[kBins + 1];        // tokens before bin j
  double bin_scale[kBins];     // of whole-number weights
  int shift[kMaxChunks];       // of a chunk's bins; kBins: none
  int use[kMaxChunks];         // chunks that have tokens of the bin
  int n_use, n, at;
  u64 top[kRowWaves];
  u64 wave_u64[kRowWaves];
  double wave_f64[kRowWaves];
  int wave_int[kRowWaves];
  int found;
  double found_mass;
  uint32_t found_key;
  u64 found_base;
  int found_count;
};

// What a selection inside a bin looks for.
enum Seek { kRank, kReach, kPass };  // the r-th token; the first whose running mass >= / > the target

template <bool kF32>
struct RowSampler {
  RowLds& s;
  const SampleArgs& a;
  const void* src;
  int row, tid, lane, wave;
  Scale sc;
  bool far;
  float mx;
  double first;       // bin of mx
  int sorted_bin = -1, sorted_n = 0;

  __device__ u64 weight(float l) const { return far ? u64{1} << 34 : sc.weight(l, sc.bin(l)); }
  __device__ bool in_bin(float l, int bin) const { return far ? l == mx : first - sc.bin(l) == bin; }

  // Every token of the bin, chunk by chunk, to f(logit, index); by all threads.
  template <class F>
  __device__ void each(int bin, F f) {
    const int nu = s.n_use;
    for (int x = 0; x < nu; ++x) {
      const int base = s.use[x] * a.chunk, stop = min(base + a.chunk, a.w.vocab);
      constexpr int kUnroll = 8;
      for (int i0 = base + tid; i0 < stop; i0 += kUnroll * kRowThreads) {
        float l[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) l[u] = logit<kF32>(src, min(i0 + u * kRowThreads, stop - 1));
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (i0 + u * kRowThreads < stop && in_bin(l[u], bin)) f(l[u], i0 + u * kRowThreads);
      }
    }
  }
  // The chunks that have tokens of the bin.
  __device__ void find_chunks(int bin) {
    __syncthreads();
    if (tid == 0) s.n_use = 0;
    __syncthreads();
    for (int c = tid; c < a.chunks; c += kRowThreads) {
      const int b = bin - s.shift[c];
      if (s.shift[c] < kBins && b >= 0 && b < kBins &&
          a.hist[(static_cast<int64_t>(row) * a.chunks + c) * kBins + b] >> kCountShift != 0)
        s.use[atomicAdd(&s.n_use, 1)] = c;
    }
    __syncthreads();
  }
  // Sum of v before this thread's, over the workgroup; total in *all.
  __device__ u64 scan(u64 v, u64* all) {
    u64 incl = v;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const u64 y = __shfl_up(incl, o, kWave);
      if (lane >= o) incl += y;
    }
    __syncthreads();
    if (lane == kWave - 1) s.wave_u64[wave] = incl;
    __syncthreads();
    u64 before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < kRowWaves; ++w) {
      if (w < wave) before += s.wave_u64[w];
      sum += s.wave_u64[w];
    }
    *all = sum;
    return before + incl - v;
  }

  // The tokens of the bin whose key has the high bits of `prefix` (all bits above
  // `bits`), sorted, with their running weight, in s.list; n of them, n <= kSort.
  __device__ void sort_list(int bin, uint32_t prefix, int bits, int n) {
    __syncthreads();
    if (tid == 0) s.n = 0;
    __syncthreads();
    each(bin, [&](float l, int i) {
      if (bits < 32 && key_of(l) >> bits != prefix) return;
      const int at = atomicAdd(&s.n, 1);
      if (at < kSort) s.list.key[at] = rank_key(l, i);
    });
    int size = kWave;
    while (size < n) size *= 2;
    for (int i = n + tid; i < size; i += kRowThreads) s.list.key[i] = 0;
    __syncthreads();
    for (int k = 2; k <= size; k *= 2)
      for (int j = k / 2; j > 0; j /= 2) {
        for (int x = tid; x < size / 2; x += kRowThreads) {
          const int i = 2 * x - (x & (j - 1)), o = i + j;
          const u64 p = s.list.key[i], q = s.list.key[o];
          if ((p < q) == ((i & k) == 0)) {  // falling
            s.list.key[i] = q;
            s.list.key[o] = p;
          }
        }
        __syncthreads();
      }
    constexpr int kEach = kSort / kRowThreads;
    u64 v[kEach], sum = 0, all;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = tid * kEach + e;
      v[e] = i < n ? weight(value_of(static_cast<uint32_t>(s.list.key[i] >> 32))) : 0;
      sum += v[e];
    }
    u64 before = scan(sum, &all);
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      before += v[e];
      s.list.upto[tid * kEach + e] = before;
    }
    __syncthreads();
  }

  // Of the first `most` tokens of the bin, the one that `seek` looks for: its place
  // (from 1) in *place, the bin's mass up to and with it in *upto; its key and index
  // by return.  The last of them if none fits.
  __device__ u64 select(int bin, Seek seek, int rank, double target, int most, int* place, double* upto) {
    const double scale = s.bin_scale[bin], before_bin = s.mass[bin];
    int n = s.count[bin + 1] - s.count[bin], skipped = 0;
    u64 skipped_w = 0;
    uint32_t prefix = 0;
    int bits = 32;
    auto fits = [&](int c, u64 w) {  // the token with this place and running weight, or one before it
      if (c >= most) return true;
      const double mass = before_bin + static_cast<double>(w) * scale;
      return seek == kRank ? c >= rank : (seek == kReach ? mass >= target : mass > target);
    };
    const bool cached = sorted_bin == bin;
    if (!cached) {
      find_chunks(bin);
      while (n > kSort && bits > 0) {
        const int width = bits == 32 ? 11 : (bits == 21 ? 11 : 10), low = bits - width;
        __syncthreads();
        for (int i = tid; i < kDigits; i += kRowThreads) {
          s.digit.weight[i] = 0;
          s.digit.count[i] = 0;
        }
        __syncthreads();
        each(bin, [&](float l, int) {
          const uint32_t k = key_of(l);
          if (bits < 32 && k >> bits != prefix) return;
          const uint32_t d = (1u << width) - 1 - ((k >> low) & ((1u << width) - 1));  // falling
          atomicAdd(&s.digit.weight[d], weight(l));
          atomicAdd(&s.digit.count[d], 1u);
        });
        __syncthreads();
        constexpr int kEach = kDigits / kRowThreads;
        u64 wsum = 0, wall;
        int csum = 0;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
          wsum += s.digit.weight[tid * kEach + e];
          csum += s.digit.count[tid * kEach + e];
        }
        u64 wbefore = skipped_w + scan(wsum, &wall), call;
        int cbefore = skipped + static_cast<int>(scan(csum, &call));
        if (tid == 0) s.found = -1;
        __syncthreads();
        for (int e = 0; e < kEach; ++e) {
          const int d = tid * kEach + e, cn = s.digit.count[d];
          const u64 wn = s.digit.weight[d];
          if (cn != 0 && !(cbefore > 0 && fits(cbefore, wbefore)) &&
              (fits(cbefore + cn, wbefore + wn) || cbefore + cn == skipped + n)) {
            s.found = d;
            s.found_base = wbefore;
            s.found_count = cbefore;
            s.n = cn;
          }
          cbefore += cn;
          wbefore += wn;
        }
        __syncthreads();
        prefix = (bits == 32 ? 0u : prefix << width) | ((1u << width) - 1 - static_cast<uint32_t>(s.found));
        skipped = s.found_count;
        skipped_w = s.found_base;
        n = s.n;
        bits = low;
      }
      if (n > kSort) return select_tie(bin, prefix, n, skipped, skipped_w, seek, rank, target, most, place, upto);
      sort_list(bin, prefix, bits, n);
      if (bits == 32) {
        sorted_bin = bin;
        sorted_n = n;
      } else {
        sorted_bin = -1;
      }
    }
    __syncthreads();
    for (int i = tid; i < n; i += kRowThreads) {
      const u64 w = skipped_w + s.list.upto[i], w0 = skipped_w + (i > 0 ? s.list.upto[i - 1] : 0);
      const int at = skipped + i + 1;
      if ((fits(at, w) || i == n - 1) && !(i > 0 && fits(at - 1, w0))) {
        s.found = at;
        s.found_base = w;
        s.at = i;
      }
    }
    __syncthreads();
    *place = s.found;
    *upto = before_bin + static_cast<double>(s.found_base) * scale;
    const u64 key = s.list.key[s.at];
    __syncthreads();
    return key;
  }

  // More than kSort tokens of one value: the place by arithmetic, the token by counting
  // through the row.
  __device__ u64 select_tie(int bin, uint32_t key, int n, int skipped, u64 skipped_w, Seek seek, int rank, double target,
                            int most, int* place, double* upto) {
    const double scale = s.bin_scale[bin], before_bin = s.mass[bin];
    const float l = value_of(key);
    const u64 w = weight(l);
    auto fits = [&](int c) {
      if (c >= most) return true;
      const double mass = before_bin + static_cast<double>(skipped_w + static_cast<u64>(c - skipped) * w) * scale;
      return seek == kRank ? c >= rank : (seek == kReach ? mass >= target : mass > target);
    };
    int lo = skipped + 1, hi = skipped + n;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (fits(mid)) hi = mid; else lo = mid + 1;
    }
    *place = lo;
    *upto = before_bin + static_cast<double>(skipped_w + static_cast<u64>(lo - skipped) * w) * scale;
    const int want = lo - skipped;  // the want-th of them, by index
    const int V = a.w.vocab, subs = (V + kSub - 1) / kSub;
    auto is_tie = [&](int i) { return i < V && logit<kF32>(src, min(i, V - 1)) == l; };
    __syncthreads();
    for (int x = wave; x < subs; x += kRowWaves) {
      int c = 0;
#pragma unroll 4
      for (int b = 0; b < kSub; b += kWave) c += __popcll(__ballot(is_tie(x * kSub + b + lane)));
      if (lane == 0) s.ties[x] = c;
    }
    __syncthreads();
    if (tid == 0) {
      int c = 0, x = 0;
      while (x < subs - 1 && c + static_cast<int>(s.ties[x]) < want) c += s.ties[x++];
      s.at = x;
      s.found_count = c;
    }
    __syncthreads();
    if (wave == 0) {
      int c = s.found_count;
      const int x = s.at;
      int hit = -1;
      for (int b = 0; b < kSub && hit < 0; b += kWave) {
        const uint64_t t = __ballot(is_tie(x * kSub + b + lane));
        const int here = __popcll(t);
        if (c + here >= want) {
          const uint64_t below = t & ((2ull << lane) - 1);
          const uint64_t b1 = __ballot((t >> lane & 1) != 0 && c + static_cast<int>(__popcll(below)) == want);
          hit = x * kSub + b + (b1 != 0 ? __builtin_ctzll(b1) : 0);
        }
        c += here;
      }
      if (lane == 0) s.found = max(hit, 0);
    }
    __syncthreads();
    const int index = s.found;
    sorted_bin = -1;
    __syncthreads();
    return rank_key(l, index);
  }

  // The first bin of 0 .. kBins - 1 that has tokens and ends at or past the target.
  template <class F>
  __device__ int find_bin(F past) {
    __syncthreads();
    if (tid == 0) s.found = kBins - 1;
    __syncthreads();
    if (tid < kBins) {
      const int c0 = s.count[tid], c1 = s.count[tid + 1];
      if (c1 > c0 && (past(c1, s.mass[tid + 1]) || c1 == s.count[kBins])) atomicMin(&s.found, tid);
    }
    __syncthreads();
    const int b = s.found;
    __syncthreads();
    return b;
  }
};

template <bool kF32>
__global__ __launch_bounds__(kRowThreads) void sample_rows_kernel(SampleArgs a) {
  __shared__ RowLds s;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, row = blockIdx.x;
  const int pr = a.w.param_row != nullptr ? a.w.param_row[row] : row;
  const float T = a.w.temperature[pr];
  const ChunkTop* tops = a.top + static_cast<int64_t>(row) * a.chunks;
  u64 top = 0;
  for (int c = tid; c < a.chunks; c += kRowThreads) {
    const ChunkTop t = tops[c];
    top = max(top, rank_key(t.max, t.index));
  }
  top = wave_max(top);
  if (lane == 0) s.top[wave] = top;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < kRowWaves; ++v) top = max(top, s.top[v]);
  const float mx = value_of(static_cast<uint32_t>(top >> 32));
  if (!(T > 0.f) || mx == -INFINITY) {
    if (tid == 0) {
      a.w.tokens[row] = static_cast<int>(0xffffffffu - static_cast<uint32_t>(top));
      if (a.w.logprobs != nullptr) a.w.logprobs[row] = 0.f;
    }
    return;
  }
  const Scale sc(T);
  const bool far = sc.far(mx);
  const double first = far ? 0.0 : sc.bin(mx);
  for (int c = tid; c < a.chunks; c += kRowThreads) {
    const float m = tops[c].max;
    int shift = kBins;
    if (far) {
      shift = m == mx ? 0 : kBins;
    } else if (!sc.far(m)) {  // (a chunk too low to bin is far below the row's largest)
      const double d = first - sc.bin(m);
      shift = d < kBins ? static_cast<int>(d) : kBins;
    }
    s.shift[c] = m == -INFINITY ? kBins : shift;
  }
  __syncthreads();
  u64 w = 0;
  int n = 0;
  double scale = 0.0;
  if (tid < kBins) {
    const u64* h = a.hist + static_cast<int64_t>(row) * a.chunks * kBins;
    for (int c = 0; c < a.chunks; ++c) {
      const int b = tid - s.shift[c];
      const u64 v = b >= 0 && s.shift[c] < kBins ? h[static_cast<int64_t>(c) * kBins + b] : 0;
      w += v & kWeightMask;
      n += static_cast<int>(v >> kCountShift);
    }
    scale = exp2(tid * -0.125) / kOne;
    s.bin_scale[tid] = scale;
  }
  // running counts and masses; the order of the sums is fixed
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

  RowSampler<kF32> rs{s, a, row_of<kF32>(a, row), row, tid, lane, wave, sc, far, mx, first};
  int kept = s.count[kBins];
  double Z = s.mass[kBins];
  const int k = a.w.top_k[pr];
  if (k > 0 && k < kept) {
    const int bin = rs.find_bin([&](int c, double) { return c >= k; });
    if (s.count[bin + 1] == k) {
      Z = s.mass[bin + 1];
      kept = k;
    } else {
      rs.select(bin, kRank, k - s.count[bin], 0.0, k - s.count[bin], &n, &Z);
      kept = k;
    }
  }
  const float top_p = a.w.top_p[pr];
  if (top_p < 1.f) {
    const double target = static_cast<double>(top_p) * Z;
    const int bin = rs.find_bin([&](int c, double m) { return c >= kept || m >= target; });
    const int base = s.count[bin];
    rs.select(bin, kReach, 0, target, min(kept - base, s.count[bin + 1] - base), &n, &Z);
    kept = base + n;
  }
  const float min_p = a.w.min_p != nullptr ? fminf(a.w.min_p[pr], 1.f) : 0.f;
  if (min_p > 0.f && !far) {
    // the bin that the least weight falls into
    const double d = first - __builtin_floor(__builtin_fma(static_cast<double>(mx), sc.c, 8.0 * log2(static_cast<double>(min_p))));
    if (d < kBins && s.count[static_cast<int>(d)] < kept) {
      const int bin = static_cast<int>(d), base = s.count[bin];
      u64 wsum = 0, all;
      int csum = 0;
      rs.find_chunks(bin);
      rs.each(bin, [&](float l, int) {
        if (exp2((static_cast<double>(l) - mx) * sc.c * 0.125) >= static_cast<double>(min_p)) {
          wsum += rs.weight(l);
          ++csum;
        }
      });
      rs.scan(csum, &all);
      csum = static_cast<int>(all);
      rs.scan(wsum, &all);
      if (base + csum < kept) {
        kept = base + csum;
        Z = s.mass[bin] + static_cast<double>(all) * s.bin_scale[bin];
      }
    }
  }
  float u = a.w.uniform[row];
  u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;  // (NaN: 0)
  const double target = static_cast<double>(u) * Z;
  const int bin = rs.find_bin([&](int c, double m) { return c >= kept || m > target; });
  const int base = s.count[bin];
  double upto;
  const u64 key = rs.select(bin, kPass, 0, target, min(kept - base, s.count[bin + 1] - base), &n, &upto);
  if (tid == 0) {
    a.w.tokens[row] = static_cast<int>(0xffffffffu - static_cast<uint32_t>(key));
    if (a.w.logprobs != nullptr) {
      const float l = value_of(static_cast<uint32_t>(key >> 32));
      // Z is in weights of the first bin's middle
      const double top_w = far ? 0.0 : __builtin_fma(static_cast<double>(mx), sc.c, -(first + 0.5)) * 0.08664339756999316;
      const double own = far ? 0.0 : (static_cast<double>(l) - mx) * sc.c * 0.08664339756999316;
      a.w.logprobs[row] = static_cast<float>(own + top_w - log(Z));
    }
  }
}

int chunks_of(int vocab, int chunk) { return (vocab + chunk - 1) / chunk; }

size_t workspace_bytes(int64_t rows, int vocab) {
  return static_cast<size_t>(rows) * chunks_of(vocab, kSmallChunk) * (sizeof(ChunkTop) + kBins * sizeof(u64)) + 256;
}

template <bool kF32>
void launch(const SampleArgs& a, hipStream_t stream) {
  const uint32_t grid = static_cast<uint32_t>(a.w.num_rows) * a.chunks;
  if (a.chunk == kSmallChunk) sample_chunks_kernel<kF32, 256><<<grid, 256, 0, stream>>>(a);
  else sample_chunks_kernel<kF32, 1024><<<grid, 1024, 0, stream>>>(a);
  sample_rows_kernel<kF32><<<a.w.num_rows, kRowThreads, 0, stream>>>(a);
}

}  // namespace
}  // namespace rlk

using namespace rlk;

extern "C" size_t rlk_sampling_workspace_bytes(int max_rows, int max_vocab) {
  if (max_rows <= 0 || max_vocab <= 0 || max_vocab > kMaxVocab) return 0;
  return workspace_bytes(max_rows, max_vocab);
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
  const size_t need = workspace_bytes(w->num_rows, w->vocab);
  if (w->workspace_bytes < need)
    return fail(RLK_EINVAL, "%s: a workspace of %zu bytes, needs %zu", what, w->workspace_bytes, need);
  SampleArgs a;
  a.w = *w;
  // few rows: small chunks, so that more CUs share a row
  a.chunk = static_cast<int64_t>(w->num_rows) * chunks_of(w->vocab, kLargeChunk) >= 2 * compute_units() ? kLargeChunk : kSmallChunk;
  a.chunks = chunks_of(w->vocab, a.chunk);
  if (static_cast<int64_t>(w->num_rows) * a.chunks > (1 << 30))
    return fail(RLK_EINVAL, "%s: %d rows exceed one launch; split the call", what, w->num_rows);
  a.hist = static_cast<u64*>(w->workspace);
  a.top = reinterpret_cast<ChunkTop*>(a.hist + static_cast<int64_t>(w->num_rows) * a.chunks * kBins);
  w->logits_fp32 ? launch<true>(a, stream) : launch<false>(a, stream);
  return launch_status(what);
}
