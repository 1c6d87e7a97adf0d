// The block-scaled 8-bit KV cache, written (RoPE fused) and read back.
//
// Work of the write.  Rows that continue one block form a run (consecutive
// rows, consecutive offsets); the scale of the (block, head) follows from the
// whole run, so one group of lanes does a whole run of one kv head's K or V:
// decides the scale, requantises the old codes and stores the new ones, with no
// exchange beyond a reduction over its lanes.  A wave does one K or V head for the
// runs that start among kRows consecutive token rows, found by one ballot over
// their slots: long runs (prompts) with all 64 lanes, runs of up to 4 rows
// (decoding sequences) four at a time with 16 lanes each.  The q heads are rotated
// by other workgroups of the same launch.
//   K: lane p of a token holds the 8 rotation pairs (8p + e, D/2 + 8p + e),
//      which are one 16-byte piece of the layout.
//   V: lane m holds dims E m .. E m + E - 1 of the 4 tokens of a quad, which
//      are E/4 16-byte pieces, every byte of them: no data leaves its lane.
//      A quad that the run fills in part is read, merged and written back.
// Bound: HBM bytes for prefill (16384 rows of 28 + 2 x 4 heads of 128 with a bias,
// 294 MB: 55 us, 5.3 TB/s), the launch and one chain of dependent reads (slots ->
// positions -> cos/sin) for decode (32 rows 4.2 us).  Numerics: the rotation as in
// rope_kv.hip (fp32 without contraction, rounded to fp16), then kv_blocks.hpp.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "kv_blocks.hpp"

namespace rlk {

int check_block_view(const rlk_kv_block_view* kv, const char* what) {
  if (kv == nullptr) return fail(RLK_EINVAL, "%s: null KV block view", what);
  if (kv->head_dim != 64 && kv->head_dim != 128)
    return fail(RLK_EUNSUPPORTED, "%s: unsupported head_dim %d (supported: 64, 128)", what,
                kv->head_dim);
  if (kv->block_size != 16 && kv->block_size != 32)
    return fail(RLK_EUNSUPPORTED, "%s: unsupported block size %d (supported: 16, 32)", what,
                kv->block_size);
  if (kv->format != RLK_KV_BLOCK_INT8 && kv->format != RLK_KV_BLOCK_FP8)
    return fail(RLK_EINVAL, "%s: unknown block format %d", what, kv->format);
  if (kv->num_blocks <= 0 || kv->num_kv_heads <= 0)
    return fail(RLK_EINVAL, "%s: bad block count %d or kv heads %d", what, kv->num_blocks,
                kv->num_kv_heads);
  if (static_cast<int64_t>(kv->num_blocks) * kv->block_size > 0x7fffffffll ||
      static_cast<int64_t>(kv->num_blocks) * kv->num_kv_heads > 0x7fffffffll)
    return fail(RLK_EINVAL, "%s: %d blocks exceed 32-bit slots", what, kv->num_blocks);
  if (kv->k == nullptr || kv->v == nullptr || kv->k_scale == nullptr || kv->v_scale == nullptr)
    return fail(RLK_EINVAL, "%s: null pointer argument", what);
  if (((reinterpret_cast<uintptr_t>(kv->k) | reinterpret_cast<uintptr_t>(kv->v)) & 15) != 0)
    return fail(RLK_EINVAL, "%s: k and v must be 16-byte aligned", what);
  return RLK_OK;
}

namespace {

struct WriteArgs {
  _Float16* qkv;
  const int32_t* positions;
  const int32_t* slots;
  const float* cos_t;
  const float* sin_t;
  const _Float16* bias;
  rlk_kv_block_view kv;
  int num_tokens, hq;
  int kv_groups;    // workgroups of the kv part, before those of the q part
};

// cos and sin of a token position for 8 rotation pairs, and their rotation
// (rounded to fp16).
template <int D>
struct Angles {
  f32x8 c, s;
  __device__ __forceinline__ Angles(const WriteArgs& a, int pos, int p0) {
    c = *reinterpret_cast<const f32x8*>(a.cos_t + static_cast<int64_t>(pos) * (D / 2) + p0);
    s = *reinterpret_cast<const f32x8*>(a.sin_t + static_cast<int64_t>(pos) * (D / 2) + p0);
  }
  __device__ __forceinline__ void rotate(f32x8& x0, f32x8& x1) const {
#pragma clang fp contract(off)
    const f32x8 y0 = x0 * c - x1 * s;
    const f32x8 y1 = x1 * c + x0 * s;
    x0 = round_f16(y0);
    x1 = round_f16(y1);
  }
};

__device__ __forceinline__ f32x8 biased(u32x4 v, const _Float16* bias, int col) {
  if (bias != nullptr)
    v = __builtin_bit_cast(u32x4, __builtin_bit_cast(f16x8, v) +
                                      __builtin_bit_cast(f16x8, load16(bias + col)));
  return unpack8(v);
}

__device__ __forceinline__ float amax8(f32x8 x, float m) {
#pragma unroll
  for (int j = 0; j < 8; ++j) m = fmaxf(m, __builtin_fabsf(x[j]));
  return m;
}

// A run: rows row0 .. row0 + n - 1 at offsets off .. off + n - 1 of block blk.
struct Run {
  int row0, n, blk, off;
};

// Maximum over a group of 16 or 64 lanes.
template <int kLanes>
__device__ __forceinline__ float lanes_max(float v) {
  v = group_max<16>(v);
  if constexpr (kLanes == 64) v = rows_max<true>(rows_max<false>(v));
  return v;
}

// The scale of the run's block and head: old (0 when the run starts the block)
// joined with what amax asks for.  ratio = old / new for the old codes.
template <bool kFp8>
__device__ __forceinline__ float join_scale(float old, float amax, float& ratio) {
  const float s = fmaxf(old, block_scale<kFp8>(amax));
  ratio = s > old ? old * inv_scale(s) : 1.f;
  return s;
}

// Codes at the grown scale; lim is that scale's: an INT8 code of 127 at 2^9 would round
// to 64 at 2^10, which no fp16 number holds.
template <bool kFp8>
__device__ __forceinline__ uint32_t requant4(uint32_t w, float ratio, float lim) {
  const f32x4 v = decode4<kFp8>(w);
  return encode4<kFp8>(v[0], v[1], v[2], v[3], ratio, lim);
}

// K of one head for a run of at most kMax rows, by kGroup lanes of which this is
// number l; pos: the run's positions.
template <int D, int BS, bool kFp8, int kGroup, int kMax>
__device__ __forceinline__ void write_k(const WriteArgs& a, const Run& r, const int* pos, int kvh, int l) {
  constexpr int kLanes = D / 16, kTok = kGroup / kLanes;  // lanes of a token, tokens in flight
  constexpr int kIts = (kMax + kTok - 1) / kTok;
  const int p = l % kLanes, sub = l / kLanes;
  const int heads = a.hq + 2 * a.kv.num_kv_heads, col = (a.hq + kvh) * D;
  const int64_t cell = static_cast<int64_t>(r.blk) * a.kv.num_kv_heads + kvh;
  const float old = r.off > 0 ? a.kv.k_scale[cell] : 0.f;
  uint8_t* dst = static_cast<uint8_t*>(a.kv.k) + cell * (BS * D) + p * 256;
  // a lane past the run repeats its last row
  u32x4 x[kIts][2];
#pragma unroll
  for (int it = 0; it < kIts; ++it) {
    const _Float16* row = a.qkv + static_cast<int64_t>(r.row0 + min(it * kTok + sub, r.n - 1)) * heads * D + col;
    x[it][0] = ld16<true>(reinterpret_cast<const u32x4*>(row + 8 * p));
    x[it][1] = ld16<true>(reinterpret_cast<const u32x4*>(row + D / 2 + 8 * p));
  }
  float amax = 0.f;
#pragma unroll
  for (int it = 0; it < kIts; ++it) {
    f32x8 x0 = biased(x[it][0], a.bias, col + 8 * p), x1 = biased(x[it][1], a.bias, col + D / 2 + 8 * p);
    Angles<D>(a, pos[min(it * kTok + sub, r.n - 1)], 8 * p).rotate(x0, x1);
    amax = amax8(x1, amax8(x0, amax));
    x[it][0] = pack8(x0);
    x[it][1] = pack8(x1);
  }
  amax = lanes_max<kGroup>(amax);
  float ratio;
  const float s = join_scale<kFp8>(old, amax, ratio), inv = inv_scale(s), lim = code_limit<kFp8>(s);
#pragma unroll
  for (int it = 0; it < kIts; ++it) {
    if (it * kTok + sub < r.n) {
      const f32x8 x0 = unpack8(x[it][0]), x1 = unpack8(x[it][1]);
      const int key = r.off + it * kTok + sub;
      const u32x4 w = {encode4<kFp8>(x0[0], x0[1], x0[2], x0[3], inv, lim),
                       encode4<kFp8>(x0[4], x0[5], x0[6], x0[7], inv, lim),
                       encode4<kFp8>(x1[0], x1[1], x1[2], x1[3], inv, lim),
                       encode4<kFp8>(x1[4], x1[5], x1[6], x1[7], inv, lim)};
      store16(dst + (key / 16) * (16 * D) + (key % 16) * 16, w);
    }
  }
  if (ratio != 1.f) {  // the same for the group's lanes: requantise the earlier offsets
    for (int key = sub; key < r.off; key += kTok) {
      u32x4* at = reinterpret_cast<u32x4*>(dst + (key / 16) * (16 * D) + (key % 16) * 16);
      u32x4 w = *at;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = requant4<kFp8>(w[e], ratio, lim);
      *at = w;
    }
  }
  if (l == 0 && (r.off == 0 || ratio != 1.f)) a.kv.k_scale[cell] = s;
}

// V of one head likewise: lane m of a row of 16 holds dims E m .. E m + E - 1;
// the rows of 16 take every kRows16-th quad of the block.
template <int D, int BS, bool kFp8, int kGroup, int kMax>
__device__ __forceinline__ void write_v(const WriteArgs& a, const Run& r, int kvh, int l) {
  constexpr int E = D / 16, kRows16 = kGroup / 16;
  // quads that a run of kMax rows can touch (it may start inside one)
  constexpr int kQuads = (kMax + 6) / 4 < BS / 4 ? (kMax + 6) / 4 : BS / 4;
  constexpr int kIts = (kQuads + kRows16 - 1) / kRows16;
  using Raw = typename std::conditional<E == 8, u32x4, u32x2>::type;  // E halves
  typedef _Float16 f16xE __attribute__((ext_vector_type(E)));
  const int m = l % 16;
  const int heads = a.hq + 2 * a.kv.num_kv_heads;
  const int col = (a.hq + a.kv.num_kv_heads + kvh) * D + E * m;
  const int64_t cell = static_cast<int64_t>(r.blk) * a.kv.num_kv_heads + kvh;
  const float old = r.off > 0 ? a.kv.v_scale[cell] : 0.f;
  uint8_t* dst = static_cast<uint8_t*>(a.kv.v) + cell * (BS * D) + m * 16;
  const int q0 = r.off / 4, q1 = (r.off + r.n - 1) / 4;  // quads of the run
  f16xE x[kIts][4];
#pragma unroll
  for (int it = 0; it < kIts; ++it)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // keys outside the run repeat one inside it
      const int j = min(max(4 * (q0 + it * kRows16 + l / 16) + i - r.off, 0), r.n - 1);
      const _Float16* row = a.qkv + static_cast<int64_t>(r.row0 + j) * heads * D;
      x[it][i] = __builtin_bit_cast(f16xE, __builtin_nontemporal_load(reinterpret_cast<const Raw*>(row + col)));
    }
  f16xE bias = {};
  if (a.bias != nullptr) bias = *reinterpret_cast<const f16xE*>(a.bias + col);
  // a quad's bytes of keys inside the run, and of those before it; the pieces of
  // quads that the run fills in part are read with its rows
  auto piece = [&](int quad, int g) {
    return reinterpret_cast<u32x4*>(dst + (quad / 4) * (16 * D) + (quad % 4) * 256 + g * 1024);
  };
  uint32_t mine[kIts], below[kIts];
  u32x4 had[kIts][E / 4];
#pragma unroll
  for (int it = 0; it < kIts; ++it) {
    const int quad = q0 + it * kRows16 + l / 16;
    const int lo = min(max(r.off - 4 * quad, 0), 4), hi = min(max(r.off + r.n - 4 * quad, 0), 4);
    below[it] = lo == 0 ? 0u : 0xffffffffu >> (32 - 8 * lo);
    mine[it] = (hi == 0 ? 0u : 0xffffffffu >> (32 - 8 * hi)) & ~below[it];
#pragma unroll
    for (int g = 0; g < E / 4; ++g)
      had[it][g] = quad <= q1 && mine[it] != 0xffffffffu ? *piece(quad, g) : u32x4{0, 0, 0, 0};
  }
  float amax = 0.f;
#pragma unroll
  for (int it = 0; it < kIts; ++it)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (a.bias != nullptr) x[it][i] += bias;
#pragma unroll
      for (int d = 0; d < E; ++d) amax = fmaxf(amax, __builtin_fabsf(static_cast<float>(x[it][i][d])));
    }
  amax = lanes_max<kGroup>(amax);
  float ratio;
  const float s = join_scale<kFp8>(old, amax, ratio), inv = inv_scale(s), lim = code_limit<kFp8>(s);
#pragma unroll
  for (int it = 0; it < kIts; ++it) {
    const int quad = q0 + it * kRows16 + l / 16;
    if (quad <= q1) {
#pragma unroll
      for (int g = 0; g < E / 4; ++g) {
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int d = 4 * g + j;
          w[j] = encode4<kFp8>(static_cast<float>(x[it][0][d]), static_cast<float>(x[it][1][d]),
                               static_cast<float>(x[it][2][d]), static_cast<float>(x[it][3][d]), inv, lim);
          if (mine[it] != 0xffffffffu) {
            const uint32_t h = had[it][g][j];
            const uint32_t keep = ratio != 1.f ? (requant4<kFp8>(h, ratio, lim) & below[it]) | (h & ~below[it]) : h;
            w[j] = (w[j] & mine[it]) | (keep & ~mine[it]);
          }
        }
        *piece(quad, g) = w;
      }
    }
  }
  if (ratio != 1.f) {
    for (int quad = l / 16; quad < q0; quad += kRows16) {
#pragma unroll
      for (int g = 0; g < E / 4; ++g) {
        u32x4 w = *piece(quad, g);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = requant4<kFp8>(w[j], ratio, lim);
        *piece(quad, g) = w;
      }
    }
  }
  if (l == 0 && (r.off == 0 || ratio != 1.f)) a.kv.v_scale[cell] = s;
}

constexpr int kWriteThreads = 256;
constexpr int kShort = 4;  // rows of a run that 16 lanes do

// The runs that start in rows chunk0 .. chunk0 + kRows - 1, for K head `unit` or
// V head unit - hkv.
template <int D, int BS, bool kFp8, int kRows>
__device__ __forceinline__ void write_chunk(const WriteArgs& a, int chunk0, int unit, int lane, int* pos) {
  // (so a run that starts in the chunk ends, at the block's end at the latest, before a
  // row that this wave sees)
  static_assert(kRows + BS <= kWave, "a chunk's rows and the last run's rest fit one wave");
  const int hkv = a.kv.num_kv_heads;
  const int row = chunk0 + lane;
  const int slot = row < a.num_tokens ? a.slots[row] : -1;
  int before = __shfl_up(slot, 1, kWave);
  if (lane == 0) before = chunk0 > 0 ? a.slots[chunk0 - 1] : -1;
  // positions of the rows, in LDS: lanes of one run need those of other rows
  pos[lane] = row < a.num_tokens ? a.positions[row] : 0;
  __builtin_amdgcn_wave_barrier();
  const bool valid = slot >= 0 && slot / BS < a.kv.num_blocks;
  // a row starts a run unless it continues the block of the row before
  const uint64_t starts = __ballot(!valid || slot % BS == 0 || slot != before + 1);
  uint64_t todo = starts & __ballot(valid) & ((1ull << kRows) - 1);
  auto rows_of = [&](int i) { return __builtin_ctzll(starts >> (i + 1)) + 1; };  // of the run from row i on
  auto run_at = [&](int i) {  // the run that starts at row chunk0 + i
    const int sl = __shfl(slot, i, kWave);
    return Run{chunk0 + i, rows_of(i), sl / BS, sl % BS};
  };
  while (todo != 0) {  // uniform over the wave
    const int i = __builtin_ctzll(todo);
    if (rows_of(i) > kShort) {  // a long run, by the whole wave
      todo &= todo - 1;
      const Run r = run_at(i);
      if (unit < hkv) write_k<D, BS, kFp8, 64, BS>(a, r, pos + i, unit, lane);
      else write_v<D, BS, kFp8, 64, BS>(a, r, unit - hkv, lane);
    } else {  // up to four short ones, one to each 16 lanes
      int mine = -1;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if (todo == 0) break;
        const int k = __builtin_ctzll(todo);
        if (rows_of(k) > kShort) break;
        if (lane / 16 == g) mine = k;
        todo &= todo - 1;
      }
      const Run r = run_at(max(mine, 0));
      if (mine >= 0) {
        if (unit < hkv) write_k<D, BS, kFp8, 16, kShort>(a, r, pos + mine, unit, lane % 16);
        else write_v<D, BS, kFp8, 16, kShort>(a, r, unit - hkv, lane % 16);
      }
    }
  }
}

// kHeads: q heads that a lane rotates with one load of cos and sin.
template <int D, int BS, bool kFp8, int kRows, int kHeads>
__global__ __launch_bounds__(kWriteThreads) void write_kv_blocks_kernel(WriteArgs a) {
  __shared__ int pos[kWriteThreads / kWave][kWave];
  const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  if (static_cast<int>(blockIdx.x) < a.kv_groups) {  // first: their chain of reads is the longer
    const int units = 2 * a.kv.num_kv_heads, w = blockIdx.x * (kWriteThreads / kWave) + wave;
    const int chunk = w / units;
    if (chunk >= (a.num_tokens + kRows - 1) / kRows) return;
    write_chunk<D, BS, kFp8, kRows>(a, chunk * kRows, w - chunk * units, lane, pos[wave]);
    return;
  }
  // q heads: 8 rotation pairs of kHeads heads per lane
  constexpr int kLanes = D / 16;
  const int64_t g = static_cast<int64_t>(blockIdx.x - a.kv_groups) * kWriteThreads + tid;
  const int per = a.hq / kHeads * kLanes;
  const int64_t t = g / per;
  if (t >= a.num_tokens) return;
  const int h = static_cast<int>(g - t * per) / kLanes * kHeads, p0 = static_cast<int>(g % kLanes) * 8;
  const int heads = a.hq + 2 * a.kv.num_kv_heads, col = h * D + p0;
  _Float16* row = a.qkv + t * heads * D;
  u32x4 v[kHeads][2];
#pragma unroll
  for (int k = 0; k < kHeads; ++k) {
    v[k][0] = ld16<true>(reinterpret_cast<const u32x4*>(row + col + k * D));
    v[k][1] = ld16<true>(reinterpret_cast<const u32x4*>(row + col + k * D + D / 2));
  }
  const Angles<D> an(a, a.positions[t], p0);
#pragma unroll
  for (int k = 0; k < kHeads; ++k) {
    f32x8 x0 = biased(v[k][0], a.bias, col + k * D), x1 = biased(v[k][1], a.bias, col + k * D + D / 2);
    an.rotate(x0, x1);
    st16<true>(reinterpret_cast<u32x4*>(row + col + k * D), pack8(x0));
    st16<true>(reinterpret_cast<u32x4*>(row + col + k * D + D / 2), pack8(x1));
  }
}

template <int D, int BS, bool kFp8>
int launch_write(WriteArgs a, hipStream_t stream) {
  // Rows of a wave: with 16 a prompt's blocks are found by fewer waves, with 4 single
  // rows have more waves.  us, 4 / 16: 32 single rows 4.2 / 9.4, 512 7.7 / 14.8, 2048
  // 20.3 / 21.9; a prompt of 512 5.3 / 5.5, 1024 8.4 / 6.8, 2048 14.2 / 9.6, 4 of 4096
  // 76 / 56; 61 single rows beside 9 prompts, 4802 rows, D = 64, 16.5 / 14.3.
  // RLK_TUNE_BLK_WRITE forces them (4 or 16; tests and tuning runs)
  const int rows = tune_knob(kBlkWrite, a.num_tokens > 1024 ? 16 : 4) == 4 ? 4 : 16;
  const int64_t waves = (static_cast<int64_t>(a.num_tokens) + rows - 1) / rows * 2 * a.kv.num_kv_heads;
  const int64_t kvg = (waves + kWriteThreads / kWave - 1) / (kWriteThreads / kWave);
  const int per = rows == 16 && a.hq % 2 == 0 ? 2 : 1;
  const int64_t qg = (static_cast<int64_t>(a.num_tokens) * (a.hq / per) * (D / 16) + kWriteThreads - 1) / kWriteThreads;
  if (kvg + qg > 0x7fffffffll)
    return fail(RLK_EINVAL, "rope_and_write_kv_blocks: %d rows exceed one launch; split the call",
                a.num_tokens);
  a.kv_groups = static_cast<int>(kvg);
  const uint32_t grid = static_cast<uint32_t>(kvg + qg);
  if (rows == 4) {
    write_kv_blocks_kernel<D, BS, kFp8, 4, 1><<<grid, kWriteThreads, 0, stream>>>(a);
  } else if (per == 2) {
    write_kv_blocks_kernel<D, BS, kFp8, 16, 2><<<grid, kWriteThreads, 0, stream>>>(a);
  } else {
    write_kv_blocks_kernel<D, BS, kFp8, 16, 1><<<grid, kWriteThreads, 0, stream>>>(a);
  }
  return launch_status("rope_and_write_kv_blocks");
}

template <int D, int BS>
int launch_write_f(const WriteArgs& a, hipStream_t stream) {
  return a.kv.format == RLK_KV_BLOCK_FP8 ? launch_write<D, BS, true>(a, stream)
                                         : launch_write<D, BS, false>(a, stream);
}

// ------------------------------------------------------------------ read back

struct ReadArgs {
  rlk_kv_block_view kv;
  const int32_t* slots;
  int n;
  _Float16* k_out;
  _Float16* v_out;
};

__device__ __forceinline__ u32x2 scaled4(f32x4 v, float s) {
  return __builtin_bit_cast(u32x2, __builtin_convertvector(v * s, f16x4));
}

// 16 lanes take 4 rows of the list for one head's K or V.  Where the 4 rows are a
// quad of the layout (lists of consecutive slots), each V piece is read once and
// gives 4 rows; other rows take theirs alone, a byte in four of what they read.
// Bound: HBM bytes for runs (16384 rows of 4 heads of 128, 50 MB: 11.3 us, 4.4 TB/s),
// address translation for single rows far apart (2048 of 8 heads in a 17 GB cache: 28 us),
// the launch and two dependent reads below (32 rows 3.7 us).
template <int D, bool kFp8>
__global__ __launch_bounds__(256) void read_kv_blocks_kernel(ReadArgs a) {
  constexpr int E = D / 16, kLanes = D / 16, kTok = 16 / kLanes;
  const int hkv = a.kv.num_kv_heads, bs = a.kv.block_size;
  const int64_t g = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int l16 = g % 16;
  const int64_t group = g / 16;
  const int i0 = static_cast<int>(group / (2 * hkv)) * 4, unit = static_cast<int>(group % (2 * hkv));
  if (i0 >= a.n) return;
  const bool is_v = unit >= hkv;
  const int kvh = is_v ? unit - hkv : unit;
  _Float16* out = is_v ? a.v_out : a.k_out;
  if (out == nullptr) return;
  int slot[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) slot[u] = i0 + u < a.n ? a.slots[i0 + u] : -1;
  auto tile_of = [&](const void* base, int blk, int off) {
    const int64_t cell = static_cast<int64_t>(blk) * hkv + kvh;
    return static_cast<const uint8_t*>(base) + cell * (bs * D) + (off / 16) * (16 * D);
  };
  auto valid = [&](int s) { return s >= 0 && s / bs < a.kv.num_blocks; };
  if (!is_v) {
    const int p = l16 % kLanes;
    // all rows are requested before the first is used; a slot outside the pool reads slot 0
    int s[4];
    float scale[4];
    u32x4 code[4];
#pragma unroll
    for (int u = 0; u < 4; u += kTok) {
      const int v = u + l16 / kLanes;
      s[u] = v == 0 ? slot[0] : (v == 1 ? slot[1] : (v == 2 ? slot[2] : slot[3]));
      const int at = valid(s[u]) ? s[u] : 0, blk = at / bs, off = at - blk * bs;
      scale[u] = a.kv.k_scale[static_cast<int64_t>(blk) * hkv + kvh];
      code[u] = load16(tile_of(a.kv.k, blk, off) + p * 256 + (off % 16) * 16);
    }
#pragma unroll
    for (int u = 0; u < 4; u += kTok) {
      if (!valid(s[u])) continue;
      const int v = u + l16 / kLanes;
      const float sc = scale[u];
      const u32x4 w = code[u];
      const u32x2 a0 = scaled4(decode4<kFp8>(w[0]), sc), a1 = scaled4(decode4<kFp8>(w[1]), sc);
      const u32x2 b0 = scaled4(decode4<kFp8>(w[2]), sc), b1 = scaled4(decode4<kFp8>(w[3]), sc);
      _Float16* o = out + (static_cast<int64_t>(i0 + v) * hkv + kvh) * D;
      st16<true>(reinterpret_cast<u32x4*>(o + 8 * p), u32x4{a0[0], a0[1], a1[0], a1[1]});
      st16<true>(reinterpret_cast<u32x4*>(o + D / 2 + 8 * p), u32x4{b0[0], b0[1], b1[0], b1[1]});
    }
    return;
  }
  auto row = [&](int u) { return out + (static_cast<int64_t>(i0 + u) * hkv + kvh) * D + E * l16; };
  if (valid(slot[0]) && slot[0] % 4 == 0 && slot[1] == slot[0] + 1 && slot[2] == slot[0] + 2 &&
      slot[3] == slot[0] + 3) {
    const int blk = slot[0] / bs, off = slot[0] - blk * bs;
    const float sc = a.kv.v_scale[static_cast<int64_t>(blk) * hkv + kvh];
    const uint8_t* at = tile_of(a.kv.v, blk, off) + (off % 16 / 4) * 256 + l16 * 16;
    f32x4 v[E];  // dim E m + d of the 4 rows
#pragma unroll
    for (int gg = 0; gg < E / 4; ++gg) {
      const u32x4 w = load16(at + gg * 1024);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * gg + j] = decode4<kFp8>(w[j]) * sc;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if constexpr (E == 8) {
        st16<true>(reinterpret_cast<u32x4*>(row(u)),
                   pack8(f32x8{v[0][u], v[1][u], v[2][u], v[3][u], v[4][u], v[5][u], v[6][u], v[7][u]}));
      } else {
        st8<true>(reinterpret_cast<u32x2*>(row(u)), scaled4(f32x4{v[0][u], v[1][u], v[2][u], v[3][u]}, 1.f));
      }
    }
    return;
  }
  float scale[4];
  u32x4 code[4][E / 4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int s = valid(slot[u]) ? slot[u] : 0, blk = s / bs, off = s - blk * bs;
    scale[u] = a.kv.v_scale[static_cast<int64_t>(blk) * hkv + kvh];
    const uint8_t* at = tile_of(a.kv.v, blk, off) + (off % 16 / 4) * 256 + l16 * 16;
#pragma unroll
    for (int gg = 0; gg < E / 4; ++gg) code[u][gg] = load16(at + gg * 1024);
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    if (!valid(slot[u])) continue;
    const float sc = scale[u];
#pragma unroll
    for (int gg = 0; gg < E / 4; ++gg) {
      const u32x4 w = code[u][gg];
      const int sh = 8 * (slot[u] % 4);  // (blocks are whole quads)
      const uint32_t b = ((w[0] >> sh) & 0xff) | (((w[1] >> sh) & 0xff) << 8) |
                         (((w[2] >> sh) & 0xff) << 16) | (((w[3] >> sh) & 0xff) << 24);
      *reinterpret_cast<u32x2*>(row(u) + 4 * gg) = scaled4(decode4<kFp8>(b), sc);
    }
  }
}

}  // namespace
}  // namespace rlk

using namespace rlk;

extern "C" int rlk_rope_and_write_kv_blocks(uint16_t* qkv, const int32_t* positions,
                                            const int32_t* slot_mapping, int num_tokens,
                                            int num_heads, const float* cos_table,
                                            const float* sin_table, const rlk_kv_block_view* kv,
                                            const uint16_t* qkv_bias, hipStream_t stream) {
  if (num_tokens <= 0) return RLK_OK;
  const char* what = "rope_and_write_kv_blocks";
  if (const int st = check_block_view(kv, what); st != RLK_OK) return st;
  if (num_heads < 0) return fail(RLK_EINVAL, "%s: bad head count %d", what, num_heads);
  if (qkv == nullptr || positions == nullptr || slot_mapping == nullptr || cos_table == nullptr ||
      sin_table == nullptr)
    return fail(RLK_EINVAL, "%s: null pointer argument", what);
  if (((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(qkv_bias) |
        reinterpret_cast<uintptr_t>(cos_table) | reinterpret_cast<uintptr_t>(sin_table)) & 15) != 0)
    return fail(RLK_EINVAL, "%s: qkv, bias and cos/sin tables must be 16-byte aligned", what);
  WriteArgs a;
  a.qkv = reinterpret_cast<_Float16*>(qkv);
  a.positions = positions;
  a.slots = slot_mapping;
  a.cos_t = cos_table;
  a.sin_t = sin_table;
  a.bias = reinterpret_cast<const _Float16*>(qkv_bias);
  a.kv = *kv;
  a.num_tokens = num_tokens;
  a.hq = num_heads;
  if (kv->head_dim == 128)
    return kv->block_size == 16 ? launch_write_f<128, 16>(a, stream) : launch_write_f<128, 32>(a, stream);
  return kv->block_size == 16 ? launch_write_f<64, 16>(a, stream) : launch_write_f<64, 32>(a, stream);
}

extern "C" int rlk_read_kv_blocks(const rlk_kv_block_view* kv, const int32_t* slots, int n,
                                  uint16_t* k_out, uint16_t* v_out, hipStream_t stream) {
  if (n <= 0) return RLK_OK;
  const char* what = "read_kv_blocks";
  if (const int st = check_block_view(kv, what); st != RLK_OK) return st;
  if (slots == nullptr) return fail(RLK_EINVAL, "%s: null pointer argument", what);
  if (((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15) != 0)
    return fail(RLK_EINVAL, "%s: outputs must be 16-byte aligned", what);
  if (k_out == nullptr && v_out == nullptr) return RLK_OK;
  const int64_t blocks = (static_cast<int64_t>((n + 3) / 4) * 2 * kv->num_kv_heads * 16 + 255) / 256;
  if (blocks > 0x7fffffffll || n > 0x7ffffff0)
    return fail(RLK_EINVAL, "%s: %d rows exceed one launch; split the call", what, n);
  const ReadArgs a = {*kv, slots, n, reinterpret_cast<_Float16*>(k_out),
                      reinterpret_cast<_Float16*>(v_out)};
  const uint32_t grid = static_cast<uint32_t>(blocks);
  const bool fp8 = kv->format == RLK_KV_BLOCK_FP8;
  if (kv->head_dim == 128) {
    if (fp8) read_kv_blocks_kernel<128, true><<<grid, 256, 0, stream>>>(a);
    else read_kv_blocks_kernel<128, false><<<grid, 256, 0, stream>>>(a);
  } else {
    if (fp8) read_kv_blocks_kernel<64, true><<<grid, 256, 0, stream>>>(a);
    else read_kv_blocks_kernel<64, false><<<grid, 256, 0, stream>>>(a);
  }
  return launch_status(what);
}
