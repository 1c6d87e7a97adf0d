// The block-scaled 8-bit KV cache, written (RoPE fused) and read back.
//
// Work of the write.  Rows that continue one block form a run (consecutive
// rows, consecutive offsets); one group of 16 lanes does a whole run of one
// kv head's K or V, so the scale of the (block, head) is decided, the old codes
// requantised and the new ones stored without any exchange beyond a row of 16
// lanes.  A wave does 4 heads of the same run, so its control flow is uniform.
// A wave looks at kRows consecutive token rows and does the runs that start
// among them; their starts are one ballot over the slots.  The q heads are
// rotated by other workgroups of the same launch.
//   K: lane p of a token holds the 8 rotation pairs (8p + e, D/2 + 8p + e),
//      which are one 16-byte piece of the layout.
//   V: lane m holds dims E m .. E m + E - 1 of the 4 tokens of a quad, which
//      are E/4 16-byte pieces, every byte of them: no data leaves its lane.
//      A quad that the run fills in part is read, merged and written back.
// Bound: HBM bytes for prefill, the launch and one chain of dependent reads
// (slots -> positions -> cos/sin) for decode.  Numerics: the rotation as in
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
  int head_groups;  // waves a chunk of rows takes: ceil(2 * hkv / 4)
};

// The 8 rotation pairs of (x0, x1) at token position pos, rounded to fp16.
template <int D>
__device__ __forceinline__ void rotate8(const WriteArgs& a, int pos, int p0, f32x8& x0, f32x8& x1) {
#pragma clang fp contract(off)
  const float* cp = a.cos_t + static_cast<int64_t>(pos) * (D / 2) + p0;
  const float* sp = a.sin_t + static_cast<int64_t>(pos) * (D / 2) + p0;
  const f32x8 c = *reinterpret_cast<const f32x8*>(cp), s = *reinterpret_cast<const f32x8*>(sp);
  const f32x8 y0 = x0 * c - x1 * s;
  const f32x8 y1 = x1 * c + x0 * s;
  x0 = round_f16(y0);
  x1 = round_f16(y1);
}

__device__ __forceinline__ f32x8 load_biased(const _Float16* row, const _Float16* bias, int col) {
  u32x4 v = load16(row + col);
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

// The scale of the run's block and head: old (0 when the run starts the block)
// joined with what amax asks for.  ratio = old / new for the old codes.
template <bool kFp8>
__device__ __forceinline__ float join_scale(float old, float amax, float& ratio) {
  const float s = fmaxf(old, block_scale<kFp8>(amax));
  ratio = s > old ? old * inv_scale(s) : 1.f;
  return s;
}

// K of one head: lane p of D / 16 lanes per token; pos: the run's positions.
template <int D, int BS, bool kFp8>
__device__ __forceinline__ void write_k(const WriteArgs& a, const Run& r, const int* pos, int kvh,
                                        int l16) {
  constexpr int kLanes = D / 16, kTok = 16 / kLanes;  // lanes per token, tokens in flight
  constexpr int kIts = BS / kTok;
  const int p = l16 % kLanes, sub = l16 / kLanes;
  const int heads = a.hq + 2 * a.kv.num_kv_heads, col = (a.hq + kvh) * D;
  const int64_t cell = static_cast<int64_t>(r.blk) * a.kv.num_kv_heads + kvh;
  const float old = r.off > 0 ? a.kv.k_scale[cell] : 0.f;
  uint8_t* dst = static_cast<uint8_t*>(a.kv.k) + cell * (BS * D) + p * 256;
  u32x4 x[kIts][2];
  float amax = 0.f;
#pragma unroll
  for (int it = 0; it < kIts; ++it) {
    if (it * kTok < r.n) {  // uniform
      const int j = min(it * kTok + sub, r.n - 1);  // a lane past the run repeats its last row
      const _Float16* row = a.qkv + static_cast<int64_t>(r.row0 + j) * heads * D;
      f32x8 x0 = load_biased(row, a.bias, col + 8 * p);
      f32x8 x1 = load_biased(row, a.bias, col + D / 2 + 8 * p);
      rotate8<D>(a, pos[j], 8 * p, x0, x1);
      amax = amax8(x1, amax8(x0, amax));
      x[it][0] = pack8(x0);
      x[it][1] = pack8(x1);
    }
  }
  amax = group_max<16>(amax);
  float ratio;
  const float s = join_scale<kFp8>(old, amax, ratio), inv = inv_scale(s), lim = code_limit<kFp8>(s);
#pragma unroll
  for (int it = 0; it < kIts; ++it) {
    if (it * kTok < r.n && it * kTok + sub < r.n) {
      const f32x8 x0 = unpack8(x[it][0]), x1 = unpack8(x[it][1]);
      const int key = r.off + it * kTok + sub;
      const u32x4 w = {encode4<kFp8>(x0[0], x0[1], x0[2], x0[3], inv, lim),
                       encode4<kFp8>(x0[4], x0[5], x0[6], x0[7], inv, lim),
                       encode4<kFp8>(x1[0], x1[1], x1[2], x1[3], inv, lim),
                       encode4<kFp8>(x1[4], x1[5], x1[6], x1[7], inv, lim)};
      store16(dst + (key / 16) * (16 * D) + (key % 16) * 16, w);
    }
  }
  if (ratio != 1.f) {  // the same for the 16 lanes: requantise the earlier offsets
    for (int key = sub; key < r.off; key += kTok) {
      u32x4* at = reinterpret_cast<u32x4*>(dst + (key / 16) * (16 * D) + (key % 16) * 16);
      u32x4 w = *at;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f32x4 v = decode4<kFp8>(w[e]);
        w[e] = encode4<kFp8>(v[0], v[1], v[2], v[3], ratio, BlockFormat<kFp8>::kMax);
      }
      *at = w;
    }
  }
  if (l16 == 0 && (r.off == 0 || ratio != 1.f)) a.kv.k_scale[cell] = s;
}

// V of one head: lane m.
template <int D, int BS, bool kFp8>
__device__ __forceinline__ void write_v(const WriteArgs& a, const Run& r, int kvh, int m) {
  constexpr int E = D / 16, kQuads = BS / 4;
  using Raw = typename std::conditional<E == 8, u32x4, u32x2>::type;  // E halves
  typedef _Float16 f16xE __attribute__((ext_vector_type(E)));
  const int heads = a.hq + 2 * a.kv.num_kv_heads;
  const int col = (a.hq + a.kv.num_kv_heads + kvh) * D + E * m;
  const int64_t cell = static_cast<int64_t>(r.blk) * a.kv.num_kv_heads + kvh;
  const float old = r.off > 0 ? a.kv.v_scale[cell] : 0.f;
  uint8_t* dst = static_cast<uint8_t*>(a.kv.v) + cell * (BS * D) + m * 16;
  const int q0 = r.off / 4, q1 = (r.off + r.n - 1) / 4;  // quads that the run touches
  f16xE x[kQuads][4];
  f16xE bias = {};
  if (a.bias != nullptr) bias = *reinterpret_cast<const f16xE*>(a.bias + col);
  float amax = 0.f;
#pragma unroll
  for (int q = 0; q < kQuads; ++q) {
    if (q <= q1 - q0) {  // uniform
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // keys outside the run repeat one inside it
        const int j = min(max(4 * (q0 + q) + i - r.off, 0), r.n - 1);
        const _Float16* row = a.qkv + static_cast<int64_t>(r.row0 + j) * heads * D;
        f16xE v = __builtin_bit_cast(f16xE, *reinterpret_cast<const Raw*>(row + col));
        if (a.bias != nullptr) v += bias;
        x[q][i] = v;
#pragma unroll
        for (int d = 0; d < E; ++d) amax = fmaxf(amax, __builtin_fabsf(static_cast<float>(v[d])));
      }
    }
  }
  amax = group_max<16>(amax);
  float ratio;
  const float s = join_scale<kFp8>(old, amax, ratio), inv = inv_scale(s), lim = code_limit<kFp8>(s);
  auto requant = [&](uint32_t w) {
    const f32x4 v = decode4<kFp8>(w);
    return encode4<kFp8>(v[0], v[1], v[2], v[3], ratio, BlockFormat<kFp8>::kMax);
  };
#pragma unroll
  for (int q = 0; q < kQuads; ++q) {
    if (q <= q1 - q0) {
      const int quad = q0 + q;
      uint8_t* at = dst + (quad / 4) * (16 * D) + (quad % 4) * 256;
      // bytes of the quad's keys inside the run, and of those before it
      const int lo = max(r.off - 4 * quad, 0), hi = min(r.off + r.n - 4 * quad, 4);
      const uint32_t below = lo == 0 ? 0u : 0xffffffffu >> (32 - 8 * lo);
      const uint32_t mine = (hi == 4 ? 0xffffffffu : 0xffffffffu >> (32 - 8 * hi)) & ~below;
#pragma unroll
      for (int g = 0; g < E / 4; ++g) {
        u32x4* piece = reinterpret_cast<u32x4*>(at + g * 1024);
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int d = 4 * g + j;
          w[j] = encode4<kFp8>(static_cast<float>(x[q][0][d]), static_cast<float>(x[q][1][d]),
                               static_cast<float>(x[q][2][d]), static_cast<float>(x[q][3][d]), inv, lim);
        }
        if (mine != 0xffffffffu) {  // uniform
          const u32x4 had = *piece;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t keep = ratio != 1.f ? (requant(had[j]) & below) | (had[j] & ~below) : had[j];
            w[j] = (w[j] & mine) | (keep & ~mine);
          }
        }
        *piece = w;
      }
    }
  }
  if (ratio != 1.f) {
    for (int quad = 0; quad < q0; ++quad) {
      uint8_t* at = dst + (quad / 4) * (16 * D) + (quad % 4) * 256;
#pragma unroll
      for (int g = 0; g < E / 4; ++g) {
        u32x4* piece = reinterpret_cast<u32x4*>(at + g * 1024);
        u32x4 w = *piece;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = requant(w[j]);
        *piece = w;
      }
    }
  }
  if (m == 0 && (r.off == 0 || ratio != 1.f)) a.kv.v_scale[cell] = s;
}

constexpr int kWriteThreads = 256;

// The runs that start in rows chunk0 .. chunk0 + kRows - 1, for 4 of the
// 2 * hkv (K heads, then V heads): head unit 4 * group + lane / 16.
template <int D, int BS, bool kFp8, int kRows>
__device__ __forceinline__ void write_chunk(const WriteArgs& a, int chunk0, int group, int lane,
                                            int* pos) {
  static_assert(kRows + BS <= kWave, "a chunk's rows and the last run's rest fit one wave");
  const int hkv = a.kv.num_kv_heads;
  const int row = chunk0 + lane;
  const int slot = row < a.num_tokens ? a.slots[row] : -1;
  int before = __shfl_up(slot, 1, kWave);
  if (lane == 0) before = chunk0 > 0 ? a.slots[chunk0 - 1] : -1;
  // positions of the rows, in LDS: the lanes of a K head need those of other
  // rows, and lanes of the wave that do a V head are not there to hand them over
  pos[lane] = row < a.num_tokens ? a.positions[row] : 0;
  __builtin_amdgcn_wave_barrier();
  const bool valid = slot >= 0 && slot / BS < a.kv.num_blocks;
  // a row starts a run unless it continues the block of the row before
  const bool start = !valid || slot % BS == 0 || slot != before + 1;
  const uint64_t starts = __ballot(start);
  uint64_t todo = __ballot(start && valid) & ((1ull << kRows) - 1);
  const int unit = 4 * group + lane / 16;
  while (todo != 0) {  // uniform over the wave
    const int i = __builtin_ctzll(todo);
    todo &= todo - 1;
    const uint64_t after = starts >> (i + 1);
    const int n = after != 0 ? __builtin_ctzll(after) + 1 : kWave - i;
    const int sl = __builtin_amdgcn_readlane(slot, i);
    const Run r = {chunk0 + i, n, sl / BS, sl % BS};
    if (unit < hkv) {
      write_k<D, BS, kFp8>(a, r, pos + i, unit, lane % 16);
    } else if (unit < 2 * hkv) {
      write_v<D, BS, kFp8>(a, r, unit - hkv, lane % 16);
    }
  }
}

template <int D, int BS, bool kFp8, int kRows>
__global__ __launch_bounds__(kWriteThreads) void write_kv_blocks_kernel(WriteArgs a) {
  __shared__ int pos[kWriteThreads / kWave][kWave];
  const int tid = threadIdx.x, lane = tid % kWave;
  if (static_cast<int>(blockIdx.x) < a.kv_groups) {
    const int w = blockIdx.x * (kWriteThreads / kWave) + tid / kWave;
    const int chunk = w / a.head_groups;
    if (chunk * kRows >= a.num_tokens) return;
    write_chunk<D, BS, kFp8, kRows>(a, chunk * kRows, w - chunk * a.head_groups, lane,
                                       pos[tid / kWave]);
    return;
  }
  // q heads: 8 rotation pairs per lane
  constexpr int kLanes = D / 16;
  const int64_t g = static_cast<int64_t>(blockIdx.x - a.kv_groups) * kWriteThreads + tid;
  const int per = a.hq * kLanes;
  const int64_t t = g / per;
  if (t >= a.num_tokens) return;
  const int h = static_cast<int>(g - t * per) / kLanes, p0 = static_cast<int>(g % kLanes) * 8;
  const int heads = a.hq + 2 * a.kv.num_kv_heads;
  _Float16* row = a.qkv + t * heads * D;
  f32x8 x0 = load_biased(row, a.bias, h * D + p0), x1 = load_biased(row, a.bias, h * D + D / 2 + p0);
  rotate8<D>(a, a.positions[t], p0, x0, x1);
  st16<true>(reinterpret_cast<u32x4*>(row + h * D + p0), pack8(x0));
  st16<true>(reinterpret_cast<u32x4*>(row + h * D + D / 2 + p0), pack8(x1));
}

template <int D, int BS, bool kFp8>
int launch_write(WriteArgs a, hipStream_t stream) {
  // RLK_TUNE_BLK_WRITE forces the rows of a wave (1 or 16; tests and tuning runs)
  const int rows = tune_knob(kBlkWrite, a.num_tokens > 1024 ? 16 : 1) == 1 ? 1 : 16;
  const int64_t waves = static_cast<int64_t>((a.num_tokens + rows - 1) / rows) * a.head_groups;
  const int64_t kvg = (waves + kWriteThreads / kWave - 1) / (kWriteThreads / kWave);
  const int64_t qg = (static_cast<int64_t>(a.num_tokens) * a.hq * (D / 16) + kWriteThreads - 1) / kWriteThreads;
  if (kvg + qg > 0x7fffffffll)
    return fail(RLK_EINVAL, "rope_and_write_kv_blocks: %d rows exceed one launch; split the call",
                a.num_tokens);
  a.kv_groups = static_cast<int>(kvg);
  const uint32_t grid = static_cast<uint32_t>(kvg + qg);
  if (rows == 1) {
    write_kv_blocks_kernel<D, BS, kFp8, 1><<<grid, kWriteThreads, 0, stream>>>(a);
  } else {
    write_kv_blocks_kernel<D, BS, kFp8, 16><<<grid, kWriteThreads, 0, stream>>>(a);
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

// 16 lanes take 4 rows of the list for one head's K or V.
template <int D, bool kFp8>
__global__ __launch_bounds__(256) void read_kv_blocks_kernel(ReadArgs a) {
  constexpr int E = D / 16, kLanes = D / 16, kTok = 16 / kLanes;
  const int hkv = a.kv.num_kv_heads, bs = a.kv.block_size;
  const int64_t g = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int l16 = g % 16;
  const int64_t group = g / 16;
  const int quad = static_cast<int>(group / (2 * hkv)), unit = static_cast<int>(group % (2 * hkv));
  if (quad * 4 >= a.n) return;
  const bool is_v = unit >= hkv;
  const int kvh = is_v ? unit - hkv : unit;
  _Float16* out = is_v ? a.v_out : a.k_out;
  if (out == nullptr) return;
  const uint8_t* base = static_cast<const uint8_t*>(is_v ? a.kv.v : a.kv.k);
  const float* scales = is_v ? a.kv.v_scale : a.kv.k_scale;
  for (int u = 0; u < 4; u += is_v ? 1 : kTok) {
    const int i = quad * 4 + u + (is_v ? 0 : l16 / kLanes);
    if (i >= a.n) continue;
    const int slot = a.slots[i];
    if (slot < 0 || slot / bs >= a.kv.num_blocks) continue;
    const int blk = slot / bs, off = slot - blk * bs;
    const int64_t cell = static_cast<int64_t>(blk) * hkv + kvh;
    const float s = scales[cell];
    const uint8_t* tile = base + cell * (bs * D) + (off / 16) * (16 * D);
    _Float16* o = out + (static_cast<int64_t>(i) * hkv + kvh) * D;
    if (!is_v) {
      const int p = l16 % kLanes;
      const u32x4 w = load16(tile + p * 256 + (off % 16) * 16);
      const u32x2 a0 = scaled4(decode4<kFp8>(w[0]), s), a1 = scaled4(decode4<kFp8>(w[1]), s);
      const u32x2 b0 = scaled4(decode4<kFp8>(w[2]), s), b1 = scaled4(decode4<kFp8>(w[3]), s);
      store16(o + 8 * p, u32x4{a0[0], a0[1], a1[0], a1[1]});
      store16(o + D / 2 + 8 * p, u32x4{b0[0], b0[1], b1[0], b1[1]});
    } else {
#pragma unroll
      for (int gg = 0; gg < E / 4; ++gg) {
        const u32x4 w = load16(tile + gg * 1024 + (off % 16 / 4) * 256 + l16 * 16);
        const int sh = 8 * (off % 4);
        const uint32_t b = ((w[0] >> sh) & 0xff) | (((w[1] >> sh) & 0xff) << 8) |
                           (((w[2] >> sh) & 0xff) << 16) | (((w[3] >> sh) & 0xff) << 24);
        *reinterpret_cast<u32x2*>(o + E * l16 + 4 * gg) = scaled4(decode4<kFp8>(b), s);
      }
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
  a.head_groups = (2 * kv->num_kv_heads + 3) / 4;
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
