// Paged prefill attention over the block-scaled 8-bit cache, for gfx950.
//
// Causal attention of a sequence's new tokens over its cached and new keys.
// Rows are (token, query head) pairs of one kv head, head fastest, so K and V
// are read and converted once for the G heads of the group; a workgroup of 4
// waves takes 128 rows, 32 per wave, and walks the keys in tiles of 64.
//   * Codes go to registers one tile ahead, become fp16 (code * scale, exact) and
//     are written to one of two LDS images in the operand order of
//     v_mfma_f32_32x32x16_f16: K as 16-byte chunks [piece][half][key], V as
//     [16-key tile][lane half][dim], each chunk the 8 keys of a lane's own
//     scores; both are read as whole contiguous rows (no bank conflicts), and
//     neither operand is transposed or exchanged anywhere.
//   * S^T = K Q^T leaves one query row per lane (its keys split over the two lane
//     halves), so the running maximum and sum are lane-local, and the scores are
//     the B operand of O^T = V^T P^T as they stand.
//   * One barrier per tile: tile t + 1 is converted between the products of
//     tile t.
// m, l and the output accumulate in fp32; P is rounded to fp16 (at most 1).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cstdint>

#include "kv_blocks.hpp"

namespace rlk {

int check_block_params(const rlk_block_attention_params* p, const char* what);

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kThreads = 256;
constexpr int kRows = 128;     // (token, head) rows of a workgroup
constexpr int kTileKeys = 64;

struct PrefillArgs {
  rlk_block_attention_params p;
  rlk_prefill_attention_work w;
  int group;  // query heads per kv head
};

// Four codes times their scale as fp16, exactly.
template <bool kFp8>
__device__ __forceinline__ u32x2 scaled_f16(uint32_t w, float s) {
  f16x4 v;
  if constexpr (kFp8) {
    const f16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, false);
    const f16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, true);
    v = f16x4{lo[0], lo[1], hi[0], hi[1]};
  } else {
    v = codes_to_f16<false>(w) * static_cast<_Float16>(s);
  }
  return __builtin_bit_cast(u32x2, v);
}

template <int D>
struct Image {
  u32x4 k[D / 16][2][kTileKeys];  // chunk (piece, half, key): 8 dims
  u32x4 v[4][2][D];               // chunk (16-key tile, lane half, dim index): 8 keys
};

// A thread's pieces of a key tile: piece i is 16-byte piece (tid + 256 i) of the
// tile's 4 layout tiles in order.
template <int D>
struct TileCodes {
  static constexpr int kPieces = D / 64;
  u32x4 k[kPieces], v[kPieces];
  float ks[kPieces], vs[kPieces];
};

template <int D, bool kFp8>
__global__ __launch_bounds__(kThreads, 2) void prefill_blocks_kernel(PrefillArgs a) {
  constexpr int E = D / 16, kPieces = D / 64, kPerTile = D;  // 16-byte pieces of a layout tile
  constexpr float kLog2e = 1.4426950408889634f;
  __shared__ Image<D> img[2];
  const rlk_block_attention_params& p = a.p;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int half = lane / 32, col = lane % 32;
  const int kvh = blockIdx.x, G = a.group;
  const int seq = a.w.seq_ids[blockIdx.z];
  if (seq < 0) return;
  const int q_len = a.w.q_len[seq], rows = q_len * G;
  // the rows with the most keys first
  const int row0 = (gridDim.y - 1 - blockIdx.y) * kRows;
  if (row0 >= rows) return;
  const int past = a.w.ctx_len[seq] - q_len, q_start = a.w.q_start[seq];
  const int bs = p.kv.block_size, tpb = bs / kTileTokens, hkv = p.kv.num_kv_heads;
  const int most = static_cast<int>(min(static_cast<int64_t>(p.max_blocks_per_seq) * bs, static_cast<int64_t>(1 << 30)));
  // keys of the workgroup's last row; those of each lane's row
  const int last_tok = min(row0 + kRows, rows) - 1;
  const int keys = min(past + last_tok / G + 1, most);
  const int row = min(row0 + wave * 32 + col, rows - 1);  // rows past the end repeat the last one
  const int tok = row / G, head = kvh * G + row - tok * G;
  const int row_keys = min(past + tok + 1, most);
  const int first_row = min(row0 + wave * 32, rows - 1);
  const int full = min(past + first_row / G + 1, most);  // keys that every row of the wave sees

  const _Float16* q = reinterpret_cast<const _Float16*>(p.q) + static_cast<int64_t>(q_start + tok) * p.q_stride + head * D;
  f16x8 qb[E];
#pragma unroll
  for (int pc = 0; pc < E; ++pc) {
    qb[pc] = __builtin_bit_cast(f16x8, load16(q + half * (D / 2) + 8 * pc));
    if (p.scale < 0.f) qb[pc] = -qb[pc];  // the maximum is taken before the scale
  }

  const int32_t* table = p.block_tables + static_cast<int64_t>(seq) * p.max_blocks_per_seq;
  const int tiles = (keys + kTileKeys - 1) / kTileKeys, last16 = (max(keys, 1) - 1) / kTileTokens;
  // block of this thread's layout tile i of key tile t (tiles past the last repeat it)
  auto entry = [&](int t, int i) {
    const int t16 = min(4 * t + (tid + kThreads * i) / kPerTile, last16);
    return table[t16 / tpb];
  };
  auto request = [&](TileCodes<D>& c, int t, const int (&id)[kPieces]) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int t16 = min(4 * t + (tid + kThreads * i) / kPerTile, last16);
      const int b = static_cast<uint32_t>(id[i]) < static_cast<uint32_t>(p.kv.num_blocks) ? id[i] : 0;
      const int64_t cell = static_cast<int64_t>(b) * hkv + kvh;
      const int64_t at = (cell * tpb + t16 % tpb) * (kTileTokens * D) + (tid % kPerTile) * 16;
      c.k[i] = load16(static_cast<const uint8_t*>(p.kv.k) + at);
      c.v[i] = load16(static_cast<const uint8_t*>(p.kv.v) + at);
      c.ks[i] = p.kv.k_scale[cell];
      c.vs[i] = p.kv.v_scale[cell];
    }
  };
  auto convert = [&](const TileCodes<D>& c, Image<D>& im, int t) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int t16 = (tid + kThreads * i) / kPerTile, piece = tid % kPerTile;
      {
        const int pc = piece / 16, key = 16 * t16 + piece % 16;
        const u32x2 a0 = scaled_f16<kFp8>(c.k[i][0], c.ks[i]), a1 = scaled_f16<kFp8>(c.k[i][1], c.ks[i]);
        const u32x2 b0 = scaled_f16<kFp8>(c.k[i][2], c.ks[i]), b1 = scaled_f16<kFp8>(c.k[i][3], c.ks[i]);
        im.k[pc][0][key] = u32x4{a0[0], a0[1], a1[0], a1[1]};
        im.k[pc][1][key] = u32x4{b0[0], b0[1], b1[0], b1[1]};
      }
      const int g = piece / 64, rho = piece / 16 % 4, m = piece % 16;
      u32x4 v = c.v[i];
      if (t * kTileKeys + kTileKeys > keys) {  // uniform: bytes past the keys may be anything
        const int keep = min(max(keys - t * kTileKeys - 16 * t16 - 4 * rho, 0), 4);
        const uint32_t mask = keep == 0 ? 0u : 0xffffffffu >> (32 - 8 * keep);
        v &= u32x4{mask, mask, mask, mask};
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        reinterpret_cast<u32x2*>(&im.v[t16][rho % 2][(4 * g + j) * 16 + m])[rho / 2] = scaled_f16<kFp8>(v[j], c.vs[i]);
    }
  };

  f32x16 o[D / 32];
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  // (below every score of fp16 rows, and far above a masked one)
  float m = -1e30f, l = 0.f;
  const float cs = __builtin_fabsf(p.scale) * kLog2e;
  TileCodes<D> codes;
  int id[kPieces];
  if (tiles > 0) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) id[i] = entry(0, i);
    request(codes, 0, id);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) id[i] = entry(1, i);
    convert(codes, img[0], 0);
    request(codes, 1, id);
  }
  for (int t = 0; t < tiles; ++t) {
    const Image<D>& im = img[t & 1];
    __syncthreads();  // tile t is written, tile t - 1 has been read
#pragma unroll
    for (int i = 0; i < kPieces; ++i) id[i] = entry(t + 2, i);
    f32x16 s[2];
#pragma unroll
    for (int kh = 0; kh < 2; ++kh) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kh][i] = 0.f;
#pragma unroll
      for (int pc = 0; pc < E; ++pc)
        s[kh] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, im.k[pc][half][32 * kh + col]),
                                                       qb[pc], s[kh], 0, 0, 0);
    }
    if (t + 1 < tiles) {
      convert(codes, img[(t + 1) & 1], t + 1);
      request(codes, t + 2, id);
    }
    // element i of half kh: key 64 t + 32 kh + 8 (i / 4) + 4 half + i % 4
    if ((t + 1) * kTileKeys > full) {
#pragma unroll
      for (int kh = 0; kh < 2; ++kh)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (t * kTileKeys + 32 * kh + 8 * (i / 4) + 4 * half + i % 4 >= row_keys) s[kh][i] = -FLT_MAX;
    }
    float mx = s[0][0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[0][i]);
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[1][i]);
    mx = rows_max<true>(mx);
    const float mn = fmaxf(m, mx);
    if (__any(mn != m)) {
      const float f = __builtin_amdgcn_exp2f((m - mn) * cs);
      l *= f;
#pragma unroll
      for (int d = 0; d < D / 32; ++d) o[d] *= f;
      m = mn;
    }
    const float mc = m * cs;
    f16x8 pb[4];
#pragma unroll
    for (int kh = 0; kh < 2; ++kh)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = __builtin_amdgcn_exp2f(fmaf(s[kh][i], cs, -mc));
        l += e;
        pb[2 * kh + i / 8][i % 8] = static_cast<_Float16>(e);
      }
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, im.v[kt][half][32 * d + col]),
                                                      pb[kt], o[d], 0, 0, 0);
  }
  l = rows_sum<true>(l);
  if (row0 + wave * 32 + col >= rows) return;  // no barrier follows
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
  const int64_t tiles = (static_cast<int64_t>(w->max_q_tiles) * RLK_PREFILL_TILE_Q * G + kRows - 1) / kRows;
  if (w->num_seqs > 65535 || tiles > 65535)
    return fail(RLK_EINVAL, "%s: %d sequences of %d query tiles exceed one launch; split the call",
                what, w->num_seqs, w->max_q_tiles);
  const PrefillArgs a = {*p, *w, G};
  const dim3 grid(p->kv.num_kv_heads, static_cast<uint32_t>(tiles), w->num_seqs);
  const bool fp8 = p->kv.format == RLK_KV_BLOCK_FP8;
  if (p->kv.head_dim == 128) {
    if (fp8) prefill_blocks_kernel<128, true><<<grid, kThreads, 0, stream>>>(a);
    else prefill_blocks_kernel<128, false><<<grid, kThreads, 0, stream>>>(a);
  } else {
    if (fp8) prefill_blocks_kernel<64, true><<<grid, kThreads, 0, stream>>>(a);
    else prefill_blocks_kernel<64, false><<<grid, kThreads, 0, stream>>>(a);
  }
  return launch_status(what);
}
