// The block-scaled 8-bit KV cache: codes, scales and byte layout shared by the
// kernels that write and read it (layout: redline_amd/rlk.h).
//
// Scales are powers of two.  x / s is then exact, so a code is one rounding of
// the fp16 value it stands for; requantising a code when the scale of its block
// grows is exact for e4m3 down to its subnormals; and a stored value, a code
// of at most 8 significant bits times 2^e, is an exact fp16 number, so no
// consumer rounds it again.  The price is up to one bit of the code range.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "device.hpp"
#include "redline_amd/rlk.h"
#include "status.hpp"

namespace rlk {

constexpr int kTileTokens = 16;  // tokens of a layout tile

// Scalar facts of a format: the largest code value, and the code limit at the
// largest scale, where code * scale must stay a finite fp16 number.
template <bool kFp8>
struct BlockFormat {
  static constexpr float kMax = kFp8 ? 448.f : 127.f;
  static constexpr float kTopScale = kFp8 ? 256.f : 1024.f;  // for amax up to 65504
  static constexpr float kTopMax = kFp8 ? 240.f : 63.f;
};

// The least power of two s >= 2^-24 with amax <= kMax * s; 0 for amax == 0.
// With kMax = m * 2^e, amax = n * 2^x: s = 2^(x - e), or twice that when n > m,
// which the addition carries into the exponent field.  (2^-24 is fp16's
// smallest spacing: no smaller scale would store anything more exactly.)
template <bool kFp8>
__device__ __forceinline__ float block_scale(float amax) {
  constexpr uint32_t qmax = __builtin_bit_cast(uint32_t, BlockFormat<kFp8>::kMax);
  constexpr uint32_t mant = qmax & 0x7fffffu, expo = (qmax >> 23) - 127;
  const uint32_t bits = __builtin_bit_cast(uint32_t, fminf(amax, 65504.f));
  const uint32_t e = (bits - mant + 0x7fffffu) >> 23;
  const uint32_t s = (e < 103 + expo ? 103 : e - expo) << 23;  // biased exponent of 2^-24: 103
  return amax > 0.f ? __builtin_bit_cast(float, s) : 0.f;
}

// 1 / s of a power-of-two scale (0 for 0).
__device__ __forceinline__ float inv_scale(float s) {
  return s > 0.f ? __builtin_bit_cast(float, (254u << 23) - __builtin_bit_cast(uint32_t, s)) : 0.f;
}

// Largest |code| that may be stored at scale s.
template <bool kFp8>
__device__ __forceinline__ float code_limit(float s) {
  return s >= BlockFormat<kFp8>::kTopScale ? BlockFormat<kFp8>::kTopMax : BlockFormat<kFp8>::kMax;
}

// Four values to four codes, rne(clamp(x * inv)), value 0 in the low byte.
// INT8: adding 1.5 * 2^23 leaves the rounded integer in the low mantissa bits.
template <bool kFp8>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, float inv,
                                            float lim) {
#pragma clang fp contract(off)
  const float x[4] = {fminf(fmaxf(a * inv, -lim), lim), fminf(fmaxf(b * inv, -lim), lim),
                      fminf(fmaxf(c * inv, -lim), lim), fminf(fmaxf(d * inv, -lim), lim)};
  if constexpr (kFp8) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true));
  } else {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = __builtin_bit_cast(uint32_t, x[i] + 12582912.f);
    const uint32_t lo = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(u[3], u[2], 0x04000c0cu);
    return lo | hi;
  }
}

// Four codes to their values (unscaled).
template <bool kFp8>
__device__ __forceinline__ f32x4 decode4(uint32_t w) {
  if constexpr (kFp8) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
    const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
    return f32x4{lo[0], lo[1], hi[0], hi[1]};
  } else {
    const int v = static_cast<int>(w);
    return f32x4{static_cast<float>((v << 24) >> 24), static_cast<float>((v << 16) >> 24),
                 static_cast<float>((v << 8) >> 24), static_cast<float>(v >> 24)};
  }
}

// Four codes to fp16, exactly (both formats' codes are fp16 numbers).
template <bool kFp8>
__device__ __forceinline__ f16x4 codes_to_f16(uint32_t w) {
  if constexpr (kFp8) {
    const f16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false);
    const f16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true);
    return f16x4{lo[0], lo[1], hi[0], hi[1]};
  } else {  // 1152 + code under an fp16 exponent byte, as in int8x8_to_f16
    const uint32_t u = w ^ 0x80808080u;
    const f16x2 lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) -
                     static_cast<_Float16>(1152);
    const f16x2 hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) -
                     static_cast<_Float16>(1152);
    return f16x4{lo[0], lo[1], hi[0], hi[1]};
  }
}

// Checks of a view that every entry point makes; RLK_OK or a failure status.
int check_block_view(const rlk_kv_block_view* kv, const char* what);

}  // namespace rlk
