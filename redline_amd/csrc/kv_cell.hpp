// One head's row into its cell of the paged cache (FP16, or INT8 with a
// per-(token, head) scale): what the cache writes share.
#pragma once

#include "device.hpp"

namespace rlk {

// The planes of one layer and how their cells are counted.
struct CellPlanes {
  void* k;
  void* v;
  void* k_scale;  // float[cells], or fp16[cells] when scale16
  void* v_scale;
  int scale16;
};

// Stores a head's D elements into `cell`: x0 = elements p0 .. p0 + 7 of this
// lane and x1 = those D/2 later, fp16 values.  Every lane of the head's
// group (D/16 lanes) calls it.
template <int D, bool kInt8>
__device__ __forceinline__ void store_cell(const CellPlanes& a, bool is_v, int64_t cell, int p0, f32x8 x0, f32x8 x1) {
#pragma clang fp contract(off)
  constexpr bool NT = true;  // streaming accesses of whole lines: measured faster at every batch size
  constexpr int kHalf = D / 2;
  constexpr int kLPH = kHalf / 8;
  if constexpr (!kInt8) {
    _Float16* dst = static_cast<_Float16*>(is_v ? a.v : a.k) + cell * D;
    st16<NT>(reinterpret_cast<u32x4*>(dst + p0), pack8(x0));
    st16<NT>(reinterpret_cast<u32x4*>(dst + kHalf + p0), pack8(x1));
  } else {
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fmaxf(__builtin_fabsf(x0[j]), __builtin_fabsf(x1[j])));
    amax = group_max<kLPH>(amax);
    float scale = amax > 0.f ? amax / 127.f : 1.f;
    if (a.scale16) scale = round_f16(scale);  // extension: quantise against the stored fp16 scale
    const float inv = 1.f / scale;
    i8x8 q0, q1;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      q0[j] = static_cast<int8_t>(__builtin_rintf(fminf(fmaxf(x0[j] * inv, -127.f), 127.f)));
      q1[j] = static_cast<int8_t>(__builtin_rintf(fminf(fmaxf(x1[j] * inv, -127.f), 127.f)));
    }
    // An INT8 cell row of D = 128 is one 128-byte line, written as two
    // 64-byte halves (the rotation pairs i and i + D/2 sit in different
    // halves).  Ordinary stores let L2 join the halves before the line goes
    // to HBM; with the streaming hint each half went out on its own (C4:
    // 63.7 against 59.4 us per call).
    int8_t* dst = static_cast<int8_t*>(is_v ? a.v : a.k) + cell * D;
    st8<false>(reinterpret_cast<u32x2*>(dst + p0), __builtin_bit_cast(u32x2, q0));
    st8<false>(reinterpret_cast<u32x2*>(dst + kHalf + p0), __builtin_bit_cast(u32x2, q1));
    if (p0 == 0) {
      void* sp = is_v ? a.v_scale : a.k_scale;
      if (a.scale16) {
        static_cast<_Float16*>(sp)[cell] = static_cast<_Float16>(scale);
      } else {
        static_cast<float*>(sp)[cell] = scale;
      }
    }
  }
}

}  // namespace rlk
