// Saturating sums of token rows, blocks and work items, as the batch tables form
// them: never negative, whatever the requests ask for.
#pragma once

#include <cstdint>

namespace rlk {

constexpr int kSat = 1 << 30;  // running sums saturate here

// min(a + b, kSat) of 0 <= a, b <= kSat.  Two saturated sums add up to 2^31, which an
// int does not hold: the sum is formed without a sign.
constexpr int sat_add(int a, int b) {
  const uint32_t s = static_cast<uint32_t>(a) + static_cast<uint32_t>(b);
  return s < static_cast<uint32_t>(kSat) ? static_cast<int>(s) : kSat;
}

}  // namespace rlk
