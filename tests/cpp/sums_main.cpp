// Host check of the batch tables' saturating sums: any way of adding up requests
// gives the least of their sum and 2^30.
#include <algorithm>
#include <cstdio>
#include <vector>

#include "batch_sums.hpp"

using rlk::kSat;
using rlk::sat_add;

static_assert(sat_add(kSat, kSat) == kSat && sat_add(kSat, 1) == kSat && sat_add(kSat - 1, 1) == kSat &&
              sat_add(kSat / 2, kSat / 2 - 1) == kSat - 1 && sat_add(0, 0) == 0);

// A scan over `lanes` values in steps of doubling distance, as a wave makes it.
static std::vector<int> scan(std::vector<int> v, int lanes) {
  for (int o = 1; o < lanes; o <<= 1) {
    const std::vector<int> before = v;
    for (int i = o; i < lanes; ++i) v[i] = sat_add(before[i], before[i - o]);
  }
  return v;
}

int main() {
  const int pick[] = {0, 1, 5, kSat / 2, kSat - 1, kSat};
  unsigned seed = 1;
  for (int trial = 0; trial < 2000; ++trial) {
    std::vector<int> v(64);
    for (int& x : v) {
      seed = seed * 1664525u + 1013904223u;
      x = pick[(seed >> 16) % 6];
      if ((seed >> 8) % 3 != 0) x = std::min(x, 5);
    }
    const std::vector<int> got = scan(v, 64);
    long long sum = 0;
    for (int i = 0; i < 64; ++i) {
      sum += v[i];
      if (got[i] != std::min<long long>(sum, kSat)) {
        std::printf("FAIL trial %d value %d: %d for %lld\n", trial, i, got[i], sum);
        return 1;
      }
    }
  }
  std::printf("PASS\n");
  return 0;
}
