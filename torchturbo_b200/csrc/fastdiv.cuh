// Division by a number that the host knows.
#pragma once
#include <stdint.h>

namespace ttb {

// n / d for 0 <= n < 2^31 by a multiplication: with 2^s >= d and m = ceil(2^(31 + s) / d), m d exceeds 2^(31 + s) by less than 2^s, so
// that n m / 2^(31 + s) stays below the next whole number.
struct FastDiv {
  uint32_t mul, shift;
  __device__ __forceinline__ int operator()(int n) const { return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * mul) >> shift); }
};
static FastDiv fast_div(int d) {
  uint32_t s = 0;
  while ((1ull << s) < static_cast<uint64_t>(d)) ++s;
  return FastDiv{static_cast<uint32_t>(((1ull << (31 + s)) + d - 1) / d), 31 + s};
}

}  // namespace ttb
