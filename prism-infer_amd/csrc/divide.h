// Division by a number that a launch fixes, as a multiplication.
#pragma once

#include "common.h"

namespace prism {

// n / d for 0 <= n < 2^31: with 2^l the smallest power of two >= d and m =
// ceil(2^(31 + l) / d), n m is above n 2^(31 + l) / d by less than n 2^l / d, so
// that its floor is n / d's.
struct Divisor {
  uint32_t m;
  int shift;
};

inline Divisor divisor(int d) {
  int l = 0;
  while ((int64_t{1} << l) < d) ++l;
  return Divisor{static_cast<uint32_t>(((uint64_t{1} << (31 + l)) + d - 1) / d), 31 + l};
}

__device__ __forceinline__ int divide(int n, Divisor d) {
  return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * d.m) >> d.shift);
}

}  // namespace prism
