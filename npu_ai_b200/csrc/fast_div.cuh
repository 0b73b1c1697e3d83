// fast_div.cuh - division of a non-negative int by a number that the host knows, by a multiplication.
#pragma once

#include <stdint.h>

namespace npub200 {

// n / d for 0 <= n < 2^31: with p = 31 + ceil(log2 d) and mul = ceil(2^p / d), n mul / 2^p is above n / d by less than 1 / d.
struct Divisor {
  uint32_t mul, shift;
  __host__ __device__ int operator()(int n) const { return int((uint64_t(uint32_t(n)) * mul) >> shift); }
};
inline Divisor divisor(int64_t d) {
  int log = 0;
  while ((int64_t(1) << log) < d) ++log;
  return Divisor{uint32_t(((uint64_t(1) << (31 + log)) + uint64_t(d) - 1) / uint64_t(d)), uint32_t(31 + log)};
}

}  // namespace npub200
