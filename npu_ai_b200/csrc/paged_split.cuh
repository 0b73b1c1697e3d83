// paged_split.cuh - the run of key tiles that each block of the paged attention takes.
#pragma once

#include "fast_div.cuh"

namespace npub200 {

// The least run with which `blocks` runs of it hold all of `total` tiles, `least` at the least, rounded up to a multiple of
// `workers`, a power of two. by_blocks divides by `blocks`; from 2^31 tiles on (a batch of long caches) it is a 64-bit division,
// which takes longer.
__host__ __device__ inline long long tiles_of_run(long long total, int blocks, Divisor by_blocks, int least, int workers) {
  const long long up = total + blocks - 1;
  long long run = up < (1ll << 31) ? (long long)by_blocks(int(up)) : up / blocks;
  run = run > least ? run : least;
  return (run + workers - 1) & -(long long)workers;
}

}  // namespace npub200
