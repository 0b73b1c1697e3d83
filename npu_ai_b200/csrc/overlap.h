// overlap.h - whether two strided tensors have a byte in common, or one holds a byte twice. Host code without torch or CUDA.
//
// A tensor is its runs of contiguous bytes at base + sum_i x_i step_i, 0 <= x_i < n_i. Two of them are compared dimension by
// dimension from the largest step down, where only those indices are followed whose bounds meet. Two dimensions of one step (views
// of one buffer, which is what interleaves) are one: only the difference of the indices counts, and where steps are longer than
// what lies within them two differences at most are left. Exact, but for tensors that take more than kOverlapSteps comparisons
// (interleaved with different steps): these count as overlapping.
#pragma once

#include <stdint.h>

#include <algorithm>

namespace npub200 {

constexpr int kOverlapDims = 5, kOverlapSteps = 4096;

struct ByteRuns {
  uintptr_t base = 0;
  int64_t run = 0;  // bytes; 0: the tensor is empty
  int dims = 0;
  int64_t n[kOverlapDims], step[kOverlapDims];  // steps in bytes, the largest first
};

// Of a tensor with up to kOverlapDims dimensions, strides >= 0.
inline ByteRuns byte_runs(const void* p, int64_t element, int dims, const int64_t* sizes, const int64_t* strides) {
  ByteRuns r;
  r.base = reinterpret_cast<uintptr_t>(p);
  r.run = element;
  for (int i = 0; i < dims; ++i) {
    if (sizes[i] == 0) {
      r.run = 0;
      return r;
    }
    if (sizes[i] == 1 || strides[i] == 0) continue;  // no bytes of their own
    const int64_t step = strides[i] * element;
    int at = r.dims++;
    for (; at > 0 && r.step[at - 1] < step; --at) r.n[at] = r.n[at - 1], r.step[at] = r.step[at - 1];
    r.n[at] = sizes[i];
    r.step[at] = step;
  }
  while (r.dims > 0 && r.step[r.dims - 1] == r.run) r.run *= r.n[--r.dims];
  return r;
}

// Bytes from the first to the last of dimension i and those within it.
inline int64_t bytes_span(const ByteRuns& r, int i) {
  int64_t span = r.run;
  for (; i < r.dims; ++i) span += (r.n[i] - 1) * r.step[i];
  return span;
}

// Dimensions i of a and j of b and those within them, b beginning `ahead` bytes behind a.
inline bool bytes_meet(const ByteRuns& a, int i, const ByteRuns& b, int j, int64_t ahead, int& left) {
  if (ahead >= bytes_span(a, i) || -ahead >= bytes_span(b, j)) return false;
  if (i == a.dims && j == b.dims) return true;
  if (--left < 0) return true;
  const int64_t sa = i < a.dims ? a.step[i] : 0, sb = j < b.dims ? b.step[j] : 0, s = std::max(sa, sb);
  const int di = i + (sa == s), dj = j + (sb == s);
  // b's index less a's, where s is the step of both; else the index of the one whose step it is, a's counted down.
  const int64_t lowest = sa == s ? 1 - a.n[i] : 0, highest = sb == s ? b.n[j] - 1 : 0;
  // -(b's span) < ahead + k s < a's span
  const auto floor_div = [](int64_t x, int64_t y) { return x >= 0 ? x / y : -((-x + y - 1) / y); };
  const int64_t first = std::max(lowest, floor_div(-bytes_span(b, dj) - ahead, s) + 1);
  const int64_t last = std::min(highest, floor_div(bytes_span(a, di) - ahead - 1, s));
  for (int64_t k = first; k <= last; ++k)
    if (bytes_meet(a, di, b, dj, ahead + k * s, left)) return true;
  return false;
}

inline bool bytes_overlap(const ByteRuns& a, const ByteRuns& b) {
  if (a.run == 0 || b.run == 0) return false;
  int left = kOverlapSteps;
  return bytes_meet(a, 0, b, 0, int64_t(b.base) - int64_t(a.base), left);
}

// Whether two elements of a tensor lie on the same bytes: windows that overlap (what a stride of 0 repeats is not asked here). Of
// each dimension, whether what lies within it meets itself one or more steps on.
inline bool bytes_repeat(const ByteRuns& a) {
  int left = kOverlapSteps;
  for (int i = 0; a.run != 0 && i < a.dims; ++i) {
    const int64_t within = bytes_span(a, i + 1);
    for (int64_t k = 1; k < a.n[i] && k * a.step[i] < within; ++k)
      if (bytes_meet(a, i + 1, a, i + 1, k * a.step[i], left)) return true;
  }
  return false;
}

}  // namespace npub200
