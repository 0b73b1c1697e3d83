// attention_masked.cuh - attention with masks, score modifiers and grouped key/value heads on B200:
//   o_i = sum_j softmax_j(s_ij) v_j over the keys j that row i may see (zeros if none),
//   s_ij = cap tanh(scale q_i.k_j / cap) - slope_h |p_i - j| + table_h[clamp(j - p_i)] + mask_ij.
// The reference sends every such call to the CPU (its attention gate, comfyui node :39-99); here prompts and single
// tokens run on the tensor cores.
//
// Every rule but the mask tensor leaves a row ONE interval [lo, hi) of keys: lengths, causal (hi = p + 1), prefix
// (hi = max(p + 1, prefix)), documents ([start, end) of the row's document). A softmax thread owns one row, so its mask
// is two registers; the CTA walks only the key tiles of the union of its rows' intervals, and only tiles that some row
// of a warp sees in part pay for masking (two compares a score). A warp none of whose rows sees a tile writes P = 0
// without reading S.
//
// One kernel, one 128-row Q tile per CTA, 64-key tiles, up to two CTAs per SM (the structure of
// attention_fwd_tcgen05_kernel with eight or sixteen softmax warps, a TMA producer warp and an MMA warp):
//   * Two softmax warps share a lane quarter (32 rows): each takes 32 of the tile's 64 keys, they exchange their row
//     maxima through shared memory, keep a partial sum each, and rescale half of the O columns each. A tile's step is a
//     chain of waits (TMEM load, maximum, exchange, exponentials, store) of which the instructions are half.
//   * Two streams of key tiles where an SM holds one CTA (two_streams in attention_masked.cu): sixteen warps, eight on the
//     even and eight on the odd tiles with running maxima, sums and O accumulators of their own, joined at the end. One
//     stream's waits are the other's work: 2x8x1024x1024x80 with a bool mask 32.5 -> 18.3 us (now 17.9).
//   * Q rows: `pack` query heads x T positions. With few queries the heads of a group that share a K/V head fill the
//     tile together (one TMA box of pack heads x T positions), so the cache is read once per group, not once per head.
//   * Keys beyond the union inside its last (or before it inside its first) tile may be stale cache memory: their V
//     rows are zeroed in shared memory before the P V product, since P = 0 times a NaN would be a NaN. Their scores are
//     replaced, not added to.
//   * Split keys (grid z): when the row tiles leave most SMs idle, each CTA takes an equal part of its tile's keys. Few
//     parts are a cluster, which joins them through its shared memory; otherwise each CTA writes its unnormalised O row,
//     max and sum to the workspace and attention_join_kernel joins the parts, either way in part order.
// What bounds it: a token against a long cache, memory (16x32/8 over 16384 keys of 128: 134 us, 6.1 of 6.5 TB/s); a long
// prompt, the waits of the softmax step's chain (1x32/8x4096x4096x128 causal: 130 us, 1.05 PFLOP/s; no pipe is full: tensor
// 54%, MUFU 55%, issue 55%, loads and stores of shared memory 11%); everything between, the same chain, 0.7 - 1.3 us a
// tile, and 2.5 - 4 us of a CTA's start and end.
// Rounding: P is rounded to bf16 for the tensor core (relative 2^-8, as in the unmasked kernel); the sums, the maxima,
// the modifiers and O are f32.
#pragma once

#include <algorithm>
#include <cfloat>
#include <climits>

#include "attention_sm100.cuh"

namespace npub200 {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaskedBN = 64;        // keys per tile
constexpr int kHalf = kMaskedBN / 2;  // keys per softmax thread: two warps share the rows of a TMEM lane quarter
constexpr int kSoftWarps = 2 * kSoftmaxWarps;  // of a stream of key tiles
constexpr int kMaxSplits = 64;
constexpr int kMaxCluster = 16;  // parts that are joined within a cluster of CTAs
constexpr int kTableMargin = 128;     // repeated ends of the distance bias in shared memory, either side
constexpr int kTableSmemMax = 10240;  // bytes: keeps two CTAs per SM

struct MaskedArgs {
  AttnArgs a;
  int G;              // query heads per key/value head
  int pack, T;        // a Q tile holds `pack` heads x T positions
  int inv_row;        // 65536 / (pack or T), rounded up: the divisor of a tile row
  int head_fast;      // tile row r = position * pack + head (1) or head * T + position (0)
  int q_bytes;        // bytes of one 64-column atom of the Q box
  int tiles;          // Q tiles along the positions
  int pairs, groups;  // (batch, head group) pairs, groups of a sequence: the grid is pairs x tiles x splits
  int splits;
  int cluster;        // the parts of a tile are a cluster, which joins them through its shared memory
  float* part_o;      // [splits][pairs][tiles][128][D] unnormalised O rows
  float2* part_ml;    // [splits][pairs][tiles][128] (max in log2 units, sum)
  int causal;
  long long q_start;
  const int* q_starts;
  long long prefix;
  const int* prefixes;
  const int* kv_lens;
  const int* docs;
  int ndocs;
  long long doc_stride;
  int gaps;           // documents may end in keys that no row sees: causal, and a start that may be below 0
  float cap_in, cap_out;  // capped score in log2 units = cap_out x tanh(cap_in x raw score)
  float cap_poly[6];      // cap_out x kTanhRatio: operands straight from the constant bank
  const float* slopes;
  const float* table;
  int max_dist;
  const void* mask;
  int mask_kind;  // 0 none, 1 bool, 2 bf16, 3 f32
  int mask_vec;   // rows can be read in 16-byte words
  int mask_row;   // the rows of a warp share one mask row
  int table_smem; // the tile's head has its distance bias in shared memory
  int out_vec;    // output rows can be written in 16-byte words
  int out_sectors;  // and in 32-byte ones (with split keys: the partial rows)
  long long m_sb, m_sh, m_sq;
};

// What a softmax thread knows of its row.
struct Row {
  int lo, hi;       // keys it may see
  int p;            // its position among the keys
  bool valid;       // a row of the output
  int head, i, b;
  float slope;      // slopes[head] * log2 e
  const uint8_t* mask;  // its mask row
  // Over the warp's rows that see something (output rows for the positions): what a tile is to all of them is decided
  // from these, without a vote.
  int lo_min, lo_max, hi_min, hi_max, p_min, p_max;
};

__device__ __forceinline__ int clamp_pos(long long x) {
  return int(min(max(x, -(1ll << 30)), 1ll << 30));
}

// The document [lo, hi) that token i lies in; false outside every document. Few borders: the warp reads them together and
// every lane looks at each; many: a binary search. Documents of no tokens are passed over.
__device__ __forceinline__ bool document_of(const int* off, int docs, int i, int lane, int& lo, int& hi) {
  lo = hi = 0;
  int below = 0;  // borders at or below i
  if (docs < 64) {
    bool above = false;
    for (int base = 0; base <= docs; base += 32) {
      const int v = off[min(base + lane, docs)];
      for (int k = 0; k < 32 && base + k <= docs; ++k) {
        const int o = __shfl_sync(0xffffffffu, v, k);
        if (o <= i) {
          lo = o;
          ++below;
        } else if (!above) {
          hi = o;
          above = true;
        }
      }
    }
  } else {
    int right = docs + 1;  // off[below - 1] <= i < off[right]
    while (below < right) {
      const int mid = (below + right) >> 1;
      if (off[mid] <= i)
        below = mid + 1;
      else
        right = mid;
    }
    if (below >= 1 && below <= docs) {
      lo = off[below - 1];
      hi = off[below];
    }
  }
  return below >= 1 && below <= docs;
}

// The row of thread r of the tile (whole warps call it).
__device__ __forceinline__ Row row_of(const MaskedArgs& m, int r, int tile, int h0, int b) {
  Row w;
  // r / pack or r / T by a multiplication (both at most 128, so the reciprocal rounded up is exact for r < 128)
  const int q = (r * m.inv_row) >> 16;
  const int s = m.head_fast ? q : r - q * m.T;
  const int g = m.head_fast ? r - q * m.pack : q;
  w.i = tile * m.T + s;
  w.head = h0 + g;
  w.b = b;
  w.valid = r < m.pack * m.T && w.i < m.a.Sq;
  if (!w.valid) w.head = h0;
  const int len = m.kv_lens != nullptr ? m.kv_lens[b] : m.a.Skv;
  const long long start = m.q_starts != nullptr ? (long long)m.q_starts[b] : m.q_start;
  const long long prefix = m.prefixes != nullptr ? (long long)m.prefixes[b] : m.prefix;
  w.slope = m.slopes != nullptr ? m.slopes[w.head] * kLog2e : 0.0f;
  w.p = w.valid ? clamp_pos(start + w.i) : 0;
  int lo = 0, hi = min(m.a.Skv, len);
  if (m.causal) hi = min(hi, max(w.p + 1, clamp_pos(prefix)));
  if (m.docs != nullptr) {
    int d0, d1;
    const bool in = document_of(m.docs + b * m.doc_stride, m.ndocs, w.i, r & 31, d0, d1);
    lo = max(d0, 0);
    hi = in ? min(hi, d1) : 0;
  }
  const bool any = w.valid && hi > lo;  // a row that sees nothing leaves the union alone
  w.lo = any ? lo : 0;
  w.hi = any ? hi : 0;
  w.lo_min = __reduce_min_sync(0xffffffffu, any ? lo : INT_MAX);
  w.lo_max = __reduce_max_sync(0xffffffffu, any ? lo : 0);
  w.hi_min = __reduce_min_sync(0xffffffffu, any ? hi : (w.valid ? 0 : INT_MAX));  // a row that sees nothing is masked
  w.hi_max = __reduce_max_sync(0xffffffffu, any ? hi : 0);
  w.p_min = __reduce_min_sync(0xffffffffu, w.valid ? w.p : INT_MAX);
  w.p_max = __reduce_max_sync(0xffffffffu, w.valid ? w.p : -INT_MAX);
  const int esz = m.mask_kind == 3 ? 4 : m.mask_kind;
  w.mask = static_cast<const uint8_t*>(m.mask) +
           ((long long)b * m.m_sb + (long long)w.head * m.m_sh + (long long)(w.valid ? w.i : 0) * m.m_sq) * esz;
  return w;
}

// Which of the 64 keys of the tile at kv0 no row of the Q tile sees, as bits, with documents and causal (whole warps call
// it). From position 0 on every key of a document is seen by its own row or by a later one of the Q tile; a start below 0
// takes each document's last keys from all its rows. Only the kernel for any modifier has this code, and those calls go
// there: even out of line it cost the others 2% (1x32/8x4096x128 causal 128.7 us without, 131.5 with it).
static __device__ __noinline__ uint64_t unseen_keys(const MaskedArgs& m, int b, int tile, int kv0, int lane) {
  const long long start = m.q_starts != nullptr ? (long long)m.q_starts[b] : m.q_start;
  const long long prefix = m.prefixes != nullptr ? (long long)m.prefixes[b] : m.prefix;
  const int i0 = tile * m.T, i1 = min(i0 + m.T, m.a.Sq);
  uint64_t bits = 0;
  if (start >= 0) return bits;
  for (int k = 0; k < kMaskedBN; k += 32) {
    const int key = kv0 + k + lane;
    int d0, d1;
    const bool in = document_of(m.docs + b * m.doc_stride, m.ndocs, key, lane, d0, d1);
    const int last = min(d1, i1) - 1;  // the document's last row in the Q tile sees the most
    const bool seen = in && last >= max(d0, i0) && (key <= clamp_pos(start + last) || key < prefix);
    bits |= uint64_t(__ballot_sync(0xffffffffu, !seen)) << k;
  }
  return bits;
}

// tanh(y) / y as a polynomial in y^2, |y| <= 1 (fit_tanh_poly.py beside this file; relative error 7e-7).
constexpr float kTanhRatio[6] = {9.999994040e-01f, -3.332909346e-01f, 1.328188479e-01f,
                                 -5.161965266e-02f, 1.676048711e-02f, -3.074449487e-03f};

// What a kernel instantiation does to the scores: nothing, one of these, or any of them as the arguments say. (One
// kernel with every branch spent as long on instruction fetches as on the instructions.)
// A mask tensor with a row of its own for each query and one whose row a warp shares are two kinds: in one kernel a few
// instructions more in either moved the other by 10% (1x24x4608x4608x128 with a bool mask of its own rows 431 us before the
// NaN tests, 465 with them, 408 in a kernel of its own).
constexpr int kFeatCap = 1, kFeatDistance = 2, kFeatMask = 4, kFeatMaskRow = 8, kFeatAny = 15;
template <int FEAT>
__device__ __forceinline__ bool has_cap(const MaskedArgs& m) {
  return FEAT == kFeatCap || (FEAT == kFeatAny && m.cap_in != 0.0f);
}
template <int FEAT>
__device__ __forceinline__ bool has_distance(const MaskedArgs& m) {
  return FEAT == kFeatDistance || FEAT == kFeatAny;
}
template <int FEAT>
__device__ __forceinline__ bool has_mask(const MaskedArgs& m) {
  return FEAT == kFeatMask || FEAT == kFeatMaskRow || (FEAT == kFeatAny && m.mask_kind != 0);
}
template <int FEAT>
__device__ __forceinline__ bool has_mask_row(const MaskedArgs& m) {
  return FEAT == kFeatMaskRow || (FEAT == kFeatAny && m.mask_row);
}

// A mask value in log2 units: -inf hides; any finite value, however low, stays finite; a NaN stays.
__device__ __forceinline__ float mask_log2(float e) { return e == -INFINITY ? e : max_nan(e * kLog2e, -FLT_MAX); }

// All bits the sign bit of byte `i` (a constant) of x.
__device__ __forceinline__ uint32_t replicate_sign(uint32_t x, uint32_t i) {
  uint32_t r;
  asm("prmt.b32 %0, %1, 0, %2;" : "=r"(r) : "r"(x), "r"(0x8888u + 0x1111u * i));
  return r;
}

// One mask row for the warp: this lane's value, key kv0 + lane, in log2 units, requested before the wait for S.
__device__ __forceinline__ float mask_row_value(const MaskedArgs& m, const Row& w, int kv0, int lane) {
  if (kv0 + lane >= m.a.Skv) return -INFINITY;
  const int at = kv0 + lane;
  if (m.mask_kind == 1) return __ldg(w.mask + at) != 0 ? 0.0f : -INFINITY;
  if (m.mask_kind == 2)
    return mask_log2(__uint_as_float(uint32_t(__ldg(reinterpret_cast<const unsigned short*>(w.mask) + at)) << 16));
  return mask_log2(__ldg(reinterpret_cast<const float*>(w.mask) + at));
}

// Rows of their own: the next tile's part of this thread's row into L1 while this tile is worked on (kHalf values of
// 1, 2 or 4 bytes; the loads themselves, held across a step, cost registers that the kernel does not have).
__device__ __forceinline__ void prefetch_mask(const MaskedArgs& m, const Row& w, int kv0) {
  if (kv0 + kHalf > m.a.Skv) return;
  const int esz = m.mask_kind == 3 ? 4 : m.mask_kind;
  const uint8_t* p = w.mask + (long long)kv0 * esz;
  for (int k = 0; k < esz; ++k) asm volatile("prefetch.global.L1 [%0];" ::"l"(p + 32 * k));
}

// 16 bytes from offset `o` (0 ... 15) of two consecutive 16-byte words.
__device__ __forceinline__ uint4 bytes_at(const uint4& a, const uint4& b, uint32_t o) {
  const bool two = o & 8u, one = o & 4u;
  const uint32_t t[6] = {two ? a.z : a.x, two ? a.w : a.y, two ? b.x : a.z,
                         two ? b.y : a.w, two ? b.z : b.x, two ? b.w : b.y};
  uint32_t u[5];
#pragma unroll
  for (int e = 0; e < 5; ++e) u[e] = one ? t[e + 1] : t[e];
  const uint32_t s = 8 * (o & 3u);
  return make_uint4(__funnelshift_r(u[0], u[1], s), __funnelshift_r(u[1], u[2], s), __funnelshift_r(u[2], u[3], s),
                    __funnelshift_r(u[3], u[4], s));
}

// A mask row's bytes from p on, 32 a call. `whole`: p is aligned and the bytes are all the row's. Otherwise the aligned
// words that hold a byte of [p, end), put together (the first and the last may hold neighbours' bytes, which share their
// 16 bytes and so their page); what lies behind the end is zeros or a neighbour's.
struct MaskBytes {
  const uint4* next;
  const uint8_t* end;
  uint32_t o;
  bool whole;
  uint4 word;
  __device__ __forceinline__ MaskBytes(const uint8_t* p, const uint8_t* row_end, bool all) : end(row_end), whole(all) {
    o = uint32_t(reinterpret_cast<uintptr_t>(p) & 15u);
    next = reinterpret_cast<const uint4*>(p - o);
    if (!whole) word = load();
  }
  __device__ __forceinline__ uint4 load() {
    const uint4 v = reinterpret_cast<const uint8_t*>(next) < end ? __ldg(next) : make_uint4(0u, 0u, 0u, 0u);
    ++next;
    return v;
  }
  __device__ __forceinline__ void take(uint4 (&v)[2]) {
    if (whole) {
      v[0] = __ldg(next);
      v[1] = __ldg(next + 1);
      next += 2;
    } else {
      const uint4 a = load(), b = load();
      v[0] = bytes_at(word, a, o);
      v[1] = bytes_at(a, b, o);
      word = b;
    }
  }
};

// The cap, the biases by distance and the mask tensor on 32 raw scores of keys from kv0 on. Returns the factor that
// takes the result to log2 units: the scale, until something that is not a multiple of a score has been added (the
// addition then carries it: one fused multiply-add a score).
template <int FEAT, int BN>
__device__ __forceinline__ float modify_scores(const MaskedArgs& m, const Row& w, int kv0, float row_mask,
                                               const float* s_table, float* s_mask, int lane, float (&s)[BN]) {
  float k = m.a.scale_log2;
  if (has_cap<FEAT>(m)) {
    float big = 0.0f;
#pragma unroll
    for (int t = 0; t < BN; t += 2) big = fmax3(big, fabsf(s[t]), fabsf(s[t + 1]));
    if (__all_sync(0xffffffffu, !w.valid || big * m.cap_in <= 1.0f)) {
      // The usual case, on the FMA pipe (the MUFU has the softmax's exponentials to do): cap tanh(y) = y P(y^2).
      const uint64_t in2 = f2_pack(m.cap_in, m.cap_in);
#pragma unroll
      for (int t = 0; t < BN; t += 2) {
        const uint64_t y = f2_mul(f2_pack(s[t], s[t + 1]), in2), z = f2_mul(y, y);
        uint64_t p = f2_pack(m.cap_poly[5], m.cap_poly[5]);
#pragma unroll
        for (int e = 4; e >= 0; --e) p = f2_fma(p, z, f2_pack(m.cap_poly[e], m.cap_poly[e]));
        f2_unpack(f2_mul(y, p), s[t], s[t + 1]);
      }
    } else {
      // tanh(y) = 1 - 2 / (1 + e^(2y)); the absolute error of a few 2^-23 stays that small next to the cap.
      const float e = 2.0f * kLog2e * m.cap_in;
#pragma unroll
      for (int t = 0; t < BN; ++t) s[t] = fmaf(-2.0f * m.cap_out, fast_rcp(1.0f + fast_exp2(e * s[t])), m.cap_out);
    }
    k = 1.0f;
  }
  if (has_distance<FEAT>(m) && m.slopes != nullptr) {
    const float rel = float(w.p - kv0);
    if (w.p_min >= kv0 + BN - 1) {  // all keys at or before their rows: linear in t
      const float base = -w.slope * rel;
#pragma unroll
      for (int t = 0; t < BN; ++t) s[t] = fmaf(w.slope, float(t), fmaf(s[t], k, base));
    } else {
#pragma unroll
      for (int t = 0; t < BN; ++t) s[t] = fmaf(s[t], k, -w.slope * fabsf(float(t) - rel));
    }
    k = 1.0f;
  }
  if (has_distance<FEAT>(m) && m.table != nullptr) {
    const int R = m.max_dist;
    const float* tab = m.table + (long long)w.head * (2 * R + 1) + R;
    const int d0 = kv0 - w.p;
    if (kv0 - w.p_max >= R || kv0 + BN - 1 - w.p_min <= -R) {  // past the table's end on either side, for every row
      const float e = __ldg(tab + (kv0 - w.p_max >= R ? R : -R)) * kLog2e;
#pragma unroll
      for (int t = 0; t < BN; ++t) s[t] = fmaf(s[t], k, e);
    } else if (m.table_smem) {
      // Log2 units, the ends repeated: no clamp a score. Rows of a warp lie within 32 positions, so some row in reach
      // keeps all within the margin; rows that are no output rows read a row's place in reach.
      const float* e = s_table + R + kTableMargin + min(max(d0, -R - kTableMargin), R + kTableMargin - BN + 1);
#pragma unroll
      for (int t = 0; t < BN; ++t) s[t] = fmaf(s[t], k, e[t]);
    } else {
#pragma unroll
      for (int t = 0; t < BN; ++t) s[t] = fmaf(s[t], k, __ldg(tab + min(max(d0 + t, -R), R)) * kLog2e);
    }
    k = 1.0f;
  }
  if (!has_mask<FEAT>(m)) return k;
  if (has_mask_row<FEAT>(m)) {  // one mask row for the warp: broadcast from shared memory
    // What it hides is replaced: -inf added to a NaN or an infinite score would not hide it.
    const uint32_t hidden = __ballot_sync(0xffffffffu, row_mask == -INFINITY);
    if (hidden == 0xffffffffu) {
#pragma unroll
      for (int t = 0; t < BN; ++t) s[t] = -INFINITY;
      return 1.0f;
    }
    s_mask[lane] = row_mask;
    const bool low = row_mask < -1e37f && row_mask != -INFINITY;
    const bool lows = __any_sync(0xffffffffu, low);
    __syncwarp();
    if (!lows) {
#pragma unroll
      for (int t = 0; t < BN; t += 4) {
        const float4 e = *reinterpret_cast<const float4*>(s_mask + t);
        s[t] = fmaf(s[t], k, e.x);
        s[t + 1] = fmaf(s[t + 1], k, e.y);
        s[t + 2] = fmaf(s[t + 2], k, e.z);
        s[t + 3] = fmaf(s[t + 3], k, e.w);
      }
      if (hidden != 0u) {
#pragma unroll
        for (int t = 0; t < BN; ++t) s[t] = (hidden >> t) & 1u ? -INFINITY : s[t];
      }
    } else {
#pragma unroll
      for (int t = 0; t < BN; ++t) {
        const float e = s_mask[t];
        s[t] = e == -INFINITY ? e : max_nan(fmaf(s[t], k, e), -FLT_MAX);
      }
    }
    return 1.0f;
  }
  const int esz = m.mask_kind == 3 ? 4 : m.mask_kind;
  // (scores of keys behind the last get any value here: no row sees them)
  MaskBytes bytes(w.mask + (long long)kv0 * esz, w.mask + (long long)m.a.Skv * esz, m.mask_vec && m.a.Skv - kv0 >= BN);
  // -inf hides; any finite value, however low, stays finite in log2 units; a NaN, of the score or the mask, stays.
  auto add = [k](float x, float e) {
    const float r = fmaf(x, k, e * kLog2e);
    return e == -INFINITY ? -INFINITY : r < -FLT_MAX ? -FLT_MAX : r;
  };
  if (m.mask_kind == 1) {
    uint4 v[BN / 16];
    bytes.take(v);
#pragma unroll
    for (int c = 0; c < BN; c += 16) {
      const uint32_t q[4] = {v[c / 16].x, v[c / 16].y, v[c / 16].z, v[c / 16].w};
#pragma unroll
      for (int t = 0; t < 16; ++t) {
        // The byte as all zeros or all ones: any of its bits carried to the sign and that replicated.
        const uint32_t keep = replicate_sign(((q[t / 4] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | q[t / 4], t % 4);
        s[c + t] = __uint_as_float((__float_as_uint(s[c + t]) & keep) | (0xff800000u & ~keep));
      }
    }
  } else if (m.mask_kind == 2) {
#pragma unroll
    for (int c = 0; c < BN; c += 16) {
      uint4 v[2];
      bytes.take(v);
      const uint32_t q[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
      for (int t = 0; t < 16; ++t)
        s[c + t] = add(s[c + t], __uint_as_float(t & 1 ? q[t / 2] & 0xFFFF0000u : q[t / 2] << 16));
    }
  } else {
#pragma unroll
    for (int c = 0; c < BN; c += 8) {
      uint4 v[2];
      bytes.take(v);
      const uint32_t q[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
      for (int t = 0; t < 8; ++t) s[c + t] = add(s[c + t], __uint_as_float(q[t]));
    }
  }
  return m.mask_kind == 1 ? k : 1.0f;
}

// Whether no row of the warp sees the key tile at kv0 (the same in both warps of the rows: neither reads S then, nor
// takes the step's barrier).
__device__ __forceinline__ bool hidden_tile(const Row& w, int kv0) {
  return w.hi_max <= kv0 || w.lo_min >= kv0 + kMaskedBN;
}

// One online-softmax step over the key tile at kv0 for this thread's row and its half of the keys: P as bf16 pairs over
// the first columns of the S buffer, the running max `mx` (log2 units, -inf while the row has seen nothing) moved only
// when the tile's max beats it by more than 8 (see softmax_step of the unmasked kernel), the running sum of this half.
// The two warps of the rows exchange their maxima through s_max[2][128] (a buffer for alternate tiles); the barrier
// also orders one warp's reads of S before the other's P over the same columns. Returns the factor for O; `move`:
// whether the max moved (the same in both warps).
// A NaN score makes its P and from then on the sum and O NaN (the maximum passes it over): the sum carries it to the end,
// through the joins too, where 0 x NaN is NaN whatever weight the part has.
template <int FEAT>
__device__ __forceinline__ float masked_softmax_step(const MaskedArgs& m, const Row& w, uint32_t s_addr, int kv0, int half,
                                                     int row, int lane, float row_mask, const float* s_table,
                                                     float* s_mask, float* s_max, int barrier, float& run_max,
                                                     float& run_sum, bool& move) {
  move = false;
  const uint32_t p_addr = s_addr + uint32_t(half * (kHalf / 2));
  if (hidden_tile(w, kv0)) {
    const uint32_t z[16] = {};
    tmem_st16(p_addr, z);
    return 1.0f;
  }
  const int key0 = kv0 + half * kHalf;
  float s[kHalf];
  {
    uint32_t r[32];
    tmem_ld32(s_addr + uint32_t(half * kHalf), r);
    tmem_wait_ld();
#pragma unroll
    for (int t = 0; t < kHalf; ++t) s[t] = __uint_as_float(r[t]);
  }
  // Partly seen: the keys [a, z) of this half as bits, a bit test a score instead of two comparisons.
  const bool partial = w.lo_max > key0 || w.hi_min < key0 + kHalf;
  uint32_t keep = 0xffffffffu;
  if (partial) {
    const int a = max(w.lo - key0, 0), z = min(w.hi - key0, kHalf);
    keep = a < z ? (0xffffffffu << a) & (0xffffffffu >> (32 - z)) : 0u;
    static_assert(kHalf == 32, "a bit a key");
    if constexpr ((FEAT & kFeatCap) != 0) {
      // The largest score chooses between the cap's two forms: stale memory must have no say in it.
#pragma unroll
      for (int t = 0; t < kHalf; ++t) s[t] = (keep >> t) & 1u ? s[t] : 0.0f;
    }
  }
  float c = m.a.scale_log2;
  if constexpr (FEAT != 0) c = modify_scores<FEAT, kHalf>(m, w, key0, row_mask, s_table, s_mask, lane, s);
  if (partial) {
#pragma unroll
    for (int t = 0; t < kHalf; ++t) s[t] = (keep >> t) & 1u ? s[t] : -INFINITY;
  }
  float mx8[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) mx8[e] = fmax3(s[e], s[8 + e], s[16 + e]);
#pragma unroll
  for (int e = 0; e < 8; ++e) mx8[e] = fmaxf(mx8[e], s[24 + e]);
  float mx = fmax3(fmax3(mx8[0], mx8[1], mx8[2]), fmax3(mx8[3], mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7])) * c;
  s_max[half * kAttnBM + row] = mx;
  named_barrier_sync(barrier, 64);
  mx = fmaxf(mx, s_max[(half ^ 1) * kAttnBM + row]);
  move = mx > run_max + m.a.rescale_thr;
  const float m_new = move ? mx : run_max;
  const float alpha = move ? fast_exp2(run_max - m_new) : 1.0f;  // 0 on the first tile with a key
  const float neg_m = m_new == -INFINITY ? 0.0f : -m_new;        // nothing seen yet: every P is 2^-inf = 0
  const uint64_t c2 = f2_pack(c, c);
  const uint64_t nm2 = f2_pack(neg_m, neg_m);
  uint64_t rs2[4] = {0ull, 0ull, 0ull, 0ull};
  uint32_t pk[16];
#pragma unroll
  for (int e2 = 0; e2 < 16; ++e2) {
    float x0, x1;
    const uint64_t sv = f2_pack(s[2 * e2], s[2 * e2 + 1]);
    f2_unpack(f2_fma(sv, c2, nm2), x0, x1);
    const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
    rs2[e2 & 3] = f2_add(rs2[e2 & 3], f2_pack(p0, p1));
    pk[e2] = pack_bf16x2(p0, p1);
  }
  tmem_st16(p_addr, pk);
  rs2[0] = f2_add(rs2[0], rs2[2]);
  rs2[1] = f2_add(rs2[1], rs2[3]);
  float r0, r1;
  f2_unpack(f2_add(rs2[0], rs2[1]), r0, r1);
  run_sum = run_sum * alpha + (r0 + r1);
  run_max = m_new;
  return alpha;
}

// The O columns of a padded head dim that each of PARTS warps of a row takes: parts in units of 16 columns.
template <int DP, int PARTS>
struct OColumns {
  static constexpr int kWidth = (DP / 16 + PARTS - 1) / PARTS * 16;  // the last parts may be narrower or empty
  static __device__ __forceinline__ int begin(int part) { return min(part * kWidth, DP); }
};

// 32 aligned bytes, a whole sector, to global memory.
__device__ __forceinline__ void st_global_v8(void* to, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// The warp's 32 O rows x inv (zeros where `zero`; o_addr 0: no O, all zeros; o_addr2 not 0: plus the rows there x inv2):
// `cols` columns from o_addr on (a multiple of 8; the padded columns are whole sixteens) as f32 or bf16 to `dst`, each
// lane's own row (null: no row). A lane holds a row and writes it itself, in whole sectors (`sectors`) or in 16-byte words:
// through shared memory and out along the rows, with the index arithmetic that takes, was slower (2x12x77x77x64 causal 4.95
// us, 4.80 in 16-byte words, 4.62 in sectors; 5 tokens against 5001 keys 12.65, 11.8, 11.6). Rolled: it runs once a tile, and
// straight-line code for every head dim and type was paid for in instruction fetches.
__device__ __forceinline__ void store_rows(uint32_t o_addr, uint32_t o_addr2, int cols, bool f32, uint8_t* dst, float inv,
                                           float inv2, bool zero, bool sectors) {
#pragma unroll 1
  for (int c = 0; c < cols; c += 16) {
    uint32_t r[16] = {}, r2[16] = {};
    if (o_addr != 0) tmem_ld16(o_addr + uint32_t(c), r);
    if (o_addr2 != 0) tmem_ld16(o_addr2 + uint32_t(c), r2);
    tmem_wait_ld();
    float o[16];
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      o[t] = __uint_as_float(r[t]) * inv;
      if (o_addr2 != 0) o[t] = fmaf(__uint_as_float(r2[t]), inv2, o[t]);
      if (zero) o[t] = 0.0f;
    }
    if (dst == nullptr) continue;
    if (sectors && c + 16 <= cols) {
      uint32_t w[8];
      if (f32) {
#pragma unroll
        for (int h = 0; h < 16; h += 8) {
#pragma unroll
          for (int t = 0; t < 8; ++t) w[t] = __float_as_uint(o[h + t]);
          st_global_v8(dst + (c + h) * 4, w);
        }
      } else {
#pragma unroll
        for (int t = 0; t < 8; ++t) w[t] = pack_bf16x2(o[2 * t], o[2 * t + 1]);
        st_global_v8(dst + c * 2, w);
      }
      continue;
    }
#pragma unroll
    for (int e = 0; e < 16; e += 8) {
      if (c + e >= cols) break;
      if (f32) {
        float4* to = reinterpret_cast<float4*>(dst + (c + e) * 4);
        to[0] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        to[1] = make_float4(o[e + 4], o[e + 5], o[e + 6], o[e + 7]);
      } else {
        *reinterpret_cast<uint4*>(dst + (c + e) * 2) =
            make_uint4(pack_bf16x2(o[e], o[e + 1]), pack_bf16x2(o[e + 2], o[e + 3]), pack_bf16x2(o[e + 4], o[e + 5]),
                       pack_bf16x2(o[e + 6], o[e + 7]));
      }
    }
  }
}

// Eight columns of an output row, from element offset `at` on.
__device__ __forceinline__ void write_columns(const MaskedArgs& m, long long at, const float (&o)[8]) {
  if (m.a.out_f32) {
    float* dst = static_cast<float*>(m.a.out) + at;
    if (m.out_vec) {
      reinterpret_cast<float4*>(dst)[0] = make_float4(o[0], o[1], o[2], o[3]);
      reinterpret_cast<float4*>(dst)[1] = make_float4(o[4], o[5], o[6], o[7]);
    } else {
#pragma unroll
      for (int t = 0; t < 8; ++t) dst[t] = o[t];
    }
  } else {
    __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(m.a.out) + at;
    if (m.out_vec) {
      *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]),
                                                  pack_bf16x2(o[4], o[5]), pack_bf16x2(o[6], o[7]));
    } else {
#pragma unroll
      for (int t = 0; t < 8; ++t) dst[t] = __float2bfloat16_rn(o[t]);
    }
  }
}

// Joins the parts of the tile's rows, which the CTAs of the cluster hold as staged rows and (max, sum) pairs in shared
// memory: with M = max of the parts' maxima, o = sum_z 2^(m_z - M) O_z / sum_z 2^(m_z - M) l_z, in part order. CTA `rank`
// takes every splits-th row, a thread eight columns.
template <int DP, int STREAMS>
__device__ __noinline__ void join_cluster(const MaskedArgs& m, const uint8_t* smem, const float2* s_ml, int tile, int h0,
                                          int bb, int rank) {
  using OPart = OColumns<DP, 2 * STREAMS>;
  const AttnArgs& args = m.a;
  const int chunks = args.D / 8, splits = m.splits;
  const int items = (m.pack * m.T - rank + splits - 1) / splits * chunks;
  for (int k = int(threadIdx.x); k < items; k += STREAMS * kSoftWarps * 32) {
    const int r = rank + k / chunks * splits, c = k % chunks * 8;
    const int q = (r * m.inv_row) >> 16;
    const int i = tile * m.T + (m.head_fast ? q : r - q * m.T), head = h0 + (m.head_fast ? r - q * m.pack : q);
    if (i >= args.Sq) continue;
    float wz[kMaxCluster], lz[kMaxCluster];
    float top = -INFINITY;
#pragma unroll
    for (int z = 0; z < kMaxCluster; ++z) {
      wz[z] = -INFINITY;
      lz[z] = 0.0f;
      if (z < splits) ld_cluster_f32x2(cluster_smem_addr(s_ml + r, uint32_t(z)), wz[z], lz[z]);
    }
#pragma unroll
    for (int z = 0; z < kMaxCluster; ++z) top = fmaxf(top, wz[z]);
    float sum = 0.0f;
#pragma unroll
    for (int z = 0; z < kMaxCluster; ++z) {
      wz[z] = wz[z] == -INFINITY ? 0.0f : fast_exp2(wz[z] - top);
      sum = fmaf(wz[z], lz[z], sum);
    }
    const int part = c / OPart::kWidth, begin = OPart::begin(part);
    const int cols = min(args.D, OPart::begin(part + 1)) - begin;
    const int warp = (part >> 1) * kSoftWarps + (part & 1) * kSoftmaxWarps + (r >> 5);
    const uint8_t* src = smem + warp * 32 * ((OPart::kWidth * 4 / 16) | 1) * 16 + (r & 31) * ((cols / 4) | 1) * 16 +
                         (c - begin) * 4;
    float o[8] = {};
#pragma unroll
    for (int z = 0; z < kMaxCluster; ++z) {
      if (wz[z] != 0.0f) {  // a part that saw nothing staged no row
        const uint32_t at = cluster_smem_addr(src, uint32_t(z));
        const float4 a = ld_cluster_f32x4(at), b = ld_cluster_f32x4(at + 16);
        const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int t = 0; t < 8; ++t) o[t] = fmaf(wz[z], v[t], o[t]);
      }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // (a NaN sum makes the row NaN, whatever its parts' weights)
#pragma unroll
    for (int t = 0; t < 8; ++t) o[t] *= inv;
    write_columns(m, (long long)bb * args.o_sb + (long long)i * args.o_ss + (long long)head * args.o_sh + c, o);
  }
}

template <int DP, int STAGES, int STREAMS>
struct MaskedLayout {
  static constexpr int BN = kMaskedBN;
  static constexpr int kNA = (DP + 63) / 64;
  static constexpr int kThreads = (STREAMS * kSoftWarps + 2) * 32;
  static constexpr int kBufs = STREAMS + 1;  // S tiles in TMEM
  static constexpr int kQAtom = kAttnBM * kAtomBytesPerRow;
  static constexpr int kKVAtom = BN * kAtomBytesPerRow;
  static constexpr int kQBytes = kNA * kQAtom;
  static constexpr int kKVBytes = kNA * kKVAtom;
  static constexpr int kKOff = kQBytes;
  static constexpr int kVOff = kKOff + STAGES * kKVBytes;
  static constexpr int kBarOff = kVOff + STAGES * kKVBytes;
  // q_full, k_full[S], v_full[S], k_empty[S], v_empty[S], s_full[kBufs], p_full[kBufs], pv_done[2], drain
  static constexpr int kNumBars = 1 + 4 * STAGES + 2 * kBufs + 2 + 1;
  static constexpr int kMiscOff = kBarOff + kNumBars * 8;   // TMEM slot, abort flag, the warps' unions
  static constexpr int kMaskOff = (kMiscOff + 16 + 4 * 8 + 15) / 16 * 16;  // the warp's part of a mask row, per softmax warp
  // row maxima [stream][tile parity][half][row]
  static constexpr int kMaxOff = kMaskOff + STREAMS * kSoftWarps * kHalf * 4;
  // both streams' sums [stream][half][row] and maxima [stream][row]
  static constexpr int kJoinOff = kMaxOff + STREAMS * 2 * 2 * kAttnBM * 4;
  // the rows' (max, sum) for the other CTAs of a cluster
  static constexpr int kMlOff = kJoinOff + (STREAMS > 1 ? 6 * kAttnBM * 4 : 0);
  // the head's distance bias (launch-sized)
  static constexpr int kTableOff = kMlOff + kAttnBM * 8;
  static constexpr int kSmemBytes = kTableOff + 1024;
  // The output rows' staging (f32 rows, an odd number of words apart) reuses Q, K and V.
  static_assert(kBarOff >= STREAMS * kSoftWarps * 32 * (OColumns<DP, 2 * STREAMS>::kWidth * 4 + 16),
                "staging of the output rows");
  static constexpr int kOCol = kBufs * BN;
  static constexpr int kTmemUsed = kOCol + STREAMS * DP;
  static_assert(kTmemUsed <= 512, "TMEM columns");
  static constexpr int kTmemCols = (kTmemUsed <= 256) ? 256 : 512;
  static constexpr bool kTwoPerSm = STREAMS == 1 && kSmemBytes <= 113 * 1024 && kTmemCols <= 256;
  static_assert(DP % 16 == 0 && DP >= 16 && DP <= 256, "padded head dim must be a multiple of 16 in [16, 256]");
  static_assert(kSmemBytes <= 232448, "shared memory budget");
};

template <int DP, int STAGES, int STREAMS, int FEAT>
__global__ void __launch_bounds__(MaskedLayout<DP, STAGES, STREAMS>::kThreads,
                                  MaskedLayout<DP, STAGES, STREAMS>::kTwoPerSm ? 2 : 1)
    attention_masked_tcgen05_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                                    const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ MaskedArgs m) {
  using L = MaskedLayout<DP, STAGES, STREAMS>;
  using OHalf = OColumns<DP, 2>;            // a stream's O, rescaled by the two warps of a row
  using OPart = OColumns<DP, 2 * STREAMS>;  // the output row, stored by all warps of a row
  constexpr int BN = L::BN;
  constexpr int kProducerWarp = STREAMS * kSoftWarps, kMmaWarp = kProducerWarp + 1;
  const AttnArgs& args = m.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = smem + L::kKOff;
  uint8_t* sV = smem + L::kVOff;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* k_full = q_full + 1;
  uint64_t* v_full = k_full + STAGES;
  uint64_t* k_empty = v_full + STAGES;
  uint64_t* v_empty = k_empty + STAGES;
  uint64_t* s_full = v_empty + STAGES;
  uint64_t* p_full = s_full + L::kBufs;
  uint64_t* pv_done = p_full + L::kBufs;
  uint64_t* drain = pv_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMiscOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMiscOff + 4);
  int* s_union = reinterpret_cast<int*>(smem + L::kMiscOff + 16);  // lo[4], hi[4]
  float* s_table = reinterpret_cast<float*>(smem + L::kTableOff);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  // All pairs' tiles of one place before the next place; causal rows see more the later they come, so those start first.
  const int pair = int(blockIdx.x);
  const int tile = m.causal ? m.tiles - 1 - int(blockIdx.y) : int(blockIdx.y);
  const int bb = pair / m.groups;
  const int h0 = (pair - bb * m.groups) * m.pack;
  const int kvh = m.pack > 1 ? pair - bb * m.groups : h0 / m.G;
  const int split = int(blockIdx.z);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      if (s > 0) mbar_init(&k_full[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int i = 0; i < L::kBufs; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], kSoftWarps);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&pv_done[i], 1);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, L::kTmemCols);
    tmem_relinquish();
    tc_fence_before();
    // Only now may the next kernel's blocks come: one that took the TMEM this block still needs would wait for this grid.
    pdl_launch_dependents();
  }
  if (warp == kProducerWarp && lane == 0) {
    mbar_init(q_full, 1);  // by the thread that loads Q, which does not wait for the barriers' owner
    mbar_init(&k_full[0], 1);
    fence_barrier_init();
    fence_proxy_async_smem();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  pdl_wait();  // q, k, v, the lengths, borders and masks may be the previous kernel's outputs; it may read out
  Row w = {};
  // Q needs nothing but the tile, and neither does the first K tile where no rule hides the first keys: both are on their
  // way while the rows are worked out (2x12x77x77x64 causal 5.12 -> 4.97 us, 2x8x4096x77x40 15.0 -> 14.75 us).
  const bool early_k = m.splits == 1 && m.docs == nullptr;
  if (warp == kProducerWarp && lane == 0) {
    int c0, c1, c2, c3;
    mbar_arrive_expect_tx(q_full, uint32_t(L::kNA * m.q_bytes));
    for (int a = 0; a < L::kNA; ++a) {
      map_coords(args.pq, a, tile * m.T, h0, bb, c0, c1, c2, c3);
      tma_load_4d(&tm_q, q_full, sQ + a * L::kQAtom, c0, c1, c2, c3);
    }
    if (early_k) {
      mbar_arrive_expect_tx(&k_full[0], uint32_t(L::kKVBytes));
      for (int a = 0; a < L::kNA; ++a) {
        map_coords(args.pk, a, 0, kvh, bb, c0, c1, c2, c3);
        tma_load_4d(&tm_k, &k_full[0], sK + a * L::kKVAtom, c0, c1, c2, c3);
      }
    }
  }
  if ((FEAT & kFeatDistance) && m.table_smem) {
    const int R = m.max_dist;
    const float* tab = m.table + (long long)h0 * (2 * R + 1) + R;
    for (int k = int(threadIdx.x); k < 2 * (R + kTableMargin) + 1; k += L::kThreads)
      s_table[k] = __ldg(tab + min(max(k - R - kTableMargin, -R), R)) * kLog2e;
  }
  // Softmax threads: row of the tile, half of the keys, stream of key tiles.
  const int row = int(threadIdx.x) & (kAttnBM - 1);
  const int half = (int(threadIdx.x) >> 7) & 1;
  const int stream = int(threadIdx.x) >> 8;
  if (warp < STREAMS * kSoftWarps) {
    w = row_of(m, row, tile, h0, bb);
    if (lane == 0 && warp < kSoftmaxWarps) {
      s_union[warp] = w.lo_min;
      s_union[4 + warp] = w.hi_max;
    }
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // The keys [key_lo, key_hi) that some row of the tile sees, and this part's tiles of them.
  const int key_lo = min(min(s_union[0], s_union[1]), min(s_union[2], s_union[3]));
  const int key_hi = max(max(s_union[4], s_union[5]), max(s_union[6], s_union[7]));
  int first = 0, nkv = 0;
  if (key_hi > key_lo) {
    const int t0 = key_lo / BN, t1 = (key_hi + BN - 1) / BN;
    const int per = (t1 - t0 + m.splits - 1) / m.splits;
    first = t0 + split * per;
    nkv = max(0, min(t1 - first, per));
  }

  if (warp == kProducerWarp) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      if (nkv > 0)
        kv_producer<L::kNA, BN, STAGES>(&tm_k, &tm_v, args, sK, sV, k_full, v_full, k_empty, v_empty, abort_flag, kvh,
                                        bb, nkv, first, early_k);
      else if (early_k)
        mbar_wait_drain(&k_full[0], 0, args.ctl);
      mbar_wait_drain(q_full, 0, args.ctl);
    }
  } else if (nkv > 0 && warp == kMmaWarp) {
    // ------------------------------------------------------------------ MMA issuer (whole warp, one elected lane issues)
    bool ok = true;
    if (args.ctl.debug & 1u) {
      if (!mbar_wait_bounded_warp(drain, 0, abort_flag, args.ctl, kStatusForced)) ok = false;
    }
    if (ok && !mbar_wait_bounded_warp(q_full, 0, abort_flag, args.ctl, kStatusTimeoutMma)) ok = false;
    tc_fence_after();
    const uint64_t q_desc = smem_desc_kmajor_sw128(smem_u32(sQ));
    const uint64_t k_desc = smem_desc_kmajor_sw128(smem_u32(sK));
    const uint64_t v_desc = smem_desc_mnmajor_sw128(smem_u32(sV), L::kKVAtom);
    auto pv_step = [&](int i) -> bool {
      const int st = i % STAGES;
      const int buf = i % L::kBufs;
      if (!mbar_wait_bounded_warp(&v_full[st], uint32_t(i / STAGES) & 1u, abort_flag, args.ctl, kStatusTimeoutMma))
        return false;
      // V rows of this tile that no row sees: zeros, whatever the cache holds there.
      const int kv0 = (first + i) * BN;
      const int live0 = max(key_lo - kv0, 0), live1 = min(key_hi - kv0, BN), end = min(args.Skv - kv0, BN);
      uint64_t gaps = 0;  // between those keys
      if constexpr (FEAT == kFeatAny) {
        if (m.gaps) gaps = unseen_keys(m, bb, tile, kv0, lane);
      }
      if (live0 > 0 || live1 < end || gaps != 0) {
        for (int c = lane; c < BN * L::kNA * 8; c += 32) {
          const int row = (c >> 3) % BN;
          if (row < live0 || row >= live1 || (gaps >> row & 1u) != 0)
            *reinterpret_cast<uint4*>(sV + st * L::kKVBytes + (c >> 3) / BN * L::kKVAtom + row * kAtomBytesPerRow +
                                      (c & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
        __syncwarp();
      }
      if (!mbar_wait_bounded_warp(&p_full[buf], uint32_t(i / L::kBufs) & 1u, abort_flag, args.ctl, kStatusTimeoutMma))
        return false;
      tc_fence_after();
      if (elect_one()) {
        issue_pv<DP, BN>(tmem_base + L::kOCol + uint32_t(i % STREAMS * DP), tmem_base + uint32_t(buf * BN),
                         v_desc + uint64_t((st * L::kKVBytes) >> 4), i >= STREAMS);
        umma_commit(&pv_done[i & 1]);
        umma_commit(&v_empty[st]);
      }
      __syncwarp();
      return true;
    };
    for (int j = 0; ok && j < nkv; ++j) {
      const int st = j % STAGES;
      const int buf = j % L::kBufs;
      if (!mbar_wait_bounded_warp(&k_full[st], uint32_t(j / STAGES) & 1u, abort_flag, args.ctl, kStatusTimeoutMma)) {
        ok = false;
        break;
      }
      tc_fence_after();
      if (elect_one()) {
        issue_s<DP, BN>(tmem_base + uint32_t(buf * BN), q_desc, k_desc + uint64_t((st * L::kKVBytes) >> 4), L::kQAtom,
                        L::kKVAtom);
        umma_commit(&s_full[buf]);
        umma_commit(&k_empty[st]);
      }
      __syncwarp();
      if (j >= STREAMS && !pv_step(j - STREAMS)) {
        ok = false;
        break;
      }
    }
    for (int i = max(nkv - STREAMS, 0); ok && i < nkv; ++i) ok = pv_step(i);
    if (!ok) {
      if (elect_one()) umma_commit(drain);
      __syncwarp();
      mbar_wait_drain(drain, 0u, args.ctl);
    }
  } else if (warp < STREAMS * kSoftWarps) {
    // ------------------------------------------------------------------ softmax / correction / epilogue
    const uint32_t lane_base = tmem_base + (uint32_t((warp & 3) * 32) << 16);
    const uint32_t o_addr = lane_base + uint32_t(L::kOCol);
    const int barrier = 1 + stream * 4 + (warp & 3);  // of the row's two warps in a stream
    float* s_mask = reinterpret_cast<float*>(smem + L::kMaskOff) + warp * kHalf;
    float* s_max = reinterpret_cast<float*>(smem + L::kMaxOff) + stream * 4 * kAttnBM;
    float run_max = -INFINITY, run_sum = 0.0f;
    bool ok = true;
    for (int j = stream; j < nkv; j += STREAMS) {
      const int buf = j % L::kBufs;
      const int kv0 = (first + j) * BN;
      float row_mask = 0.0f;
      if (has_mask<FEAT>(m)) {
        if (has_mask_row<FEAT>(m))
          row_mask = mask_row_value(m, w, kv0 + half * kHalf, lane);
        else
          prefetch_mask(m, w, kv0 + STREAMS * BN + half * kHalf);
      }
      if (ok && !mbar_wait_bounded_warp(&s_full[buf], uint32_t(j / L::kBufs) & 1u, abort_flag, args.ctl,
                                        kStatusTimeoutEpilogue))
        ok = false;
      if (!ok) {  // aborted: the other warp of the rows may still come to this step's barrier
        if (!hidden_tile(w, kv0)) named_barrier_sync(barrier, 64);
        continue;
      }
      tc_fence_after();
      bool move;
      const float alpha =
          masked_softmax_step<FEAT>(m, w, lane_base + uint32_t(buf * BN), kv0, half, row, lane, row_mask, s_table, s_mask,
                                      s_max + (j / STREAMS & 1) * 2 * kAttnBM, barrier, run_max, run_sum, move);
      if (j >= STREAMS && __any_sync(0xffffffffu, move)) {
        if (!mbar_wait_bounded_warp(&pv_done[(j - STREAMS) & 1], uint32_t((j - STREAMS) >> 1) & 1u, abort_flag, args.ctl,
                                    kStatusTimeoutEpilogue)) {
          ok = false;
          continue;
        }
        tc_fence_after();
#pragma unroll 1
        for (int c = OHalf::begin(half); c < OHalf::begin(half + 1); c += 16)
          rescale_o_row<16>(o_addr + uint32_t(stream * DP + c), alpha);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[buf]);
    }
    // The last P V of each stream; without a tile the loads that the rows' staging would race with.
    if (ok && nkv == 0)
      ok = mbar_wait_bounded_warp(q_full, 0, abort_flag, args.ctl, kStatusTimeoutEpilogue) &&
           (!early_k || mbar_wait_bounded_warp(&k_full[0], 0, abort_flag, args.ctl, kStatusTimeoutEpilogue));
    for (int i = max(nkv - STREAMS, 0); ok && i < nkv; ++i)
      ok = mbar_wait_bounded_warp(&pv_done[i & 1], uint32_t(i >> 1) & 1u, abort_flag, args.ctl, kStatusTimeoutEpilogue);
    // The row's sum is both halves', and with two streams the row is joined: with M the larger maximum, 2^(m - M) weighs
    // each stream's O and sum. (Aborted warps take the barrier, too.)
    float weight[2] = {1.0f, 0.0f};
    if constexpr (STREAMS == 1) {
      float* s_sum = s_max + (nkv & 1) * 2 * kAttnBM;
      s_sum[half * kAttnBM + row] = run_sum;
      named_barrier_sync(barrier, 64);
      run_sum += s_sum[(half ^ 1) * kAttnBM + row];
    } else {
      float* s_join = reinterpret_cast<float*>(smem + L::kJoinOff) + row;
      s_join[(2 * stream + half) * kAttnBM] = run_sum;
      s_join[(4 + stream) * kAttnBM] = run_max;  // the same in both halves
      named_barrier_sync(1 + 8 + (warp & 3), 128);
      run_max = fmaxf(s_join[4 * kAttnBM], s_join[5 * kAttnBM]);
      run_sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float top = s_join[(4 + e) * kAttnBM];
        weight[e] = top == -INFINITY ? 0.0f : fast_exp2(top - run_max);
        run_sum = fmaf(s_join[2 * e * kAttnBM] + s_join[(2 * e + 1) * kAttnBM], weight[e], run_sum);
      }
    }
    float2* s_ml = reinterpret_cast<float2*>(smem + L::kMlOff);
    if (m.cluster && warp < kSoftmaxWarps) s_ml[row] = make_float2(ok ? run_max : -INFINITY, run_sum);
    if (ok && __any_sync(0xffffffffu, w.valid)) {
      tc_fence_after();
      // The row has seen no key. (A score that is NaN leaves the maximum alone, but not the sum: such a row is NaN.)
      const bool empty = run_max == -INFINITY && run_sum == 0.0f;
      const bool wide = m.splits > 1 || args.out_f32;  // f32 rows
      const int esz = wide ? 4 : 2;
      const int part = 2 * stream + half;
      const int begin = OPart::begin(part);
      const int cols = min(args.D, OPart::begin(part + 1)) - begin;  // this warp's, maybe none
      const long long obase =
          (long long)bb * args.o_sb + (long long)w.i * args.o_ss + (long long)w.head * args.o_sh + begin;
      uint8_t* stage = smem + warp * 32 * ((OPart::kWidth * 4 / 16) | 1) * 16;
      uint8_t* dst = nullptr;
      if (m.splits > 1 && !m.cluster) {
        const long long at = (((long long)split * m.pairs + pair) * m.tiles + tile) * kAttnBM + row;
        if (w.valid && part == 0) m.part_ml[at] = make_float2(run_max, empty ? 0.0f : run_sum);
        if (w.valid && !empty) dst = reinterpret_cast<uint8_t*>(m.part_o + at * args.D + begin);
      } else if (w.valid && !m.cluster) {
        dst = static_cast<uint8_t*>(args.out) + obase * esz;
      }
      const float inv = m.splits > 1 ? 1.0f : 1.0f / run_sum;
      const uint32_t o_at = nkv > 0 ? o_addr + uint32_t(begin) : 0u;
      const uint32_t o_at2 = STREAMS > 1 && nkv > 1 ? o_addr + uint32_t(DP + begin) : 0u;
      if (cols <= 0) {
        // nothing of the true head dim in this half
      } else if (m.splits > 1 ? nkv > 0 : m.out_vec != 0) {
        // (in a cluster to the staged rows in shared memory, from where the other CTAs read them)
        store_rows(o_at, o_at2, cols, wide, m.cluster ? stage + lane * ((cols / 4) | 1) * 16 : dst, inv * weight[0],
                   inv * weight[1], empty, !m.cluster && m.out_sectors);
      } else if (m.splits == 1) {
        // Output rows that 16-byte words do not reach.
        for (int c = 0; c < cols; c += 8) {
          float o[8] = {};
#pragma unroll
          for (int e = 0; e < STREAMS; ++e) {
            if ((e == 0 ? o_at : o_at2) == 0) break;
            uint32_t r[8];
            tmem_ld8((e == 0 ? o_at : o_at2) + uint32_t(c), r);
            tmem_wait_ld();
#pragma unroll
            for (int t = 0; t < 8; ++t) o[t] = empty ? 0.0f : fmaf(__uint_as_float(r[t]), inv * weight[e], o[t]);
          }
          if (w.valid) {
#pragma unroll
            for (int t = 0; t < 8; ++t) {
              if (wide)
                reinterpret_cast<float*>(dst)[c + t] = o[t];
              else
                reinterpret_cast<__nv_bfloat16*>(dst)[c + t] = __float2bfloat16_rn(o[t]);
            }
          }
        }
      }
    }
    tc_fence_before();
  }

  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem_base, L::kTmemCols);
  }
  if (m.cluster) {  // (after TMEM is free: a CTA that waits for it elsewhere may belong to this cluster)
    cluster_sync();
    if (warp < STREAMS * kSoftWarps)
      join_cluster<DP, STREAMS>(m, smem, reinterpret_cast<const float2*>(smem + L::kMlOff), tile, h0, bb, split);
    cluster_sync();  // no CTA leaves while another reads its rows
  }
}

template <int DP, int STAGES, int STREAMS, int FEAT>
int launch_masked(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const MaskedArgs& m, dim3 grid,
                  cudaStream_t st, int device) {
  static bool configured[64] = {false};
  auto kern = attention_masked_tcgen05_kernel<DP, STAGES, STREAMS, FEAT>;
  using L = MaskedLayout<DP, STAGES, STREAMS>;
  static_assert(L::kSmemBytes + kTableSmemMax <= (L::kTwoPerSm ? 113 * 1024 : 232448), "room for the distance bias");
  const int smem = L::kSmemBytes + (m.table_smem ? (2 * (m.max_dist + kTableMargin) + 1) * 4 : 0);
  if (!configured[device]) {
    if (int rc = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 L::kSmemBytes + kTableSmemMax),
                            "cudaFuncSetAttribute(masked attention smem)"))
      return rc;
    if (int rc = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1),
                            "cudaFuncSetAttribute(masked attention cluster)"))
      return rc;
    configured[device] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(L::kThreads);
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = grid.z;
  cfg.attrs = attr;
  cfg.numAttrs = m.cluster ? 2 : 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, mq, mk, mv, m), "masked attention kernel launch");
}

template <int FEAT>
int launch_masked_for(int64_t D, int streams, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                      const MaskedArgs& m, dim3 grid, cudaStream_t st, int dev) {
  if (streams == 2) {
    if (D <= 64) return launch_masked<64, 5, 2, FEAT>(mq, mk, mv, m, grid, st, dev);
    if (D <= 96) return launch_masked<96, 4, 2, FEAT>(mq, mk, mv, m, grid, st, dev);
    if (D <= 128) return launch_masked<128, 4, 2, FEAT>(mq, mk, mv, m, grid, st, dev);
    return launch_masked<160, 3, 2, FEAT>(mq, mk, mv, m, grid, st, dev);
  }
  // The padded head dims with a kernel; the columns between D and its pad are TMA zeros.
  if (D <= 32) return launch_masked<32, 5, 1, FEAT>(mq, mk, mv, m, grid, st, dev);
  if (D <= 48) return launch_masked<48, 5, 1, FEAT>(mq, mk, mv, m, grid, st, dev);
  if (D <= 64) return launch_masked<64, 5, 1, FEAT>(mq, mk, mv, m, grid, st, dev);
  if (D <= 80) return launch_masked<80, 2, 1, FEAT>(mq, mk, mv, m, grid, st, dev);
  if (D <= 96) return launch_masked<96, 2, 1, FEAT>(mq, mk, mv, m, grid, st, dev);
  if (D <= 128) return launch_masked<128, 2, 1, FEAT>(mq, mk, mv, m, grid, st, dev);
  if (D <= 160) return launch_masked<160, 2, 1, FEAT>(mq, mk, mv, m, grid, st, dev);
  if (D <= 192) return launch_masked<192, 2, 1, FEAT>(mq, mk, mv, m, grid, st, dev);
  return launch_masked<256, 2, 1, FEAT>(mq, mk, mv, m, grid, st, dev);
}

// The instantiations (attention_masked.cu and attention_masked_*.cu, one set of features each).
extern template int launch_masked_for<0>(int64_t, int, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&,
                                         const MaskedArgs&, dim3, cudaStream_t, int);
extern template int launch_masked_for<kFeatCap>(int64_t, int, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&,
                                                const MaskedArgs&, dim3, cudaStream_t, int);
extern template int launch_masked_for<kFeatDistance>(int64_t, int, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&,
                                                     const MaskedArgs&, dim3, cudaStream_t, int);
extern template int launch_masked_for<kFeatMask>(int64_t, int, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&,
                                                 const MaskedArgs&, dim3, cudaStream_t, int);
extern template int launch_masked_for<kFeatMaskRow>(int64_t, int, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&,
                                                    const MaskedArgs&, dim3, cudaStream_t, int);
extern template int launch_masked_for<kFeatAny>(int64_t, int, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&,
                                                const MaskedArgs&, dim3, cudaStream_t, int);

}  // namespace npub200
