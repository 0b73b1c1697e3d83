// attention_masked.cu - attention with masks, score modifiers and grouped key/value heads on B200:
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
// One kernel, one 128-row Q tile per CTA, 64-key tiles, up to two CTAs per SM (the structure and the roles of
// attention_fwd_tcgen05_kernel: softmax warps 0-3, TMA producer warp 4, MMA warp 5):
//   * Q rows: `pack` query heads x T positions. With few queries the heads of a group that share a K/V head fill the
//     tile together (one TMA box of pack heads x T positions), so the cache is read once per group, not once per head.
//   * Keys beyond the union inside its last (or before it inside its first) tile may be stale cache memory: their V
//     rows are zeroed in shared memory before the P V product, since P = 0 times a NaN would be a NaN. Their scores are
//     replaced, not added to.
//   * Split keys (grid z): when the row tiles leave most SMs idle, each CTA takes an equal part of its tile's keys and
//     writes its unnormalised O row, max and sum to the workspace; attention_join_kernel joins the parts in part order.
// Rounding: P is rounded to bf16 for the tensor core (relative 2^-9, as in the unmasked kernel); the sums, the maxima,
// the modifiers and O are f32.
#include <algorithm>
#include <cfloat>
#include <cstring>

#include "attention_sm100.cuh"

namespace npub200 {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaskedBN = 64;        // keys per tile
constexpr int kMaskedThreads = 192;
constexpr int kMaxSplits = 64;

struct MaskedArgs {
  AttnArgs a;
  int G;              // query heads per key/value head
  int pack, T;        // a Q tile holds `pack` heads x T positions
  int head_fast;      // tile row r = position * pack + head (1) or head * T + position (0)
  int q_bytes;        // bytes of one 64-column atom of the Q box
  int tiles;          // Q tiles along the positions
  int splits;
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
  float cap_in, cap_out;  // tanh argument = cap_in / (2 log2 e) x raw score; capped score in log2 units = cap_out x tanh
  const float* slopes;
  const float* table;
  int max_dist;
  const void* mask;
  int mask_kind;  // 0 none, 1 bool, 2 bf16, 3 f32
  int mask_vec;   // rows can be read in 16-byte words
  long long m_sb, m_sh, m_sq;
};

// What a softmax thread knows of its row.
struct Row {
  int lo, hi;       // keys it may see
  int p;            // its position among the keys
  bool valid;       // a row of the output
  int head, i, b;
  float slope;      // slopes[head] * log2 e
};

__device__ __forceinline__ int clamp_pos(long long x) {
  return int(min(max(x, -(1ll << 30)), 1ll << 30));
}

__device__ __forceinline__ Row row_of(const MaskedArgs& m, int r, int tile, int h0, int b) {
  Row w;
  const int s = m.head_fast ? r / m.pack : r % m.T;
  const int g = m.head_fast ? r - s * m.pack : r / m.T;
  w.i = tile * m.T + s;
  w.head = h0 + g;
  w.b = b;
  w.valid = r < m.pack * m.T && w.i < m.a.Sq;
  w.lo = 0;
  w.hi = 0;
  w.p = 0;
  w.slope = 0.0f;
  if (!w.valid) {
    w.head = h0;
    return w;
  }
  w.p = clamp_pos((m.q_starts != nullptr ? (long long)m.q_starts[b] : m.q_start) + w.i);
  int hi = m.a.Skv;
  if (m.kv_lens != nullptr) hi = min(hi, m.kv_lens[b]);
  if (m.causal) {
    const long long prefix = m.prefixes != nullptr ? (long long)m.prefixes[b] : m.prefix;
    hi = min(hi, max(w.p + 1, clamp_pos(prefix)));
  }
  int lo = 0;
  if (m.docs != nullptr) {
    // Last border at or below i: documents of no tokens are passed over.
    const int* off = m.docs + b * m.doc_stride;
    int left = 0, right = m.ndocs + 1;  // off[left - 1] <= i < off[right]
    while (left < right) {
      const int mid = (left + right) >> 1;
      if (off[mid] <= w.i)
        left = mid + 1;
      else
        right = mid;
    }
    if (left >= 1 && left <= m.ndocs) {
      lo = max(off[left - 1], 0);
      hi = min(hi, off[left]);
    } else {
      hi = 0;
    }
  }
  w.lo = lo;
  w.hi = max(hi, lo);
  if (w.hi == w.lo) w.lo = w.hi = 0;  // sees nothing: leaves the union alone
  if (m.slopes != nullptr) w.slope = m.slopes[w.head] * kLog2e;
  return w;
}

// Raw scores -> log2 units with the cap, the biases and the mask tensor applied.
template <int BN>
__device__ __forceinline__ void modify_scores(const MaskedArgs& m, const Row& w, int kv0, float (&s)[BN]) {
  if (m.cap_in != 0.0f) {
    // tanh(y) = 1 - 2 / (1 + e^(2y)); the absolute error of a few 2^-23 stays that small next to the cap.
#pragma unroll
    for (int t = 0; t < BN; ++t)
      s[t] = m.cap_out * (1.0f - __fdividef(2.0f, 1.0f + fast_exp2(m.cap_in * s[t])));
  } else {
#pragma unroll
    for (int t = 0; t < BN; ++t) s[t] *= m.a.scale_log2;
  }
  if (m.slopes != nullptr) {
    const float rel = float(w.p - kv0);
#pragma unroll
    for (int t = 0; t < BN; ++t) s[t] = fmaf(-w.slope, fabsf(float(t) - rel), s[t]);
  }
  if (m.table != nullptr) {
    const int R = m.max_dist;
    const float* tab = m.table + (long long)w.head * (2 * R + 1) + R;
    const int d0 = kv0 - w.p;
    if (__all_sync(0xffffffffu, d0 >= R || d0 + BN - 1 <= -R)) {  // the whole tile past the table's end on one side
      const float e = __ldg(tab + (d0 >= R ? R : -R)) * kLog2e;
#pragma unroll
      for (int t = 0; t < BN; ++t) s[t] += e;
    } else {
#pragma unroll
      for (int t = 0; t < BN; ++t) s[t] = fmaf(__ldg(tab + min(max(d0 + t, -R), R)), kLog2e, s[t]);
    }
  }
  if (m.mask_kind == 0) return;
  const long long off = (long long)w.b * m.m_sb + (long long)w.head * m.m_sh + (long long)(w.valid ? w.i : 0) * m.m_sq + kv0;
  const int n = m.a.Skv - kv0;  // readable keys from here
  // -inf hides; any finite value, however low, stays finite in log2 units.
  auto add = [](float x, float e) { return e == -INFINITY ? -INFINITY : fmaxf(fmaf(e, kLog2e, x), -FLT_MAX); };
  if (m.mask_kind == 1) {
    const uint8_t* p = static_cast<const uint8_t*>(m.mask) + off;
    if (m.mask_vec && n >= BN) {
#pragma unroll
      for (int c = 0; c < BN; c += 16) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p + c));
        const uint32_t q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int t = 0; t < 16; ++t)
          if (((q[t / 4] >> (8 * (t % 4))) & 0xffu) == 0) s[c + t] = -INFINITY;
      }
    } else {
#pragma unroll
      for (int t = 0; t < BN; ++t)
        if (t >= n || __ldg(p + t) == 0) s[t] = -INFINITY;
    }
  } else if (m.mask_kind == 2) {
    const unsigned short* p = static_cast<const unsigned short*>(m.mask) + off;
    if (m.mask_vec && n >= BN) {
#pragma unroll
      for (int c = 0; c < BN; c += 8) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p + c));
        const uint32_t q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int t = 0; t < 8; ++t)
          s[c + t] = add(s[c + t], __uint_as_float(t & 1 ? q[t / 2] & 0xFFFF0000u : q[t / 2] << 16));
      }
    } else {
#pragma unroll
      for (int t = 0; t < BN; ++t)
        s[t] = t < n ? add(s[t], __uint_as_float(uint32_t(__ldg(p + t)) << 16)) : -INFINITY;
    }
  } else {
    const float* p = static_cast<const float*>(m.mask) + off;
    if (m.mask_vec && n >= BN) {
#pragma unroll
      for (int c = 0; c < BN; c += 4) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(p + c));
        s[c] = add(s[c], v.x);
        s[c + 1] = add(s[c + 1], v.y);
        s[c + 2] = add(s[c + 2], v.z);
        s[c + 3] = add(s[c + 3], v.w);
      }
    } else {
#pragma unroll
      for (int t = 0; t < BN; ++t) s[t] = t < n ? add(s[t], __ldg(p + t)) : -INFINITY;
    }
  }
}

// One online-softmax step over the key tile at kv0 for this thread's row (see softmax_step of the unmasked kernel): P
// over the first BN/2 columns of its S, the running max `mx` (log2 units, -inf while the row has seen nothing) moved
// only when the tile's max beats it by more than 8, the running sum. Returns the factor for O; `move`: whether the max
// moved.
template <int BN, bool SCORES>
__device__ __forceinline__ float masked_softmax_step(const MaskedArgs& m, const Row& w, uint32_t s_addr, int kv0,
                                                     float& run_max, float& run_sum, bool& move) {
  move = false;
  if (__all_sync(0xffffffffu, w.hi <= kv0 || w.lo >= kv0 + BN)) {
    const uint32_t z[16] = {};
#pragma unroll
    for (int c = 0; c < BN / 32; ++c) tmem_st16(s_addr + uint32_t(c * 16), z);
    return 1.0f;
  }
  float s[BN];
#pragma unroll
  for (int c = 0; c < BN; c += 32) {
    uint32_t r[32];
    tmem_ld32(s_addr + uint32_t(c), r);
#pragma unroll
    for (int t = 0; t < 32; ++t) s[c + t] = __uint_as_float(r[t]);
  }
  tmem_wait_ld();
  if constexpr (SCORES) modify_scores<BN>(m, w, kv0, s);
  if (__any_sync(0xffffffffu, w.lo > kv0 || w.hi < kv0 + BN)) {
    const int a = w.lo - kv0, z = w.hi - kv0;
#pragma unroll
    for (int t = 0; t < BN; ++t)
      if (t < a || t >= z) s[t] = -INFINITY;
  }
  float mx8[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) mx8[e] = s[e];
#pragma unroll
  for (int t = 8; t + 16 <= BN; t += 16)
#pragma unroll
    for (int e = 0; e < 8; ++e) mx8[e] = fmax3(mx8[e], s[t + e], s[t + 8 + e]);
  if constexpr ((BN - 8) % 16 != 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) mx8[e] = fmaxf(mx8[e], s[BN - 8 + e]);
  }
  const float c = SCORES ? 1.0f : m.a.scale_log2;
  const float mx =
      fmax3(fmax3(mx8[0], mx8[1], mx8[2]), fmax3(mx8[3], mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7])) * c;
  move = mx > run_max + m.a.rescale_thr;
  const float m_new = move ? mx : run_max;
  const float alpha = move ? fast_exp2(run_max - m_new) : 1.0f;   // 0 on the first tile with a key
  const float neg_m = m_new == -INFINITY ? 0.0f : -m_new;         // nothing seen yet: every P is 2^-inf = 0
  const uint64_t c2 = f2_pack(c, c);
  const uint64_t nm2 = f2_pack(neg_m, neg_m);
  uint64_t rs2[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
  for (int c32 = 0; c32 < BN / 32; ++c32) {
    uint32_t pk[16];
#pragma unroll
    for (int e2 = 0; e2 < 16; ++e2) {
      float x0, x1;
      const uint64_t sv = f2_pack(s[c32 * 32 + 2 * e2], s[c32 * 32 + 2 * e2 + 1]);
      f2_unpack(SCORES ? f2_add(sv, nm2) : f2_fma(sv, c2, nm2), x0, x1);
      const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
      rs2[e2 & 3] = f2_add(rs2[e2 & 3], f2_pack(p0, p1));
      pk[e2] = pack_bf16x2(p0, p1);
    }
    tmem_st16(s_addr + uint32_t(c32 * 16), pk);
  }
  rs2[0] = f2_add(rs2[0], rs2[2]);
  rs2[1] = f2_add(rs2[1], rs2[3]);
  float r0, r1;
  f2_unpack(f2_add(rs2[0], rs2[1]), r0, r1);
  run_sum = run_sum * alpha + (r0 + r1);
  run_max = m_new;
  return alpha;
}

// Unnormalised O row (f32, D columns) of a split part to the workspace.
template <int DP>
__device__ __forceinline__ void store_part_row(uint32_t o_addr, float* dst, int D, bool store) {
#pragma unroll
  for (int cc = 0; cc < DP; cc += 16) {
    uint32_t r[16];
    tmem_ld16(o_addr + uint32_t(cc), r);
    tmem_wait_ld();
    if (store) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (cc + 4 * t < D)  // D is a multiple of 8
          reinterpret_cast<float4*>(dst + cc)[t] =
              make_float4(__uint_as_float(r[4 * t]), __uint_as_float(r[4 * t + 1]), __uint_as_float(r[4 * t + 2]),
                          __uint_as_float(r[4 * t + 3]));
    }
  }
}

template <int DP, int STAGES>
struct MaskedLayout {
  static constexpr int BN = kMaskedBN;
  static constexpr int kNA = (DP + 63) / 64;
  static constexpr int kQAtom = kAttnBM * kAtomBytesPerRow;
  static constexpr int kKVAtom = BN * kAtomBytesPerRow;
  static constexpr int kQBytes = kNA * kQAtom;
  static constexpr int kKVBytes = kNA * kKVAtom;
  static constexpr int kKOff = kQBytes;
  static constexpr int kVOff = kKOff + STAGES * kKVBytes;
  static constexpr int kBarOff = kVOff + STAGES * kKVBytes;
  // q_full, k_full[S], v_full[S], k_empty[S], v_empty[S], s_full[2], p_full[2], pv_done[2], drain
  static constexpr int kNumBars = 1 + 4 * STAGES + 6 + 1;
  static constexpr int kMiscOff = kBarOff + kNumBars * 8;   // TMEM slot, abort flag, the warps' unions
  static constexpr int kSmemBytes = kMiscOff + 16 + 4 * 8 + 1024;
  static constexpr int kOCol = 2 * BN;
  static constexpr int kTmemUsed = kOCol + DP;
  static constexpr int kTmemCols = (kTmemUsed <= 256) ? 256 : 512;
  static constexpr bool kTwoPerSm = kSmemBytes <= 113 * 1024 && kTmemCols <= 256;
  static_assert(DP % 16 == 0 && DP >= 16 && DP <= 256, "padded head dim must be a multiple of 16 in [16, 256]");
  static_assert(kSmemBytes <= 232448, "shared memory budget");
};

template <int DP, int STAGES, bool SCORES>
__global__ void __launch_bounds__(kMaskedThreads, MaskedLayout<DP, STAGES>::kTwoPerSm ? 2 : 1)
    attention_masked_tcgen05_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                                    const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ MaskedArgs m) {
  using L = MaskedLayout<DP, STAGES>;
  constexpr int BN = L::BN;
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
  uint64_t* p_full = s_full + 2;
  uint64_t* pv_done = p_full + 2;
  uint64_t* drain = pv_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMiscOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMiscOff + 4);
  int* s_union = reinterpret_cast<int*>(smem + L::kMiscOff + 16);  // lo[4], hi[4]

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  // Causal rows see more the later they come: the longest tiles start first.
  const int tile = m.causal ? int(gridDim.x) - 1 - int(blockIdx.x) : int(blockIdx.x);
  const int groups = args.H / m.pack;
  const int bb = int(blockIdx.y) / groups;
  const int h0 = (int(blockIdx.y) - bb * groups) * m.pack;
  const int kvh = h0 / m.G;
  const int split = int(blockIdx.z);

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], kSoftmaxWarps);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 5) {
    tmem_alloc(tmem_slot, L::kTmemCols);
    tmem_relinquish();
    tc_fence_before();
  }
  if (warp == 4 && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  pdl_launch_dependents();
  pdl_wait();  // q, k, v, the lengths, borders and masks may be the previous kernel's outputs; it may read out
  Row w = {};
  if (warp < kSoftmaxWarps) {
    w = row_of(m, int(threadIdx.x), tile, h0, bb);
    const int lo = __reduce_min_sync(0xffffffffu, w.hi > w.lo ? w.lo : INT_MAX);
    const int hi = __reduce_max_sync(0xffffffffu, w.hi);
    if (lane == 0) {
      s_union[warp] = lo;
      s_union[4 + warp] = hi;
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

  if (nkv > 0 && warp == 4) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      int c0, c1, c2, c3;
      mbar_arrive_expect_tx(q_full, uint32_t(L::kNA * m.q_bytes));
      for (int a = 0; a < L::kNA; ++a) {
        map_coords(args.pq, a, tile * m.T, h0, bb, c0, c1, c2, c3);
        tma_load_4d(&tm_q, q_full, sQ + a * L::kQAtom, c0, c1, c2, c3);
      }
      kv_producer<L::kNA, BN, STAGES>(&tm_k, &tm_v, args, sK, sV, k_full, v_full, k_empty, v_empty, abort_flag, kvh, bb,
                                      nkv, first);
      mbar_wait_drain(q_full, 0, args.ctl);
    }
  } else if (nkv > 0 && warp == 5) {
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
      const int buf = i & 1;
      if (!mbar_wait_bounded_warp(&v_full[st], uint32_t(i / STAGES) & 1u, abort_flag, args.ctl, kStatusTimeoutMma))
        return false;
      // V rows of this tile that no row sees: zeros, whatever the cache holds there.
      const int kv0 = (first + i) * BN;
      const int live0 = max(key_lo - kv0, 0), live1 = min(key_hi - kv0, BN), end = min(args.Skv - kv0, BN);
      if (live0 > 0 || live1 < end) {
        for (int c = lane; c < BN * L::kNA * 8; c += 32) {
          const int row = (c >> 3) % BN;
          if (row < live0 || row >= live1)
            *reinterpret_cast<uint4*>(sV + st * L::kKVBytes + (c >> 3) / BN * L::kKVAtom + row * kAtomBytesPerRow +
                                      (c & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
        __syncwarp();
      }
      if (!mbar_wait_bounded_warp(&p_full[buf], uint32_t(i >> 1) & 1u, abort_flag, args.ctl, kStatusTimeoutMma))
        return false;
      tc_fence_after();
      if (elect_one()) {
        issue_pv<DP, BN>(tmem_base + L::kOCol, tmem_base + uint32_t(buf * BN),
                         v_desc + uint64_t((st * L::kKVBytes) >> 4), i > 0);
        umma_commit(&pv_done[buf]);
        umma_commit(&v_empty[st]);
      }
      __syncwarp();
      return true;
    };
    for (int j = 0; ok && j < nkv; ++j) {
      const int st = j % STAGES;
      const int buf = j & 1;
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
      if (j >= 1 && !pv_step(j - 1)) {
        ok = false;
        break;
      }
    }
    if (ok && !pv_step(nkv - 1)) ok = false;
    if (!ok) {
      if (elect_one()) umma_commit(drain);
      __syncwarp();
      mbar_wait_drain(drain, 0u, args.ctl);
    }
  } else if (warp < kSoftmaxWarps) {
    // ------------------------------------------------------------------ softmax / correction / epilogue
    const uint32_t lane_base = tmem_base + (uint32_t(warp * 32) << 16);
    float run_max = -INFINITY, run_sum = 0.0f;
    bool ok = true;
    for (int j = 0; j < nkv; ++j) {
      const int buf = j & 1;
      if (!mbar_wait_bounded_warp(&s_full[buf], uint32_t(j >> 1) & 1u, abort_flag, args.ctl, kStatusTimeoutEpilogue)) {
        ok = false;
        break;
      }
      tc_fence_after();
      bool move;
      const float alpha = masked_softmax_step<BN, SCORES>(m, w, lane_base + uint32_t(buf * BN), (first + j) * BN, run_max,
                                                          run_sum, move);
      if (j > 0 && __any_sync(0xffffffffu, move)) {
        if (!mbar_wait_bounded_warp(&pv_done[(j - 1) & 1], uint32_t((j - 1) >> 1) & 1u, abort_flag, args.ctl,
                               kStatusTimeoutEpilogue)) {
          ok = false;
          break;
        }
        tc_fence_after();
        rescale_o_row<DP>(lane_base + uint32_t(L::kOCol), alpha);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[buf]);
    }
    if (ok && nkv > 0)
      ok = mbar_wait_bounded_warp(&pv_done[(nkv - 1) & 1], uint32_t((nkv - 1) >> 1) & 1u, abort_flag, args.ctl,
                                  kStatusTimeoutEpilogue);
    const bool any_row = __any_sync(0xffffffffu, w.valid);
    if (ok && any_row) {
      tc_fence_after();
      const bool empty = run_max == -INFINITY;  // the row has seen no key
      const uint32_t o_addr = lane_base + uint32_t(L::kOCol);
      if (m.splits > 1) {
        const long long at = (((long long)split * gridDim.y + blockIdx.y) * m.tiles + tile) * kAttnBM + threadIdx.x;
        if (w.valid) m.part_ml[at] = make_float2(run_max, empty ? 0.0f : run_sum);
        if (nkv > 0) store_part_row<DP>(o_addr, m.part_o + at * args.D, args.D, w.valid && !empty);
      } else {
        const long long obase = (long long)bb * args.o_sb + (long long)w.i * args.o_ss + (long long)w.head * args.o_sh;
        if (nkv > 0) store_o_at<DP>(o_addr, args, w.valid && !empty, obase, 1.0f / run_sum);
        if (w.valid && empty) {
          for (int c = 0; c < args.D; ++c) {
            if (args.out_f32)
              static_cast<float*>(args.out)[obase + c] = 0.0f;
            else
              static_cast<__nv_bfloat16*>(args.out)[obase + c] = __float2bfloat16_rn(0.0f);
          }
        }
      }
    }
    tc_fence_before();
  }

  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem_base, L::kTmemCols);
  }
}

// Joins the split parts of a row: with M = max of the parts' maxima, o = sum_z 2^(m_z - M) O_z / sum_z 2^(m_z - M) l_z in
// part order. One warp per row; a few KB per row from L2.
__global__ void __launch_bounds__(128) attention_join_kernel(const __grid_constant__ MaskedArgs m, int rows, int pairs) {
  pdl_launch_dependents();
  pdl_wait();
  const AttnArgs& args = m.a;
  const int lane = threadIdx.x & 31;
  const int row = int(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= rows) return;
  // rows run (b, i, h), h fastest
  const int h = row % args.H;
  const int i = row / args.H % args.Sq;
  const int b = row / args.H / args.Sq;
  const int groups = args.H / m.pack;
  const int g = h % m.pack;
  const int tile = i / m.T, s = i - tile * m.T;
  const int r = m.head_fast ? s * m.pack + g : g * m.T + s;
  const long long at = (((long long)(b * groups + h / m.pack)) * m.tiles + tile) * kAttnBM + r;
  const long long step = (long long)pairs * m.tiles * kAttnBM;  // rows between parts
  float mz[2], lz[2];
  float top = -INFINITY;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int z = lane + 32 * k;
    const float2 ml = z < m.splits ? m.part_ml[at + z * step] : make_float2(-INFINITY, 0.0f);
    mz[k] = ml.x;
    lz[k] = ml.y;
    top = fmaxf(top, ml.x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float wz[2], sum = 0.0f;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    wz[k] = mz[k] == -INFINITY ? 0.0f : fast_exp2(mz[k] - top);
    sum += wz[k] * lz[k];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
  const long long obase = (long long)b * args.o_sb + (long long)i * args.o_ss + (long long)h * args.o_sh;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int c = half * 128 + lane * 4;
    if (half * 128 >= args.D) break;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int z = 0; z < m.splits; ++z) {
      const float wt = __shfl_sync(0xffffffffu, z < 32 ? wz[0] : wz[1], z & 31);
      if (wt != 0.0f && c < args.D) {  // parts that saw nothing wrote no O
        const float4 v = *reinterpret_cast<const float4*>(m.part_o + (at + z * step) * args.D + c);
        acc.x = fmaf(wt, v.x, acc.x);
        acc.y = fmaf(wt, v.y, acc.y);
        acc.z = fmaf(wt, v.z, acc.z);
        acc.w = fmaf(wt, v.w, acc.w);
      }
    }
    if (c < args.D) {
      const float v[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if (args.out_f32)
          static_cast<float*>(args.out)[obase + c + t] = v[t];
        else
          static_cast<__nv_bfloat16*>(args.out)[obase + c + t] = __float2bfloat16_rn(v[t]);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------------------------
struct MaskedPlan {
  int pack, T, splits;
  int64_t tiles, pairs;
  size_t ml_bytes, bytes;  // workspace: (max, sum) pairs first, then the O rows
};

int check_masked_sizes(int64_t B, int64_t H, int64_t Hk, int64_t Sq, int64_t Skv, int64_t D, int variant) {
  if (B <= 0 || H <= 0 || Hk <= 0 || Sq <= 0 || Skv <= 0 || D <= 0)
    return fail(kErrInvalid, "attention sizes must be positive (B=%lld H=%lld Hkv=%lld Sq=%lld Skv=%lld D=%lld)",
                (long long)B, (long long)H, (long long)Hk, (long long)Sq, (long long)Skv, (long long)D);
  if (H % Hk != 0)
    return fail(kErrInvalid, "%lld query heads are not a multiple of %lld key/value heads", (long long)H, (long long)Hk);
  if (D % 8 != 0 || D > 256)
    return fail(kErrUnsupported, "head dim %lld is not a multiple of 8 in [8, 256]", (long long)D);
  if (variant < 0 || variant > kMaxSplits)
    return fail(kErrUnsupported, "masked attention variant %d (0 or the number of key splits up to %d)", variant,
                kMaxSplits);
  if (Sq > INT32_MAX / 2 || Skv > INT32_MAX / 2) return fail(kErrInvalid, "sequence too long");
  if (H > 65535 || B > 65535 || B * H > 65535)
    return fail(kErrUnsupported, "batch*heads = %lld x %lld exceeds 65535", (long long)B, (long long)H);
  return kOk;
}

int plan_masked(int64_t B, int64_t H, int64_t Hk, int64_t Sq, int64_t Skv, int64_t D, int variant, int sms,
                MaskedPlan* out) {
  const int64_t G = H / Hk;
  MaskedPlan p;
  memset(&p, 0, sizeof(p));
  // One head per tile, or the whole group where that needs fewer tiles (few queries).
  p.pack = 1;
  p.T = kAttnBM;
  if (G > 1 && G <= kAttnBM) {
    const int64_t T = kAttnBM / G;
    if ((Sq + T - 1) / T < G * ((Sq + kAttnBM - 1) / kAttnBM)) {
      p.pack = int(G);
      p.T = int(T);
    }
  }
  p.tiles = (Sq + p.T - 1) / p.T;
  p.pairs = B * H / p.pack;
  const int64_t ctas = p.tiles * p.pairs;
  const int64_t key_tiles = (Skv + kMaskedBN - 1) / kMaskedBN;
  p.splits = 1;
  if (variant > 0) {
    p.splits = variant;
  } else if (2 * ctas <= 2 * sms && key_tiles >= 8) {
    p.splits = int(std::max<int64_t>(1, std::min<int64_t>({2 * sms / ctas, key_tiles / 4, kMaxSplits})));
  }
  if (p.splits > 1) {
    if (B * H * Sq > INT32_MAX / kMaxSplits)
      return fail(kErrUnsupported, "too many rows to split their keys (%lld)", (long long)(B * H * Sq));
    const int64_t rows = p.splits * ctas * kAttnBM;
    p.ml_bytes = size_t(rows) * sizeof(float2);
    p.bytes = p.ml_bytes + size_t(rows) * size_t(D) * sizeof(float);
  }
  *out = p;
  return kOk;
}

template <int DP, int STAGES, bool SCORES>
int launch_masked(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const MaskedArgs& m, dim3 grid,
                  cudaStream_t st, int device) {
  static bool configured[64] = {false};
  auto kern = attention_masked_tcgen05_kernel<DP, STAGES, SCORES>;
  constexpr int smem = MaskedLayout<DP, STAGES>::kSmemBytes;
  if (!configured[device]) {
    if (int rc = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
                            "cudaFuncSetAttribute(masked attention smem)"))
      return rc;
    configured[device] = true;
  }
  return check_cuda(launch_pdl(kern, grid, dim3(kMaskedThreads), smem, st, mq, mk, mv, m),
                    "masked attention kernel launch");
}

template <bool SCORES>
int launch_masked_for(int64_t D, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                      const MaskedArgs& m, dim3 grid, cudaStream_t st, int dev) {
  // The padded head dims with a kernel; the columns between D and its pad are TMA zeros.
  if (D <= 32) return launch_masked<32, 5, SCORES>(mq, mk, mv, m, grid, st, dev);
  if (D <= 48) return launch_masked<48, 5, SCORES>(mq, mk, mv, m, grid, st, dev);
  if (D <= 64) return launch_masked<64, 5, SCORES>(mq, mk, mv, m, grid, st, dev);
  if (D <= 80) return launch_masked<80, 2, SCORES>(mq, mk, mv, m, grid, st, dev);
  if (D <= 96) return launch_masked<96, 2, SCORES>(mq, mk, mv, m, grid, st, dev);
  if (D <= 128) return launch_masked<128, 2, SCORES>(mq, mk, mv, m, grid, st, dev);
  if (D <= 160) return launch_masked<160, 2, SCORES>(mq, mk, mv, m, grid, st, dev);
  if (D <= 192) return launch_masked<192, 2, SCORES>(mq, mk, mv, m, grid, st, dev);
  return launch_masked<256, 2, SCORES>(mq, mk, mv, m, grid, st, dev);
}

}  // namespace

int attention_masked_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t sq, int64_t skv,
                               int64_t head_dim, int variant, size_t* bytes) {
  if (int rc = check_masked_sizes(batch, heads, kv_heads, sq, skv, head_dim, variant)) return rc;
  const DeviceInfo* dev = nullptr;
  if (int rc = current_device_info(&dev)) return rc;
  MaskedPlan plan;
  if (int rc = plan_masked(batch, heads, kv_heads, sq, skv, head_dim, variant, dev->sms, &plan)) return rc;
  *bytes = plan.bytes;
  return kOk;
}

int attention_masked_launch(const AttnMaskedProblem& mp, cudaStream_t stream) {
  const AttnProblem& p = mp.base;
  npub200_attention_mods none;
  memset(&none, 0, sizeof(none));
  const npub200_attention_mods& o = mp.mods != nullptr ? *mp.mods : none;
  if (p.q == nullptr || p.k == nullptr || p.v == nullptr || p.o == nullptr)
    return fail(kErrInvalid, "attention tensor pointer is null");
  if (int rc = check_masked_sizes(p.B, p.H, mp.kv_heads, p.Sq, p.Skv, p.D, p.variant)) return rc;
  if (!(p.scale > 0.0f)) return fail(kErrInvalid, "attention scale must be positive (got %g)", double(p.scale));
  for (const void* ptr : {p.q, p.k, p.v})
    if (reinterpret_cast<uintptr_t>(ptr) & 15u) return fail(kErrInvalid, "q/k/v base addresses must be 16-byte aligned");
  if (!(o.softcap >= 0.0f) || o.softcap > FLT_MAX)
    return fail(kErrInvalid, "softcap must be 0 (none) or positive and finite (got %g)", double(o.softcap));
  if (!o.causal && (o.prefix != 0 || o.prefixes != nullptr))
    return fail(kErrInvalid, "a prefix needs the causal mask");
  if (o.doc_offsets != nullptr) {
    if (p.Sq != p.Skv) return fail(kErrInvalid, "documents need as many queries as keys (got %lld and %lld)",
                                   (long long)p.Sq, (long long)p.Skv);
    if (o.docs < 0 || o.docs > INT32_MAX / 2 || o.doc_stride < 0)
      return fail(kErrInvalid, "bad document count or stride");
  }
  if (o.distance_bias != nullptr && (o.max_distance < 0 || o.max_distance > (1 << 24)))
    return fail(kErrInvalid, "max_distance must be in [0, 2^24] (got %d)", o.max_distance);
  if (o.mask != nullptr) {
    if (o.mask_dtype != NPUB200_DTYPE_BOOL && o.mask_dtype != NPUB200_DTYPE_BF16 && o.mask_dtype != NPUB200_DTYPE_F32)
      return fail(kErrInvalid, "unknown mask dtype code %d", o.mask_dtype);
    if (o.mask_sb < 0 || o.mask_sh < 0 || o.mask_sq < 0) return fail(kErrInvalid, "mask strides must not be negative");
  }
  const DeviceInfo* dev = nullptr;
  if (int rc = current_device_info(&dev)) return rc;
  MaskedPlan plan;
  if (int rc = plan_masked(p.B, p.H, mp.kv_heads, p.Sq, p.Skv, p.D, p.variant, dev->sms, &plan)) return rc;
  if (plan.bytes > 0) {
    if (mp.workspace == nullptr || mp.workspace_bytes < plan.bytes)
      return fail(kErrInvalid, "this attention needs a %zu-byte workspace (its keys are split), got %zu", plan.bytes,
                  mp.workspace_bytes);
    if (reinterpret_cast<uintptr_t>(mp.workspace) & 15u) return fail(kErrInvalid, "workspace must be 16-byte aligned");
  }

  MaskedArgs m;
  memset(&m, 0, sizeof(m));
  AttnArgs& a = m.a;
  CUtensorMap mq, mk, mv;
  m.G = int(p.H / mp.kv_heads);
  m.pack = plan.pack;
  m.T = int(std::min<int64_t>(plan.T, p.Sq));  // one tile of fewer rows for fewer queries
  if (int rc = encode_bshd_map(p.q, p.D, p.Sq, p.H, p.B, p.q_ss, p.q_sh, p.q_sb, m.T, &mq, &a.pq, m.pack)) return rc;
  if (int rc = encode_bshd_map(p.k, p.D, p.Skv, mp.kv_heads, p.B, p.k_ss, p.k_sh, p.k_sb, kMaskedBN, &mk, &a.pk))
    return rc;
  if (int rc = encode_bshd_map(p.v, p.D, p.Skv, mp.kv_heads, p.B, p.v_ss, p.v_sh, p.v_sb, kMaskedBN, &mv, &a.pv))
    return rc;
  m.head_fast = a.pq.h < a.pq.s;
  m.q_bytes = m.pack * m.T * kAtomBytesPerRow;
  m.tiles = int(plan.tiles);
  m.splits = plan.splits;
  m.part_ml = static_cast<float2*>(mp.workspace);
  m.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(mp.workspace) + plan.ml_bytes);
  a.Sq = int(p.Sq);
  a.Skv = int(p.Skv);
  a.H = int(p.H);
  a.scale_log2 = p.scale * kLog2e;
  a.rescale_thr = 8.0f;
  a.out = p.o;
  a.o_sb = p.o_sb;
  a.o_ss = p.o_ss;
  a.o_sh = p.o_sh;
  a.out_f32 = p.out_f32;
  a.D = int(p.D);
  a.ctl.status = dev->status;
  a.ctl.timeout_ns = wait_timeout_ns();
  a.ctl.debug = p.debug;
  m.causal = o.causal != 0;
  m.q_start = o.q_start;
  m.q_starts = o.q_starts;
  m.prefix = o.prefix;
  m.prefixes = o.prefixes;
  m.kv_lens = o.kv_lens;
  m.docs = o.doc_offsets;
  m.ndocs = int(o.docs);
  m.doc_stride = o.doc_stride;
  if (o.softcap > 0.0f) {
    m.cap_in = 2.0f * kLog2e * p.scale / o.softcap;
    m.cap_out = o.softcap * kLog2e;
  }
  m.slopes = o.slopes;
  m.table = o.distance_bias;
  m.max_dist = o.max_distance;
  m.mask = o.mask;
  if (o.mask != nullptr) {
    m.mask_kind = o.mask_dtype == NPUB200_DTYPE_BOOL ? 1 : o.mask_dtype == NPUB200_DTYPE_BF16 ? 2 : 3;
    const int64_t esz = m.mask_kind == 3 ? 4 : m.mask_kind;
    m.m_sb = o.mask_sb;
    m.m_sh = o.mask_sh;
    m.m_sq = o.mask_sq;
    m.mask_vec = ((reinterpret_cast<uintptr_t>(o.mask) | uintptr_t(o.mask_sb * esz) | uintptr_t(o.mask_sh * esz) |
                   uintptr_t(o.mask_sq * esz)) & 15u) == 0;
  }
  const dim3 grid{unsigned(plan.tiles), unsigned(plan.pairs), unsigned(plan.splits)};
  const bool scores = o.softcap > 0.0f || o.slopes != nullptr || o.distance_bias != nullptr || o.mask != nullptr;
  if (int rc = scores ? launch_masked_for<true>(p.D, mq, mk, mv, m, grid, stream, dev->device)
                      : launch_masked_for<false>(p.D, mq, mk, mv, m, grid, stream, dev->device))
    return rc;
  if (plan.splits == 1) return kOk;
  const int64_t rows = p.B * p.H * p.Sq;
  return check_cuda(launch_pdl(attention_join_kernel, dim3(unsigned((rows + 3) / 4)), dim3(128), 0, stream, m, int(rows),
                               int(plan.pairs)),
                    "attention join kernel launch");
}

}  // namespace npub200
