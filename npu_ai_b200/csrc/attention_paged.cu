// attention_paged.cu - attention of a few new tokens of each sequence over a key/value cache in pages.
//
//   o_i = sum_j softmax_j(s_ij) v_j over the keys j that row i sees; s_ij = scale q_i . k_j, then the cap, then the bias.
//
// One pass over the keys with the running maximum and sum of the softmax: for a tile of keys with row maximum t,
//   m' = max(m, t), l' = l 2^(m - m') + sum_j 2^(s_j - m'), o' = o 2^(m - m') + sum_j 2^(s_j - m') v_j,
// and parts (m, l, o) of one row's keys join the same way. Scores are kept in log2 units.
//
// Bound by memory: each key and value is read once and does 4 G flops a value for the G query heads of its head, far below
// what the tensor cores need to be busy. So the design is about loads in flight and an even split:
//   * A worker is `wr` warps, 16 rows each; the rows of a (sequence, key/value head) are its G heads x the new tokens. Few
//     rows take one warp, more share the keys of one load among 2 or 4 warps. Rows of 16 waste the matrix instruction's
//     rows, not time: mma.sync m16n8k16 on registers keeps the whole softmax in one warp, without the round trips through
//     TMEM and shared memory that a tcgen05 tile of 128 rows would add to each tile of keys.
//   * Every worker takes an equal run of tiles of 16 wr keys of the whole batch, found on the device from kv_lens, so
//     ragged lengths leave no worker idle and a captured graph follows them. A run starts and ends anywhere in a sequence;
//     parts of a row's keys go to the workspace and the join kernel adds them up in order of keys.
//   * A tile's keys and values are rows anywhere in memory: cp.async of 16 bytes a lane takes any page size and layout,
//     into a ring of 3 to 6 tiles. (A bulk copy a row, one instruction a lane, was the first form: the copy engine takes
//     one in about 17 cycles, 16 bytes a cycle at 128 columns where 23 are the memory's rate.) Rows in shared memory are
//     16 bytes longer than the head, so that ldmatrix reads 8 of them without a bank conflict.
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <cstring>

#include "internal.h"

namespace npub200 {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWarps = 4;      // of a block
constexpr int kSub = 16;       // keys of one step of the matrix instructions; a tile is `wr` of them
constexpr int kMaxStages = 6;  // of a ring
constexpr int kJoinWarps = 8;
// The row maximum moves only when a tile's beats it by this much (log2 units): P stays within 2^8 of 1, which bf16 holds
// with the same relative rounding, and the O registers are rescaled once in a while instead of once a tile.
constexpr float kRescale = 8.0f;

struct PagedArgs {
  const __nv_bfloat16* q;
  long long q_sb, q_ss, q_sh;
  const __nv_bfloat16* k;
  long long k_sp, k_ss, k_sh;
  const __nv_bfloat16* v;
  long long v_sp, v_ss, v_sh;
  const int32_t* table;
  long long table_stride;
  int pages, page_size, capacity;
  const int32_t* lens;
  const int32_t* q_starts;
  void* out;
  long long o_sb, o_ss, o_sh;
  int out_f32, out_vec;  // out_vec: pairs of output columns may be written together
  int B, Hk, G, Sq, D;
  int causal;
  float scale_log2;     // scores to log2 units
  float cap_in, cap_out;  // softcap: cap_out tanh(cap_in q.k), cap_out 0: none
  const float* slopes;
  int workers;              // of the grid
  int rows, row_tiles, slot_rows;  // rows of a (sequence, kv head), tiles of 16 wr rows, rows of a part in the workspace
  int min_span;             // least tiles of a worker's run
  // What there is to join: of each item where there are no more items than workers, else of the item that begins in each
  // worker's run and goes on behind it. (sequence, kv head and row tile, parts or 0, worker of the first)
  int4* rec;
  int rec_items;
  float2* part_ml;          // [2 workers][slot_rows] (m, l); part 0 of a worker continues an item, part 1 begins one
  float* part_o;            // [2 workers][slot_rows][D]
};

__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16 bytes from global to shared memory, or zeros where `ok` is false.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {  // all but the last N groups of this thread are there
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Layout of a block's shared memory for head dims up to DP and workers of WR warps.
template <int DP, int WR>
struct PagedLayout {
  static constexpr int kTile = kSub * WR;                // keys of a tile
  static constexpr int kRow = DP * 2 + 16;               // bytes of a key's (value's) row
  static constexpr int kStage = 2 * kTile * kRow;        // the keys, then their values
  static constexpr int kBlocks = DP <= 128 ? 2 : 1;      // resident on an SM
  // As many as 227 KB hold: 69 to 112 KB in flight on an SM, of which some 40 KB cover the latency at full rate.
  static constexpr int kStages = DP == 64 ? 6 : DP == 96 ? 4 : DP == 128 ? 3 : DP == 160 ? 5 : DP == 192 ? 4 : 3;
  static constexpr int kRing = kStages * kStage;
  static constexpr int kSmem = kWarps / WR * kRing;
};

// The keys that row tile `rt` of a sequence sees at most, and the row's own bounds.
struct Sequence {
  int len;         // valid keys
  long long p0;    // position of query 0
};
__device__ __forceinline__ int sequence_len(const PagedArgs& a, int b) { return min(max(a.lens[b], 0), a.capacity); }
__device__ __forceinline__ Sequence sequence_of(const PagedArgs& a, int b) {
  Sequence s;
  s.len = sequence_len(a, b);
  s.p0 = a.q_starts != nullptr ? (long long)a.q_starts[b] : (long long)s.len - a.Sq;
  return s;
}
// Keys that the query at position p sees.
__device__ __forceinline__ int keys_seen(const PagedArgs& a, int len, long long p) {
  return a.causal ? int(max(0ll, min((long long)len, p + 1))) : len;
}
// A sequence without keys still has rows to write: it counts one tile.
template <int KT>
__device__ __forceinline__ int tiles_of(int len) {
  return max(1, (len + KT - 1) / KT);
}

// A worker's place in its run of tiles: the item (sequence b, rest = kv head * row_tiles + row tile) and the tiles of it
// that belong to the run.
template <int KT>
struct Cursor {
  int b, rest;
  int t, t1;        // next tile, end of the run's tiles within the item
  int tiles;        // of the item
  int seen;         // keys that some row of the item's row tile sees
  Sequence seq;
  long long left;   // tiles of the run behind this item

  __device__ __forceinline__ void enter(const PagedArgs& a, int t0, long long run) {
    seq = sequence_of(a, b);
    tiles = tiles_of<KT>(seq.len);
    t = t0;
    t1 = int(min((long long)tiles, t0 + run));
    left = run - (t1 - t0);
    const int last = min(a.rows, (rest % a.row_tiles + 1) * KT) - 1;  // (a row tile has as many rows as a tile has keys)
    seen = keys_seen(a, seq.len, seq.p0 + last / a.G);
  }
  // The next item of the run; false when there is none.
  __device__ __forceinline__ bool next(const PagedArgs& a) {
    if (left <= 0) return false;
    if (++rest == a.Hk * a.row_tiles) {
      rest = 0;
      ++b;
    }
    enter(a, 0, left);
    return true;
  }
  // End of the tiles that have a key to see.
  __device__ __forceinline__ int visible_end() const { return min(t1, (seen + KT - 1) / KT); }
};

__device__ __forceinline__ long long shfl_ll(long long v, int lane) { return __shfl_sync(0xffffffffu, v, lane); }

template <int DP, int WR, bool MODS>
__global__ void __launch_bounds__(kWarps * 32, PagedLayout<DP, WR>::kBlocks) attention_paged_kernel(const PagedArgs a) {
  using L = PagedLayout<DP, WR>;
  constexpr int KT = L::kTile;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint32_t s_valid[kWarps][kMaxStages][2];  // which of a stage's keys are there, as each warp found
  const int lane = int(threadIdx.x) & 31, warp = int(threadIdx.x) >> 5;
  const int role = warp % WR;  // this warp's 16 rows of the worker's
  const int worker = int(blockIdx.x) * (kWarps / WR) + warp / WR;
  const uint32_t ring = smem_u32(smem) + (warp / WR) * L::kRing;
  pdl_wait();
  pdl_launch_dependents();

  // The worker's run: an equal share of all tiles.
  const long long per_tile = (long long)a.Hk * a.row_tiles;
  long long total = 0;
  for (int b = lane; b < a.B; b += 32) total += tiles_of<KT>(sequence_len(a, b));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  total *= per_tile;
  const long long span = max((total + a.workers - 1) / a.workers, (long long)a.min_span);
  const long long u0 = worker * span, u1 = min(total, u0 + span);
  int4 rec = make_int4(0, 0, 0, worker);
  if (u0 < u1) {
    Cursor<KT> at;
    long long base = 0;
    for (int c = 0; c < a.B; c += 32) {
      const long long mine = c + lane < a.B ? per_tile * tiles_of<KT>(sequence_len(a, c + lane)) : 0;
      long long upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, base + upto > u0);
      if (hit != 0) {
        const int f = __ffs(int(hit)) - 1;
        at.b = c + f;
        base += shfl_ll(upto, f) - shfl_ll(mine, f);
        break;
      }
      base += shfl_ll(upto, 31);
    }
    const int tiles0 = tiles_of<KT>(sequence_len(a, at.b));
    at.rest = int((u0 - base) / tiles0);
    at.enter(a, int((u0 - base) - (long long)at.rest * tiles0), u1 - u0);

    // ---- the loader, kStages - 1 tiles ahead: each lane looks up the page of one key (two of 64), the warps of a worker
    // copy a share each
    constexpr int kKeys = KT <= 32 ? 1 : 2;
    Cursor<KT> ld = at;
    bool more = true;  // the loader has a tile
    int ld_end = ld.visible_end(), ld_stage = 0;
    int page[kKeys];
    const auto seek = [&]() {  // to the next tile with keys, and the pages of this lane's keys of it
      while (ld.t >= ld_end) {
        if (!ld.next(a)) {
          more = false;
          return;
        }
        ld_end = ld.visible_end();
      }
#pragma unroll
      for (int x = 0; x < kKeys; ++x) {
        const int j = ld.t * KT + lane + 32 * x;
        page[x] = lane < KT && j < ld.seen ? a.table[ld.b * a.table_stride + j / a.page_size] : -1;
      }
    };
    const auto issue = [&]() {
      if (more) {
        const int kvh = ld.rest / a.row_tiles;
        const __nv_bfloat16* src[2] = {a.k + kvh * a.k_sh, a.v + kvh * a.v_sh};
        long long off[kKeys][2];  // of this lane's keys and values
#pragma unroll
        for (int x = 0; x < kKeys; ++x) {
          const bool ok = page[x] >= 0 && page[x] < a.pages;
          const uint32_t mask = __ballot_sync(0xffffffffu, ok);
          if (lane == 0) s_valid[warp][ld_stage][x] = mask;
          const int slot = (ld.t * KT + lane + 32 * x) % a.page_size;
          off[x][0] = ok ? page[x] * a.k_sp + slot * a.k_ss : -1;
          off[x][1] = ok ? page[x] * a.v_sp + slot * a.v_ss : -1;
        }
        constexpr int kChunks = DP / 8;  // 16-byte pieces of a row
        const uint32_t stage = ring + ld_stage * L::kStage;
#pragma unroll
        for (int which = 0; which < 2; ++which)
#pragma unroll
          for (int i = 0; i < kSub * kChunks / 32; ++i) {
            const int idx = (i * WR + role) * 32 + lane, row = idx / kChunks, c = idx - row * kChunks;
            long long o = __shfl_sync(0xffffffffu, off[0][which], row & 31);
            if constexpr (kKeys == 2) {
              const long long hi = __shfl_sync(0xffffffffu, off[1][which], row & 31);
              o = row >= 32 ? hi : o;
            }
            const bool ok = o >= 0 && c * 8 < a.D;
            copy16(stage + (which * KT + row) * L::kRow + c * 16, src[which] + (ok ? o + c * 8 : 0), ok);
          }
        ld_stage = ld_stage + 1 == L::kStages ? 0 : ld_stage + 1;
        ++ld.t;
        seek();
      }
      copy_commit();  // (an empty group behind the last tile: the waits count groups)
    };
    seek();
#pragma unroll
    for (int i = 0; i < L::kStages - 1; ++i) issue();

    // ---- the items of the run
    const int g = lane >> 2, c2 = (lane & 3) * 2;
    int stage = 0;
    do {
      const int kvh = at.rest / a.row_tiles, r0 = (at.rest % a.row_tiles) * 16 * WR + role * 16;
      int lim[2];
      long long p[2];
      float slope[2];
      uint32_t qf[DP / 16][4];
      {
        const __nv_bfloat16* qp[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int r = r0 + g + 8 * x;
          const bool in = r < a.rows;
          const int i = in ? r / a.G : 0, h = kvh * a.G + (in ? r - i * a.G : 0);
          p[x] = at.seq.p0 + i;
          lim[x] = in ? keys_seen(a, at.seq.len, p[x]) : at.seq.len;
          slope[x] = MODS && a.slopes != nullptr ? a.slopes[h] * kLog2e : 0.0f;
          qp[x] = in ? a.q + ((long long)at.b * a.q_sb + (long long)i * a.q_ss + (long long)h * a.q_sh + c2) : nullptr;
        }
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int col = s * 16 + (e >> 1) * 8;
            qf[s][e] = qp[e & 1] != nullptr && col < a.D ? *reinterpret_cast<const uint32_t*>(qp[e & 1] + col) : 0u;
          }
      }
      int lim_min = min(lim[0], lim[1]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) lim_min = min(lim_min, __shfl_xor_sync(0xffffffffu, lim_min, o));
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
      float o[DP / 8][4];
#pragma unroll
      for (int n = 0; n < DP / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;

      const int first = at.t, end = at.visible_end();
      for (int t = first; t < end; ++t) {
        copy_wait<L::kStages - 2>();
        if constexpr (WR == 1) {
          __syncwarp();
        } else {  // the other warps' copies of this tile are there, and they are done with the tile before
          named_barrier_sync(1 + warp / WR, WR * 32);
        }
        issue();
        const uint32_t stage_k = ring + stage * L::kStage;
#pragma unroll 1
        for (int sub = 0; sub < WR; ++sub) {
        const int j0 = t * KT + sub * kSub;
        const uint32_t valid = (s_valid[warp][stage][sub >> 1] >> ((sub & 1) * 16)) & 0xffffu;
        const uint32_t base_k = stage_k + sub * kSub * L::kRow;
        // S = Q K^T: two blocks of 8 keys, even and odd steps in sums of their own (half the chain)
        float s4[2][2][4];
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int e = 0; e < 4; ++e) s4[x][y][e] = 0.0f;
        const uint32_t ka = base_k + ((lane & 7) + ((lane >> 4) & 1) * 8) * L::kRow + ((lane >> 3) & 1) * 16;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
          uint32_t kf[4];
          ldmatrix_x4(ka + s * 32, kf);
          mma_bf16(s4[s & 1][0], qf[s], kf[0], kf[1]);
          mma_bf16(s4[s & 1][1], qf[s], kf[2], kf[3]);
        }
        float x[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float dot = s4[0][n][e] + s4[1][n][e];
            if constexpr (MODS) {
              x[n][e] = a.cap_out != 0.0f ? a.cap_out * tanhf(dot * a.cap_in) : dot * a.scale_log2;
              if (a.slopes != nullptr) {
                const long long j = j0 + n * 8 + c2 + (e & 1);
                x[n][e] = fmaf(-slope[e >> 1], fabsf(float(p[e >> 1] - j)), x[n][e]);
              }
            } else {
              x[n][e] = dot * a.scale_log2;
            }
          }
        if (valid != 0xffffu || j0 + kSub > lim_min) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int j = n * 8 + c2 + (e & 1);
              if (j0 + j >= lim[e >> 1] || ((valid >> j) & 1u) == 0) x[n][e] = -INFINITY;
            }
        }
        float top[2];
        bool moved = false;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          top[r] = fmaxf(fmaxf(x[0][2 * r], x[0][2 * r + 1]), fmaxf(x[1][2 * r], x[1][2 * r + 1]));
          top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
          top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
          moved = moved || top[r] > m[r] + kRescale;
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float mr = top[r] > m[r] + kRescale ? top[r] : m[r];
            const float f = mr == m[r] ? 1.0f : fast_exp2(m[r] - mr);
            m[r] = mr;
            l[r] *= f;
#pragma unroll
            for (int n = 0; n < DP / 8; ++n) {
              o[n][2 * r] *= f;
              o[n][2 * r + 1] *= f;
            }
          }
        }
        uint32_t pf[4];
        {
          float w[2][4];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float mu = m[r] == -INFINITY ? 0.0f : m[r];  // nothing seen yet: every weight is 0
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                w[n][2 * r + e] = fast_exp2(x[n][2 * r + e] - mu);
                l[r] += w[n][2 * r + e];
              }
          }
          // P rounded to bf16 for the tensor core: 2^-8 relative at most; the sum takes the unrounded values.
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            pf[2 * n] = pack_bf16x2(w[n][0], w[n][1]);
            pf[2 * n + 1] = pack_bf16x2(w[n][2], w[n][3]);
          }
        }
        // O += P V
        const uint32_t va = base_k + KT * L::kRow + ((lane & 7) + ((lane >> 3) & 1) * 8) * L::kRow + ((lane >> 4) & 1) * 16;
#pragma unroll
        for (int n = 0; n < DP / 16; ++n) {
          uint32_t vf[4];
          ldmatrix_x4_trans(va + n * 32, vf);
          mma_bf16(o[2 * n], pf, vf[0], vf[1]);
          mma_bf16(o[2 * n + 1], pf, vf[2], vf[3]);
        }
        }
        stage = stage + 1 == L::kStages ? 0 : stage + 1;
      }

      // ---- the item's rows, or the run's part of them
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      }
      const bool whole = first == 0 && at.t1 == at.tiles;
      if (first == 0 && !whole) {
        const long long item_end = u1 - (at.t1 - first) + at.tiles;  // the run ends in this item
        rec = make_int4(at.b, at.rest, int((item_end - 1) / span) - worker + 1, worker);
      }
      if (a.rec_items && first == 0 && role == 0 && lane == 0)
        a.rec[at.b * (a.Hk * a.row_tiles) + at.rest] = whole ? make_int4(0, 0, 0, 0) : rec;
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int r = r0 + g + 8 * y;
        if (r >= a.rows) continue;
        if (whole) {
          const float inv = l[y] == 0.0f ? 0.0f : 1.0f / l[y];  // (a NaN sum makes the row NaN)
          const int i = r / a.G, h = kvh * a.G + (r - i * a.G);
          const long long at0 = (long long)at.b * a.o_sb + (long long)i * a.o_ss + (long long)h * a.o_sh + c2;
#pragma unroll
          for (int n = 0; n < DP / 8; ++n) {
            if (n * 8 >= a.D) break;
            const float v0 = o[n][2 * y] * inv, v1 = o[n][2 * y + 1] * inv;
            if (a.out_f32) {
              float* d = static_cast<float*>(a.out) + at0 + n * 8;
              if (a.out_vec) {
                *reinterpret_cast<float2*>(d) = make_float2(v0, v1);
              } else {
                d[0] = v0;
                d[1] = v1;
              }
            } else {
              __nv_bfloat16* d = static_cast<__nv_bfloat16*>(a.out) + at0 + n * 8;
              if (a.out_vec) {
                *reinterpret_cast<uint32_t*>(d) = pack_bf16x2(v0, v1);
              } else {
                d[0] = __float2bfloat16_rn(v0);
                d[1] = __float2bfloat16_rn(v1);
              }
            }
          }
        } else {
          const long long part = ((long long)worker * 2 + (first == 0)) * a.slot_rows + (role * 16 + g + 8 * y);
          if (c2 == 0) a.part_ml[part] = make_float2(m[y], l[y]);
#pragma unroll
          for (int n = 0; n < DP / 8; ++n) {
            if (n * 8 >= a.D) break;
            *reinterpret_cast<float2*>(a.part_o + part * a.D + n * 8 + c2) = make_float2(o[n][2 * y], o[n][2 * y + 1]);
          }
        }
      }
    } while (at.next(a));
  }
  if (!a.rec_items && role == 0 && lane == 0) a.rec[worker] = rec;
}

// Joins the parts of the item of record blockIdx.x. Eight warps take the parts in turn, a lane 4 (8 above 128) columns.
__global__ void __launch_bounds__(kJoinWarps * 32) attention_paged_join_kernel(const PagedArgs a, int row_tile) {
  __shared__ float s_acc[kJoinWarps][256];
  __shared__ float s_inv;
  const int lane = int(threadIdx.x) & 31, warp = int(threadIdx.x) >> 5;
  pdl_wait();
  pdl_launch_dependents();
  const int4 rec = a.rec[blockIdx.x];
  const int parts = rec.z, w = rec.w;
  if (parts == 0) return;
  const int kvh = rec.y / a.row_tiles, r0 = (rec.y % a.row_tiles) * row_tile;
  const int rows = min(a.rows - r0, row_tile);
  const auto part_row = [&](int z) { return ((long long)(w + z) * 2 + (z == 0)) * a.slot_rows; };
  for (int row = int(blockIdx.y); row < rows; row += int(gridDim.y)) {
    float top = -INFINITY;
    for (int z = lane; z < parts; z += 32) top = fmaxf(top, a.part_ml[part_row(z) + row].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float sum = 0.0f;
    if (warp == 0) {
      for (int z = lane; z < parts; z += 32) {
        const float2 ml = a.part_ml[part_row(z) + row];
        sum = fmaf(ml.x == -INFINITY ? 0.0f : fast_exp2(ml.x - top), ml.y, sum);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) s_inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    }
    float acc[2][4] = {};
    for (int z = warp; z < parts; z += kJoinWarps) {
      const long long at = part_row(z) + row;
      const float mz = a.part_ml[at].x;
      const float wt = mz == -INFINITY ? 0.0f : fast_exp2(mz - top);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int col = lane * 4 + k * 128;
        if (col < a.D) {
          const float4 x = *reinterpret_cast<const float4*>(a.part_o + at * a.D + col);
          acc[k][0] = fmaf(wt, x.x, acc[k][0]);
          acc[k][1] = fmaf(wt, x.y, acc[k][1]);
          acc[k][2] = fmaf(wt, x.z, acc[k][2]);
          acc[k][3] = fmaf(wt, x.w, acc[k][3]);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) s_acc[warp][k * 128 + lane * 4 + e] = acc[k][e];
    __syncthreads();
    const int col = int(threadIdx.x);
    if (col < a.D) {
      float x = 0.0f;
#pragma unroll
      for (int k = 0; k < kJoinWarps; ++k) x += s_acc[k][col];
      x *= s_inv;
      const int r = r0 + row, i = r / a.G, h = kvh * a.G + (r - i * a.G);
      const long long at = (long long)rec.x * a.o_sb + (long long)i * a.o_ss + (long long)h * a.o_sh + col;
      if (a.out_f32)
        static_cast<float*>(a.out)[at] = x;
      else
        static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(x);
    }
    __syncthreads();  // s_acc and s_inv are written again for the next row
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------------------------
struct PagedPlan {
  int wr, blocks, workers;
  int64_t rows, row_tiles, slot_rows;
  size_t ml_offset, o_offset, bytes;
};

int check_paged_sizes(int64_t H, int64_t Hk, int64_t Sq, int64_t D) {
  if (H <= 0 || Hk <= 0 || Sq <= 0 || D <= 0)
    return fail(kErrInvalid, "attention sizes must be positive (H=%lld Hkv=%lld Sq=%lld D=%lld)", (long long)H,
                (long long)Hk, (long long)Sq, (long long)D);
  if (H % Hk != 0)
    return fail(kErrInvalid, "%lld query heads are not a multiple of %lld key/value heads", (long long)H, (long long)Hk);
  if (D % 8 != 0 || D > 256)
    return fail(kErrUnsupported, "head dim %lld is not a multiple of 8 in [8, 256]", (long long)D);
  if (H > 65535 || Sq > (1 << 24) || H * Sq > (1 << 30))
    return fail(kErrUnsupported, "too many rows (%lld heads x %lld tokens)", (long long)H, (long long)Sq);
  return kOk;
}

PagedPlan plan_paged(int64_t H, int64_t Hk, int64_t Sq, int64_t D, int sms) {
  PagedPlan p;
  p.rows = H / Hk * Sq;
  p.wr = p.rows <= 16 ? 1 : p.rows <= 32 ? 2 : 4;
  p.row_tiles = (p.rows + 16 * p.wr - 1) / (16 * p.wr);
  p.slot_rows = p.rows < 16 * p.wr ? p.rows : 16 * p.wr;
  p.blocks = sms * (D <= 128 ? 2 : 1);
  p.workers = p.blocks * (kWarps / p.wr);
  const size_t parts = size_t(p.workers) * 2 * size_t(p.slot_rows);
  p.ml_offset = (size_t(p.workers) * sizeof(int4) + 255) / 256 * 256;
  p.o_offset = (p.ml_offset + parts * sizeof(float2) + 255) / 256 * 256;
  p.bytes = p.o_offset + parts * size_t(D) * sizeof(float);
  return p;
}

template <int DP, int WR, bool MODS>
int launch_paged(const PagedArgs& a, int blocks, cudaStream_t stream, int device) {
  using L = PagedLayout<DP, WR>;
  static_assert(L::kStages <= kMaxStages && L::kSmem + 2048 <= 227 * 1024 / L::kBlocks, "shared memory of the SM");
  static std::atomic<bool> ready[64] = {};
  if (!ready[device]) {
    if (int rc = check_cuda(cudaFuncSetAttribute(attention_paged_kernel<DP, WR, MODS>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem),
                            "paged attention shared memory"))
      return rc;
    ready[device] = true;
  }
  return check_cuda(launch_pdl(attention_paged_kernel<DP, WR, MODS>, dim3(unsigned(blocks)), dim3(kWarps * 32), L::kSmem,
                               stream, a),
                    "paged attention kernel launch");
}

template <int WR, bool MODS>
int launch_paged_dim(const PagedArgs& a, int blocks, cudaStream_t stream, int device) {
  if (a.D <= 64) return launch_paged<64, WR, MODS>(a, blocks, stream, device);
  if (a.D <= 96) return launch_paged<96, WR, MODS>(a, blocks, stream, device);
  if (a.D <= 128) return launch_paged<128, WR, MODS>(a, blocks, stream, device);
  if (a.D <= 160) return launch_paged<160, WR, MODS>(a, blocks, stream, device);
  if (a.D <= 192) return launch_paged<192, WR, MODS>(a, blocks, stream, device);
  return launch_paged<256, WR, MODS>(a, blocks, stream, device);
}

template <bool MODS>
int launch_paged_for(const PagedArgs& a, int wr, int blocks, cudaStream_t stream, int device) {
  if (wr == 1) return launch_paged_dim<1, MODS>(a, blocks, stream, device);
  if (wr == 2) return launch_paged_dim<2, MODS>(a, blocks, stream, device);
  return launch_paged_dim<4, MODS>(a, blocks, stream, device);
}

}  // namespace

int attention_paged_workspace(int64_t heads, int64_t kv_heads, int64_t sq, int64_t head_dim, size_t* bytes) {
  if (int rc = check_paged_sizes(heads, kv_heads, sq, head_dim)) return rc;
  const DeviceInfo* dev = nullptr;
  if (int rc = current_device_info(&dev)) return rc;
  *bytes = plan_paged(heads, kv_heads, sq, head_dim, dev->sms).bytes;
  return kOk;
}

int attention_paged_launch(const AttnPagedProblem& p, cudaStream_t stream) {
  if (int rc = check_paged_cache(p.cache, p.batch, "paged attention")) return rc;
  const npub200_paged_cache& c = *p.cache;
  if (p.batch < 0 || p.sq < 0 || p.batch > INT32_MAX)
    return fail(kErrInvalid, "paged attention: bad batch or number of tokens (%lld, %lld)", (long long)p.batch,
                (long long)p.sq);
  if (int rc = check_paged_sizes(p.heads, c.kv_heads, p.sq == 0 ? 1 : p.sq, c.head_dim)) return rc;
  if (p.out_dtype != NPUB200_DTYPE_BF16 && p.out_dtype != NPUB200_DTYPE_F32)
    return fail(kErrInvalid, "unknown output dtype code %d", p.out_dtype);
  if (p.variant < 0 || p.variant > (1 << 20))
    return fail(kErrUnsupported, "paged attention variant %d (0 or the least number of tiles of a split up to 2^20)",
                p.variant);
  if (!(p.scale > 0.0f && p.scale * kLog2e <= FLT_MAX))
    return fail(kErrInvalid, "attention scale must be positive and finite, times log2 e too (got %g)", double(p.scale));
  if (!(p.softcap == 0.0f || (p.softcap >= 1e-30f && p.softcap <= 1e30f)))
    return fail(kErrInvalid, "softcap must be 0 (none) or positive, within [1e-30, 1e30] (got %g)", double(p.softcap));
  const float cap_in = p.softcap > 0.0f ? p.scale / p.softcap : 0.0f;
  if (p.softcap > 0.0f && !(cap_in >= FLT_MIN && cap_in <= FLT_MAX))
    return fail(kErrInvalid, "attention scale %g over softcap %g is not a normal number", double(p.scale),
                double(p.softcap));
  if (p.batch == 0 || p.sq == 0) return kOk;
  if (p.q == nullptr || p.out == nullptr || p.kv_lens == nullptr)
    return fail(kErrInvalid, "paged attention: q, out or kv_lens is null");
  if (p.q_sb < 0 || p.q_ss < 0 || p.q_sh < 0 || p.o_sb < 0 || p.o_ss < 0 || p.o_sh < 0)
    return fail(kErrInvalid, "paged attention: negative stride");
  if ((reinterpret_cast<uintptr_t>(p.q) & 15u) || (p.q_sb | p.q_ss | p.q_sh) % 8 != 0)
    return fail(kErrInvalid, "paged attention: q needs a 16-byte aligned base and strides in multiples of 8 elements");
  if (c.pages > 0 && ((reinterpret_cast<uintptr_t>(c.k) & 15u) || (reinterpret_cast<uintptr_t>(c.v) & 15u) ||
                      (c.k_sp | c.k_ss | c.k_sh | c.v_sp | c.v_ss | c.v_sh) % 8 != 0))
    return fail(kErrInvalid, "paged attention: pages need 16-byte aligned bases and strides in multiples of 8 elements");
  const int esize = p.out_dtype == NPUB200_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(p.out) % uintptr_t(esize)) return fail(kErrInvalid, "paged attention: out is misaligned");
  const DeviceInfo* dev = nullptr;
  if (int rc = current_device_info(&dev)) return rc;
  const PagedPlan plan = plan_paged(p.heads, c.kv_heads, p.sq, c.head_dim, dev->sms);
  if (p.workspace == nullptr || p.workspace_bytes < plan.bytes)
    return fail(kErrInvalid, "paged attention needs a %zu-byte workspace, got %zu", plan.bytes, p.workspace_bytes);
  if (reinterpret_cast<uintptr_t>(p.workspace) & 15u) return fail(kErrInvalid, "workspace must be 16-byte aligned");

  PagedArgs a;
  memset(&a, 0, sizeof(a));
  a.q = static_cast<const __nv_bfloat16*>(p.q);
  a.q_sb = p.q_sb, a.q_ss = p.q_ss, a.q_sh = p.q_sh;
  a.k = static_cast<const __nv_bfloat16*>(c.k);
  a.k_sp = c.k_sp, a.k_ss = c.k_ss, a.k_sh = c.k_sh;
  a.v = static_cast<const __nv_bfloat16*>(c.v);
  a.v_sp = c.v_sp, a.v_ss = c.v_ss, a.v_sh = c.v_sh;
  a.table = c.table;
  a.table_stride = c.table_stride;
  a.pages = int(c.pages);
  a.page_size = int(c.page_size);
  a.capacity = int(c.table_width * c.page_size);
  a.lens = p.kv_lens;
  a.q_starts = p.q_starts;
  a.out = p.out;
  a.o_sb = p.o_sb, a.o_ss = p.o_ss, a.o_sh = p.o_sh;
  a.out_f32 = p.out_dtype == NPUB200_DTYPE_F32;
  a.out_vec = ((reinterpret_cast<uintptr_t>(p.out) | uintptr_t(p.o_sb * esize) | uintptr_t(p.o_ss * esize) |
                uintptr_t(p.o_sh * esize)) &
               uintptr_t(2 * esize - 1)) == 0;
  a.B = int(p.batch);
  a.Hk = int(c.kv_heads);
  a.G = int(p.heads / c.kv_heads);
  a.Sq = int(p.sq);
  a.D = int(c.head_dim);
  a.causal = p.causal != 0;
  a.scale_log2 = p.scale * kLog2e;
  a.cap_in = cap_in;
  a.cap_out = p.softcap * kLog2e;
  a.slopes = p.slopes;
  a.workers = plan.workers;
  a.rows = int(plan.rows);
  a.row_tiles = int(plan.row_tiles);
  a.slot_rows = int(plan.slot_rows);
  a.min_span = p.variant > 0 ? p.variant : 4;
  const int64_t items = p.batch * c.kv_heads * plan.row_tiles;
  a.rec_items = items <= plan.workers;
  uint8_t* ws = static_cast<uint8_t*>(p.workspace);
  a.rec = reinterpret_cast<int4*>(ws);
  a.part_ml = reinterpret_cast<float2*>(ws + plan.ml_offset);
  a.part_o = reinterpret_cast<float*>(ws + plan.o_offset);
  const bool mods = p.softcap > 0.0f || p.slopes != nullptr;
  if (int rc = mods ? launch_paged_for<true>(a, plan.wr, plan.blocks, stream, dev->device)
                    : launch_paged_for<false>(a, plan.wr, plan.blocks, stream, dev->device))
    return rc;
  // A block joins one row of an item, or all of them when there are items enough to fill the GPU.
  const int64_t split = items >= dev->sms ? 1 : plan.slot_rows;
  return check_cuda(launch_pdl(attention_paged_join_kernel, dim3(unsigned(std::min<int64_t>(items, plan.workers)), unsigned(split)),
                               dim3(kJoinWarps * 32), 0, stream, a, 16 * plan.wr),
                    "paged attention join kernel launch");
}

}  // namespace npub200
