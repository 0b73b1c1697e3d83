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
//   * A worker is WR warps, 16 rows each; the rows of a (sequence, key/value head) are its G heads x the new tokens. Few
//     rows take one warp, more share the keys of one load among 2 or 4 warps. Rows of 16 waste the matrix instruction's
//     rows, not time: mma.sync m16n8k16 on registers keeps the whole softmax in one warp, without the round trips through
//     TMEM and shared memory that a tcgen05 tile of 128 rows would add to each tile of keys.
//   * One block an SM. Every block takes an equal run of tiles of the whole batch, found on the device from kv_lens, so
//     ragged lengths leave no SM idle and a captured graph follows them, and its workers equal shares of it. Shares start
//     and end anywhere in a sequence; the parts of a row's keys are joined in order of keys, first those of a block through
//     its shared memory, then those of several blocks through the workspace by the join kernel.
//   * A tile's keys and values are rows anywhere in memory: cp.async of 16 bytes a lane takes any page size and layout.
//     (A bulk copy a row, one instruction a lane, was the first form: the copy engine takes one in about 17 cycles, 16
//     bytes a cycle at 128 columns where 23 are the memory's rate.) Keys and values wait in one ring, a half tile each.
//     Rows in shared memory are 16 bytes longer than the head, so that ldmatrix reads 8 of them without a bank conflict.
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <cstring>

#include "internal.h"

namespace npub200 {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWarps = 8;  // of a block
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
  int out_f32, out_vec;  // out_vec: pairs (1) or four (2) output columns may be written together
  int B, Hk, G, Sq, D;
  int causal;
  float scale_log2;       // scores to log2 units
  float cap_in, cap_out;  // softcap: cap_out tanh(cap_in q.k), cap_out 0: none
  const float* slopes;
  int rows, row_tiles, slot_rows;  // rows of a (sequence, kv head), tiles of 16 WR rows, rows of a part
  int min_span;           // least tiles of a block's run
  // What there is to join: of each item where there are no more items than blocks, else of the item that begins in each
  // block's run and goes on behind it. (sequence, kv head and row tile, parts or 0, block of the first)
  int4* rec;
  int rec_items;
  float2* part_ml;  // [2 blocks][slot_rows] (m, l); part 0 of a block continues an item, part 1 begins one
  float* part_o;    // [2 blocks][slot_rows][D]
  float* head_o;    // [blocks][workers][slot_rows][D] O of the items that end within a worker's share
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
  // Keys of a tile: what keeps its scores in registers next to O and Q. 16 for one warp took 30% longer at 64 columns,
  // where the softmax of a tile and not its load decided.
  static constexpr int kTile = WR == 1 ? (DP <= 128 ? 32 : 16) : 16 * WR;
  static constexpr int kRow = DP * 2 + 16;  // bytes of a key's (value's) row
  static constexpr int kHalf = kTile * kRow;  // the keys or the values of a tile
  static constexpr int kWorkers = kWarps / WR;
  // As many as an SM holds next to the static tables: 130 to 170 KB in flight, of which some 40 KB cover the latency at the
  // full rate.
  static constexpr int kFit = 219 * 1000 / (kWorkers * kHalf);
  static constexpr int kHalves = kFit < 8 ? kFit : 8;
  static constexpr int kRing = kHalves * kHalf;
  static constexpr int kSmem = kWorkers * kRing;
  // The ring takes the O rows of the share's last part, 8 floats longer so that their stores spread over the banks.
  static_assert(kHalves >= 3 && kRing >= 16 * WR * (DP + 8) * 4, "ring");
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

// A worker's place in its share of tiles: the item (sequence b, rest = kv head * row_tiles + row tile) and the tiles of it
// that belong to the share.
template <int KT>
struct Cursor {
  int b, rest;
  int t, t1;       // next tile, end of the share's tiles within the item
  int tiles;       // of the item
  int seen;        // keys that some row of the item's row tile sees
  Sequence seq;
  long long left;  // tiles of the share behind this item

  __device__ __forceinline__ void enter(const PagedArgs& a, int row_tile, int t0, long long run) {
    seq = sequence_of(a, b);
    tiles = tiles_of<KT>(seq.len);
    t = t0;
    t1 = int(min((long long)tiles, t0 + run));
    left = run - (t1 - t0);
    const int last = min(a.rows, (rest % a.row_tiles + 1) * row_tile) - 1;
    seen = keys_seen(a, seq.len, seq.p0 + last / a.G);
  }
  // The next item of the share; false when there is none.
  __device__ __forceinline__ bool next(const PagedArgs& a, int row_tile) {
    if (left <= 0) return false;
    if (++rest == a.Hk * a.row_tiles) {
      rest = 0;
      ++b;
    }
    enter(a, row_tile, 0, left);
    return true;
  }
  // End of the tiles that have a key to see.
  __device__ __forceinline__ int visible_end() const { return min(t1, (seen + KT - 1) / KT); }
};

// a / b for a >= 0, b > 0; nearly always both fit 32 bits, where the division takes a fraction of the time.
__device__ __forceinline__ long long divide(long long a, long long b) {
  return ((a | b) >> 32) == 0 ? (long long)(uint32_t(a) / uint32_t(b)) : a / b;
}

// cap_out tanh(y): below 1 tanh(y) / y as a polynomial in y^2 (fit_tanh_poly.py beside this file; relative error 7e-7), which
// keeps small values' relative accuracy, e^2y above.
__device__ __forceinline__ float capped(float y, float cap_out) {
  constexpr float kTanhRatio[6] = {9.999994040e-01f, -3.332909346e-01f, 1.328188479e-01f,
                                   -5.161965266e-02f, 1.676048711e-02f, -3.074449487e-03f};
  const float z = y * y;
  float p = kTanhRatio[5];
#pragma unroll
  for (int i = 4; i >= 0; --i) p = fmaf(p, z, kTanhRatio[i]);
  const float e = fast_exp2(2.0f * kLog2e * fabsf(y));  // (infinity ends at 1)
  const float far = copysignf(1.0f - 2.0f * fast_rcp(1.0f + e), y);
  return cap_out * (z <= 1.0f ? p * y : far);
}

// Output columns col ... col + N - 1 (N = 2 or 4) of the row that starts at `base`.
template <int N>
__device__ __forceinline__ void write_out(const PagedArgs& a, long long base, int col, const float (&x)[N]) {
  if (a.out_f32) {
    float* d = static_cast<float*>(a.out) + base + col;
    if (N == 4 && a.out_vec == 2) {
      *reinterpret_cast<float4*>(d) = make_float4(x[0], x[1], x[N - 2], x[N - 1]);
    } else if (N == 2 && a.out_vec) {
      *reinterpret_cast<float2*>(d) = make_float2(x[0], x[1]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) d[i] = x[i];
    }
  } else {
    __nv_bfloat16* d = static_cast<__nv_bfloat16*>(a.out) + base + col;
    if (N == 4 && a.out_vec == 2) {
      *reinterpret_cast<uint2*>(d) = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[N - 2], x[N - 1]));
    } else if (N == 2 && a.out_vec) {
      *reinterpret_cast<uint32_t*>(d) = pack_bf16x2(x[0], x[1]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) d[i] = __float2bfloat16_rn(x[i]);
    }
  }
}
__device__ __forceinline__ long long out_row(const PagedArgs& a, int b, int kvh, int r) {
  const int i = r / a.G, h = kvh * a.G + (r - i * a.G);
  return (long long)b * a.o_sb + (long long)i * a.o_ss + (long long)h * a.o_sh;
}

// A part of an item's keys that a worker is done with, or nothing (b < 0).
struct Part {
  int b, rest;
  int rem;            // tiles of the item behind it
  uint8_t begins, ends, in_ring;  // holds the item's first tile, its last; where its O rows are
};

template <int DP, int WR, bool MODS>
__global__ void __launch_bounds__(kWarps * 32, 1) attention_paged_kernel(const PagedArgs a) {
  using L = PagedLayout<DP, WR>;
  constexpr int KT = L::kTile, H = L::kHalves, NW = L::kWorkers, ROWS = 16 * WR;
  constexpr int kKeys = KT <= 32 ? 1 : 2;  // keys of a tile a lane looks up
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long s_off[kWarps][KT][2];      // where the keys and values of the tile in issue are; < 0: nowhere
  __shared__ uint32_t s_valid[kWarps][H][kKeys];  // which of a tile's keys are there, as each warp found
  __shared__ Part s_part[NW][2];                  // parts to join: of the item a share continues, of the one it begins
  __shared__ float2 s_ml[NW][2][ROWS];
  const int lane = int(threadIdx.x) & 31, warp = int(threadIdx.x) >> 5;
  const int role = warp % WR, wk = warp / WR;  // this warp's 16 rows of its worker's
  uint8_t* const ring = smem + wk * L::kRing;
  const uint32_t ring_at = smem_u32(ring);
  const auto worker_sync = [&]() {
    if constexpr (WR == 1) {
      __syncwarp();
    } else {
      named_barrier_sync(1 + wk, WR * 32);
    }
  };
  if (role == 0 && lane < 2) s_part[wk][lane].b = -1;
  __syncwarp();
  pdl_wait();
  pdl_launch_dependents();

  // ---- the block's run: an equal share of all tiles, and the worker's of it
  const long long per_tile = (long long)a.Hk * a.row_tiles;
  const auto scan = [&](int c, int& mine) {  // tiles of sequence c + lane, and of all from c up to it (below 2^31)
    mine = c + lane < a.B ? tiles_of<KT>(sequence_len(a, c + lane)) : 0;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    return upto;
  };
  int mine;
  int upto = scan(0, mine);
  long long total = __shfl_sync(0xffffffffu, upto, 31);
  if (a.B > 32) {
    long long more = 0;
    for (int b = 32 + lane; b < a.B; b += 32) more += tiles_of<KT>(sequence_len(a, b));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) more += __shfl_xor_sync(0xffffffffu, more, o);
    total += more;
  }
  total *= per_tile;
  const long long span = max(divide(total + gridDim.x - 1, gridDim.x), (long long)a.min_span);
  const long long c0 = blockIdx.x * span, run = max(0ll, min(total, c0 + span) - c0);
  const long long u0 = c0 + run * wk / NW, u1 = c0 + run * (wk + 1) / NW;
  if (u0 < u1) {
    Cursor<KT> at;
    long long base = 0;
    for (int c = 0;;) {
      const unsigned hit = __ballot_sync(0xffffffffu, base + upto * per_tile > u0);
      if (hit != 0) {
        const int f = __ffs(int(hit)) - 1;
        at.b = c + f;
        base += __shfl_sync(0xffffffffu, upto - mine, f) * per_tile;
        break;
      }
      base += __shfl_sync(0xffffffffu, upto, 31) * per_tile;
      c += 32;
      upto = scan(c, mine);
    }
    const int tiles0 = tiles_of<KT>(sequence_len(a, at.b));
    at.rest = int(divide(u0 - base, tiles0));
    at.enter(a, ROWS, int((u0 - base) - (long long)at.rest * tiles0), u1 - u0);

    // ---- the loader, H - 1 halves ahead: each lane looks up the page of a key, the warps of a worker copy a share each
    struct Ahead {
      int page[kKeys];
      int t, kvh;  // t < 0: behind the last tile
    };
    Cursor<KT> ld = at;
    int ld_end = ld.visible_end();
    const auto seek = [&]() {  // to the next tile with keys, if any
      while (ld.t >= ld_end) {
        if (!ld.next(a, ROWS)) {
          ld_end = INT32_MAX;
          ld.t = -1;
          return;
        }
        ld_end = ld.visible_end();
      }
    };
    const auto peek = [&](Ahead& x) {  // takes that tile and has its pages looked up
      x.t = ld.t;
      if (x.t < 0) return;
      x.kvh = ld.rest / a.row_tiles;
#pragma unroll
      for (int y = 0; y < kKeys; ++y) {
        const int key = lane + 32 * y, j = x.t * KT + key;
        x.page[y] = key < KT && j < ld.seen ? a.table[ld.b * a.table_stride + j / a.page_size] : -1;
      }
      ++ld.t;
      seek();
    };
    constexpr int kChunks = DP / 8;  // 16-byte pieces of a row
    int in = 0;                      // the half of the ring that the next copy goes to
    const auto copy_half = [&](const Ahead& x, int which) {
      if (x.t >= 0) {
        const __nv_bfloat16* src = which ? a.v + x.kvh * a.v_sh : a.k + x.kvh * a.k_sh;
        const uint32_t dst = ring_at + in * L::kHalf;
#pragma unroll
        for (int i = 0; i < KT * kChunks / (32 * WR); ++i) {
          const int idx = (i * WR + role) * 32 + lane, row = idx / kChunks, c = idx - row * kChunks;
          const long long o = s_off[warp][row][which];
          const bool ok = o >= 0 && c * 8 < a.D;
          copy16(dst + row * L::kRow + c * 16, src + (ok ? o + c * 8 : 0), ok);
        }
        in = in + 1 == H ? 0 : in + 1;
      }
      copy_commit();  // (an empty group behind the last tile: the waits count groups)
    };
    const auto issue_k = [&](const Ahead& x) {
      if (x.t >= 0) {
        __syncwarp();  // the table's last reads
#pragma unroll
        for (int y = 0; y < kKeys; ++y) {
          const int key = lane + 32 * y, slot = (x.t * KT + key) % a.page_size;
          const bool ok = x.page[y] >= 0 && x.page[y] < a.pages;
          const uint32_t valid = __ballot_sync(0xffffffffu, ok);
          if (lane == 0) s_valid[warp][in][y] = valid;
          if (key < KT) {
            s_off[warp][key][0] = ok ? x.page[y] * a.k_sp + slot * a.k_ss : -1;
            s_off[warp][key][1] = ok ? x.page[y] * a.v_sp + slot * a.v_ss : -1;
          }
        }
        __syncwarp();
      }
      copy_half(x, 0);
    };
    const auto issue_v = [&](const Ahead& x) { copy_half(x, 1); };

    Ahead next;
    {
      Ahead pre[(H - 1) / 2];  // all look-ups of the start in flight together
      seek();
#pragma unroll
      for (int i = 0; i < (H - 1) / 2; ++i) peek(pre[i]);
      peek(next);
#pragma unroll
      for (int i = 0; i < (H - 1) / 2; ++i) {
        issue_k(pre[i]);
        issue_v(pre[i]);
      }
      if constexpr (H % 2 == 0) issue_k(next);
    }
    // The half that is loaded where the keys of a tile (the values) have been waited for: H - 1 behind them.
    const auto issue_at_keys = [&]() {
      if constexpr (H % 2 == 1) {
        issue_k(next);
      } else {
        issue_v(next);
        peek(next);
      }
    };
    const auto issue_at_values = [&]() {
      if constexpr (H % 2 == 1) {
        issue_v(next);
        peek(next);
      } else {
        issue_k(next);
      }
    };

    // ---- the items of the share
    const int g = lane >> 2, c2 = (lane & 3) * 2;
    int out_half = 0;  // the half of the ring that is used next
    do {
      const int kvh = at.rest / a.row_tiles, r0 = (at.rest % a.row_tiles) * ROWS + role * 16;
      int lim[2];
      long long p[2];
      float slope[2];
      uint32_t qf[DP / 16][4];
      {
        const __nv_bfloat16* qp[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int r = r0 + g + 8 * x;
          const bool ok = r < a.rows;
          const int i = ok ? r / a.G : 0, h = kvh * a.G + (ok ? r - i * a.G : 0);
          p[x] = at.seq.p0 + i;
          lim[x] = ok ? keys_seen(a, at.seq.len, p[x]) : at.seq.len;
          slope[x] = MODS && a.slopes != nullptr ? a.slopes[h] * kLog2e : 0.0f;
          qp[x] = ok ? a.q + ((long long)at.b * a.q_sb + (long long)i * a.q_ss + (long long)h * a.q_sh + c2) : nullptr;
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
        // S = Q K^T, 8 keys a block of x
        copy_wait<H - 2>();
        worker_sync();  // the tile's keys are there, whoever copied them, and all are done with the half before
        uint32_t valid[kKeys];
#pragma unroll
        for (int y = 0; y < kKeys; ++y) valid[y] = s_valid[warp][out_half][y];
        issue_at_keys();
        float x[KT / 8][4];
#pragma unroll
        for (int n = 0; n < KT / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[n][e] = 0.0f;
        {
          const uint32_t ka = ring_at + out_half * L::kHalf + ((lane & 7) + ((lane >> 4) & 1) * 8) * L::kRow + ((lane >> 3) & 1) * 16;
#pragma unroll
          for (int s = 0; s < DP / 16; ++s)
#pragma unroll
            for (int n = 0; n < KT / 16; ++n) {
              uint32_t kf[4];
              ldmatrix_x4(ka + n * 16 * L::kRow + s * 32, kf);
              mma_bf16(x[2 * n], qf[s], kf[0], kf[1]);
              mma_bf16(x[2 * n + 1], qf[s], kf[2], kf[3]);
            }
        }
        out_half = out_half + 1 == H ? 0 : out_half + 1;
        const int j0 = t * KT;
#pragma unroll
        for (int n = 0; n < KT / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (MODS) {
              x[n][e] = a.cap_out != 0.0f ? capped(x[n][e] * a.cap_in, a.cap_out) : x[n][e] * a.scale_log2;
              if (a.slopes != nullptr) {
                const long long j = j0 + n * 8 + c2 + (e & 1);
                x[n][e] = fmaf(-slope[e >> 1], fabsf(float(p[e >> 1] - j)), x[n][e]);
              }
            } else {
              x[n][e] *= a.scale_log2;
            }
          }
        bool all = j0 + KT <= lim_min;
#pragma unroll
        for (int y = 0; y < kKeys; ++y) all = all && valid[y] == (KT < 32 ? (1u << (KT & 31)) - 1u : 0xffffffffu);
        if (!all) {
#pragma unroll
          for (int n = 0; n < KT / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int j = n * 8 + c2 + (e & 1);
              if (j0 + j >= lim[e >> 1] || ((valid[n / 4] >> (j & 31)) & 1u) == 0) x[n][e] = -INFINITY;
            }
        }
        float top[2];
        bool moved = false;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          top[r] = fmaxf(x[0][2 * r], x[0][2 * r + 1]);
#pragma unroll
          for (int n = 1; n < KT / 8; ++n) top[r] = fmax3(top[r], x[n][2 * r], x[n][2 * r + 1]);
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
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float mu = m[r] == -INFINITY ? 0.0f : m[r];  // nothing seen yet: every weight is 0
#pragma unroll
          for (int n = 0; n < KT / 8; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              x[n][2 * r + e] = fast_exp2(x[n][2 * r + e] - mu);
              l[r] += x[n][2 * r + e];
            }
        }
        // O += P V; P rounded to bf16 for the tensor core, 2^-8 relative at most, the sum takes the unrounded weights
        copy_wait<H - 2>();
        worker_sync();
        issue_at_values();
        const uint32_t va = ring_at + out_half * L::kHalf + ((lane & 7) + ((lane >> 3) & 1) * 8) * L::kRow + ((lane >> 4) & 1) * 16;
#pragma unroll
        for (int n = 0; n < KT / 16; ++n) {
          const uint32_t pf[4] = {pack_bf16x2(x[2 * n][0], x[2 * n][1]), pack_bf16x2(x[2 * n][2], x[2 * n][3]),
                                  pack_bf16x2(x[2 * n + 1][0], x[2 * n + 1][1]),
                                  pack_bf16x2(x[2 * n + 1][2], x[2 * n + 1][3])};
#pragma unroll
          for (int c = 0; c < DP / 16; ++c) {
            uint32_t vf[4];
            ldmatrix_x4_trans(va + n * 16 * L::kRow + c * 32, vf);
            mma_bf16(o[2 * c], pf, vf[0], vf[1]);
            mma_bf16(o[2 * c + 1], pf, vf[2], vf[3]);
          }
        }
        out_half = out_half + 1 == H ? 0 : out_half + 1;
      }

      // ---- the item's rows, or the share's part of them
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      }
      const bool begins = first == 0, ends = at.t1 == at.tiles, last = at.left <= 0;
      if (begins && ends) {
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int r = r0 + g + 8 * y;
          if (r >= a.rows) continue;
          const float inv = l[y] == 0.0f ? 0.0f : 1.0f / l[y];  // (a NaN sum makes the row NaN)
          const long long row = out_row(a, at.b, kvh, r);
#pragma unroll
          for (int n = 0; n < DP / 8; ++n) {
            if (n * 8 >= a.D) break;
            write_out<2>(a, row, n * 8 + c2, {o[n][2 * y] * inv, o[n][2 * y + 1] * inv});
          }
        }
        if (a.rec_items && role == 0 && lane == 0)
          a.rec[at.b * (a.Hk * a.row_tiles) + at.rest] = make_int4(0, 0, 0, 0);
      } else {
        // The share's last part waits in the ring, which nobody needs any more; the end of an item before it does not.
        if (last) worker_sync();
        float* const dst = last ? reinterpret_cast<float*>(ring)
                                : a.head_o + ((long long)blockIdx.x * NW + wk) * a.slot_rows * a.D;
        const int ld_o = last ? DP + 8 : a.D;
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int r = role * 16 + g + 8 * y;
          if (r >= a.slot_rows) continue;
          if (c2 == 0) s_ml[wk][begins][r] = make_float2(m[y], l[y]);
#pragma unroll
          for (int n = 0; n < DP / 8; ++n) {
            if (n * 8 >= a.D) break;
            *reinterpret_cast<float2*>(dst + (long long)r * ld_o + n * 8 + c2) = make_float2(o[n][2 * y], o[n][2 * y + 1]);
          }
        }
        if (role == 0 && lane == 0)
          s_part[wk][begins] = Part{at.b, at.rest, at.tiles - at.t1, uint8_t(begins), uint8_t(ends), uint8_t(last)};
      }
    } while (at.next(a, ROWS));
  }
  __syncthreads();

  // ---- the block's parts, in order of keys: chains of one item each, joined here; what goes on in another block, or came
  // from one, is a part of the block's
  const Part mine_p = lane < 2 * NW ? s_part[lane >> 1][lane & 1] : Part{-1, 0, 0, 0, 0, 0};
  const uint32_t present = __ballot_sync(0xffffffffu, mine_p.b >= 0);
  const uint32_t starts = (__ballot_sync(0xffffffffu, mine_p.begins) & present) | (present & (0u - present));
  const int chains = __popc(starts), units = a.slot_rows * (a.D / 4);
  for (int i = int(threadIdx.x); i < chains * units; i += kWarps * 32) {
    int c = i / units;
    const int u = i - c * units, r = u / (a.D / 4), col = (u - r * (a.D / 4)) * 4;
    uint32_t rest = starts;
    for (; c > 0; --c) rest &= rest - 1;
    const int z0 = __ffs(int(rest)) - 1;
    rest &= rest - 1;
    const int z1 = rest != 0 ? __ffs(int(rest)) - 1 : 32;  // the chain's parts are those present in [z0, z1)
    const uint32_t parts = present & (0xffffffffu << z0) & (z1 < 32 ? (1u << z1) - 1u : 0xffffffffu);
    const Part head = s_part[z0 >> 1][z0 & 1];
    const int zl = 31 - __clz(int(parts));
    const Part tail = s_part[zl >> 1][zl & 1];
    float top = -INFINITY;
    for (uint32_t w = parts; w != 0; w &= w - 1) {
      const int z = __ffs(int(w)) - 1;
      top = fmaxf(top, s_ml[z >> 1][z & 1][r].x);
    }
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sum = 0.0f;
    for (uint32_t w = parts; w != 0; w &= w - 1) {
      const int z = __ffs(int(w)) - 1;
      const float2 ml = s_ml[z >> 1][z & 1][r];
      const float wt = ml.x == -INFINITY ? 0.0f : fast_exp2(ml.x - top);
      sum = fmaf(wt, ml.y, sum);
      const float4 v = s_part[z >> 1][z & 1].in_ring
                           ? *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem + (z >> 1) * L::kRing) +
                                                              r * (DP + 8) + col)
                           : *reinterpret_cast<const float4*>(
                                 a.head_o + (((long long)blockIdx.x * NW + (z >> 1)) * a.slot_rows + r) * a.D + col);
      acc[0] = fmaf(wt, v.x, acc[0]);
      acc[1] = fmaf(wt, v.y, acc[1]);
      acc[2] = fmaf(wt, v.z, acc[2]);
      acc[3] = fmaf(wt, v.w, acc[3]);
    }
    const int kvh = head.rest / a.row_tiles, row = (head.rest % a.row_tiles) * ROWS + r;
    if (row < a.rows) {
      if (head.begins && tail.ends) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        write_out<4>(a, out_row(a, head.b, kvh, row), col, {acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv});
      } else {
        const long long part = ((long long)blockIdx.x * 2 + head.begins) * a.slot_rows + r;
        if (col == 0) a.part_ml[part] = make_float2(top, sum);
        *reinterpret_cast<float4*>(a.part_o + part * a.D + col) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      }
    }
    if (u == 0 && head.begins) {
      const int4 mine_rec =
          tail.ends ? make_int4(0, 0, 0, 0)
                    : make_int4(head.b, head.rest, int(divide(c0 + run + tail.rem - 1, span)) - int(blockIdx.x) + 1,
                                int(blockIdx.x));
      if (a.rec_items)
        a.rec[head.b * (a.Hk * a.row_tiles) + head.rest] = mine_rec;
      else if (!tail.ends)
        a.rec[blockIdx.x] = mine_rec;
    }
  }
  // The block begins no item that goes on behind it: its record says so.
  if (!a.rec_items && threadIdx.x == 0) {
    const int zl = present != 0 ? 31 - __clz(int(present)) : 0;
    const Part tail = s_part[zl >> 1][zl & 1];
    const uint32_t z0 = starts != 0 ? 31 - __clz(int(starts)) : 0;  // the last chain's first part
    if (present == 0 || tail.ends || !s_part[z0 >> 1][z0 & 1].begins) a.rec[blockIdx.x] = make_int4(0, 0, 0, 0);
  }
}

// Joins the parts of the item of record blockIdx.x. Eight warps take the parts in turn, a lane 4 (8 above 128) columns.
__global__ void __launch_bounds__(kJoinWarps * 32) attention_paged_join_kernel(const PagedArgs a, int row_tile) {
  __shared__ float s_acc[kJoinWarps][256];
  __shared__ float s_inv;
  const int lane = int(threadIdx.x) & 31, warp = int(threadIdx.x) >> 5;
  pdl_wait();
  pdl_launch_dependents();
  const int4 rec = a.rec[blockIdx.x];
  const int parts = rec.z, blk = rec.w;
  if (parts == 0) return;
  const int kvh = rec.y / a.row_tiles, r0 = (rec.y % a.row_tiles) * row_tile;
  const int rows = min(a.rows - r0, row_tile);
  const auto part_row = [&](int z) { return ((long long)(blk + z) * 2 + (z == 0)) * a.slot_rows; };
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
      const long long at = out_row(a, rec.x, kvh, r0 + row) + col;
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
  int wr, blocks;
  int64_t rows, row_tiles, slot_rows;
  size_t ml_offset, o_offset, head_offset, bytes;
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
  // The scores of 64 keys next to O and Q of more than 128 columns do not fit a thread's registers.
  p.wr = p.rows <= 16 ? 1 : p.rows <= 32 || D > 128 ? 2 : 4;
  p.row_tiles = (p.rows + 16 * p.wr - 1) / (16 * p.wr);
  p.slot_rows = p.rows < 16 * p.wr ? p.rows : 16 * p.wr;
  p.blocks = sms;
  const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  const size_t row = size_t(p.slot_rows) * size_t(D) * sizeof(float);
  p.ml_offset = up(size_t(p.blocks) * sizeof(int4));
  p.o_offset = up(p.ml_offset + size_t(p.blocks) * 2 * size_t(p.slot_rows) * sizeof(float2));
  p.head_offset = up(p.o_offset + size_t(p.blocks) * 2 * row);
  p.bytes = p.head_offset + size_t(p.blocks) * (kWarps / p.wr) * row;
  return p;
}

template <int DP, int WR, bool MODS>
int launch_paged(const PagedArgs& a, int blocks, cudaStream_t stream, int device) {
  using L = PagedLayout<DP, WR>;
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
  if constexpr (WR <= 2) {
    if (a.D <= 160) return launch_paged<160, WR, MODS>(a, blocks, stream, device);
    if (a.D <= 192) return launch_paged<192, WR, MODS>(a, blocks, stream, device);
    return launch_paged<256, WR, MODS>(a, blocks, stream, device);
  }
  return fail(kErrUnsupported, "paged attention: no kernel for these rows");  // (plan_paged asks for none)
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
  const uintptr_t out_align = reinterpret_cast<uintptr_t>(p.out) | uintptr_t(p.o_sb * esize) | uintptr_t(p.o_ss * esize) |
                              uintptr_t(p.o_sh * esize);
  a.out_vec = out_align % uintptr_t(4 * esize) == 0 ? 2 : out_align % uintptr_t(2 * esize) == 0 ? 1 : 0;
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
  a.rows = int(plan.rows);
  a.row_tiles = int(plan.row_tiles);
  a.slot_rows = int(plan.slot_rows);
  a.min_span = p.variant > 0 ? p.variant : 8;
  const int64_t items = p.batch * c.kv_heads * plan.row_tiles;
  a.rec_items = items <= plan.blocks;
  uint8_t* ws = static_cast<uint8_t*>(p.workspace);
  a.rec = reinterpret_cast<int4*>(ws);
  a.part_ml = reinterpret_cast<float2*>(ws + plan.ml_offset);
  a.part_o = reinterpret_cast<float*>(ws + plan.o_offset);
  a.head_o = reinterpret_cast<float*>(ws + plan.head_offset);
  const bool mods = p.softcap > 0.0f || p.slopes != nullptr;
  if (int rc = mods ? launch_paged_for<true>(a, plan.wr, plan.blocks, stream, dev->device)
                    : launch_paged_for<false>(a, plan.wr, plan.blocks, stream, dev->device))
    return rc;
  // A block joins one row of an item, or all of them when there are items enough to fill the GPU.
  const int64_t split = items >= dev->sms ? 1 : plan.slot_rows;
  return check_cuda(launch_pdl(attention_paged_join_kernel, dim3(unsigned(std::min<int64_t>(items, plan.blocks)), unsigned(split)),
                               dim3(kJoinWarps * 32), 0, stream, a, 16 * plan.wr),
                    "paged attention join kernel launch");
}

}  // namespace npub200
