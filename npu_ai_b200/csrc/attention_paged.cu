// attention_paged.cu - attention of a few new tokens of each sequence over a key/value cache in pages.
//
//   o_i = sum_j softmax_j(s_ij) v_j over the keys j that row i sees; s_ij = scale q_i . k_j, then the cap, then the bias.
//
// One pass over the keys with the running maximum and sum of the softmax: for a tile of keys with row maximum t,
//   m' = max(m, t), l' = l 2^(m - m') + sum_j 2^(s_j - m'), o' = o 2^(m - m') + sum_j 2^(s_j - m') v_j,
// and parts (m, l, o) of one row's keys join the same way. Scores are kept in log2 units.
//
// Bound by memory: each element of a key or value is read once and takes part in 2 G flops, a multiplication and an addition for
// each of the G query heads of its head, far below what the tensor cores need to be busy. So the design is about loads in
// flight, few instructions a key and an even split:
//   * Keys are the rows of the matrix instructions: S^T = K Q^T and O^T = V^T P^T with mma.sync m16n8k16, 16 keys (16
//     columns of the head) against 8 rows of queries. The rows of a (sequence, key/value head) are its G heads x the new
//     tokens, mostly 8 or fewer, so nothing is padded to the 64 or 128 rows of a tcgen05 tile, and the softmax of a tile
//     stays in one warp's registers without round trips through TMEM and shared memory. More rows share the keys of one
//     load among the 2 or 4 warps of a worker.
//   * Every block takes an equal run of tiles of the whole batch, found on the device from kv_lens, so ragged lengths leave
//     no SM idle and a captured graph follows them, and its workers equal shares of it. Shares start and end anywhere in a
//     sequence; the parts of a row's keys are joined in order of keys, first those of a block through its shared memory,
//     then those of several blocks through the workspace by the join kernel. What is left: 24 of the 148 SMs are done with equal
//     runs 9% after the others (16 x 16384 keys: after 123 to 125 us, the median 114, by globaltimer stamps of each block;
//     in a plain read of as many bytes the same SMs are not behind).
//   * Pages of a multiple of 16 slots are read by TMA, a box of 64 columns x 16 (32) slots a copy; other pages and layouts
//     that a tensor map does not take by cp.async, 16 bytes a lane, which costs as many instructions as all the arithmetic.
//     (A bulk copy a row was the first form: the copy engine takes one in about 17 cycles, 16 bytes a cycle at 128 columns
//     where 23 are the memory's rate.) Keys and values wait in one ring, a half tile each, swizzled in 128-byte rows, which
//     ldmatrix reads without a bank conflict.
// Measured (GPU time of a call with its join, a graph of calls): one token, 16 x 32/8 heads x 16384 keys (ragged) x 128 134 us,
// 6.1 TB/s, 94% of the measured copy rate; 1 x 131071 keys 94 us, 5.7 TB/s; 777 keys x 64 8.6 us: launches, the run from
// kv_lens, the page table, the first keys and the join's records after each other.
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <cstring>
#include <type_traits>

#include "attention_sm100.cuh"
#include "fast_div.cuh"
#include "internal.h"
#include "paged_split.cuh"

namespace npub200 {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWarps = 4;  // of a block that use the tiles
constexpr int kLoadWarps = 2;  // that load them by TMA: each the half of the workers
// On an SM; the grid is as many as are resident (three times as many took 15% longer at 131072 keys).
constexpr int kBlocks = 2;
constexpr int kMaxHalves = 8;  // of a ring
constexpr int kJoinWarps = 8;
constexpr int kJoinMaxRecs = 1024;  // blocks whose records the join kernel looks through
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
  MapPos pk, pv;  // where the slot, head and page are among the coordinates of the tensor maps
  int box_rows;   // slots of a box: a whole tile's where the page is a multiple of it, else 16
  const int32_t* table;
  long long table_stride;
  int pages, page_size, capacity;
  Divisor by_page;
  const int32_t* lens;
  const int32_t* q_starts;
  void* out;
  long long o_sb, o_ss, o_sh;
  int out_f32, out_vec;  // out_vec: four output columns may be written together
  int B, Hk, G, Sq, D;
  Divisor by_g;
  int causal;
  float scale_log2;       // scores to log2 units
  float cap_in, cap_out;  // softcap: cap_out tanh(cap_in q.k), cap_out 0: none
  const float* slopes;
  int rows, row_tiles, slot_rows;  // rows of a (sequence, kv head), tiles of a worker's rows, rows of a part
  Divisor by_row_tiles, by_slot_rows;
  int min_span, round_span;  // least tiles of a block's run; 1: a whole number of them for each worker
  Divisor by_blocks;
  // What there is to join: of the item that begins in each block's run and goes on behind it. (sequence, kv head and row
  // tile, parts or 0, -)
  int4* rec;
  float2* part_ml;  // [2 blocks][slot_rows] (m, l); part 0 of a block continues an item, part 1 begins one
  float* part_o;    // [2 blocks][slot_rows][D]
  float* head_o;    // [blocks][workers][slot_rows][D] O of the items that end within a worker's share
  KernelCtl ctl;
};

// Four 8 x 8 matrices, a row of one at each lane's address.
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
// An 8 x 8 matrix of two-byte values across the warp, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
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
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0));
}
// Arrives on the barrier when this thread's copies so far are there.
__device__ __forceinline__ void copy_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void copy_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Layout for head dims up to DP, workers of WR warps and NB blocks of 8 rows a warp.
template <int DP, int WR, int NB>
struct PagedLayout {
  static constexpr int kAtoms = (DP + 63) / 64;           // 128-byte columns of a row
  static constexpr int kTile = DP <= 128 ? 32 : 16;       // keys of a tile
  static constexpr int kAtom = kTile * 128;               // bytes of one column of the keys (values) of a tile
  static constexpr int kHalf = kAtoms * kAtom;
  static constexpr int kWorkers = kWarps / WR;
  static constexpr int kRows = 8 * NB * WR;
  // As many as half an SM holds next to the static tables: 96 KB a block (64 KB with one worker), of which each worker uses one
  // half while the others are on their way: 112 to 160 KB in flight on the SM, where some 40 KB cover the latency at the
  // full rate.
  static constexpr int kFit = 104 * 1024 / (kWorkers * kHalf);
  static constexpr int kHalves = kFit < kMaxHalves ? kFit : kMaxHalves;
  static constexpr int kRing = kHalves * kHalf;
  static constexpr int kSmem = kWorkers * kRing + 1024;   // (the swizzle wants 1024-byte boundaries)
  // The ring takes the O rows of the share's last part, 4 floats longer so that their stores spread over the banks.
  static_assert(kHalves >= 3 && kRing >= kRows * (DP + 4) * 4, "ring");
};

// The keys of a sequence.
struct Sequence {
  int len;       // valid keys
  long long p0;  // position of query 0
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
    const int last = min(a.rows, (rest - a.by_row_tiles(rest) * a.row_tiles + 1) * row_tile) - 1;
    seen = keys_seen(a, seq.len, seq.p0 + a.by_g(last));
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

// tanh(y) for |y| <= 1: y times a polynomial in y^2 (fit_tanh_poly.py beside this file; relative error 7e-7), which keeps small
// values' relative accuracy; and for any y, by e^2y above 1.
__device__ __forceinline__ float tanh_small(float y) {
  constexpr float kTanhRatio[6] = {9.999994040e-01f, -3.332909346e-01f, 1.328188479e-01f,
                                   -5.161965266e-02f, 1.676048711e-02f, -3.074449487e-03f};
  const float z = y * y;
  float p = kTanhRatio[5];
#pragma unroll
  for (int i = 4; i >= 0; --i) p = fmaf(p, z, kTanhRatio[i]);
  return p * y;
}
__device__ __forceinline__ float tanh_any(float y) {
  const float e = fast_exp2(2.0f * kLog2e * fabsf(y));  // (infinity ends at 1)
  const float far = copysignf(1.0f - 2.0f * fast_rcp(1.0f + e), y);
  return fabsf(y) <= 1.0f ? tanh_small(y) : far;
}

__device__ __forceinline__ long long out_row(const PagedArgs& a, int b, int kvh, int r) {
  const int i = a.by_g(r), h = kvh * a.G + (r - i * a.G);
  return (long long)b * a.o_sb + (long long)i * a.o_ss + (long long)h * a.o_sh;
}
__device__ __forceinline__ void write_out(const PagedArgs& a, long long at, float x) {
  if (a.out_f32)
    static_cast<float*>(a.out)[at] = x;
  else
    static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(x);
}
__device__ __forceinline__ void write_out4(const PagedArgs& a, long long at, const float (&x)[4]) {
  if (!a.out_vec) {
#pragma unroll
    for (int i = 0; i < 4; ++i) write_out(a, at + i, x[i]);
  } else if (a.out_f32) {
    *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + at) =
        make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
  }
}

// A part of an item's keys that a worker is done with, or nothing (b < 0).
struct Part {
  int b, rest;
  int rem;                        // tiles of the item behind it
  uint8_t begins, ends, in_ring;  // holds the item's first tile, its last; where its O rows are
};

// A worker's share of tiles, as its warps hand it to the one that loads.
struct Share {
  int b, rest, t;
  long long tiles;
};

// The loads of half a block's workers by TMA: a warp, a lane for each worker, H halves ahead of it. Boxes of 64 columns and
// box_rows slots; a page that is not there is outside the map, which reads as zeros. (The warps that use the tiles spent 480
// cycles on each half where they issued the loads themselves, as much as on its arithmetic.)
template <typename L, int WR>
__device__ __forceinline__ void load_pages(const PagedArgs& a, const CUtensorMap* map_k, const CUtensorMap* map_v,
                                           const Share* shares, uint8_t* smem, uint64_t (*full)[L::kHalves],
                                           uint64_t (*empty)[L::kHalves], uint32_t (*valid)[L::kHalves], int* abort) {
  constexpr int KT = L::kTile, H = L::kHalves;
  const int lane = int(threadIdx.x) & 31;
  Cursor<KT> ld = {};
  const int half = int(threadIdx.x) / 32 - kWarps;  // (a box takes a lane some 80 cycles, and lanes take turns)
  bool more = lane < L::kWorkers && lane % kLoadWarps == half && shares[lane].tiles > 0;
  int end = 0, t = 0, head = 0, seen = 0, page[KT / 16];
  const auto peek = [&]() {  // takes the next tile with keys, if any, and has its pages looked up
    while (ld.t >= end) {
      if (!ld.next(a, L::kRows)) {
        more = false;
        return;
      }
      end = ld.visible_end();
    }
    t = ld.t++;
    head = a.by_row_tiles(ld.rest);
    seen = ld.seen;
    const int32_t* const row = a.table + ld.b * a.table_stride;
#pragma unroll
    for (int i = 0; i < KT / 16; ++i) page[i] = t * KT + i * 16 < seen ? row[a.by_page(t * KT + i * 16)] : -1;
  };
  if (more) {
    ld.b = shares[lane].b;
    ld.rest = shares[lane].rest;
    ld.enter(a, L::kRows, shares[lane].t, shares[lane].tiles);
    end = ld.visible_end();
    peek();
  }
  int in = 0, in_values = 0, issued = 0;
  uint32_t phase = 0;
  uint64_t since = globaltimer_ns();
  uint32_t polls = 0;
  while (__any_sync(0xffffffffu, more)) {
    const bool ready = more && (issued < H || mbar_test_wait(&empty[lane][in], phase ^ 1u));
    if (ready) {
      uint64_t* const bar = &full[lane][in];
      uint32_t bits = 0;
      int c[KT / 16][3];
      const int slot0 = t * KT - a.by_page(t * KT) * a.page_size;
      const MapPos& pos = in_values ? a.pv : a.pk;
#pragma unroll
      for (int i = 0; i < KT / 16; ++i) {
        const bool ok = page[i] >= 0 && page[i] < a.pages;
        const int n = min(16, seen - t * KT - i * 16);  // (no page was looked up where there is no key)
        bits |= ok ? ((1u << n) - 1u) << (16 * i) : 0u;
        int slot = slot0 + 16 * i;
        slot -= slot >= a.page_size ? a.by_page(slot) * a.page_size : 0;
        const int at = ok ? page[i] : a.pages;
        c[i][0] = pos.s == 1 ? slot : pos.h == 1 ? head : at;
        c[i][1] = pos.s == 2 ? slot : pos.h == 2 ? head : at;
        c[i][2] = pos.s == 3 ? slot : pos.h == 3 ? head : at;
      }
      valid[lane][in] = bits;
      mbar_arrive_expect_tx(bar, L::kHalf);
      uint8_t* const dst = smem + lane * L::kRing + in * L::kHalf;
#pragma unroll
      for (int i = 0; i < KT / 16; ++i)
        if (i % (a.box_rows / 16) == 0)
#pragma unroll
          for (int k = 0; k < L::kAtoms; ++k)
            tma_load_4d(in_values ? map_v : map_k, bar, dst + k * L::kAtom + i * 2048, k * 64, c[i][0], c[i][1], c[i][2]);
      ++issued;
      if (++in == H) {
        in = 0;
        phase ^= 1u;
      }
      if (in_values) peek();
      in_values ^= 1;
    }
    if (__any_sync(0xffffffffu, ready)) {
      polls = 0;
    } else if ((++polls & 63u) == 0) {
      if (polls == 64) since = globaltimer_ns();
      const bool late = globaltimer_ns() - since > a.ctl.timeout_ns;
      if (late && lane == 0) atomicOr(a.ctl.status, kStatusTimeoutProducer);
      if (late) *reinterpret_cast<volatile int*>(abort) = 1;
      if (__any_sync(0xffffffffu, late || *reinterpret_cast<volatile int*>(abort))) break;
    }
  }
  // The copies in flight write to this block's memory: it stays until they are done, whether they are used or not (the others
  // may have given up).
  for (int i = 0; i < min(issued, H); ++i) {
    in = in == 0 ? H - 1 : in - 1;
    phase ^= in == H - 1 ? 1u : 0u;
    mbar_wait_drain(&full[lane][in], phase, a.ctl);
  }
}

template <int DP, int WR, int NB, bool MODS, bool TMA>
__global__ void __launch_bounds__((kWarps + (TMA ? kLoadWarps : 0)) * 32, kBlocks)
    attention_paged_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                           const PagedArgs a) {
  using L = PagedLayout<DP, WR, NB>;
  constexpr int KT = L::kTile, H = L::kHalves, NW = L::kWorkers, ROWS = L::kRows;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t s_full[NW][H], s_empty[NW][H], s_never;
  __shared__ uint32_t s_valid[NW][H];      // which keys of a tile are there
  __shared__ Share s_share[NW];
  __shared__ Part s_part[NW][2];           // parts to join: of the item a share continues, of the one it begins
  __shared__ float2 s_ml[NW][2][ROWS];     // (m, l) of their rows
  __shared__ int s_abort;
  const int lane = int(threadIdx.x) & 31, warp = int(threadIdx.x) >> 5;
  const int role = warp % WR, wk = warp / WR;  // this warp's rows of its worker's
  uint8_t* const smem = smem_raw + ((0u - smem_u32(smem_raw)) & 1023u);
  uint8_t* const ring = smem + wk * L::kRing;
  const uint32_t ring_at = smem_u32(ring);
  if (threadIdx.x < NW * H) {
    // A tile's half is there when its copies are: TMA's bytes, or the copies of each lane, and the word of the lane that
    // says which keys are valid.
    mbar_init(&s_full[0][threadIdx.x], TMA ? 1u : 32u * WR + 1u);
    mbar_init(&s_empty[0][threadIdx.x], WR);
  }
  if (threadIdx.x < 2 * NW) s_part[threadIdx.x >> 1][threadIdx.x & 1].b = -1;
  if (threadIdx.x == 0) {
    s_abort = 0;
    mbar_init(&s_never, 1);
    fence_barrier_init();
  }
  __syncthreads();
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
  long long span = 0, c0 = 0, run = 0;
  if (TMA && warp >= kWarps) {
    __syncthreads();
    load_pages<L, WR>(a, &map_k, &map_v, s_share, smem, s_full, s_empty, s_valid, &s_abort);
  } else {
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
    // Whole tiles for every worker: 7 for four took as long as 8, and there were more parts to join (1 x 8192 keys, 8 heads
    // 15.9 us, 14.4 with 8).
    span = tiles_of_run(total, int(gridDim.x), a.by_blocks, a.min_span, a.round_span ? NW : 1);
    c0 = blockIdx.x * span;
    run = max(0ll, min(total, c0 + span) - c0);
    const long long u0 = c0 + run * wk / NW, u1 = c0 + run * (wk + 1) / NW;
    Cursor<KT> at = {};
    if (u0 < u1) {
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
    }
    if constexpr (TMA) {
      if (role == 0 && lane == 0) s_share[wk] = Share{at.b, at.rest, at.t, u1 - u0};
      __syncthreads();
    }
    if (u0 < u1) {
      // ---- loads by cp.async: H - 1 halves ahead, the warps of a worker a share each. A lane looks up the page of its key.
      Cursor<KT> ld = at;
      int ld_end = ld.visible_end();
      int page = -1, next_t = -1;  // of the tile that goes out next; next_t < 0: behind the last
      int next_head = 0;
      const auto peek = [&]() {    // takes the next tile with keys, if any, and has its pages looked up
        while (ld.t >= ld_end) {
          if (!ld.next(a, ROWS)) {
            next_t = -1;
            return;
          }
          ld_end = ld.visible_end();
        }
        next_t = ld.t++;
        next_head = a.by_row_tiles(ld.rest);
        const int j = next_t * KT + lane;
        page = lane < KT && j < ld.seen ? a.table[ld.b * a.table_stride + a.by_page(j)] : -1;
      };
      int in = 0, in_values = 0;  // the half of the ring that is filled next, with keys or values
      int filled = 0;             // how many are ahead of the one that is used, up to H - 1
      uint32_t in_phase = 0;
      // (Its code stands once: with the fill of the ring written out in front of the loop the start took 2 us more for
      // fetching instructions.)
      const auto issue = [&]() -> bool {
        if (next_t < 0) return true;
        if (WR > 1 && !mbar_wait_bounded_warp(&s_empty[wk][in], in_phase ^ 1u, &s_abort, a.ctl, kStatusTimeoutProducer))
          return false;
        uint64_t* const bar = &s_full[wk][in];
        const bool ok = page >= 0 && page < a.pages;
        const uint32_t valid = __ballot_sync(0xffffffffu, ok);
        if (role == 0 && lane == 0) {
          s_valid[wk][in] = valid;
          mbar_arrive(bar);
        }
        const long long sp = in_values ? a.v_sp : a.k_sp, ss = in_values ? a.v_ss : a.k_ss;
        const __nv_bfloat16* src = in_values ? a.v + next_head * a.v_sh : a.k + next_head * a.k_sh;
        const int j = next_t * KT + lane;
        const long long off = ok ? page * sp + (j - a.by_page(j) * a.page_size) * ss : -1;  // < 0: nowhere
        // Eight lanes a row, four rows a copy, the columns of 64 after each other; of the last 64 only what the head's columns
        // reach, where that is half of them four lanes a row.
        constexpr int kLast = DP % 64 == 32 && KT >= 8 * WR ? 4 : 8, kFull = kLast == 8 ? L::kAtoms : L::kAtoms - 1;
        const uint32_t dst = ring_at + in * L::kHalf;
        const auto copy = [&](auto lanes, int first, int last) {  // lanes a row; columns of 64
          constexpr int N = decltype(lanes)::value, ROWS4 = 32 / N;
          long long o[KT / (ROWS4 * WR)];  // (all of them first: between the copies each would wait for the copy before it)
#pragma unroll
          for (int i = 0; i < KT / (ROWS4 * WR); ++i) o[i] = __shfl_sync(0xffffffffu, off, (i * WR + role) * ROWS4 + lane / N);
#pragma unroll
          for (int i = 0; i < KT / (ROWS4 * WR); ++i) {
            const int row = (i * WR + role) * ROWS4 + lane / N;
            const uint32_t to = dst + row * 128 + (((lane % N) ^ (row & 7)) << 4);
#pragma unroll
            for (int c = first; c < last; ++c) {
              const int col = c * 64 + (lane % N) * 8;
              const bool there = o[i] >= 0 && col < a.D;
              copy16(to + c * L::kAtom, src + (there ? o[i] + col : 0), there);
            }
          }
        };
        copy(std::integral_constant<int, 8>{}, 0, kFull);
        if constexpr (kLast == 4) copy(std::integral_constant<int, 4>{}, kFull, L::kAtoms);
        copy_arrive(bar);
        if (++in == H) {
          in = 0;
          in_phase ^= 1u;
        }
        if (in_values) peek();
        in_values ^= 1;
        return true;
      };
      if constexpr (!TMA) peek();
      bool good = true;
      if (a.ctl.debug & 1u) good = mbar_wait_bounded_warp(&s_never, 0, &s_abort, a.ctl, kStatusForced);

      // ---- the items of the share
      const int g = lane >> 2, c2 = (lane & 3) * 2;
      // ldmatrix: this lane's row of a half, and the four swizzled 16-byte columns that it reads of each 64
      const int k_row = (lane & 7) + ((lane >> 3) & 1) * 8, v_row = (lane & 7) + (lane >> 4) * 8;
      uint32_t k_col[4], v_col[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        k_col[i] = k_row * 128 + (((2 * i + (lane >> 4)) ^ (lane & 7)) << 4);
        v_col[i] = v_row * 128 + (((2 * i + ((lane >> 3) & 1)) ^ (lane & 7)) << 4);
      }
      const float sc = MODS ? 1.0f : a.scale_log2;
      constexpr uint32_t kAll = 0xffffffffu >> (32 - KT);
      int used = 0;  // the half of the ring that is used next
      uint32_t phase = 0;
      while (good) {
        const int kvh = a.by_row_tiles(at.rest), r0 = (at.rest - kvh * a.row_tiles) * ROWS + role * 8 * NB;
        uint32_t qf[DP / 16][NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const int r = r0 + nb * 8 + g;
          const bool ok = r < a.rows;
          const int i = ok ? a.by_g(r) : 0, h = kvh * a.G + (ok ? r - i * a.G : 0);
          const __nv_bfloat16* qp = a.q + ((long long)at.b * a.q_sb + (long long)i * a.q_ss + (long long)h * a.q_sh + c2);
#pragma unroll
          for (int s = 0; s < DP / 16; ++s)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int col = s * 16 + e * 8;
              qf[s][nb][e] = ok && col < a.D ? *reinterpret_cast<const uint32_t*>(qp + col) : 0u;
            }
        }
        // this lane's rows of the scores: c2 and c2 + 1 of each block
        int lim[NB][2], lim_min = INT32_MAX;
        // Of the sequence's positions the one next to the row's: what distances are counted from. (An int would do; the capped
        // form came out slower with it, 64 short caches 52.3 us instead of 51.5.)
        long long near[NB][2];
        float slope[NB][2], m[NB][2], l[NB][2], o[DP / 16][NB][4];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int r = r0 + nb * 8 + c2 + y;
            const bool ok = r < a.rows;
            const int i = ok ? a.by_g(r) : 0;
            const long long p = at.seq.p0 + i;
            lim[nb][y] = ok ? keys_seen(a, at.seq.len, p) : at.seq.len;
            near[nb][y] = max(0ll, min(p, (long long)at.seq.len - 1));
            lim_min = min(lim_min, lim[nb][y]);
            slope[nb][y] = MODS && a.slopes != nullptr ? a.slopes[kvh * a.G + (ok ? r - i * a.G : 0)] * kLog2e : 0.0f;
            m[nb][y] = -INFINITY;
            l[nb][y] = 0.0f;
          }
#pragma unroll
          for (int s = 0; s < DP / 16; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[s][nb][e] = 0.0f;
        }
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) lim_min = min(lim_min, __shfl_xor_sync(0xffffffffu, lim_min, d));

        const int first = at.t, halves = 2 * max(0, at.visible_end() - first);
        uint32_t valid = 0;
        float x[KT / 16][NB][4];
#pragma unroll 1
        for (int half = 0; half < halves && good; ++half) {  // a tile's keys, then its values
          if constexpr (TMA) {
            good = mbar_wait_bounded_warp(&s_full[wk][used], phase, &s_abort, a.ctl, kStatusTimeoutEpilogue);
          } else {
#pragma unroll 1
            for (;;) {
              const bool full = filled == H - 1;
              if (full) {
                good = mbar_wait_bounded_warp(&s_full[wk][used], phase, &s_abort, a.ctl, kStatusTimeoutEpilogue);
                if (!good) break;
              }
              good = issue();
              if (full || !good) break;
              ++filled;
            }
          }
          if (!good) break;
          const uint32_t half_at = ring_at + used * L::kHalf;
          if ((half & 1) == 0) {
            valid = s_valid[wk][used];
            // S^T = K Q^T, 16 keys a block of x; with one block of rows even and odd steps are sums of their own, half the
            // chain of instructions that wait for each other
            float odd[KT / 16][4];
#pragma unroll
            for (int n = 0; n < KT / 16; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                odd[n][e] = 0.0f;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) x[n][nb][e] = 0.0f;
              }
#pragma unroll
            for (int s = 0; s < DP / 16; ++s)
#pragma unroll
              for (int n = 0; n < KT / 16; ++n) {
                uint32_t kf[4];
                ldmatrix_x4(half_at + k_col[s & 3] + (s >> 2) * L::kAtom + n * 2048, kf);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
                  mma_bf16(NB == 1 && (s & 1) ? odd[n] : x[n][nb], kf, qf[s][nb][0], qf[s][nb][1]);
              }
            if constexpr (NB == 1) {
#pragma unroll
              for (int n = 0; n < KT / 16; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[n][0][e] += odd[n][e];
            }
            const int j0 = (first + (half >> 1)) * KT;
            if constexpr (MODS) {
              if (a.cap_out != 0.0f) {
                float big = 0.0f;
#pragma unroll
                for (int n = 0; n < KT / 16; ++n)
#pragma unroll
                  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                      x[n][nb][e] *= a.cap_in;
                      big = max_nan(big, fabsf(x[n][nb][e]));
                    }
                const bool small = __all_sync(0xffffffffu, big <= 1.0f);  // (mostly: the cap is for the rare large score)
#pragma unroll
                for (int n = 0; n < KT / 16; ++n)
#pragma unroll
                  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                      x[n][nb][e] = a.cap_out * (small ? tanh_small(x[n][nb][e]) : tanh_any(x[n][nb][e]));
              } else {
#pragma unroll
                for (int n = 0; n < KT / 16; ++n)
#pragma unroll
                  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[n][nb][e] *= a.scale_log2;
              }
              if (a.slopes != nullptr) {
                // Before the first key and behind the last all distances grow alike, which the softmax does not see: they
                // are counted from the key next to the row, so that they stay below the number of keys (with p itself a row
                // 2^30 past 1000 keys had the same distance, in f32, to 64 of them). Exact up to 2^24 keys, off by half a
                // step of f32 beyond.
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                  for (int y = 0; y < 2; ++y) {
                    const float ahead = float(near[nb][y] - j0 - g);
#pragma unroll
                    for (int n = 0; n < KT / 16; ++n)
#pragma unroll
                      for (int e = 0; e < 4; e += 2)
                        x[n][nb][e + y] = fmaf(-slope[nb][y], fabsf(ahead - float(n * 16 + e * 4)), x[n][nb][e + y]);
                  }
              }
            }
            if (j0 + KT > lim_min || valid != kAll) {
#pragma unroll
              for (int n = 0; n < KT / 16; ++n)
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const int j = n * 16 + g + (e >> 1) * 8;
                    if (j0 + j >= lim[nb][e & 1] || ((valid >> j) & 1u) == 0) x[n][nb][e] = -INFINITY;
                  }
            }
            float top[NB][2];
            bool moved = false;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                top[nb][y] = fmaxf(x[0][nb][y], x[0][nb][2 + y]);
#pragma unroll
                for (int n = 1; n < KT / 16; ++n) top[nb][y] = fmax3(top[nb][y], x[n][nb][y], x[n][nb][2 + y]);
              }
#pragma unroll
            for (int d = 4; d < 32; d <<= 1)
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int y = 0; y < 2; ++y) top[nb][y] = fmaxf(top[nb][y], __shfl_xor_sync(0xffffffffu, top[nb][y], d));
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                top[nb][y] *= sc;
                moved = moved || top[nb][y] > m[nb][y] + kRescale;
              }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                  const float to = top[nb][y] > m[nb][y] + kRescale ? top[nb][y] : m[nb][y];
                  const float f = to == m[nb][y] ? 1.0f : fast_exp2(m[nb][y] - to);
                  m[nb][y] = to;
                  l[nb][y] *= f;
#pragma unroll
                  for (int s = 0; s < DP / 16; ++s) {
                    o[s][nb][y] *= f;
                    o[s][nb][2 + y] *= f;
                  }
                }
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                const float mu = m[nb][y] == -INFINITY ? 0.0f : m[nb][y];  // nothing seen yet: every weight is 0
#pragma unroll
                for (int n = 0; n < KT / 16; ++n)
#pragma unroll
                  for (int e = 0; e < 4; e += 2) {
                    x[n][nb][e + y] = fast_exp2(fmaf(x[n][nb][e + y], sc, -mu));
                    l[nb][y] += x[n][nb][e + y];
                  }
              }
          } else {
            // O^T += V^T P^T; P rounded to bf16 for the tensor core, 2^-8 relative at most, the sum takes the unrounded
            // weights. (The error of a bf16 output against 64 bits, relative to its size, is 0.0023 on long caches, 0.0017 of it
            // the output's own rounding; P in two bf16 parts would need twice the instructions of this product.)
            const bool all = valid == kAll;
#pragma unroll
            for (int n = 0; n < KT / 16; ++n) {
              uint32_t pf[NB][2];
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) {
                pf[nb][0] = transposed(pack_bf16x2(x[n][nb][0], x[n][nb][1]));
                pf[nb][1] = transposed(pack_bf16x2(x[n][nb][2], x[n][nb][3]));
              }
              const uint32_t w = valid >> (n * 16 + c2);
              const uint32_t k0 = (w & 1u ? 0xffffu : 0u) | (w & 2u ? 0xffff0000u : 0u);
              const uint32_t k1 = (w & 0x100u ? 0xffffu : 0u) | (w & 0x200u ? 0xffff0000u : 0u);
#pragma unroll
              for (int s = 0; s < DP / 16; ++s) {
                uint32_t vf[4];
                ldmatrix_x4_trans(half_at + v_col[s & 3] + (s >> 2) * L::kAtom + n * 2048, vf);
                if (!all) {  // slots behind the last key may hold anything: zeros, for 0 times NaN is NaN
                  vf[0] &= k0;
                  vf[1] &= k0;
                  vf[2] &= k1;
                  vf[3] &= k1;
                }
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) mma_bf16(o[s][nb], vf, pf[nb][0], pf[nb][1]);
              }
            }
          }
          __syncwarp();  // all lanes are done with the half
          if ((TMA || WR > 1) && lane == 0) mbar_arrive(&s_empty[wk][used]);
          if (++used == H) {
            used = 0;
            phase ^= 1u;
          }
        }
        if (!good) break;

        // ---- the item's rows, or the share's part of them
#pragma unroll
        for (int d = 4; d < 32; d <<= 1)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int y = 0; y < 2; ++y) l[nb][y] += __shfl_xor_sync(0xffffffffu, l[nb][y], d);
        const bool begins = first == 0, ends = at.t1 == at.tiles, last = at.left <= 0;
        if (begins && ends) {
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const int r = r0 + nb * 8 + c2 + y;
              if (r >= a.rows) continue;
              const float inv = l[nb][y] == 0.0f ? 0.0f : 1.0f / l[nb][y];  // (a NaN sum makes the row NaN)
              const long long row = out_row(a, at.b, kvh, r) + g;
              if (a.out_f32) {
                float* const d = static_cast<float*>(a.out) + row;
#pragma unroll
                for (int s = 0; s < DP / 8; ++s)
                  if (s * 8 < a.D) d[s * 8] = o[s / 2][nb][(s & 1) * 2 + y] * inv;
              } else {
                __nv_bfloat16* const d = static_cast<__nv_bfloat16*>(a.out) + row;
#pragma unroll
                for (int s = 0; s < DP / 8; ++s)
                  if (s * 8 < a.D) d[s * 8] = __float2bfloat16_rn(o[s / 2][nb][(s & 1) * 2 + y] * inv);
              }
            }
        } else {
          // The share's last part waits in the ring, which nobody needs any more; the end of an item before it does not.
          if (WR > 1 && NW > 1 && last) {  // (once the worker's other warps are done with the half used last)
            const int before = used == 0 ? H - 1 : used - 1;
            good = mbar_wait_bounded_warp(&s_empty[wk][before], used == 0 ? phase ^ 1u : phase, &s_abort, a.ctl,
                                          kStatusTimeoutEpilogue);
            if (!good) break;
          }
          // (The only worker's parts are the block's.)
          const long long slot = ((long long)blockIdx.x * 2 + begins) * a.slot_rows;
          float* const dst = NW == 1 ? a.part_o + slot * a.D
                             : last  ? reinterpret_cast<float*>(ring)
                                     : a.head_o + ((long long)blockIdx.x * NW + wk) * a.slot_rows * a.D;
          const int ld_o = NW > 1 && last ? DP + 4 : a.D;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const int r = (role * NB + nb) * 8 + c2 + y;
              if (r >= a.slot_rows) continue;
              if (g == 0) (NW == 1 ? a.part_ml[slot + r] : s_ml[wk][begins][r]) = make_float2(m[nb][y], l[nb][y]);
              float* const row = dst + r * ld_o + g;
#pragma unroll
              for (int s = 0; s < DP / 8; ++s)
                if (s * 8 < a.D) row[s * 8] = o[s / 2][nb][(s & 1) * 2 + y];
            }
          if (role == 0 && lane == 0)
            s_part[wk][begins] = Part{at.b, at.rest, at.tiles - at.t1, uint8_t(begins), uint8_t(ends), uint8_t(last)};
        }
        if (!at.next(a, ROWS)) break;
      }
      if (!TMA && !good) copy_wait_all();  // copies in flight write to this block's memory: it stays until they are done
    }
  }
  __syncthreads();

  // ---- the block's parts, in order of keys: chains of one item each, joined here, a warp a row; what goes on in another
  // block, or came from one, is a part of the block's. (Loops, for the code that runs once is as slow as it is long.)
  constexpr int PARTS = 2 * NW;
  const Part mine_p = lane < PARTS ? s_part[lane / 2][lane & 1] : Part{-1, 0, 0, 0, 0, 0};
  const uint32_t present = s_abort ? 0u : __ballot_sync(0xffffffffu, mine_p.b >= 0);
  const uint32_t begin_bits = __ballot_sync(0xffffffffu, mine_p.begins) & present;
  const uint32_t starts = begin_bits | (present & (0u - present));
  if (warp == 0 && lane == (present != 0 ? 31 - __clz(int(present)) : 0)) {
    // Only the last chain goes on in another block: when it begins here, it is the block's to join.
    const bool joins = present != 0 && !mine_p.ends && ((begin_bits >> (31 - __clz(int(starts)))) & 1u);
    a.rec[blockIdx.x] =
        joins ? make_int4(mine_p.b, mine_p.rest, int(divide(c0 + run + mine_p.rem - 1, span)) - int(blockIdx.x) + 1, 0)
              : make_int4(0, 0, 0, 0);
  }
  if constexpr (NW > 1) {
    if (present == 0 || warp >= kWarps) return;
#pragma unroll 1
    for (int r = warp; r < a.slot_rows; r += kWarps)
#pragma unroll 1
      for (int col = lane * 4; col < a.D; col += 128) {
        float acc[4], top = -INFINITY, sum = 0.0f;
        int begins = 0;
#pragma unroll 1
        for (uint32_t w = present; w != 0; w &= w - 1) {
          const int z = __ffs(int(w)) - 1;
          const Part part = s_part[z / 2][z & 1];
          const float2 ml = s_ml[z / 2][z & 1][r];
          const float* const src = part.in_ring
                                       ? reinterpret_cast<const float*>(smem + (z / 2) * L::kRing) + r * (DP + 4)
                                       : a.head_o + (((long long)blockIdx.x * NW + z / 2) * a.slot_rows + r) * a.D;
          const float4 v = *reinterpret_cast<const float4*>(src + col);
          if ((starts >> z) & 1u) {
            begins = part.begins;
            top = -INFINITY;
            sum = acc[0] = acc[1] = acc[2] = acc[3] = 0.0f;
          }
          const float to = fmaxf(top, ml.x), base = to == -INFINITY ? 0.0f : to;
          const float f0 = fast_exp2(top - base), f1 = fast_exp2(ml.x - base);
          top = to;
          sum = fmaf(f1, ml.y, sum * f0);
          acc[0] = fmaf(f1, v.x, acc[0] * f0);
          acc[1] = fmaf(f1, v.y, acc[1] * f0);
          acc[2] = fmaf(f1, v.z, acc[2] * f0);
          acc[3] = fmaf(f1, v.w, acc[3] * f0);
          const uint32_t behind = w & (w - 1);
          if (behind != 0 && (starts & behind & (0u - behind)) == 0) continue;  // the chain goes on
          const int kvh = a.by_row_tiles(part.rest), row = (part.rest - kvh * a.row_tiles) * ROWS + r;
          if (row >= a.rows) continue;
          if (begins && part.ends) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // (a NaN sum makes the row NaN)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] *= inv;
            write_out4(a, out_row(a, part.b, kvh, row) + col, acc);
          } else {
            const long long at = ((long long)blockIdx.x * 2 + begins) * a.slot_rows + r;
            if (col == 0) a.part_ml[at] = make_float2(top, sum);
            *reinterpret_cast<float4*>(a.part_o + at * a.D + col) = make_float4(acc[0], acc[1], acc[2], acc[3]);
          }
        }
      }
  }
}

// Joins the parts of the items that go on from block to block. WARPS warps share a row, the parts in turn: all eight of a
// block where there are few rows, each with many parts, one where there are many rows. A lane takes 4 (8 above 128) columns.
// A block looks through all records for its rows.
template <int WARPS>
__global__ void __launch_bounds__(kJoinWarps * 32) attention_paged_join_kernel(const PagedArgs a, int recs, int row_tile) {
  __shared__ float s_acc[WARPS > 1 ? WARPS : 1][256];
  __shared__ float s_inv;
  __shared__ int s_list[kJoinMaxRecs], s_count[kJoinWarps];
  const int lane = int(threadIdx.x) & 31, warp = int(threadIdx.x) >> 5;
  pdl_wait();
  pdl_launch_dependents();
  int items = 0;
  for (int i0 = 0; i0 < recs; i0 += kJoinWarps * 32) {  // the records with something to join, in order
    const int i = i0 + int(threadIdx.x);
    const bool some = i < recs && a.rec[i].z != 0;
    const unsigned mask = __ballot_sync(0xffffffffu, some);
    if (lane == 0) s_count[warp] = __popc(mask);
    __syncthreads();
    int before = items;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) {
      before += w < warp ? s_count[w] : 0;
      items += s_count[w];
    }
    if (some) s_list[before + __popc(mask & ((1u << lane) - 1u))] = i;
    __syncthreads();
  }
  constexpr int kTeams = kJoinWarps / WARPS;  // of a block
  for (int task = int(blockIdx.x) * kTeams + warp / WARPS; task < items * a.slot_rows; task += int(gridDim.x) * kTeams) {
    const int item = a.by_slot_rows(task), row = task - item * a.slot_rows;
    const int blk = s_list[item];
    const int4 rec = a.rec[blk];
    const int parts = rec.z;
    const int kvh = a.by_row_tiles(rec.y), r = (rec.y - kvh * a.row_tiles) * row_tile + row;
    if (r >= a.rows) continue;
    const auto part_row = [&](int z) { return ((long long)(blk + z) * 2 + (z == 0)) * a.slot_rows + row; };
    float top = -INFINITY;
    for (int z = lane; z < parts; z += 32) top = fmaxf(top, a.part_ml[part_row(z)].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float sum = 0.0f;
    if (WARPS == 1 || warp == 0) {
      for (int z = lane; z < parts; z += 32) {
        const float2 ml = a.part_ml[part_row(z)];
        sum = fmaf(ml.x == -INFINITY ? 0.0f : fast_exp2(ml.x - top), ml.y, sum);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // (a NaN sum makes the row NaN)
    if (WARPS > 1 && threadIdx.x == 0) s_inv = inv;
    float acc[2][4] = {};
#pragma unroll 4
    for (int z = WARPS == 1 ? 0 : warp; z < parts; z += WARPS) {
      const long long at = part_row(z);
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
    if constexpr (WARPS == 1) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int col = lane * 4 + k * 128;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[k][e] *= inv;
        if (col < a.D) write_out4(a, out_row(a, rec.x, kvh, r) + col, acc[k]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) s_acc[warp][k * 128 + lane * 4 + e] = acc[k][e];
      __syncthreads();
      const int col = int(threadIdx.x);
      if (col < a.D) {
        float x = 0.0f;
#pragma unroll
        for (int k = 0; k < WARPS; ++k) x += s_acc[k][col];
        write_out(a, out_row(a, rec.x, kvh, r) + col, x * s_inv);
      }
      __syncthreads();  // s_acc and s_inv are written again for the next row
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------------------------
struct PagedPlan {
  int wr, nb, blocks;
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
  // Two blocks of rows a warp from 33 rows on, where reading the keys from shared memory for each block decides (4 x 16 tokens,
  // 32/8 heads, 9000 keys: 68 us, 110 with one); above 128 columns their O does not fit the registers. With 20 rows two warps
  // of two blocks took 25 us, four of one 16.
  p.nb = p.rows > 32 && D <= 128 ? 2 : 1;
  p.wr = p.rows <= 8 ? 1 : p.rows <= 16 ? 2 : 4;
  const int64_t tile = 8 * p.nb * p.wr;
  p.row_tiles = (p.rows + tile - 1) / tile;
  p.slot_rows = p.rows < tile ? p.rows : tile;
  p.blocks = sms * kBlocks;
  const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  const size_t row = size_t(p.slot_rows) * size_t(D) * sizeof(float);
  p.ml_offset = up(size_t(p.blocks) * sizeof(int4));
  p.o_offset = up(p.ml_offset + size_t(p.blocks) * 2 * size_t(p.slot_rows) * sizeof(float2));
  p.head_offset = up(p.o_offset + size_t(p.blocks) * 2 * row);
  p.bytes = p.head_offset + size_t(p.blocks) * (kWarps / p.wr) * row;
  return p;
}

template <int DP, int WR, int NB, bool MODS, bool TMA>
int launch_paged(const CUtensorMap& mk, const CUtensorMap& mv, const PagedArgs& a, int blocks, cudaStream_t stream,
                 int device) {
  constexpr int smem = PagedLayout<DP, WR, NB>::kSmem;
  static std::atomic<bool> ready[64] = {};
  if (!ready[device]) {
    if (int rc = check_cuda(cudaFuncSetAttribute(attention_paged_kernel<DP, WR, NB, MODS, TMA>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
                            "paged attention shared memory"))
      return rc;
    ready[device] = true;
  }
  return check_cuda(launch_pdl(attention_paged_kernel<DP, WR, NB, MODS, TMA>, dim3(unsigned(blocks)),
                               dim3((kWarps + (TMA ? kLoadWarps : 0)) * 32), smem, stream, mk, mv, a),
                    "paged attention kernel launch");
}

template <int WR, int NB, bool MODS, bool TMA>
int launch_paged_dim(const CUtensorMap& mk, const CUtensorMap& mv, const PagedArgs& a, int blocks, cudaStream_t stream,
                     int device) {
  if (a.D <= 64) return launch_paged<64, WR, NB, MODS, TMA>(mk, mv, a, blocks, stream, device);
  if (a.D <= 96) return launch_paged<96, WR, NB, MODS, TMA>(mk, mv, a, blocks, stream, device);
  if (a.D <= 128) return launch_paged<128, WR, NB, MODS, TMA>(mk, mv, a, blocks, stream, device);
  if constexpr (NB == 1) {
    if (a.D <= 160) return launch_paged<160, WR, 1, MODS, TMA>(mk, mv, a, blocks, stream, device);
    if (a.D <= 192) return launch_paged<192, WR, 1, MODS, TMA>(mk, mv, a, blocks, stream, device);
    return launch_paged<256, WR, 1, MODS, TMA>(mk, mv, a, blocks, stream, device);
  }
  return fail(kErrUnsupported, "paged attention: no kernel for these rows");  // (plan_paged asks for none)
}

template <bool MODS, bool TMA>
int launch_paged_rows(const CUtensorMap& mk, const CUtensorMap& mv, const PagedArgs& a, const PagedPlan& p,
                      cudaStream_t stream, int device) {
  if (p.nb == 2) return launch_paged_dim<4, 2, MODS, TMA>(mk, mv, a, p.blocks, stream, device);
  if (p.wr == 1) return launch_paged_dim<1, 1, MODS, TMA>(mk, mv, a, p.blocks, stream, device);
  if (p.wr == 2) return launch_paged_dim<2, 1, MODS, TMA>(mk, mv, a, p.blocks, stream, device);
  return launch_paged_dim<4, 1, MODS, TMA>(mk, mv, a, p.blocks, stream, device);
}

template <bool MODS>
int launch_paged_for(const CUtensorMap& mk, const CUtensorMap& mv, const PagedArgs& a, const PagedPlan& p, bool tma,
                     cudaStream_t stream, int device) {
  return tma ? launch_paged_rows<MODS, true>(mk, mv, a, p, stream, device)
             : launch_paged_rows<MODS, false>(mk, mv, a, p, stream, device);
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
  if (dev->sms > 160) return fail(kErrUnsupported, "paged attention: more than 160 SMs");
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
               uintptr_t(4 * esize - 1)) == 0;
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
  a.by_page = divisor(c.page_size);
  a.by_g = divisor(a.G);
  a.by_row_tiles = divisor(a.row_tiles);
  a.by_slot_rows = divisor(a.slot_rows);
  a.min_span = p.variant > 0 ? p.variant : 1;
  a.round_span = p.variant == 0;
  a.by_blocks = divisor(plan.blocks);
  uint8_t* ws = static_cast<uint8_t*>(p.workspace);
  a.rec = reinterpret_cast<int4*>(ws);
  a.part_ml = reinterpret_cast<float2*>(ws + plan.ml_offset);
  a.part_o = reinterpret_cast<float*>(ws + plan.o_offset);
  a.head_o = reinterpret_cast<float*>(ws + plan.head_offset);
  a.ctl.status = dev->status;
  a.ctl.timeout_ns = wait_timeout_ns();
  a.ctl.debug = p.debug;
  // TMA takes 16 slots of a page at a time, and maps of positive strides below 2^40 bytes. Heads that are no multiple of 128
  // columns are copied faster by cp.async where there is much to read: TMA moves the empty part of a column of 64 too (80, 96,
  // 160), and its two warps have twice the half tiles to issue for the same bytes (64). One token, 32/8 heads, ragged, by TMA and by
  // cp.async: 16 x 16384 keys of 64 99 and 89 us; 16 x 8000 of 80 72 and 65, of 96 77 and 70, of 160 113 and 108; of 128 and
  // 256 level (72 and 73, 135 and 133). With little to read TMA starts sooner (777 keys of 64 8.7 us, 9.6 by cp.async; of 128
  // 9.1 and 10.1). How much that is only the device knows: the table's width, which the lengths end at, stands for it here, so
  // short caches under a table for long ones are copied by cp.async.
  const bool few_keys = p.batch * c.kv_heads * (a.capacity / 32 + 1) <= int64_t(plan.blocks) * 8;
  CUtensorMap mk, mv;
  memset(&mk, 0, sizeof(mk));
  memset(&mv, 0, sizeof(mv));
  const auto strided = [&](int64_t sp, int64_t ss, int64_t sh) {
    const auto fits = [](int64_t n, int64_t s) { return n == 1 || (s > 0 && s < (int64_t(1) << 38)); };
    return fits(c.pages, sp) && fits(c.page_size, ss) && fits(c.kv_heads, sh);
  };
  const bool tma = (c.head_dim % 128 == 0 || few_keys) && c.page_size % 16 == 0 && c.pages > 0 &&
                   strided(c.k_sp, c.k_ss, c.k_sh) && strided(c.v_sp, c.v_ss, c.v_sh);
  const int tile = c.head_dim <= 128 ? 32 : 16;  // (PagedLayout::kTile)
  a.box_rows = c.page_size % tile == 0 ? tile : 16;
  if (tma) {
    if (int rc = encode_bshd_map(c.k, c.head_dim, c.page_size, c.kv_heads, c.pages, c.k_ss, c.k_sh, c.k_sp, a.box_rows, &mk,
                                 &a.pk))
      return rc;
    if (int rc = encode_bshd_map(c.v, c.head_dim, c.page_size, c.kv_heads, c.pages, c.v_ss, c.v_sh, c.v_sp, a.box_rows, &mv,
                                 &a.pv))
      return rc;
  }
  const bool mods = p.softcap > 0.0f || p.slopes != nullptr;
  if (int rc = mods ? launch_paged_for<true>(mk, mv, a, plan, tma, stream, dev->device)
                    : launch_paged_for<false>(mk, mv, a, plan, tma, stream, dev->device))
    return rc;
  // As many rows can be left to join as items begin, one a block at most.
  const int64_t items = std::min<int64_t>(p.batch * c.kv_heads * plan.row_tiles, plan.blocks);
  static_assert(kBlocks * 160 <= kJoinMaxRecs, "records of the join kernel");
  const int64_t rows = items * plan.slot_rows;
  const bool few = rows <= 2 * dev->sms;
  const int64_t join_blocks = std::min<int64_t>(few ? rows : (rows + kJoinWarps - 1) / kJoinWarps, 2 * dev->sms);
  return check_cuda(launch_pdl(few ? attention_paged_join_kernel<kJoinWarps> : attention_paged_join_kernel<1>,
                               dim3(unsigned(join_blocks)), dim3(kJoinWarps * 32), 0, stream, a, plan.blocks, 8 * plan.nb * plan.wr),
                    "paged attention join kernel launch");
}

}  // namespace npub200
