// attention_sm100.cuh - device pieces shared by the attention kernels (attention_sm100.cu, attention_masked.cu): the
// TMA coordinates of a strided (batch, seq, head, dim) tensor, the K/V producer, the S = Q K^T and O += P V issue
// loops, and the O row's rescale and store.
#pragma once

#include "internal.h"

namespace npub200 {

constexpr int kAttnBM = 128;           // query rows per Q tile (one softmax warpgroup, one TMEM lane per row)
constexpr int kSoftmaxWarps = 4;       // per Q tile
constexpr int kAtomBytesPerRow = 128;  // one 128-byte swizzle atom row: 64 bf16

struct MapPos {
  int s, h, b;  // position (1..3) of the seq / head / batch dimension in the tensor map
};

struct AttnArgs {
  int Sq, Skv, H, nkv;
  float scale_log2;     // scale * log2(e)
  float rescale_thr;    // lazy-rescale threshold in log2 units
  void* out;
  long long o_sb, o_ss, o_sh;
  int out_f32;
  int D;                // true head dim (output columns)
  MapPos pq, pk, pv;
  KernelCtl ctl;
};

// Coordinates (dim, then the three outer dims in the map's order) of 64-column atom `atom` of row s of (b, h).
__device__ __forceinline__ void map_coords(const MapPos& p, int atom, int s, int h, int b, int& c0, int& c1, int& c2,
                                           int& c3) {
  c0 = atom * 64;
  c1 = p.s == 1 ? s : (p.h == 1 ? h : b);
  c2 = p.s == 2 ? s : (p.h == 2 ? h : b);
  c3 = p.s == 3 ? s : (p.h == 3 ? h : b);
}

// ---------------------------------------------------------------------------------------------------------------
// Producer: the nkv K and V tiles from tile `first` on of one (b, h) pair into STAGES-deep rings, K one tile ahead
// of V (K_j is needed a whole softmax step before V_j; `first_k_issued`: the first K is on its way). On an abort it
// waits for the loads it issued before returning, so shared memory is not released under an in-flight copy.
// ---------------------------------------------------------------------------------------------------------------
template <int NA, int BN, int STAGES>
__device__ __forceinline__ void kv_producer(const CUtensorMap* tm_k, const CUtensorMap* tm_v, const AttnArgs& args,
                                            uint8_t* sK, uint8_t* sV, uint64_t* k_full, uint64_t* v_full,
                                            uint64_t* k_empty, uint64_t* v_empty, volatile int* abort_flag, int hh,
                                            int bb, int nkv, int first = 0, bool first_k_issued = false) {
  constexpr int kAtom = BN * kAtomBytesPerRow;
  constexpr int kTile = NA * kAtom;
  int issued_k = 0, issued_v = 0;
  bool ok = true;
  int c0, c1, c2, c3;
  for (int j = 0; j <= nkv; ++j) {
    if (j == 0 && first_k_issued) {
      ++issued_k;
    } else if (j < nkv) {
      const int st = j % STAGES;
      if (!mbar_wait_bounded(&k_empty[st], (uint32_t(j / STAGES) & 1u) ^ 1u, abort_flag, args.ctl,
                             kStatusTimeoutProducer)) {
        ok = false;
        break;
      }
      mbar_arrive_expect_tx(&k_full[st], kTile);
      for (int a = 0; a < NA; ++a) {
        map_coords(args.pk, a, (first + j) * BN, hh, bb, c0, c1, c2, c3);
        tma_load_4d(tm_k, &k_full[st], sK + st * kTile + a * kAtom, c0, c1, c2, c3);
      }
      ++issued_k;
    }
    if (j >= 1) {
      const int i = j - 1;
      const int st = i % STAGES;
      if (!mbar_wait_bounded(&v_empty[st], (uint32_t(i / STAGES) & 1u) ^ 1u, abort_flag, args.ctl,
                             kStatusTimeoutProducer)) {
        ok = false;
        break;
      }
      mbar_arrive_expect_tx(&v_full[st], kTile);
      for (int a = 0; a < NA; ++a) {
        map_coords(args.pv, a, (first + i) * BN, hh, bb, c0, c1, c2, c3);
        tma_load_4d(tm_v, &v_full[st], sV + st * kTile + a * kAtom, c0, c1, c2, c3);
      }
      ++issued_v;
    }
  }
  if (!ok) {
    for (int i = max(0, issued_k - STAGES); i < issued_k; ++i)
      mbar_wait_drain(&k_full[i % STAGES], uint32_t(i / STAGES) & 1u, args.ctl);
    for (int i = max(0, issued_v - STAGES); i < issued_v; ++i)
      mbar_wait_drain(&v_full[i % STAGES], uint32_t(i / STAGES) & 1u, args.ctl);
  }
}

// S = Q K_j^T for one Q tile: K-major over the head dim, atoms of 64 columns, +32 B per 16 columns in an atom.
template <int DP, int BN>
__device__ __forceinline__ void issue_s(uint32_t d_tmem, uint64_t q_desc, uint64_t k_desc, int q_atom_bytes,
                                        int kv_atom_bytes) {
  constexpr uint32_t kIdescS = idesc_bf16_f32(kAttnBM, BN, false);
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk)
    umma_f16_ss(d_tmem, q_desc + uint64_t(((kk >> 2) * q_atom_bytes + (kk & 3) * 32) >> 4),
                k_desc + uint64_t(((kk >> 2) * kv_atom_bytes + (kk & 3) * 32) >> 4), kIdescS, kk > 0 ? 1u : 0u);
}

// O += P V_j: P from TMEM (16 keys = 8 columns of bf16 pairs per K step), V MN-major (head dim contiguous), 16 keys
// = 16 rows of 128 B further per K step.
template <int DP, int BN>
__device__ __forceinline__ void issue_pv(uint32_t o_tmem, uint32_t p_tmem, uint64_t v_desc, bool accumulate) {
  constexpr uint32_t kIdescO = idesc_bf16_f32(kAttnBM, DP, true);
#pragma unroll
  for (int kk = 0; kk < BN / 16; ++kk)
    umma_f16_ts(o_tmem, p_tmem + uint32_t(kk * 8), v_desc + uint64_t((kk * 16 * kAtomBytesPerRow) >> 4), kIdescO,
                (accumulate || kk > 0) ? 1u : 0u);
}

// O row *= alpha (TMEM columns from o_addr). Warp-wide: lanes whose max did not move pass alpha = 1.
template <int DP>
__device__ __forceinline__ void rescale_o_row(uint32_t o_addr, float alpha) {
#pragma unroll
  for (int cc = 0; cc < DP; cc += 16) {
    uint32_t r[16];
    tmem_ld16(o_addr + uint32_t(cc), r);
    tmem_wait_ld();
#pragma unroll
    for (int t = 0; t < 16; ++t) r[t] = __float_as_uint(__uint_as_float(r[t]) * alpha);
    tmem_st16(o_addr + uint32_t(cc), r);
  }
  tmem_wait_st();
}

// O row (TMEM columns from o_addr) x inv_l to the output: its first D columns at element offset `obase`, bf16 or f32,
// 16-byte vector stores where aligned. Rows with `store` false only drain TMEM (tcgen05.ld is warp-wide).
template <int DP>
__device__ __forceinline__ void store_o_at(uint32_t o_addr, const AttnArgs& args, bool store, long long obase,
                                           float inv_l) {
#pragma unroll
  for (int cc = 0; cc < DP; cc += 16) {
    uint32_t r[16];
    tmem_ld16(o_addr + uint32_t(cc), r);
    tmem_wait_ld();
    if (store) {
      float o[16];
#pragma unroll
      for (int t = 0; t < 16; ++t) o[t] = __uint_as_float(r[t]) * inv_l;
      const int ncols = min(16, args.D - cc);
      if (args.out_f32) {
        float* dst = static_cast<float*>(args.out) + obase + cc;
        if (ncols == 16 && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
#pragma unroll
          for (int t = 0; t < 4; ++t)
            reinterpret_cast<float4*>(dst)[t] = make_float4(o[4 * t], o[4 * t + 1], o[4 * t + 2], o[4 * t + 3]);
        } else {
#pragma unroll
          for (int t = 0; t < 16; ++t)
            if (t < ncols) dst[t] = o[t];
        }
      } else {
        __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(args.out) + obase + cc;
        if (ncols >= 8 && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
          uint4 v0;
          v0.x = pack_bf16x2(o[0], o[1]);
          v0.y = pack_bf16x2(o[2], o[3]);
          v0.z = pack_bf16x2(o[4], o[5]);
          v0.w = pack_bf16x2(o[6], o[7]);
          reinterpret_cast<uint4*>(dst)[0] = v0;
          if (ncols == 16) {
            uint4 v1;
            v1.x = pack_bf16x2(o[8], o[9]);
            v1.y = pack_bf16x2(o[10], o[11]);
            v1.z = pack_bf16x2(o[12], o[13]);
            v1.w = pack_bf16x2(o[14], o[15]);
            reinterpret_cast<uint4*>(dst)[1] = v1;
          } else {
#pragma unroll
            for (int t = 8; t < 16; ++t)
              if (t < ncols) dst[t] = __float2bfloat16_rn(o[t]);
          }
        } else {
#pragma unroll
          for (int t = 0; t < 16; ++t)
            if (t < ncols) dst[t] = __float2bfloat16_rn(o[t]);
        }
      }
    }
  }
}

// The O row of query `grow` of pair (bb, hh); rows past Sq are not stored.
template <int DP>
__device__ __forceinline__ void store_o_row(uint32_t o_addr, const AttnArgs& args, int grow, int bb, int hh,
                                            float inv_l) {
  store_o_at<DP>(o_addr, args, grow < args.Sq,
                 (long long)bb * args.o_sb + (long long)grow * args.o_ss + (long long)hh * args.o_sh, inv_l);
}

// Host: 4-D map (dim, then seq/head/batch sorted by stride) over a strided tensor with a box of 64 dim-elements (one
// 128-byte swizzle atom) x `rows` sequence rows x `heads` heads.
int encode_bshd_map(const void* base, int64_t D, int64_t S, int64_t H, int64_t B, int64_t ss, int64_t sh, int64_t sb,
                    int rows, CUtensorMap* out, MapPos* pos, int heads = 1);

}  // namespace npub200
