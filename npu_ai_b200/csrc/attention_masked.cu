// attention_masked.cu - host side of the masked attention (attention_masked.cuh holds the kernel and its reasons): argument
// checks, the launch plan, and the kernel that joins split keys.
#include <algorithm>
#include <cfloat>
#include <cstring>

#include "attention_masked.cuh"

namespace npub200 {

namespace {

// Joins the split parts of a row: with M = max of the parts' maxima, o = sum_z 2^(m_z - M) O_z / sum_z 2^(m_z - M) l_z.
// WARPS warps take a row's parts in turn (4: few rows, a block each; 1: many rows, four a block), all loads of a warp
// issued before the weights are known: the join is bound by latency (two round trips to L2), not by its few KB a row.
// Measured: 160 rows of 27 parts, a token step 18.2 -> 12.4 us with four warps a row; 16384 rows of 2 parts 40 us with
// a block each, 5 us with a warp each. The sum runs in a fixed order.
constexpr int kJoinBlockWarps = 4;
constexpr int kJoinFewRows = 2048;  // about two waves of blocks

template <int WARPS>
__global__ void __launch_bounds__(32 * kJoinBlockWarps)
    attention_join_kernel(const __grid_constant__ MaskedArgs m, int rows) {
  constexpr int kJoinWarps = WARPS;
  __shared__ float s_acc[WARPS][256];
  pdl_launch_dependents();
  pdl_wait();
  const AttnArgs& args = m.a;
  const int lane = threadIdx.x & 31, warp = WARPS > 1 ? int(threadIdx.x >> 5) : 0;
  const int out_row = WARPS > 1 ? int(blockIdx.x) : int(blockIdx.x) * kJoinBlockWarps + int(threadIdx.x >> 5);
  if (out_row >= rows) return;  // (whole warps, and only where they share nothing)
  // rows run (b, i, h), h fastest
  const int h = out_row % args.H;
  const int bi = out_row / args.H;
  const int b = bi / args.Sq, i = bi - b * args.Sq;
  const int g = h % m.pack;
  const int tile = i / m.T, s = i - tile * m.T;
  const int r = m.head_fast ? s * m.pack + g : g * m.T + s;
  const long long at = (((long long)(b * m.groups + h / m.pack)) * m.tiles + tile) * kAttnBM + r;
  const long long step = (long long)m.pairs * m.tiles * kAttnBM;  // rows between parts
  float mz[2], lz[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int z = lane + 32 * k;
    const float2 ml = z < m.splits ? m.part_ml[at + z * step] : make_float2(-INFINITY, 0.0f);
    mz[k] = ml.x;
    lz[k] = ml.y;
  }
  const int c = lane * 8;  // this lane's columns
  float acc[8] = {};
  float wz[2], sum = 0.0f;
  for (int z0 = warp; z0 < m.splits; z0 += 8 * kJoinWarps) {
    float4 v[8][2];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int z = z0 + k * kJoinWarps;
      v[k][0] = v[k][1] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (z < m.splits && c < args.D) {
        const float4* p = reinterpret_cast<const float4*>(m.part_o + (at + z * step) * args.D + c);
        v[k][0] = p[0];
        v[k][1] = p[1];
      }
    }
    if (z0 == warp) {
      float top = fmaxf(mz[0], mz[1]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
      for (int k = 0; k < 2; ++k) wz[k] = mz[k] == -INFINITY ? 0.0f : fast_exp2(mz[k] - top);
      sum = fmaf(wz[0], lz[0], wz[1] * lz[1]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int z = z0 + k * kJoinWarps;
      const float wt = z < m.splits ? __shfl_sync(0xffffffffu, z < 32 ? wz[0] : wz[1], z & 31) : 0.0f;
      if (wt != 0.0f) {  // a part that saw nothing wrote no O: whatever was read there is dropped
        const float* e = &v[k][0].x;
#pragma unroll
        for (int t = 0; t < 8; ++t) acc[t] = fmaf(wt, e[t], acc[t]);
      }
    }
  }
  const long long obase = (long long)b * args.o_sb + (long long)i * args.o_ss + (long long)h * args.o_sh;
  if constexpr (WARPS == 1) {
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // (a NaN sum makes the row NaN, whatever its parts' weights)
    if (c < args.D) {
#pragma unroll
      for (int t = 0; t < 8; ++t) acc[t] *= inv;
      write_columns(m, obase + c, acc);
    }
  } else {
#pragma unroll
    for (int t = 0; t < 8; ++t) s_acc[warp][c + t] = acc[t];
    __syncthreads();
    // (a warp without a part has no sum: warp 0 always has one)
    __shared__ float s_inv;
    if (threadIdx.x == 0) s_inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    __syncthreads();
    const int col = int(threadIdx.x) * 2;
    if (col < args.D) {
      float o[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float x = 0.0f;
#pragma unroll
        for (int k = 0; k < kJoinWarps; ++k) x += s_acc[k][col + t];
        o[t] = x * s_inv;
      }
      if (args.out_f32) {
        float* dst = static_cast<float*>(args.out) + obase + col;
        dst[0] = o[0];
        dst[1] = o[1];
      } else if (m.out_vec) {
        *reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(args.out) + obase + col) = pack_bf16x2(o[0], o[1]);
      } else {
        __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(args.out) + obase + col;
        dst[0] = __float2bfloat16_rn(o[0]);
        dst[1] = __float2bfloat16_rn(o[1]);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------------------------
struct MaskedPlan {
  int pack, T, splits, streams, cluster;
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

// Two streams of key tiles in a CTA where an SM holds one CTA anyway (by its size, or because there are no more) and each
// stream has two tiles at least. 2x8x1024x1024x80 with a mask of its own rows: 32.5 us with one stream, 18.3 with two.
bool two_streams(int64_t D, int64_t ctas, int64_t tiles, int sms) {
  return D <= 160 && (D > 128 || ctas <= sms) && tiles >= 4;
}

// Few parts are joined by a cluster: no workspace, no second launch. The GPU time is that of the second kernel or less
// (2 x 13 parts 6.8 us, with the second kernel 7.1), and the call takes some 4 us less on the host, which is what a small
// call waits for. Clusters that do not all find a place at once wait for a second wave: 35 x 4 parts of 32 tiles took 35 us,
// through the workspace 25; 8 x 16 parts 21.7 and 13.0.
bool in_cluster(int64_t ctas, int64_t parts, int sms) {
  return parts > 1 && parts <= kMaxCluster && (parts <= 4 ? 8 : 28) * ctas * parts <= 7 * sms;
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
  if (p.tiles > 65535) return fail(kErrUnsupported, "too many queries (%lld)", (long long)Sq);
  const int64_t key_tiles = (Skv + kMaskedBN - 1) / kMaskedBN;
  const int64_t slots = (D <= 128 ? 2 : 1) * int64_t(sms);  // resident CTAs
  p.splits = 1;
  if (variant > 0) {
    p.splits = variant;
  } else if (2 * ctas <= slots && key_tiles >= 4) {
    if (key_tiles * ctas >= 32 * slots) {
      // Many long rows: parts of at least 32 tiles, several waves of them, which evens out ragged lengths.
      p.splits = int(std::min<int64_t>(5 * slots / (2 * ctas), kMaxSplits));
    } else {
      // The number of parts with the least time, in us: a tile after the other 1.2, 1.5 where two streams share the SM's
      // units; a join 2.8, and 0.4 a MB of partial results within a cluster, 0.8 through the workspace. Measured against
      // the choice: 1x4x1024x1024x64 16.0 us whole, 13.7 / 12.4 / 13.7 in 2 / 4 / 8 parts; 1x8x512x512x128 11.2 whole,
      // 13.1 in 2; 3x16/8x16x410x72 9.7 whole, 10.8 / 9.5 in 2 / 4; 7x10/5x1x8124x64 30.5 / 25.3 in 4 / 8; 8 pairs of 20
      // rows over 79 tiles 92.6 whole, 13.7 / 13.0 / 12.7 in 12 / 16 / 27.
      double best = 0;
      const int64_t most = std::min<int64_t>({slots / ctas, key_tiles, kMaxSplits});
      for (int wish : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {  // (every number would take a microsecond)
        const int per = int((key_tiles + std::min<int64_t>(wish, most) - 1) / std::min<int64_t>(wish, most));
        const int64_t parts = (int(key_tiles) + per - 1) / per;  // no part without a tile
        double us = two_streams(D, ctas * parts, per, sms) ? 1.5 * ((per + 1) / 2) : 1.2 * per;
        if (parts > 1) us += 2.8 + (in_cluster(ctas, parts, sms) ? 0.4e-6 : 0.8e-6) * double(B * H * Sq * parts * D * 4);
        if (wish == 1 || us < best) {
          best = us;
          p.splits = int(parts);
        }
        if (wish >= most) break;
      }
    }
  }
  p.streams = two_streams(D, ctas * p.splits, key_tiles / p.splits, sms) ? 2 : 1;
  p.cluster = in_cluster(ctas, p.splits, sms);
  if (p.splits > 1 && !p.cluster) {
    if (B * H * Sq > INT32_MAX / kMaxSplits)
      return fail(kErrUnsupported, "too many rows to split their keys (%lld)", (long long)(B * H * Sq));
    const int64_t rows = p.splits * ctas * kAttnBM;
    p.ml_bytes = size_t(rows) * sizeof(float2);
    p.bytes = p.ml_bytes + size_t(rows) * size_t(D) * sizeof(float);
  }
  *out = p;
  return kOk;
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
  if (!(p.scale > 0.0f && p.scale * kLog2e <= FLT_MAX))
    return fail(kErrInvalid, "attention scale must be positive and finite, times log2 e too (got %g)", double(p.scale));
  for (const void* ptr : {p.q, p.k, p.v})
    if (reinterpret_cast<uintptr_t>(ptr) & 15u) return fail(kErrInvalid, "q/k/v base addresses must be 16-byte aligned");
  if (!(o.softcap == 0.0f || (o.softcap >= 1e-30f && o.softcap <= 1e30f)))
    return fail(kErrInvalid, "softcap must be 0 (none) or positive, within [1e-30, 1e30] (got %g)", double(o.softcap));
  // What the kernel computes with has to be a normal number: the cap times log2 e and its polynomial's coefficients are
  // within that range, the scale over the cap, and that times 2 log2 e, only for scales that belong to the cap.
  const float cap_in = o.softcap > 0.0f ? p.scale / o.softcap : 1.0f;
  if (!(cap_in >= FLT_MIN && 2.0f * kLog2e * cap_in <= FLT_MAX))
    return fail(kErrInvalid, "attention scale %g over softcap %g is not a normal number", double(p.scale),
                double(o.softcap));
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
  const int divisor = m.head_fast ? m.pack : m.T;
  m.inv_row = (65536 + divisor - 1) / divisor;
  m.q_bytes = m.pack * m.T * kAtomBytesPerRow;
  m.tiles = int(plan.tiles);
  m.pairs = int(plan.pairs);
  m.groups = int(p.H / plan.pack);
  const int out_size = p.out_f32 ? 4 : 2;
  const uintptr_t out_align = reinterpret_cast<uintptr_t>(p.o) | uintptr_t(p.o_sb * out_size) | uintptr_t(p.o_ss * out_size) |
                              uintptr_t(p.o_sh * out_size);
  m.out_vec = (out_align & 15u) == 0;
  m.splits = plan.splits;
  m.cluster = plan.cluster;
  m.part_ml = static_cast<float2*>(mp.workspace);
  m.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(mp.workspace) + plan.ml_bytes);
  m.out_sectors = plan.splits > 1 ? p.D % 8 == 0 && ((reinterpret_cast<uintptr_t>(m.part_o) | uintptr_t(p.D * 4)) & 31u) == 0
                                  : (out_align & 31u) == 0;
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
  m.q_start = std::min<int64_t>(std::max<int64_t>(o.q_start, -(int64_t(1) << 40)), int64_t(1) << 40);  // + a query index
  m.q_starts = o.q_starts;
  m.prefix = o.prefix;
  m.prefixes = o.prefixes;
  m.kv_lens = o.kv_lens;
  m.docs = o.doc_offsets;
  m.ndocs = int(o.docs);
  m.doc_stride = o.doc_stride;
  m.gaps = o.doc_offsets != nullptr && o.causal && (o.q_starts != nullptr || o.q_start < 0);
  if (o.softcap > 0.0f) {
    m.cap_in = cap_in;
    m.cap_out = o.softcap * kLog2e;
    for (int i = 0; i < 6; ++i) m.cap_poly[i] = m.cap_out * kTanhRatio[i];
  }
  m.slopes = o.slopes;
  m.table = o.distance_bias;
  m.max_dist = o.max_distance;
  m.table_smem = o.distance_bias != nullptr && m.pack == 1 && (2 * (m.max_dist + kTableMargin) + 1) * 4 <= kTableSmemMax;
  m.mask = o.mask;
  if (o.mask != nullptr) {
    m.mask_kind = o.mask_dtype == NPUB200_DTYPE_BOOL ? 1 : o.mask_dtype == NPUB200_DTYPE_BF16 ? 2 : 3;
    const int64_t esz = m.mask_kind == 3 ? 4 : m.mask_kind;
    m.m_sb = o.mask_sb;
    m.m_sh = o.mask_sh;
    m.m_sq = o.mask_sq;
    m.mask_vec = ((reinterpret_cast<uintptr_t>(o.mask) | uintptr_t(o.mask_sb * esz) | uintptr_t(o.mask_sh * esz) |
                   uintptr_t(o.mask_sq * esz)) & 15u) == 0;
    m.mask_row = (o.mask_sq == 0 || p.Sq == 1) && (o.mask_sh == 0 || m.pack == 1);
  }
  const dim3 grid{unsigned(plan.pairs), unsigned(plan.tiles), unsigned(plan.splits)};
  const int feats = m.gaps ? kFeatAny
                           : (o.softcap > 0.0f ? kFeatCap : 0) | (o.slopes || o.distance_bias ? kFeatDistance : 0) |
                                 (o.mask == nullptr ? 0 : m.mask_row ? kFeatMaskRow : kFeatMask);
  auto launch = feats == 0               ? launch_masked_for<0>
                : feats == kFeatCap      ? launch_masked_for<kFeatCap>
                : feats == kFeatDistance ? launch_masked_for<kFeatDistance>
                : feats == kFeatMask     ? launch_masked_for<kFeatMask>
                : feats == kFeatMaskRow  ? launch_masked_for<kFeatMaskRow>
                                         : launch_masked_for<kFeatAny>;
  if (int rc = launch(p.D, plan.streams, mq, mk, mv, m, grid, stream, dev->device)) return rc;
  if (plan.splits == 1 || plan.cluster) return kOk;
  const int rows = int(p.B * p.H * p.Sq);
  const bool few = rows <= kJoinFewRows;
  return check_cuda(launch_pdl(few ? attention_join_kernel<4> : attention_join_kernel<1>,
                               dim3(unsigned(few ? rows : (rows + kJoinBlockWarps - 1) / kJoinBlockWarps)),
                               dim3(32 * kJoinBlockWarps), 0, stream, m, rows),
                    "attention join kernel launch");
}

}  // namespace npub200
