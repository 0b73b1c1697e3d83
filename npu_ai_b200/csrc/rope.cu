// rope.cu - rotary positions, and the append of new keys and values to the pages of a cache with the keys (and queries)
// rotated on the way.
//
// Pair j of a head (values j and j + r/2, or 2j and 2j + 1 when interleaved) at position p turns by a = p f_j:
//   u' = m (u cos a - v sin a), v' = m (v cos a + u sin a); the inverse turns by -a.
// Far positions need the angle in 64 bits: p f_j in f32 is off by up to p f_j 2^-24, 0.06 rad at a million. It is reduced
// in 64 bits to turns in [-1/2, 1/2] and only then rounded to f32 for sincospif. The rotation runs in f32 (whatever the
// input's type) and is rounded once.
//
// Bound by memory: each value is read once and written once. A block owns a few tokens and a chunk of their heads; it works
// out its tokens' (cos, sin) once into shared memory, a thread takes those of one place of a head into registers and walks over
// the heads. (With a table read for each vector 16384 x 40 x 128 took 72 us instead of 56: eight lanes' reads of it met in the
// same banks.) 56.3 us are 6.0 TB/s, 91% of the measured copy rate; pairs next to each other 55.1 us; 8192 tokens of f32 to
// bf16 42.0 us, 92%; the append of 2 x 8192 tokens with 32 + 8 + 8 heads of 128 75 us, 82%: its start (positions, the page table,
// the angles) passes without loads in flight.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "fast_div.cuh"
#include "internal.h"

namespace npub200 {

namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeMaxTokens = 16;         // tokens of a block
constexpr int kRopeTableBytes = 32 * 1024;  // (cos, sin) of a block's tokens
constexpr int kRopeBlockBytes = 128 * 1024;  // source bytes of a block, at most, where there are enough tokens

// Element (b, s, h, e) at b*sb + s*ss + h*sh + e.
struct RopeRows {
  const void* p;
  long long sb, ss, sh;
};

struct RopeArgs {
  RopeRows src[3];  // queries (or the only tensor), new keys, new values
  RopeRows dst[3];  // their destinations; of keys and values the pages: sb is the page's stride, ss the slot's
  int heads[3];
  long long tokens;
  int seq, dim, half, rot_units, units;  // units of a head: rot_units rotated ones, the rest copied
  int block_tokens, chunk;               // tokens and heads of a block
  int places, groups;                    // units of a block's tokens, threads that share the heads of one
  Divisor by_units, by_places, by_seq, by_half;
  int inverse;
  float magnitude;
  const double* freqs;
  long long start;
  const int32_t* starts;
  const int32_t* positions;
  long long pos_sb, pos_ss;
  // pages
  const int32_t* counts;
  const int32_t* table;
  long long table_stride, pages, capacity;
  int page_size;
};

// V values as they lie in memory, and as f32.
template <typename T, int V>
struct Values {
  static constexpr int kWords = V * int(sizeof(T)) / 4 > 0 ? V * int(sizeof(T)) / 4 : 1;
  uint32_t w[kWords];

  __device__ __forceinline__ void load(const T* p) {
    if constexpr (sizeof(T) == 4) {
      if constexpr (V >= 4) {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(p + i);
          w[i] = x.x, w[i + 1] = x.y, w[i + 2] = x.z, w[i + 3] = x.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = __float_as_uint(p[i]);
      }
    } else if constexpr (V == 8) {
      const uint4 x = *reinterpret_cast<const uint4*>(p);
      w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else if constexpr (V == 4) {
      const uint2 x = *reinterpret_cast<const uint2*>(p);
      w[0] = x.x, w[1] = x.y;
    } else {  // one or two values, which need not lie on a 4-byte boundary
      w[0] = *reinterpret_cast<const uint16_t*>(p);
      if constexpr (V == 2) w[0] |= uint32_t(*reinterpret_cast<const uint16_t*>(p + 1)) << 16;
    }
  }
  __device__ __forceinline__ void unpack(float (&f)[V]) const {
#pragma unroll
    for (int i = 0; i < V; ++i)
      f[i] = sizeof(T) == 4 ? __uint_as_float(w[i])
                            : __uint_as_float(i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
  }
};

template <typename T, int V>
__device__ __forceinline__ void store_values(T* p, const float (&f)[V]) {
  if constexpr (sizeof(T) == 4) {
    if constexpr (V >= 4) {
#pragma unroll
      for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) p[i] = f[i];
    }
  } else if constexpr (V == 8) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                                              pack_bf16x2(f[6], f[7]));
  } else if constexpr (V == 4) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = __float2bfloat16_rn(f[i]);
  }
}

// What a block keeps of each of its tokens.
struct RopeToken {
  long long dst[3];  // offset of the token's first head in each destination; < 0: nothing is written
};

// V values a vector. Half layout: a rotated unit is the vectors at j and j + r/2; interleaved: one vector of V/2 pairs.
template <typename TIn, typename TOut, int V, bool IL, bool PAGED>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeArgs a) {
  extern __shared__ float2 s_turn[];  // [block_tokens][half] (m cos, m sin)
  __shared__ RopeToken s_token[kRopeMaxTokens];
  const int tid = int(threadIdx.x);
  const long long first = (long long)blockIdx.x * a.block_tokens;
  const int n = int(min((long long)a.block_tokens, a.tokens - first));
  pdl_wait();
  pdl_launch_dependents();
  __shared__ long long s_pos[kRopeMaxTokens];
  if (tid < n) {
    const long long token = first + tid, b = token / a.seq, s = token - b * a.seq;
    s_pos[tid] = a.positions != nullptr ? (long long)a.positions[b * a.pos_sb + s * a.pos_ss]
                                        : s + (a.starts != nullptr ? (long long)a.starts[b] : a.start);
  }
  __syncthreads();
  if (tid < n) {
    const long long token = first + tid, b = token / a.seq, s = token - b * a.seq;
    RopeToken t;
    t.dst[0] = b * a.dst[0].sb + s * a.dst[0].ss;
    if constexpr (PAGED) {
      const long long p = s_pos[tid];
      long long page = -1, slot = 0;
      if (p >= 0 && p < a.capacity && (a.counts == nullptr || s < a.counts[b])) {
        const uint32_t at = uint32_t(p) / uint32_t(a.page_size);  // the capacity is at most 2^30
        slot = p - (long long)at * a.page_size;
        page = a.table[b * a.table_stride + at];
      }
      const bool in = page >= 0 && page < a.pages;
#pragma unroll
      for (int k = 1; k < 3; ++k) t.dst[k] = in ? page * a.dst[k].sb + slot * a.dst[k].ss : -1;
    }
    s_token[tid] = t;
  }
  for (int i = tid; i < n * a.half; i += kRopeThreads) {
    const int t = a.by_half(i), j = i - t * a.half;
    double turns = double(s_pos[t]) * (a.freqs[j] * 0.15915494309189535);  // 1 / (2 pi)
    turns -= rint(turns);
    float sn, cs;
    sincospif(float(2.0 * turns), &sn, &cs);
    s_turn[i] = make_float2(cs * a.magnitude, (a.inverse ? -sn : sn) * a.magnitude);
  }
  __syncthreads();

  // A thread keeps one place of a head (a token's unit: V or 2 V values) with its angles in registers and walks over the
  // heads, the threads with the same place sharing them.
  constexpr int TENSORS = PAGED ? 3 : 1;
  const int h0 = int(blockIdx.y) * a.chunk;
  const int heads = min(a.chunk, a.heads[0] + (PAGED ? a.heads[1] + a.heads[2] : 0) - h0);
  for (int place = tid - a.by_places(tid) * min(a.places, kRopeThreads), group = a.by_places(tid); place < a.places && group < a.groups;
       place += a.places > kRopeThreads ? kRopeThreads : a.places) {
    const int tok = a.by_units(place), unit = place - tok * a.units;
    if (tok >= n) break;
    const bool rotated = unit < a.rot_units, pair = !IL && rotated;
    const int e = IL || rotated ? unit * V : 2 * a.half + (unit - a.rot_units) * V;  // the unit's first value
    constexpr int ANGLES = IL ? V / 2 : V;
    float cs[ANGLES], sn[ANGLES];
    if (rotated) {
#pragma unroll
      for (int i = 0; i < ANGLES; ++i) {
        const float2 w = s_turn[tok * a.half + unit * ANGLES + i];
        cs[i] = w.x;
        sn[i] = w.y;
      }
    }
    const int token = int(first) + tok;  // (fewer than 2^31 tokens)
    const long long b = a.by_seq(token), s = token - b * a.seq;
    const TIn* src[TENSORS];
    TOut* dst[TENSORS];  // null: nothing is written
#pragma unroll
    for (int k = 0; k < TENSORS; ++k) {
      const long long at = s_token[tok].dst[k];
      src[k] = static_cast<const TIn*>(a.src[k].p) + (b * a.src[k].sb + s * a.src[k].ss + e);
      dst[k] = at < 0 ? nullptr : static_cast<TOut*>(const_cast<void*>(a.dst[k].p)) + (at + e);
    }
    // Units whose loads are in flight together, of one tensor or the next: 64 bytes a thread.
    constexpr int UNIT = V * int(sizeof(TIn)) * (IL ? 1 : 2), UN = UNIT >= 64 ? 1 : UNIT >= 16 ? 64 / UNIT : 4;
    for (int h = h0 + group; h < h0 + heads; h += UN * a.groups) {
      Values<TIn, V> lo[UN], hi[UN];
      TOut* out[UN];
      bool turn[UN];
#pragma unroll
      for (int k = 0; k < UN; ++k) {
        int hk = h + k * a.groups;
        out[k] = nullptr;
        if (hk >= h0 + heads) continue;
        const TIn* in = src[0];
        long long in_sh = a.src[0].sh, out_sh = a.dst[0].sh;
        out[k] = dst[0];
        turn[k] = rotated;
        if constexpr (PAGED) {
          if (hk >= a.heads[0]) {
            const bool value = hk >= a.heads[0] + a.heads[1];
            hk -= a.heads[0] + (value ? a.heads[1] : 0);
            in = src[value ? 2 : 1];
            in_sh = value ? a.src[2].sh : a.src[1].sh;
            out[k] = dst[value ? 2 : 1];
            out_sh = value ? a.dst[2].sh : a.dst[1].sh;
            turn[k] = rotated && !value;
          }
        }
        if (out[k] == nullptr) continue;
        out[k] += hk * out_sh;
        lo[k].load(in + hk * in_sh);
        if (pair) hi[k].load(in + hk * in_sh + a.half);
      }
#pragma unroll
      for (int k = 0; k < UN; ++k) {
        if (out[k] == nullptr) continue;
        float u[V], v[V];
        lo[k].unpack(u);
        if (pair) hi[k].unpack(v);
        if (turn[k]) {
          if constexpr (IL) {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
              const float x = u[2 * i], y = u[2 * i + 1];
              u[2 * i] = x * cs[i] - y * sn[i];
              u[2 * i + 1] = y * cs[i] + x * sn[i];
            }
          } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const float x = u[i], y = v[i];
              u[i] = x * cs[i] - y * sn[i];
              v[i] = y * cs[i] + x * sn[i];
            }
          }
        }
        store_values<TOut, V>(out[k], u);
        if (pair) store_values<TOut, V>(out[k] + a.half, v);
      }
    }
  }
}

// Whether vectors of V values of a tensor lie on the boundary that their loads need.
bool rows_fit(const RopeRows& r, int V, int esize) {
  const uintptr_t bytes = uintptr_t(std::min(16, V * esize));
  return ((reinterpret_cast<uintptr_t>(r.p) | uintptr_t(r.sb * esize) | uintptr_t(r.ss * esize) | uintptr_t(r.sh * esize)) &
          (bytes - 1)) == 0;
}

template <typename TIn, typename TOut, int V, bool IL, bool PAGED>
int launch_rope(const RopeArgs& a, dim3 grid, size_t smem, cudaStream_t stream) {
  return check_cuda(launch_pdl(rope_kernel<TIn, TOut, V, IL, PAGED>, grid, dim3(kRopeThreads), smem, stream, a),
                    "rope kernel launch");
}

template <typename TIn, typename TOut, bool PAGED>
int launch_rope_for(RopeArgs& a, int rot, bool interleaved, cudaStream_t stream, int sms) {
  // The widest vectors that every tensor's alignment and the rotated part's width allow; pairs lie within a vector or in
  // two of them, so a rotated part that is no whole number of vectors takes narrower ones.
  // (Half layout: two vectors a unit, and angles for each: with 8 values 80 registers and three blocks an SM, 16384 x 40 x 128
  // 64 us, with 4 values 56.)
  int V = interleaved ? 8 : 4;
  for (; V > (interleaved ? 2 : 1); V = V == 8 ? 4 : interleaved ? 2 : 1) {
    bool fit = a.dim % V == 0 && (interleaved ? rot : rot / 2) % V == 0;
    for (int k = 0; k < (PAGED ? 3 : 1); ++k)
      if (a.heads[k] > 0) fit = fit && rows_fit(a.src[k], V, sizeof(TIn)) && rows_fit(a.dst[k], V, sizeof(TOut));
    if (fit) break;
  }
  a.half = rot / 2;
  a.rot_units = (interleaved ? rot : a.half) / V;
  a.units = a.rot_units + (a.dim - rot) / V;
  const int heads = a.heads[0] + (PAGED ? a.heads[1] + a.heads[2] : 0);
  long long tb = kRopeBlockBytes / ((long long)heads * a.dim * (int)sizeof(TIn));
  if (a.half > 0) tb = std::min<long long>(tb, kRopeTableBytes / (a.half * (int)sizeof(float2)));
  tb = std::max<long long>(1, std::min<long long>(tb, kRopeMaxTokens));
  while (tb & (tb - 1)) tb &= tb - 1;  // a power of two, whose units mostly divide the threads: with 9 tokens 144 of 256 worked
  while (tb > 1 && (a.tokens + tb - 1) / tb < 2 * sms) tb /= 2;
  a.block_tokens = int(tb);
  const long long blocks = (a.tokens + tb - 1) / tb;
  // Few tokens: their heads go to several blocks, of one unit a thread at least.
  const long long wish = std::min<long long>(std::max<long long>(1, sms / blocks),
                                             std::max<long long>(1, (long long)heads * a.units * tb / kRopeThreads));
  a.chunk = int((heads + wish - 1) / wish);
  a.places = a.block_tokens * a.units;
  a.groups = std::max(1, kRopeThreads / a.places);
  a.by_units = divisor(a.units);
  a.by_places = divisor(std::min(a.places, kRopeThreads));
  a.by_seq = divisor(a.seq);
  a.by_half = divisor(std::max(1, a.half));
  const dim3 grid(unsigned(blocks), unsigned((heads + a.chunk - 1) / a.chunk));
  const size_t smem = size_t(tb) * a.half * sizeof(float2);
  if (interleaved) {
    if (V == 8) return launch_rope<TIn, TOut, 8, true, PAGED>(a, grid, smem, stream);
    if (V == 4) return launch_rope<TIn, TOut, 4, true, PAGED>(a, grid, smem, stream);
    return launch_rope<TIn, TOut, 2, true, PAGED>(a, grid, smem, stream);
  }
  if (V == 4) return launch_rope<TIn, TOut, 4, false, PAGED>(a, grid, smem, stream);
  return launch_rope<TIn, TOut, 1, false, PAGED>(a, grid, smem, stream);
}

// What rope and the append ask of a rotation; `dim` is the head's.
int check_rotation(const npub200_rotation& r, int64_t dim, const char* what) {
  if (r.rot_dim < 0 || r.rot_dim % 2 != 0 || r.rot_dim > dim)
    return fail(kErrInvalid, "%s: rot_dim must be even and within the head dim %lld (got %lld)", what, (long long)dim,
                (long long)r.rot_dim);
  if (r.rot_dim > 0 && r.freqs == nullptr) return fail(kErrInvalid, "%s: frequencies are null", what);
  if (reinterpret_cast<uintptr_t>(r.freqs) & 7u) return fail(kErrInvalid, "%s: frequencies must be 8-byte aligned", what);
  if (!std::isfinite(r.magnitude)) return fail(kErrInvalid, "%s: magnitude must be finite", what);
  return kOk;
}

int check_rope_sizes(int64_t batch, int64_t seq, int64_t heads, int64_t dim, const char* what) {
  if (batch < 0 || seq < 0 || heads < 0 || dim <= 0)
    return fail(kErrInvalid, "%s: bad sizes (batch=%lld seq=%lld heads=%lld head_dim=%lld)", what, (long long)batch,
                (long long)seq, (long long)heads, (long long)dim);
  if (dim % 2 != 0 || dim > 1024)
    return fail(kErrUnsupported, "%s: head dim %lld is not an even number up to 1024", what, (long long)dim);
  if (heads > 65535) return fail(kErrUnsupported, "%s: more than 65535 heads (%lld)", what, (long long)heads);
  if (seq > INT32_MAX || batch > INT32_MAX || (seq > 0 && batch > INT32_MAX / seq))
    return fail(kErrUnsupported, "%s: more than 2^31 - 1 tokens (%lld x %lld)", what, (long long)batch, (long long)seq);
  return kOk;
}

int check_rows(const void* p, int64_t sb, int64_t ss, int64_t sh, int esize, const char* what, const char* name) {
  if (p == nullptr) return fail(kErrInvalid, "%s: %s is null", what, name);
  if (reinterpret_cast<uintptr_t>(p) % uintptr_t(esize)) return fail(kErrInvalid, "%s: %s is misaligned", what, name);
  if (sb < 0 || ss < 0 || sh < 0) return fail(kErrInvalid, "%s: %s has a negative stride", what, name);
  return kOk;
}

int dtype_bytes(int code) { return code == NPUB200_DTYPE_BF16 ? 2 : code == NPUB200_DTYPE_F32 ? 4 : 0; }

}  // namespace

int rope_launch(const RopeProblem& p, cudaStream_t stream) {
  const char* what = "rope";
  const int in = dtype_bytes(p.in_dtype), out = dtype_bytes(p.out_dtype);
  if (in == 0 || out == 0) return fail(kErrInvalid, "rope: unknown dtype code %d or %d", p.in_dtype, p.out_dtype);
  if (int rc = check_rope_sizes(p.batch, p.seq, p.heads, p.head_dim, what)) return rc;
  if (p.rotation == nullptr) return fail(kErrInvalid, "rope: rotation is null");
  if (int rc = check_rotation(*p.rotation, p.head_dim, what)) return rc;
  if (p.starts != nullptr && p.positions != nullptr) return fail(kErrInvalid, "rope: both starts and positions are given");
  if (p.pos_sb < 0 || p.pos_ss < 0) return fail(kErrInvalid, "rope: positions have a negative stride");
  if (p.start < INT32_MIN || p.start > INT32_MAX)
    return fail(kErrInvalid, "rope: start %lld does not fit 32 bits", (long long)p.start);
  if (p.batch == 0 || p.seq == 0 || p.heads == 0) return kOk;
  if (int rc = check_rows(p.x, p.x_sb, p.x_ss, p.x_sh, in, what, "x")) return rc;
  if (int rc = check_rows(p.out, p.o_sb, p.o_ss, p.o_sh, out, what, "out")) return rc;
  const DeviceInfo* dev = nullptr;
  if (int rc = current_device_info(&dev)) return rc;
  RopeArgs a;
  memset(&a, 0, sizeof(a));
  a.src[0] = RopeRows{p.x, p.x_sb, p.x_ss, p.x_sh};
  a.dst[0] = RopeRows{p.out, p.o_sb, p.o_ss, p.o_sh};
  a.heads[0] = int(p.heads);
  a.tokens = p.batch * p.seq;
  a.seq = int(p.seq);
  a.dim = int(p.head_dim);
  a.inverse = p.rotation->inverse != 0;
  a.magnitude = p.rotation->magnitude;
  a.freqs = p.rotation->freqs;
  a.start = p.start;
  a.starts = p.starts;
  a.positions = p.positions;
  a.pos_sb = p.pos_sb;
  a.pos_ss = p.pos_ss;
  const int rot = int(p.rotation->rot_dim);
  const bool il = p.rotation->interleaved != 0;
  if (in == 2 && out == 2) return launch_rope_for<__nv_bfloat16, __nv_bfloat16, false>(a, rot, il, stream, dev->sms);
  if (in == 2) return launch_rope_for<__nv_bfloat16, float, false>(a, rot, il, stream, dev->sms);
  if (out == 2) return launch_rope_for<float, __nv_bfloat16, false>(a, rot, il, stream, dev->sms);
  return launch_rope_for<float, float, false>(a, rot, il, stream, dev->sms);
}

int check_paged_cache(const npub200_paged_cache* c, int64_t batch, const char* what) {
  if (c == nullptr) return fail(kErrInvalid, "%s: cache is null", what);
  if (c->pages < 0 || c->page_size <= 0 || c->kv_heads <= 0 || c->head_dim <= 0 || c->table_width < 0 ||
      c->table_stride < 0)
    return fail(kErrInvalid, "%s: bad cache sizes (pages=%lld page_size=%lld kv_heads=%lld head_dim=%lld table=%lld/%lld)",
                what, (long long)c->pages, (long long)c->page_size, (long long)c->kv_heads, (long long)c->head_dim,
                (long long)c->table_width, (long long)c->table_stride);
  constexpr int64_t most = (int64_t(1) << 30) - 32;  // (32 sequences have fewer than 2^31 tiles of 16)
  if (c->pages > INT32_MAX || c->page_size > most || (c->table_width > 0 && c->page_size > most / c->table_width))
    return fail(kErrUnsupported, "%s: more than 2^31 - 1 pages (%lld) or 2^30 - 32 tokens in a sequence's pages (%lld x %lld)",
                what, (long long)c->pages, (long long)c->table_width, (long long)c->page_size);
  if (c->kv_heads > 65535) return fail(kErrUnsupported, "%s: more than 65535 heads (%lld)", what, (long long)c->kv_heads);
  if (c->pages > 0) {
    if (int rc = check_rows(c->k, c->k_sp, c->k_ss, c->k_sh, 2, what, "k pages")) return rc;
    if (int rc = check_rows(c->v, c->v_sp, c->v_ss, c->v_sh, 2, what, "v pages")) return rc;
  }
  if (c->table == nullptr && c->table_width > 0 && batch > 0) return fail(kErrInvalid, "%s: page table is null", what);
  return kOk;
}

int paged_append_launch(const PagedAppendProblem& p, cudaStream_t stream) {
  const char* what = "paged_append";
  const int in = dtype_bytes(p.in_dtype);
  if (in == 0) return fail(kErrInvalid, "paged_append: unknown dtype code %d", p.in_dtype);
  if (int rc = check_paged_cache(p.cache, p.batch, what)) return rc;
  const npub200_paged_cache& c = *p.cache;
  if (int rc = check_rope_sizes(p.batch, p.seq, p.heads + 2 * c.kv_heads, c.head_dim, what)) return rc;
  if (p.heads < 0) return fail(kErrInvalid, "paged_append: bad number of query heads (%lld)", (long long)p.heads);
  if (p.rotation != nullptr)
    if (int rc = check_rotation(*p.rotation, c.head_dim, what)) return rc;
  if (p.heads > 0 && p.rotation == nullptr)
    return fail(kErrInvalid, "paged_append: queries are only taken to be rotated, and there is no rotation");
  if (p.batch == 0 || p.seq == 0) return kOk;
  if (p.starts == nullptr) return fail(kErrInvalid, "paged_append: starts are null");
  if (int rc = check_rows(p.k, p.k_sb, p.k_ss, p.k_sh, in, what, "k")) return rc;
  if (int rc = check_rows(p.v, p.v_sb, p.v_ss, p.v_sh, in, what, "v")) return rc;
  if (p.heads > 0) {
    if (int rc = check_rows(p.q, p.q_sb, p.q_ss, p.q_sh, in, what, "q")) return rc;
    if (int rc = check_rows(p.q_out, p.o_sb, p.o_ss, p.o_sh, 2, what, "q_out")) return rc;
  }
  const DeviceInfo* dev = nullptr;
  if (int rc = current_device_info(&dev)) return rc;
  RopeArgs a;
  memset(&a, 0, sizeof(a));
  a.src[0] = RopeRows{p.q, p.q_sb, p.q_ss, p.q_sh};
  a.src[1] = RopeRows{p.k, p.k_sb, p.k_ss, p.k_sh};
  a.src[2] = RopeRows{p.v, p.v_sb, p.v_ss, p.v_sh};
  a.dst[0] = RopeRows{p.q_out, p.o_sb, p.o_ss, p.o_sh};
  a.dst[1] = RopeRows{c.k, c.k_sp, c.k_ss, c.k_sh};
  a.dst[2] = RopeRows{c.v, c.v_sp, c.v_ss, c.v_sh};
  a.heads[0] = int(p.heads);
  a.heads[1] = a.heads[2] = int(c.kv_heads);
  a.tokens = p.batch * p.seq;
  a.seq = int(p.seq);
  a.dim = int(c.head_dim);
  a.starts = p.starts;
  a.counts = p.counts;
  a.table = c.table;
  a.table_stride = c.table_stride;
  a.pages = c.pages;
  a.page_size = int(c.page_size);
  a.capacity = c.table_width * c.page_size;
  int rot = 0;
  bool il = false;
  if (p.rotation != nullptr) {
    a.inverse = p.rotation->inverse != 0;
    a.magnitude = p.rotation->magnitude;
    a.freqs = p.rotation->freqs;
    rot = int(p.rotation->rot_dim);
    il = p.rotation->interleaved != 0;
  }
  return in == 2 ? launch_rope_for<__nv_bfloat16, __nv_bfloat16, true>(a, rot, il, stream, dev->sms)
                 : launch_rope_for<float, __nv_bfloat16, true>(a, rot, il, stream, dev->sms);
}

}  // namespace npub200
