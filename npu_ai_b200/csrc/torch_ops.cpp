// torch_ops.cpp - the GEMM, the fused and the masked attention, rotary positions and the paged cache as torch operators
// (torch.ops.npub200.gemm / .attention / .attention_masked / .rope / .paged_append / .attention_paged).
//
// The reference hands each request to its NPU as one XRT command: NpuProgram.submit_gemm / submit_attn
// (npu/xdna1_program.py:441-473) with three buffer objects and 13 int32 parameters. Here the same requests are
// operators registered with the torch dispatcher (TORCH_LIBRARY), so torch code, CUDA-graph capture and
// torch.compile-free callers see them as ordinary ops on CUDA tensors. Each one checks its tensors, then calls
// the library's C ABI (include/npu_b200.h) on at::cuda::getCurrentCUDAStream() of the tensors' device; nothing is
// computed here and there is no CPU kernel (CPU tensors are refused by the dispatcher). Errors raise like the
// reference's runner: an invalid request is a ValueError, anything else a RuntimeError.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <type_traits>
#include <vector>

#include "npu_b200.h"
#include "overlap.h"

namespace {

void check_rc(int rc, const char* what) {
  if (rc == NPUB200_OK) return;
  const char* msg = npub200_last_error();
  // EINVAL: the request itself (the reference's ValueError for shapes its programs cannot take,
  // npu/xdna1_gemm.py:227-229); anything else, a legal request without a variant or a device failure, is a
  // RuntimeError (a failed NPU command, npu/xdna1_program.py:475-479), as in the ctypes binding.
  TORCH_CHECK_VALUE(rc != NPUB200_EINVAL, what, ": ", msg);
  TORCH_CHECK(false, what, ": ", msg, " (code ", rc, ")");
}

int dtype_code(const at::Tensor& t, const char* name) {
  if (t.scalar_type() == at::kBFloat16) return NPUB200_DTYPE_BF16;
  if (t.scalar_type() == at::kFloat) return NPUB200_DTYPE_F32;
  TORCH_CHECK_VALUE(false, name, " must be bf16 or f32, got ", t.scalar_type());
  return -1;
}

void check_operand(const at::Tensor& t, const at::Tensor& ref, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.device() == ref.device(), name, " must be a CUDA tensor on ", ref.device());
  TORCH_CHECK_VALUE(t.scalar_type() == at::kBFloat16, name, " must be bf16, got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() >= 1 && t.stride(-1) == 1, name, " must have a contiguous last dimension");
}

void* stream_of(const at::Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// out[M, N] = act(x[M, K] . w[N, K]^T (+ bias)) (+ residual), act an NPUB200_ACT_* code or 0 for none; bf16 operands, f32
// accumulation, bias in f32.
// Replaces NpuGemm.matmul_t (npu/xdna1_gemm.py:349-422) / NpuProgram.submit_gemm (npu/xdna1_program.py:451-454).
at::Tensor gemm(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& bias,
                const std::optional<at::Tensor>& out, int64_t variant, std::optional<at::ScalarType> out_dtype,
                int64_t weight_handle, const std::optional<at::Tensor>& residual, int64_t activation) {
  check_operand(x, x, "x");
  check_operand(w, x, "w");
  TORCH_CHECK_VALUE(x.dim() == 2 && w.dim() == 2, "gemm takes 2-D x [M, K] and w [N, K]");
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  TORCH_CHECK_VALUE(w.size(1) == K, "K mismatch: x has ", K, ", w has ", w.size(1));
  const c10::cuda::CUDAGuard guard(x.device());
  at::Tensor y;
  if (out.has_value()) {
    y = *out;
    TORCH_CHECK_VALUE(y.is_cuda() && y.device() == x.device() && y.dim() == 2 && y.size(0) == M && y.size(1) == N &&
                          y.stride(1) == 1,
                      "out must be an [M, N] CUDA matrix with contiguous rows on x's device");
  } else {
    y = at::empty({M, N}, x.options().dtype(out_dtype.value_or(at::kFloat)));
  }
  const int out_code = dtype_code(y, "out");
  const void* b_ptr = nullptr;
  int b_code = NPUB200_DTYPE_BF16;
  if (bias.has_value()) {
    const at::Tensor& b = *bias;
    TORCH_CHECK_VALUE(b.is_cuda() && b.device() == x.device() && b.numel() == N && b.is_contiguous(),
                      "bias must be a contiguous [N] CUDA vector on x's device");
    b_code = dtype_code(b, "bias");
    b_ptr = b.data_ptr();
  }
  void* st = stream_of(x);
  if (residual.has_value() || activation != 0) {
    const void* r_ptr = nullptr;
    int64_t ldr = 0;
    if (residual.has_value()) {
      const at::Tensor& r = *residual;
      check_operand(r, x, "residual");
      TORCH_CHECK_VALUE(r.dim() == 2 && r.size(0) == M && r.size(1) == N, "residual must be [M, N]");
      r_ptr = r.data_ptr();
      ldr = r.stride(0);
    }
    size_t ws_bytes = 0;
    check_rc(npub200_gemm_workspace_size(x.data_ptr(), x.stride(0), M, K, w.data_ptr(), w.stride(0), N,
                                         int(variant), &ws_bytes),
             "npub200::gemm");
    at::Tensor ws;
    if (ws_bytes) ws = at::empty({int64_t(ws_bytes)}, x.options().dtype(at::kByte));
    void* ws_ptr = ws_bytes ? ws.data_ptr() : nullptr;
    if (activation != 0)
      check_rc(npub200_gemm_act(x.data_ptr(), x.stride(0), M, K, w.data_ptr(), w.stride(0), N, b_ptr, b_code,
                                int(activation), r_ptr, ldr, y.data_ptr(), y.stride(0), out_code, ws_ptr, ws_bytes,
                                int(variant), st),
               "npub200::gemm");
    else
      check_rc(npub200_gemm_residual(x.data_ptr(), x.stride(0), M, K, w.data_ptr(), w.stride(0), N, b_ptr, b_code,
                                     r_ptr, ldr, y.data_ptr(), y.stride(0), out_code, ws_ptr, ws_bytes, int(variant),
                                     st),
               "npub200::gemm");
    return y;
  }
  size_t ws_bytes = 0;
  check_rc(npub200_gemm_workspace_size(x.data_ptr(), x.stride(0), M, K, weight_handle ? nullptr : w.data_ptr(),
                                       w.stride(0), N, int(variant), &ws_bytes),
           "npub200::gemm");
  at::Tensor ws;
  if (ws_bytes) ws = at::empty({int64_t(ws_bytes)}, x.options().dtype(at::kByte));
  void* ws_ptr = ws_bytes ? ws.data_ptr() : nullptr;
  if (weight_handle != 0) {
    check_rc(npub200_gemm_w(x.data_ptr(), x.stride(0), M, K, weight_handle, b_ptr, b_code, y.data_ptr(), y.stride(0),
                            out_code, ws_ptr, ws_bytes, int(variant), st),
             "npub200::gemm");
  } else {
    check_rc(npub200_gemm(x.data_ptr(), x.stride(0), M, K, w.data_ptr(), w.stride(0), N, b_ptr, b_code, y.data_ptr(),
                          y.stride(0), out_code, ws_ptr, ws_bytes, int(variant), st),
             "npub200::gemm");
  }
  return y;
}

// (batch, seq, head) element strides of a (B, S, H*d) tensor or, head-major, a (B, H, S, d) tensor.
void bsh_strides(const at::Tensor& t, bool head_major, int64_t d, int64_t* sb, int64_t* ss, int64_t* sh) {
  *sb = t.stride(0);
  if (head_major) {
    *sh = t.stride(1);
    *ss = t.stride(2);
  } else {
    *ss = t.stride(1);
    *sh = d;
  }
}

void check_layout(const at::Tensor& t, bool head_major, int64_t B, int64_t H, int64_t S, int64_t d,
                  int64_t row_stride, const char* name) {
  if (head_major) {
    TORCH_CHECK_VALUE(t.dim() == 4 && t.size(0) == B && t.size(1) == H && t.size(2) == S && t.size(3) == d, name,
                      " must be (B, H, S, d) = (", B, ", ", H, ", ", S, ", ", d, "), got ", t.sizes());
  } else {
    TORCH_CHECK_VALUE(t.dim() == 3 && t.size(0) == B && t.size(1) == S && t.size(2) == H * d, name,
                      " must be (B, S, H*d) = (", B, ", ", S, ", ", H * d, "), got ", t.sizes());
  }
  const int64_t rs = head_major ? t.stride(2) : t.stride(1);
  TORCH_CHECK_VALUE(row_stride <= 0 || row_stride == rs, name, " row stride ", rs, " differs from the declared ",
                    row_stride);
}

// softmax(q k^T * scale) v for every (batch, head) pair in one launch. Replaces NpuGemm.attention /
// _attention_fused (npu/xdna1_gemm.py:499-752) and NpuProgram.submit_attn (npu/xdna1_program.py:461-473). The
// declared row strides are checked against the tensors (0: take the tensor's); scale <= 0 means d^-0.5.
at::Tensor attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const std::optional<at::Tensor>& out,
                     int64_t B, int64_t H, int64_t Sq, int64_t Skv, int64_t d, int64_t q_row_stride,
                     int64_t kv_row_stride, int64_t o_row_stride, bool head_major_in, bool head_major_out,
                     double scale, int64_t variant, std::optional<at::ScalarType> out_dtype) {
  check_operand(q, q, "q");
  check_operand(k, q, "k");
  check_operand(v, q, "v");
  check_layout(q, head_major_in, B, H, Sq, d, q_row_stride, "q");
  check_layout(k, head_major_in, B, H, Skv, d, kv_row_stride, "k");
  check_layout(v, head_major_in, B, H, Skv, d, kv_row_stride, "v");
  const c10::cuda::CUDAGuard guard(q.device());
  at::Tensor o;
  if (out.has_value()) {
    o = *out;
    TORCH_CHECK_VALUE(o.is_cuda() && o.device() == q.device() && o.stride(-1) == 1,
                      "out must be a CUDA tensor on q's device with a contiguous last dimension");
  } else {
    o = head_major_out ? at::empty({B, H, Sq, d}, q.options().dtype(out_dtype.value_or(at::kFloat)))
                       : at::empty({B, Sq, H * d}, q.options().dtype(out_dtype.value_or(at::kFloat)));
  }
  check_layout(o, head_major_out, B, H, Sq, d, o_row_stride, "out");
  int64_t qs[3], ks[3], vs[3], os[3];
  bsh_strides(q, head_major_in, d, &qs[0], &qs[1], &qs[2]);
  bsh_strides(k, head_major_in, d, &ks[0], &ks[1], &ks[2]);
  bsh_strides(v, head_major_in, d, &vs[0], &vs[1], &vs[2]);
  bsh_strides(o, head_major_out, d, &os[0], &os[1], &os[2]);
  const float s = scale > 0 ? float(scale) : float(1.0 / std::sqrt(double(d)));
  check_rc(npub200_attention(q.data_ptr(), qs[0], qs[1], qs[2], k.data_ptr(), ks[0], ks[1], ks[2], v.data_ptr(),
                             vs[0], vs[1], vs[2], o.data_ptr(), os[0], os[1], os[2], dtype_code(o, "out"), B, H, Sq,
                             Skv, d, s, int(variant), stream_of(q)),
           "npub200::attention");
  return o;
}

// A device vector of n values of a masked attention (lengths, positions, slopes): its pointer, or null when absent.
template <typename T>
const T* vector_ptr(const std::optional<at::Tensor>& t, const at::Tensor& q, int64_t n, const char* name) {
  if (!t.has_value()) return nullptr;
  const at::ScalarType want = std::is_same_v<T, float> ? at::kFloat : at::kInt;
  TORCH_CHECK_VALUE(t->is_cuda() && t->device() == q.device() && t->scalar_type() == want && t->dim() == 1 &&
                        t->size(0) == n && t->is_contiguous(),
                    name, " must be a contiguous ", want, " vector of ", n, " values on ", q.device());
  return static_cast<const T*>(t->data_ptr());
}

// Attention with masks, score modifiers and grouped key/value heads (npub200_attention_masked): (B, S, H*d) tensors, or
// (B, H, S, d) when head-major. Defaults: kv_heads 0 what k's shape says, scale 0 d^-0.5, no q_start the last query at
// the last key, softcap 0 none. The workspace of split keys comes from torch's allocator, one per call.
at::Tensor attention_masked(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                            const std::optional<at::Tensor>& out_arg, std::optional<at::ScalarType> out_dtype,
                            int64_t heads, int64_t kv_heads, bool head_major_in, bool head_major_out, double scale,
                            int64_t variant, bool causal, std::optional<int64_t> q_start,
                            const std::optional<at::Tensor>& q_starts,
                            int64_t prefix, const std::optional<at::Tensor>& prefixes,
                            const std::optional<at::Tensor>& kv_lens, const std::optional<at::Tensor>& doc_offsets,
                            double softcap, const std::optional<at::Tensor>& slopes,
                            const std::optional<at::Tensor>& distance_bias, const std::optional<at::Tensor>& mask) {
  check_operand(q, q, "q");
  check_operand(k, q, "k");
  check_operand(v, q, "v");
  TORCH_CHECK_VALUE(q.dim() == (head_major_in ? 4 : 3) && k.dim() == q.dim() && v.dim() == q.dim(),
                    "attention operands must be ", head_major_in ? "(B, H, S, d)" : "(B, S, H*d)");
  TORCH_CHECK_VALUE(heads > 0 && (head_major_in || q.size(2) % heads == 0), "q's last dimension is not a multiple of heads=",
                    heads);
  const int64_t B = q.size(0), Sq = q.size(head_major_in ? 2 : 1), Skv = k.size(head_major_in ? 2 : 1);
  const int64_t d = head_major_in ? q.size(3) : q.size(2) / heads;
  const int64_t Hk = head_major_in ? k.size(1) : (d > 0 && k.size(2) % d == 0 ? k.size(2) / d : 0);
  TORCH_CHECK_VALUE(Hk > 0 && heads % Hk == 0 && (kv_heads == 0 || kv_heads == Hk), "k/v hold ", Hk,
                    " heads: kv_heads must be that, and a divisor of heads=", heads, " (got ", kv_heads, ")");
  kv_heads = Hk;
  TORCH_CHECK_VALUE(k.size(0) == B && k.size(-1) == (head_major_in ? d : Hk * d) && v.sizes() == k.sizes(), "k/v shapes ",
                    k.sizes(), ", ", v.sizes(), " do not match q's ", q.sizes());
  check_layout(q, head_major_in, B, heads, Sq, d, 0, "q");
  check_layout(k, head_major_in, B, kv_heads, Skv, d, 0, "k");
  check_layout(v, head_major_in, B, kv_heads, Skv, d, 0, "v");
  const c10::cuda::CUDAGuard guard(q.device());
  at::Tensor out;
  if (out_arg.has_value()) {
    out = *out_arg;
    check_layout(out, head_major_out, B, heads, Sq, d, 0, "attention output");
    TORCH_CHECK_VALUE(out.is_cuda() && out.device() == q.device() && out.stride(-1) == 1,
                      "attention output must be a CUDA tensor on q's device with a contiguous last dimension");
  } else {
    const auto opts = q.options().dtype(out_dtype.value_or(at::kFloat));
    out = head_major_out ? at::empty({B, heads, Sq, d}, opts) : at::empty({B, Sq, heads * d}, opts);
  }
  const int out_code = dtype_code(out, "attention output");
  if (scale <= 0) {
    TORCH_CHECK_VALUE(scale == 0, "attention scale must be positive (got ", scale, ")");
    scale = 1.0 / std::sqrt(double(d));
  }
  npub200_attention_mods m = {};
  m.causal = causal ? 1 : 0;
  m.q_start = q_start.value_or(Skv - Sq);
  m.q_starts = vector_ptr<int32_t>(q_starts, q, B, "q_starts");
  m.prefix = prefix;
  m.prefixes = vector_ptr<int32_t>(prefixes, q, B, "prefixes");
  m.kv_lens = vector_ptr<int32_t>(kv_lens, q, B, "kv_lens");
  m.softcap = float(softcap);
  m.slopes = vector_ptr<float>(slopes, q, heads, "slopes");
  if (doc_offsets.has_value()) {
    const at::Tensor& t = *doc_offsets;
    TORCH_CHECK_VALUE(t.is_cuda() && t.device() == q.device() && t.scalar_type() == at::kInt && t.is_contiguous() &&
                          (t.dim() == 1 || (t.dim() == 2 && t.size(0) == B)) && t.size(-1) >= 1,
                      "doc_offsets must be a contiguous int32 [n + 1] or [B, n + 1] tensor on q's device");
    m.doc_offsets = static_cast<const int32_t*>(t.data_ptr());
    m.docs = t.size(-1) - 1;
    m.doc_stride = t.dim() == 2 ? t.size(1) : 0;
  }
  if (distance_bias.has_value()) {
    const at::Tensor& t = *distance_bias;
    TORCH_CHECK_VALUE(t.is_cuda() && t.device() == q.device() && t.scalar_type() == at::kFloat && t.is_contiguous() &&
                          t.dim() == 2 && t.size(0) == heads && t.size(1) % 2 == 1 && t.size(1) <= (1 << 25),
                      "distance_bias must be a contiguous f32 [heads, 2R + 1] tensor on q's device");
    m.distance_bias = static_cast<const float*>(t.data_ptr());
    m.max_distance = int32_t(t.size(1) / 2);
  }
  if (mask.has_value()) {
    const at::Tensor& t = *mask;
    TORCH_CHECK_VALUE(t.is_cuda() && t.device() == q.device() && (t.dim() == 4 || t.dim() == 2),
                      "mask must be a tensor of 2 or 4 dimensions on q's device");
    const int64_t off = t.dim() - 4;  // a 2-D mask is [Sq, Skv]
    const auto size = [&](int64_t i) { return i + off < 0 ? int64_t(1) : t.size(i + off); };
    const auto stride = [&](int64_t i) { return size(i) > 1 ? t.stride(i + off) : int64_t(0); };
    TORCH_CHECK_VALUE((size(0) == 1 || size(0) == B) && (size(1) == 1 || size(1) == heads) &&
                          (size(2) == 1 || size(2) == Sq) && size(3) == Skv && (Skv == 1 || t.stride(-1) == 1),
                      "mask ", t.sizes(), " does not broadcast to (", B, ", ", heads, ", ", Sq, ", ", Skv,
                      ") with contiguous keys");
    m.mask = t.data_ptr();
    m.mask_dtype = t.scalar_type() == at::kBool ? NPUB200_DTYPE_BOOL : dtype_code(t, "mask");
    m.mask_sb = stride(0);
    m.mask_sh = stride(1);
    m.mask_sq = stride(2);
  }
  size_t ws_bytes = 0;
  check_rc(npub200_attention_masked_workspace_size(B, heads, kv_heads, Sq, Skv, d, int(variant), &ws_bytes),
           "npub200::attention_masked");
  at::Tensor ws;
  if (ws_bytes) ws = at::empty({int64_t(ws_bytes)}, q.options().dtype(at::kByte));
  int64_t qs[3], ks[3], vs[3], os[3];
  bsh_strides(q, head_major_in, d, &qs[0], &qs[1], &qs[2]);
  bsh_strides(k, head_major_in, d, &ks[0], &ks[1], &ks[2]);
  bsh_strides(v, head_major_in, d, &vs[0], &vs[1], &vs[2]);
  bsh_strides(out, head_major_out, d, &os[0], &os[1], &os[2]);
  check_rc(npub200_attention_masked(q.data_ptr(), qs[0], qs[1], qs[2], k.data_ptr(), ks[0], ks[1], ks[2], v.data_ptr(),
                                    vs[0], vs[1], vs[2], out.data_ptr(), os[0], os[1], os[2], out_code, B,
                                    heads, kv_heads, Sq, Skv, d, float(scale), &m, ws_bytes ? ws.data_ptr() : nullptr,
                                    ws_bytes, int(variant), stream_of(q)),
           "npub200::attention_masked");
  return out;
}

// An uninitialised CUDA tensor, and a workspace of the current stream's, without the way through the dispatcher (1 us each on the
// host, which is what a small call waits for).
at::Tensor empty_like_device(at::IntArrayRef size, at::ScalarType dtype, const at::Tensor& ref) {
  return at::Tensor(at::detail::empty_cuda(size, dtype, ref.device(), std::nullopt));
}
c10::DataPtr workspace(size_t bytes) { return c10::cuda::CUDACachingAllocator::get()->allocate(bytes); }

// (batch, seq, head) element strides of a tensor of heads, and the checks of its shape: (B, S, heads * d), or (B, heads, S, d)
// when head-major. A dimension of one element has no stride of its own.
struct HeadRows {
  int64_t sb, ss, sh;
};
HeadRows head_rows(const at::Tensor& t, const at::Tensor& ref, bool head_major, int64_t heads, int64_t d, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.device() == ref.device(), name, " must be a CUDA tensor on ", ref.device());
  const bool ok = head_major ? t.dim() == 4 && t.size(1) == heads && t.size(3) == d
                             : t.dim() == 3 && t.size(2) == heads * d;
  TORCH_CHECK_VALUE(ok && heads > 0, name, " must be ", head_major ? "(B, heads, S, d)" : "(B, S, heads*d)", " with ", heads,
                    " heads of ", d, ", got ", t.sizes());
  TORCH_CHECK_VALUE(t.size(-1) <= 1 || t.stride(-1) == 1, name, " must have a contiguous last dimension");
  const auto stride = [&](int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : int64_t(0); };
  return head_major ? HeadRows{stride(0), stride(2), stride(1)} : HeadRows{stride(0), stride(1), d};
}

// Positions of the tokens: none (a plain start), int32 [B] (of each sequence's first token) or int32 [B, S].
struct Positions {
  const int32_t* starts = nullptr;
  const int32_t* each = nullptr;
  int64_t sb = 0, ss = 0;
};
Positions positions_of(const std::optional<at::Tensor>& t, const at::Tensor& x, int64_t B, int64_t S) {
  Positions p;
  if (!t.has_value()) return p;
  TORCH_CHECK_VALUE(t->is_cuda() && t->device() == x.device() && t->scalar_type() == at::kInt &&
                        ((t->dim() == 1 && t->size(0) == B && (B <= 1 || t->stride(0) == 1)) ||
                         (t->dim() == 2 && t->size(0) == B && t->size(1) == S)),
                    "positions must be int32, contiguous [", B, "] or [", B, ", ", S, "], on ", x.device(), ", got ",
                    t->scalar_type(), " ", t->sizes(), " on ", t->device());
  const int32_t* ptr = static_cast<const int32_t*>(t->data_ptr());
  if (t->dim() == 1) {
    p.starts = ptr;
  } else {
    p.each = ptr;
    p.sb = t->stride(0);
    p.ss = t->stride(1);
  }
  return p;
}

npub200_rotation rotation_of(const at::Tensor& freqs, const at::Tensor& x, bool interleaved, bool inverse, double magnitude) {
  TORCH_CHECK_VALUE(freqs.is_cuda() && freqs.device() == x.device() && freqs.scalar_type() == at::kDouble &&
                        freqs.dim() == 1 && freqs.is_contiguous(),
                    "freqs must be a contiguous float64 vector (radians a position of each pair) on ", x.device(), ", got ",
                    freqs.scalar_type(), " ", freqs.sizes(), " on ", freqs.device());
  npub200_rotation r = {};
  r.freqs = static_cast<const double*>(freqs.data_ptr());
  r.rot_dim = 2 * freqs.numel();
  r.interleaved = interleaved ? 1 : 0;
  r.inverse = inverse ? 1 : 0;
  r.magnitude = float(magnitude);
  return r;
}

// The bytes of a tensor of an operator (up to four dimensions).
npub200::ByteRuns runs_of(const at::Tensor& t) {
  TORCH_CHECK_VALUE(t.dim() <= npub200::kOverlapDims, "a tensor of ", t.dim(), " dimensions");
  return npub200::byte_runs(t.data_ptr(), t.element_size(), int(t.dim()), t.sizes().data(), t.strides().data());
}

// Whether b is a itself: the same elements in the same places, so that who reads one of them is who writes it.
bool same_tensor(const at::Tensor& a, const at::Tensor& b) {
  if (a.data_ptr() != b.data_ptr() || a.scalar_type() != b.scalar_type() || a.sizes() != b.sizes()) return false;
  for (int64_t i = 0; i < a.dim(); ++i)
    if (a.size(i) > 1 && a.stride(i) != b.stride(i)) return false;
  return true;
}

// A tensor that a kernel writes: no element twice, and `from` itself or nothing of it.
void check_written(const at::Tensor& t, const char* name, const at::Tensor* from = nullptr) {
  TORCH_CHECK_VALUE(at::has_internal_overlap(t) != at::MemOverlap::Yes && !npub200::bytes_repeat(runs_of(t)), name,
                    " must not hold an element twice");
  TORCH_CHECK_VALUE(from == nullptr || same_tensor(t, *from) || !npub200::bytes_overlap(runs_of(t), runs_of(*from)), name,
                    " must be the input itself or share no element with it: they overlap");
}

// Two tensors of which one is written while the other is read, or both are written: nothing in common.
void check_apart(const npub200::ByteRuns& a, const npub200::ByteRuns& b, const char* names) {
  TORCH_CHECK_VALUE(!npub200::bytes_overlap(a, b), names, " must not overlap");
}

// What was written has another version now, by which autograd and graph tools tell (inference tensors have none).
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Rotary positions (npub200_rope): x (B, S, heads * d), or (B, heads, S, d) when head-major, like the result.
at::Tensor rope(const at::Tensor& x, const at::Tensor& freqs, int64_t heads, const std::optional<at::Tensor>& out_arg,
                std::optional<at::ScalarType> out_dtype, int64_t start, const std::optional<at::Tensor>& positions,
                bool interleaved, double magnitude, bool inverse, bool head_major) {
  TORCH_CHECK_VALUE(heads > 0 && x.dim() == (head_major ? 4 : 3) && (head_major || x.size(2) % heads == 0),
                    "x must be ", head_major ? "(B, heads, S, d)" : "(B, S, heads*d)", " with heads=", heads, ", got ",
                    x.sizes());
  const int64_t d = head_major ? x.size(3) : x.size(2) / heads;
  const int64_t B = x.size(0), S = x.size(head_major ? 2 : 1);
  const HeadRows xr = head_rows(x, x, head_major, heads, d, "x");
  const int x_code = dtype_code(x, "x");
  const npub200_rotation r = rotation_of(freqs, x, interleaved, inverse, magnitude);
  const Positions p = positions_of(positions, x, B, S);
  const c10::cuda::CUDAGuard guard(x.device());
  at::Tensor out;
  if (out_arg.has_value()) {
    out = *out_arg;
    TORCH_CHECK_VALUE(out.sizes() == x.sizes(), "out must have x's shape ", x.sizes(), ", got ", out.sizes());
    check_written(out, "out", &x);
  } else {
    out = empty_like_device(x.sizes(), out_dtype.value_or(x.scalar_type()), x);
  }
  const HeadRows orr = head_rows(out, x, head_major, heads, d, "out");
  check_rc(npub200_rope(x.data_ptr(), xr.sb, xr.ss, xr.sh, x_code, out.data_ptr(), orr.sb, orr.ss, orr.sh,
                        dtype_code(out, "out"), B, S, heads, d, &r, start, p.starts, p.each, p.sb, p.ss, stream_of(x)),
           "npub200::rope");
  if (out_arg.has_value()) written(out);
  return out;
}

// The pages of a cache: [pages, page_size, kv_heads, d] bf16 views of any strides, and each sequence's table of them.
npub200_paged_cache cache_of(const at::Tensor& k_pages, const at::Tensor& v_pages, const at::Tensor& table, int64_t B) {
  TORCH_CHECK_VALUE(k_pages.is_cuda() && k_pages.dim() == 4 && k_pages.scalar_type() == at::kBFloat16 &&
                        v_pages.device() == k_pages.device() && v_pages.scalar_type() == at::kBFloat16 &&
                        v_pages.sizes() == k_pages.sizes(),
                    "k_pages and v_pages must be bf16 CUDA tensors [pages, page_size, kv_heads, d] of one shape, got ",
                    k_pages.scalar_type(), " ", k_pages.sizes(), " and ", v_pages.scalar_type(), " ", v_pages.sizes());
  TORCH_CHECK_VALUE(k_pages.size(3) <= 1 || (k_pages.stride(3) == 1 && v_pages.stride(3) == 1),
                    "k_pages and v_pages must have a contiguous last dimension");
  TORCH_CHECK_VALUE(table.is_cuda() && table.device() == k_pages.device() && table.scalar_type() == at::kInt &&
                        table.dim() == 2 && table.size(0) == B && (table.size(1) <= 1 || table.stride(1) == 1),
                    "page_table must be int32 [", B, ", pages] with contiguous rows on ", k_pages.device(), ", got ",
                    table.scalar_type(), " ", table.sizes(), " on ", table.device());
  const auto stride = [](const at::Tensor& t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : int64_t(0); };
  npub200_paged_cache c = {};
  c.k = k_pages.data_ptr();
  c.k_sp = stride(k_pages, 0), c.k_ss = stride(k_pages, 1), c.k_sh = stride(k_pages, 2);
  c.v = v_pages.data_ptr();
  c.v_sp = stride(v_pages, 0), c.v_ss = stride(v_pages, 1), c.v_sh = stride(v_pages, 2);
  c.pages = k_pages.size(0);
  c.page_size = k_pages.size(1);
  c.kv_heads = k_pages.size(2);
  c.head_dim = k_pages.size(3);
  c.table = static_cast<const int32_t*>(table.data_ptr());
  c.table_stride = stride(table, 0);
  c.table_width = table.size(1);
  return c;
}

// Appends new keys and values to the pages, keys and queries rotated on the way (npub200_paged_append). Returns the rotated
// queries, or nothing without them.
std::optional<at::Tensor> paged_append(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_pages,
                                       const at::Tensor& v_pages, const at::Tensor& page_table, const at::Tensor& starts,
                                       const std::optional<at::Tensor>& counts, const std::optional<at::Tensor>& q,
                                       int64_t heads, const std::optional<at::Tensor>& q_out,
                                       const std::optional<at::Tensor>& freqs, bool interleaved, double magnitude,
                                       bool head_major) {
  TORCH_CHECK_VALUE(k.dim() == (head_major ? 4 : 3), "k must be ", head_major ? "(B, heads, S, d)" : "(B, S, heads*d)",
                    ", got ", k.sizes());
  const int64_t B = k.size(0), S = k.size(head_major ? 2 : 1);
  const npub200_paged_cache c = cache_of(k_pages, v_pages, page_table, B);
  const HeadRows kr = head_rows(k, k_pages, head_major, c.kv_heads, c.head_dim, "k");
  const HeadRows vr = head_rows(v, k_pages, head_major, c.kv_heads, c.head_dim, "v");
  const int code = dtype_code(k, "k");
  TORCH_CHECK_VALUE(v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type(), "v must have k's shape and type, got ",
                    v.scalar_type(), " ", v.sizes());
  check_written(k_pages, "k_pages");
  check_written(v_pages, "v_pages");
  const npub200::ByteRuns kp = runs_of(k_pages), vp = runs_of(v_pages), k_runs = runs_of(k), v_runs = runs_of(v);
  check_apart(kp, vp, "k_pages and v_pages");
  check_apart(kp, k_runs, "k_pages and k");
  check_apart(kp, v_runs, "k_pages and v");
  check_apart(vp, k_runs, "v_pages and k");
  check_apart(vp, v_runs, "v_pages and v");
  const int32_t* starts_ptr = vector_ptr<int32_t>(starts, k_pages, B, "starts");
  const int32_t* counts_ptr = vector_ptr<int32_t>(counts, k_pages, B, "counts");
  npub200_rotation r = {};
  if (freqs.has_value()) r = rotation_of(*freqs, k_pages, interleaved, false, magnitude);
  const c10::cuda::CUDAGuard guard(k_pages.device());
  std::optional<at::Tensor> out;
  HeadRows qr = {}, orr = {};
  if (q.has_value()) {
    TORCH_CHECK_VALUE(freqs.has_value(), "q is taken to be rotated: it needs freqs");
    qr = head_rows(*q, k_pages, head_major, heads, c.head_dim, "q");
    TORCH_CHECK_VALUE(q->size(0) == B && q->size(head_major ? 2 : 1) == S && q->scalar_type() == k.scalar_type(),
                      "q must have k's batch, tokens and type, got ", q->scalar_type(), " ", q->sizes());
    const npub200::ByteRuns q_runs = runs_of(*q);
    check_apart(kp, q_runs, "k_pages and q");
    check_apart(vp, q_runs, "v_pages and q");
    if (q_out.has_value()) {
      TORCH_CHECK_VALUE(q_out->sizes() == q->sizes() && q_out->scalar_type() == at::kBFloat16,
                        "q_out must be bf16 with q's shape ", q->sizes(), ", got ", q_out->scalar_type(), " ", q_out->sizes());
      check_written(*q_out, "q_out", &*q);
      const npub200::ByteRuns out_runs = runs_of(*q_out);
      check_apart(out_runs, k_runs, "q_out and k");
      check_apart(out_runs, v_runs, "q_out and v");
      check_apart(out_runs, kp, "q_out and k_pages");
      check_apart(out_runs, vp, "q_out and v_pages");
      out = *q_out;
    } else {
      out = empty_like_device(q->sizes(), at::kBFloat16, k_pages);
    }
    orr = head_rows(*out, k_pages, head_major, heads, c.head_dim, "q_out");
  } else {
    TORCH_CHECK_VALUE(!q_out.has_value(), "q_out is given without q");
  }
  check_rc(npub200_paged_append(q.has_value() ? q->data_ptr() : nullptr, qr.sb, qr.ss, qr.sh,
                                q.has_value() ? out->data_ptr() : nullptr, orr.sb, orr.ss, orr.sh, q.has_value() ? heads : 0,
                                k.data_ptr(), kr.sb, kr.ss, kr.sh, v.data_ptr(), vr.sb, vr.ss, vr.sh, code, &c, starts_ptr,
                                counts_ptr, B, S, freqs.has_value() ? &r : nullptr, stream_of(k_pages)),
           "npub200::paged_append");
  written(k_pages);
  written(v_pages);
  if (q_out.has_value()) written(*out);
  return out;
}

// Attention over a cache in pages (npub200_attention_paged). Defaults: scale 0 d^-0.5, softcap 0 none. The workspace comes
// from torch's allocator, one per call.
at::Tensor attention_paged(const at::Tensor& q, const at::Tensor& k_pages, const at::Tensor& v_pages,
                           const at::Tensor& page_table, const at::Tensor& kv_lens, const std::optional<at::Tensor>& out_arg,
                           std::optional<at::ScalarType> out_dtype, int64_t heads, double scale, bool causal,
                           const std::optional<at::Tensor>& q_starts, double softcap,
                           const std::optional<at::Tensor>& slopes, bool head_major_in, bool head_major_out,
                           int64_t variant) {
  TORCH_CHECK_VALUE(q.scalar_type() == at::kBFloat16 && q.dim() == (head_major_in ? 4 : 3), "q must be bf16 ",
                    head_major_in ? "(B, heads, S, d)" : "(B, S, heads*d)", ", got ", q.scalar_type(), " ", q.sizes());
  const int64_t B = q.size(0), S = q.size(head_major_in ? 2 : 1);
  const npub200_paged_cache c = cache_of(k_pages, v_pages, page_table, B);
  const int64_t d = c.head_dim;
  const HeadRows qr = head_rows(q, k_pages, head_major_in, heads, d, "q");
  TORCH_CHECK_VALUE(scale >= 0, "attention scale must be positive (got ", scale, ")");
  if (scale == 0) scale = 1.0 / std::sqrt(double(d));
  TORCH_CHECK_VALUE(softcap == 0 || float(softcap) != 0, "softcap must be 0 (none) or within [1e-30, 1e30] (got ", softcap, ")");
  const int tiles = int(std::clamp<int64_t>(variant, -1, INT32_MAX));  // (what an int does not hold stays out of range)
  const c10::cuda::CUDAGuard guard(k_pages.device());
  at::Tensor out;
  const auto shape = head_major_out ? std::vector<int64_t>{B, heads, S, d} : std::vector<int64_t>{B, S, heads * d};
  if (out_arg.has_value()) {
    out = *out_arg;
    TORCH_CHECK_VALUE(out.sizes() == at::IntArrayRef(shape), "attention output must be ", at::IntArrayRef(shape), ", got ",
                      out.sizes());
    check_written(out, "out", &q);
    const npub200::ByteRuns out_runs = runs_of(out);
    check_apart(out_runs, runs_of(k_pages), "out and k_pages");
    check_apart(out_runs, runs_of(v_pages), "out and v_pages");
  } else {
    out = empty_like_device(shape, out_dtype.value_or(at::kFloat), k_pages);
  }
  const HeadRows orr = head_rows(out, k_pages, head_major_out, heads, d, "attention output");
  const int out_code = dtype_code(out, "attention output");
  const int32_t* lens = vector_ptr<int32_t>(kv_lens, k_pages, B, "kv_lens");
  const int32_t* starts = vector_ptr<int32_t>(q_starts, k_pages, B, "q_start");
  const float* slopes_ptr = vector_ptr<float>(slopes, k_pages, heads, "slopes");
  if (B == 0 || S == 0) return out;
  size_t ws_bytes = 0;
  check_rc(npub200_attention_paged_workspace_size(heads, c.kv_heads, S, d, &ws_bytes), "npub200::attention_paged");
  const c10::DataPtr ws = workspace(ws_bytes);  // (of this call's own: calls on other streams and captured graphs share none)
  check_rc(npub200_attention_paged(q.data_ptr(), qr.sb, qr.ss, qr.sh, &c, lens, out.data_ptr(), orr.sb, orr.ss, orr.sh,
                                   out_code, B, heads, S, float(scale), causal ? 1 : 0, starts, float(softcap), slopes_ptr,
                                   ws.get(), ws_bytes, tiles, stream_of(k_pages)),
           "npub200::attention_paged");
  if (out_arg.has_value()) written(out);
  return out;
}

}  // namespace

TORCH_LIBRARY(npub200, m) {
  m.def("gemm(Tensor x, Tensor w, Tensor? bias=None, Tensor? out=None, int variant=0, ScalarType? out_dtype=None, "
        "int weight_handle=0, Tensor? residual=None, int activation=0) -> Tensor");
  m.def("attention(Tensor q, Tensor k, Tensor v, Tensor? out, int B, int H, int Sq, int Skv, int d, "
        "int q_row_stride, int kv_row_stride, int o_row_stride, bool head_major_in, bool head_major_out, "
        "float scale, int variant, ScalarType? out_dtype=None) -> Tensor");
  m.def("attention_masked(Tensor q, Tensor k, Tensor v, Tensor? out, ScalarType? out_dtype, int heads, int kv_heads=0, "
        "bool head_major_in=False, bool head_major_out=False, float scale=0., int variant=0, bool causal=False, "
        "int? q_start=None, Tensor? q_starts=None, int prefix=0, Tensor? prefixes=None, Tensor? kv_lens=None, "
        "Tensor? doc_offsets=None, float softcap=0., Tensor? slopes=None, Tensor? distance_bias=None, "
        "Tensor? mask=None) -> Tensor");
  m.def("rope(Tensor x, Tensor freqs, int heads, Tensor(a!)? out=None, ScalarType? out_dtype=None, int start=0, "
        "Tensor? positions=None, bool interleaved=False, float magnitude=1., bool inverse=False, "
        "bool head_major=False) -> Tensor(a!)");
  m.def("paged_append(Tensor k, Tensor v, Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor page_table, Tensor starts, "
        "Tensor? counts=None, Tensor? q=None, int heads=0, Tensor(c!)? q_out=None, Tensor? freqs=None, "
        "bool interleaved=False, float magnitude=1., bool head_major=False) -> Tensor(c!)?");
  m.def("attention_paged(Tensor q, Tensor k_pages, Tensor v_pages, Tensor page_table, Tensor kv_lens, Tensor(a!)? out, "
        "ScalarType? out_dtype, int heads, float scale=0., bool causal=True, Tensor? q_starts=None, float softcap=0., "
        "Tensor? slopes=None, bool head_major_in=False, bool head_major_out=False, int variant=0) -> Tensor(a!)");
}

TORCH_LIBRARY_IMPL(npub200, CUDA, m) {
  m.impl("gemm", &gemm);
  m.impl("attention", &attention);
  m.impl("attention_masked", &attention_masked);
  m.impl("rope", &rope);
  m.impl("paged_append", &paged_append);
  m.impl("attention_paged", &attention_paged);
}
