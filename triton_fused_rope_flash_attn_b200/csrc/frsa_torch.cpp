// PyTorch C++ extension over the C ABI (include/frsa.h): the host side of the
// product path. It does in C++ what the reference's autograd wrapper does in
// Python before its Triton launches (fa_rope_full .py:1011-1138): shape and
// dtype checks, output and scratch allocation (torch's caching allocator, on
// the tensors' device), and the launch on torch's current stream. The C-ABI
// entry points are bound at run time from the loaded libfrsa.so (bind()), so
// this module has no link-time dependency on it.
//
// Each function returns its tensors plus the FRSA status code; the Python
// layer turns a non-zero code into FrsaError, as it does for direct C-ABI
// calls.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cmath>
#include <cstdint>
#include <map>
#include <mutex>
#include <utility>

#include "frsa.h"

namespace {

using FwdFn = int (*)(const frsa_attn_args*, void*);
using WsFn = size_t (*)(const frsa_attn_args*);

FwdFn g_fwd = nullptr;
FwdFn g_bwd = nullptr;
WsFn g_ws = nullptr;

void bind(int64_t fwd, int64_t bwd, int64_t ws) {
  g_fwd = reinterpret_cast<FwdFn>(fwd);
  g_bwd = reinterpret_cast<FwdFn>(bwd);
  g_ws = reinterpret_cast<WsFn>(ws);
}

int32_t dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return FRSA_DTYPE_BF16;
    case at::kHalf: return FRSA_DTYPE_F16;
    case at::kFloat: return FRSA_DTYPE_F32;
    default: TORCH_CHECK_TYPE(false, "unsupported compute dtype ", t.scalar_type());
  }
  return -1;
}

void check_inputs(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                  const at::Tensor& cosp, const at::Tensor& sinp, int64_t flags) {
  TORCH_CHECK(g_fwd && g_bwd && g_ws, "frsa extension: C ABI not bound (call bind first)");
  TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor (there is no CPU path)");
  TORCH_CHECK(q.dim() == 4, "q must be [B, H, N, D]");
  TORCH_CHECK(k.sizes() == q.sizes() && v.sizes() == q.sizes(), "q, k, v shapes differ");
  TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                   "q, k, v dtypes differ");
  TORCH_CHECK(k.device() == q.device() && v.device() == q.device(), "q, k, v devices differ");
  if (flags & FRSA_FLAG_NO_ROPE) return;   // tables unused
  TORCH_CHECK_TYPE(cosp.scalar_type() == at::kFloat && sinp.scalar_type() == at::kFloat,
                   "COSP/SINP must be float32");
  TORCH_CHECK(cosp.device() == q.device() && sinp.device() == q.device(),
              "RoPE tables must be on the same device as Q");
  TORCH_CHECK(cosp.dim() == 2 && cosp.sizes() == sinp.sizes(), "COSP/SINP must be [N_pos, D/2]");
}

// q, k and v are read in place through strided TMA maps when their d stride
// is 1, their other strides are multiples of 16 bytes and their data 16-byte
// aligned (e.g. the q, k, v views of a [B, N, 3, H, D] projection output);
// otherwise a contiguous copy is made.
bool tma_strided_ok(const at::Tensor& t) {
  if (t.stride(3) != 1) return false;
  const int64_t e = t.element_size();
  for (int d = 0; d < 3; ++d)
    if (t.size(d) > 1 && (t.stride(d) < 1 || (t.stride(d) * e) % 16 != 0)) return false;
  return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0;
}

at::Tensor readable(const at::Tensor& t) { return tma_strided_ok(t) ? t : t.contiguous(); }

void set_strides(int64_t* dst, const at::Tensor& t) {
  if (t.is_contiguous()) {
    dst[0] = dst[1] = dst[2] = 0;
    return;
  }
  // Size-1 dimensions may carry any stride; give them a valid one.
  const int64_t e = t.element_size(), unit = 16 / e;
  for (int d = 0; d < 3; ++d) dst[d] = (t.size(d) > 1) ? t.stride(d) : unit;
}

void fill_shape(frsa_attn_args& a, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                const at::Tensor& cosp, const at::Tensor& sinp, bool has_cls, double scale,
                int64_t flags) {
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  set_strides(a.q_strides, q);
  set_strides(a.k_strides, k);
  set_strides(a.v_strides, v);
  a.flags = static_cast<int32_t>(flags);
  const bool rope = (flags & FRSA_FLAG_NO_ROPE) == 0;
  a.cosp = rope ? cosp.data_ptr<float>() : nullptr;
  a.sinp = rope ? sinp.data_ptr<float>() : nullptr;
  a.B = q.size(0);
  a.H = q.size(1);
  a.N = q.size(2);
  a.D = q.size(3);
  a.n_pos = rope ? cosp.size(0) : 0;
  a.has_cls = has_cls ? 1 : 0;
  a.io_dtype = a.compute_dtype = dtype_code(q);
  a.scale = scale > 0 ? static_cast<float>(scale) : static_cast<float>(1.0 / std::sqrt(double(a.D)));
}

// O and LSE of softmax(R(q) R(k)^T * scale) v. scale <= 0: 1/sqrt(D).
std::tuple<at::Tensor, at::Tensor, int64_t> fwd(const at::Tensor& q_in, const at::Tensor& k_in,
                                                const at::Tensor& v_in, const at::Tensor& cosp_in,
                                                const at::Tensor& sinp_in, bool has_cls,
                                                double scale, int64_t flags) {
  check_inputs(q_in, k_in, v_in, cosp_in, sinp_in, flags);
  const c10::cuda::CUDAGuard guard(q_in.device());
  const at::Tensor q = readable(q_in), k = readable(k_in), v = readable(v_in);
  const bool rope = (flags & FRSA_FLAG_NO_ROPE) == 0;
  const at::Tensor cosp = rope ? cosp_in.contiguous() : cosp_in;
  const at::Tensor sinp = rope ? sinp_in.contiguous() : sinp_in;
  at::Tensor o = at::empty(q.sizes(), q.options());
  at::Tensor lse = at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat));
  frsa_attn_args a{};
  fill_shape(a, q, k, v, cosp, sinp, has_cls, scale, flags);
  a.o = o.data_ptr();
  a.lse = lse.data_ptr<float>();
  const int rc = g_fwd(&a, at::cuda::getCurrentCUDAStream().stream());
  return {o, lse, rc};
}

// dQ, dK, dV (and Delta into delta_out when given). scale <= 0: 1/sqrt(D).
std::tuple<at::Tensor, at::Tensor, at::Tensor, int64_t> bwd(
    const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in,
    const at::Tensor& o_in, const at::Tensor& lse_in, const at::Tensor& do_in,
    const at::Tensor& cosp_in, const at::Tensor& sinp_in, bool has_cls,
    const c10::optional<at::Tensor>& delta_out, double scale, int64_t flags) {
  check_inputs(q_in, k_in, v_in, cosp_in, sinp_in, flags);
  TORCH_CHECK(o_in.sizes() == q_in.sizes() && do_in.sizes() == q_in.sizes(),
              "o and dO must have q's shape");
  TORCH_CHECK_TYPE(o_in.scalar_type() == q_in.scalar_type() &&
                       do_in.scalar_type() == q_in.scalar_type(),
                   "o and dO must have q's dtype");
  TORCH_CHECK_TYPE(lse_in.scalar_type() == at::kFloat, "lse must be float32");
  const c10::cuda::CUDAGuard guard(q_in.device());
  const at::Tensor q = readable(q_in), k = readable(k_in), v = readable(v_in);
  const at::Tensor o = o_in.contiguous(), lse = lse_in.contiguous(), d_o = do_in.contiguous();
  const bool rope = (flags & FRSA_FLAG_NO_ROPE) == 0;
  const at::Tensor cosp = rope ? cosp_in.contiguous() : cosp_in;
  const at::Tensor sinp = rope ? sinp_in.contiguous() : sinp_in;
  at::Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()),
             dv = at::empty(v.sizes(), v.options());
  frsa_attn_args a{};
  fill_shape(a, q, k, v, cosp, sinp, has_cls, scale, flags);
  a.o = const_cast<void*>(o.data_ptr());
  a.lse = const_cast<float*>(lse.data_ptr<float>());
  a.d_o = d_o.data_ptr();
  a.dq = dq.data_ptr();
  a.dk = dk.data_ptr();
  a.dv = dv.data_ptr();
  if (delta_out.has_value()) {
    TORCH_CHECK(delta_out->is_contiguous() && delta_out->scalar_type() == at::kFloat &&
                    delta_out->numel() == q.size(0) * q.size(1) * q.size(2),
                "delta_out must be a contiguous float32 [B, H, N] tensor");
    a.delta = delta_out->data_ptr<float>();
  }
  at::Tensor ws;
  const size_t ws_bytes = g_ws(&a);
  if (ws_bytes > 0) {
    ws = at::empty({static_cast<int64_t>((ws_bytes + 3) / 4)}, q.options().dtype(at::kFloat));
    a.workspace = ws.data_ptr();
    a.workspace_bytes = ws_bytes;
  }
  const int rc = g_bwd(&a, at::cuda::getCurrentCUDAStream().stream());
  return {dq, dk, dv, rc};
}

// ---------------------------------------------------------------- serving

using AppendFn = int (*)(const frsa_paged_append_args*, void*);
using DecodeFn = int (*)(const frsa_paged_decode_args*, void*);
using DecodeWsFn = size_t (*)();
using PromptFn = int (*)(const frsa_prompt_args*, void*);

AppendFn g_append = nullptr;
DecodeFn g_decode = nullptr;
DecodeWsFn g_decode_ws = nullptr;
PromptFn g_prompt = nullptr;

void bind_serving(int64_t append, int64_t decode, int64_t decode_ws, int64_t prompt) {
  g_append = reinterpret_cast<AppendFn>(append);
  g_decode = reinterpret_cast<DecodeFn>(decode);
  g_decode_ws = reinterpret_cast<DecodeWsFn>(decode_ws);
  g_prompt = reinterpret_cast<PromptFn>(prompt);
}

int32_t serve_dtype(const at::Tensor& t) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf,
                   "the serving operators take bfloat16 or float16, got ", t.scalar_type());
  return t.scalar_type() == at::kBFloat16 ? FRSA_DTYPE_BF16 : FRSA_DTYPE_F16;
}

// Neither a gradient nor a forward-mode tangent is asked of a tensor.
void check_no_grad(const at::Tensor& t, const char* name) {
  TORCH_CHECK(!(t.requires_grad() && at::GradMode::is_enabled()), name,
              " requires a gradient: the serving operators have no backward, call them under "
              "torch.no_grad()");
  TORCH_CHECK(!t._fw_grad(/*level=*/0).defined(), name,
              " has a forward-mode tangent: the serving operators have no derivative");
}

// A [tokens, heads, D] tensor: on q's device, of q's type, without derivatives.
void check_tokens(const at::Tensor& t, const at::Tensor& q, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == q.device(), name,
              " must be a CUDA tensor on q's device (there is no CPU path)");
  TORCH_CHECK(t.dim() == 3, name, " must be [tokens, heads, D]");
  TORCH_CHECK_TYPE(t.scalar_type() == q.scalar_type(), name, " must have q's dtype");
  TORCH_CHECK(t.size(2) == q.size(2), name, " must have q's head dim");
  check_no_grad(t, name);
}

void check_cache(const at::Tensor& c, const at::Tensor& q, const at::Tensor& k_cache,
                 const char* name) {
  TORCH_CHECK(c.is_cuda() && c.device() == q.device(), name,
              " must be a CUDA tensor on q's device (there is no CPU path)");
  TORCH_CHECK(c.dim() == 4 && c.size(3) == q.size(2), name,
              " must be [pages, kv heads, page_size, D] with q's head dim");
  TORCH_CHECK_TYPE(c.scalar_type() == q.scalar_type(), name, " must have q's dtype");
  TORCH_CHECK(c.sizes() == k_cache.sizes() && c.strides() == k_cache.strides(),
              "k_cache and v_cache must have the same shape and strides");
  TORCH_CHECK(c.stride(3) == 1 && tma_strided_ok(c), name,
              " must have a unit d stride, other strides that are multiples of 16 bytes and "
              "16-byte aligned data");
  check_no_grad(c, name);
}

// An int32 index array on q's device, contiguous.
at::Tensor index_array(const at::Tensor& t, const at::Tensor& q, int64_t n, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == q.device(), name, " must be on q's device");
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt, name, " must be int32");
  TORCH_CHECK(t.dim() == 1 && (n < 0 || t.size(0) == n), name, " has the wrong shape");
  return t.contiguous();
}

at::Tensor table_array(const at::Tensor& t, const at::Tensor& q, int64_t B) {
  TORCH_CHECK(t.is_cuda() && t.device() == q.device(), "block_table must be on q's device");
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt, "block_table must be int32");
  TORCH_CHECK(t.dim() == 2 && t.size(0) == B && t.size(1) >= 1,
              "block_table must be [sequences, pages per sequence]");
  return t.stride(1) == 1 || t.size(1) == 1 ? t : t.contiguous();
}

// Strided [tokens, heads, D] rows are read in place where 16-byte loads and
// TMA can address them, otherwise copied once.
at::Tensor readable_tokens(const at::Tensor& t) {
  if (t.is_contiguous() && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0) return t;
  bool ok = t.stride(2) == 1 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0;
  for (int d = 0; d < 2; ++d) ok = ok && (t.size(d) <= 1 || (t.stride(d) > 0 && t.stride(d) % 8 == 0));
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

// (first, second) strides of a tensor's leading dimensions; an extent of one
// may carry any stride, so it gets the packed one.
template <int N>
void lead_strides(int64_t (&dst)[N], const at::Tensor& t) {
  int64_t packed = t.size(N);
  for (int d = N - 1; d >= 0; --d) {
    dst[d] = t.size(d) > 1 ? t.stride(d) : packed;
    packed *= t.size(d);
  }
}

// A kernel has written t: as torch's in-place operations do, raise its version
// (an inference tensor has none).
void mark_written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// An output of q's type (or `type`) on q's device, without the dispatcher.
at::Tensor output(at::IntArrayRef sizes, const at::Tensor& q, c10::optional<at::ScalarType> type = {}) {
  return at::detail::empty_cuda(sizes, type.value_or(q.scalar_type()), q.device(), c10::nullopt);
}

float scale_of(const c10::optional<double>& scale, int64_t D) {
  const float s = static_cast<float>(scale.has_value() ? *scale : 1.0 / std::sqrt(double(D)));
  // (the kernels' exponentials are to the base 2)
  TORCH_CHECK_VALUE(s > 0 && std::isfinite(s * 1.4426950408889634f),
                    "scale must be positive and finite in float32");
  return s;
}

// The split decode's scratch: one per (device, stream), made and zeroed on its
// first use there and left ready by every call, so calls on one stream share
// it in stream order. While a graph is captured each call gets its own (its
// zeroing is captured with it). Kept until the process ends.
at::Tensor decode_workspace(const at::Tensor& q, c10::cuda::CUDAStream stream) {
  const auto opts = q.options().dtype(at::kByte);
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None)
    return at::zeros({static_cast<int64_t>(g_decode_ws())}, opts);
  static std::mutex* mu = new std::mutex;
  static auto* kept = new std::map<std::pair<int, cudaStream_t>, at::Tensor>;
  std::lock_guard<std::mutex> lock(*mu);
  at::Tensor& ws = (*kept)[{static_cast<int>(q.device().index()), stream.stream()}];
  if (!ws.defined()) ws = at::zeros({static_cast<int64_t>(g_decode_ws())}, opts);
  return ws;
}

std::tuple<at::Tensor, at::Tensor, int64_t> paged_append(
    const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in,
    const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& block_table,
    const at::Tensor& start_lens, const at::Tensor& cosp, const at::Tensor& sinp,
    const c10::optional<at::Tensor>& cu_seqlens, const c10::optional<at::Tensor>& positions) {
  TORCH_CHECK(g_append, "frsa extension: C ABI not bound (call bind_serving first)");
  check_tokens(q_in, q_in, "q");
  check_tokens(k_in, q_in, "k");
  check_tokens(v_in, q_in, "v");
  check_cache(k_cache, q_in, k_cache, "k_cache");
  check_cache(v_cache, q_in, k_cache, "v_cache");
  TORCH_CHECK(k_in.sizes() == v_in.sizes() && k_in.size(0) == q_in.size(0) &&
                  k_in.size(1) == k_cache.size(1),
              "k and v must be [tokens, kv heads, D] with q's tokens and the cache's kv heads");
  TORCH_CHECK_TYPE(cosp.scalar_type() == at::kFloat && sinp.scalar_type() == at::kFloat,
                   "COSP/SINP must be float32");
  TORCH_CHECK(cosp.dim() == 2 && cosp.sizes() == sinp.sizes() && cosp.size(1) * 2 == q_in.size(2),
              "COSP/SINP must be [N_pos, D/2]");
  TORCH_CHECK(cosp.device() == q_in.device() && sinp.device() == q_in.device(),
              "RoPE tables must be on the same device as Q");
  check_no_grad(cosp, "COSP");
  check_no_grad(sinp, "SINP");
  const c10::cuda::CUDAGuard guard(q_in.device());
  const int64_t T = q_in.size(0), B = start_lens.numel();
  frsa_paged_append_args a{};
  const at::Tensor bt = table_array(block_table, q_in, B);
  const at::Tensor sl = index_array(start_lens, q_in, -1, "start_lens");
  at::Tensor cu, pos;
  if (cu_seqlens.has_value()) cu = index_array(*cu_seqlens, q_in, B + 1, "cu_seqlens");
  else TORCH_CHECK(T == B, "without cu_seqlens there is one token per sequence");
  if (positions.has_value()) pos = index_array(*positions, q_in, T, "positions");
  at::Tensor q_out = output(q_in.sizes(), q_in);
  at::Tensor k_out = output(k_in.sizes(), q_in);
  a.dtype = serve_dtype(q_in);
  if (T == 0 || q_in.size(1) == 0) return {q_out, k_out, 0};
  const at::Tensor q = readable_tokens(q_in), k = readable_tokens(k_in), v = readable_tokens(v_in);
  const at::Tensor c = cosp.contiguous(), s = sinp.contiguous();
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.q_out = q_out.data_ptr();
  a.k_out = k_out.data_ptr();
  a.k_cache = k_cache.data_ptr();
  a.v_cache = v_cache.data_ptr();
  a.block_table = bt.data_ptr<int32_t>();
  a.start_lens = sl.data_ptr<int32_t>();
  a.cu_seqlens = cu.defined() ? cu.data_ptr<int32_t>() : nullptr;
  a.positions = pos.defined() ? pos.data_ptr<int32_t>() : nullptr;
  a.cosp = c.data_ptr<float>();
  a.sinp = s.data_ptr<float>();
  a.T = T;
  a.B = B;
  a.Hq = q.size(1);
  a.Hkv = k.size(1);
  a.D = q.size(2);
  a.n_pos = c.size(0);
  a.num_pages = k_cache.size(0);
  a.page_size = k_cache.size(2);
  a.max_pages = bt.size(1);
  a.block_table_stride = bt.size(0) > 1 ? bt.stride(0) : bt.size(1);
  lead_strides(a.q_strides, q);
  lead_strides(a.k_strides, k);
  lead_strides(a.v_strides, v);
  lead_strides(a.cache_strides, k_cache);
  const int rc = g_append(&a, at::cuda::getCurrentCUDAStream().stream());
  if (rc == FRSA_OK) {
    mark_written(k_cache);
    mark_written(v_cache);
  }
  return {q_out, k_out, rc};
}

std::tuple<at::Tensor, at::Tensor, int64_t> paged_decode(
    const at::Tensor& q_in, const at::Tensor& k_cache, const at::Tensor& v_cache,
    const at::Tensor& block_table, const at::Tensor& seq_lens, const c10::optional<double>& scale,
    bool with_lse) {
  TORCH_CHECK(g_decode && g_decode_ws, "frsa extension: C ABI not bound (call bind_serving first)");
  check_tokens(q_in, q_in, "q");
  check_cache(k_cache, q_in, k_cache, "k_cache");
  check_cache(v_cache, q_in, k_cache, "v_cache");
  const c10::cuda::CUDAGuard guard(q_in.device());
  const int64_t B = q_in.size(0);
  const at::Tensor bt = table_array(block_table, q_in, B);
  const at::Tensor sl = index_array(seq_lens, q_in, B, "seq_lens");
  at::Tensor o = output(q_in.sizes(), q_in), lse;
  if (with_lse) lse = output({B, q_in.size(1)}, q_in, at::kFloat);
  frsa_paged_decode_args a{};
  a.dtype = serve_dtype(q_in);
  if (scale.has_value()) a.scale = scale_of(scale, 1);
  if (B == 0 || q_in.size(1) == 0) return {o, lse, 0};
  const at::Tensor q = readable_tokens(q_in);
  const c10::cuda::CUDAStream stream = at::cuda::getCurrentCUDAStream();
  const at::Tensor ws = decode_workspace(q, stream);
  a.q = q.data_ptr();
  a.k_cache = k_cache.data_ptr();
  a.v_cache = v_cache.data_ptr();
  a.o = o.data_ptr();
  a.lse = with_lse ? lse.data_ptr<float>() : nullptr;
  a.block_table = bt.data_ptr<int32_t>();
  a.seq_lens = sl.data_ptr<int32_t>();
  a.workspace = ws.data_ptr();
  a.workspace_bytes = static_cast<size_t>(ws.numel());
  a.B = B;
  a.Hq = q.size(1);
  a.Hkv = k_cache.size(1);
  a.D = q.size(2);
  a.num_pages = k_cache.size(0);
  a.page_size = k_cache.size(2);
  a.max_pages = bt.size(1);
  a.block_table_stride = bt.size(0) > 1 ? bt.stride(0) : bt.size(1);
  lead_strides(a.q_strides, q);
  lead_strides(a.cache_strides, k_cache);
  if (!scale.has_value()) a.scale = scale_of(scale, a.D);
  const int rc = g_decode(&a, stream.stream());
  return {o, lse, rc};
}

std::tuple<at::Tensor, at::Tensor, int64_t> prompt(const at::Tensor& q_in, const at::Tensor& k_in,
                                                   const at::Tensor& v_in,
                                                   const at::Tensor& cu_seqlens,
                                                   const c10::optional<double>& scale,
                                                   bool with_lse) {
  TORCH_CHECK(g_prompt, "frsa extension: C ABI not bound (call bind_serving first)");
  check_tokens(q_in, q_in, "q");
  check_tokens(k_in, q_in, "k");
  check_tokens(v_in, q_in, "v");
  TORCH_CHECK(k_in.sizes() == v_in.sizes() && k_in.size(0) == q_in.size(0),
              "k and v must be [tokens, kv heads, D] with q's tokens");
  const c10::cuda::CUDAGuard guard(q_in.device());
  const at::Tensor cu = index_array(cu_seqlens, q_in, -1, "cu_seqlens");
  TORCH_CHECK(cu.size(0) >= 1, "cu_seqlens must hold at least one boundary");
  const int64_t T = q_in.size(0), Hq = q_in.size(1);
  frsa_prompt_args a{};
  a.dtype = serve_dtype(q_in);
  if (scale.has_value()) a.scale = scale_of(scale, 1);
  if (T == 0 || Hq == 0 || cu.size(0) == 1) {   // no sequence: every token belongs to none
    at::Tensor o = at::zeros(q_in.sizes(), q_in.options()), lse;
    if (with_lse) lse = at::full({Hq, T}, -INFINITY, q_in.options().dtype(at::kFloat));
    return {o, lse, 0};
  }
  at::Tensor o = output(q_in.sizes(), q_in), lse;
  if (with_lse) lse = output({Hq, T}, q_in, at::kFloat);
  const at::Tensor q = readable_tokens(q_in), k = readable_tokens(k_in), v = readable_tokens(v_in);
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.o = o.data_ptr();
  a.lse = with_lse ? lse.data_ptr<float>() : nullptr;
  a.cu_seqlens = cu.data_ptr<int32_t>();
  a.T = T;
  a.B = cu.size(0) - 1;
  a.Hq = Hq;
  a.Hkv = k.size(1);
  a.D = q.size(2);
  lead_strides(a.q_strides, q);
  lead_strides(a.k_strides, k);
  lead_strides(a.v_strides, v);
  if (!scale.has_value()) a.scale = scale_of(scale, a.D);
  const int rc = g_prompt(&a, at::cuda::getCurrentCUDAStream().stream());
  return {o, lse, rc};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "PyTorch host side of the fused 2D-RoPE attention (C ABI include/frsa.h)";
  m.def("bind", &bind, "bind the C-ABI entry points (frsa_fwd, frsa_bwd, frsa_bwd_workspace_bytes)");
  m.def("fwd", &fwd, "forward: (o, lse, status)");
  m.def("bwd", &bwd, "backward: (dq, dk, dv, status)");
  m.def("bind_serving", &bind_serving,
        "bind the serving entry points (frsa_paged_append, frsa_paged_decode, "
        "frsa_paged_decode_workspace_bytes, frsa_prompt_fwd)");
  m.def("paged_append", &paged_append, "append to a paged cache: (q, k, status)");
  m.def("paged_decode", &paged_decode, "one token over a paged cache: (o, lse, status)");
  m.def("prompt", &prompt, "causal attention over packed prompts: (o, lse, status)");
}
