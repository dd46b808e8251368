// C ABI of the serving operators (include/frsa.h): argument checks, tensor
// maps and launches. Part of frsa_api.cu's translation unit.

namespace {

// Head counts, head dim and type that the serving kernels share.
int serve_common(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int32_t dtype) {
  constexpr int64_t kMost = int64_t(1) << 30;
  if (B < 1 || Hq < 1 || Hkv < 1 || D < 1 || B > kMost || Hq > 65535 || Hq % Hkv != 0)
    return FRSA_ERR_BAD_SHAPE;
  if (D % 8 != 0 || D > 128) return FRSA_ERR_UNSUPPORTED_D;
  if (dtype != FRSA_DTYPE_BF16 && dtype != FRSA_DTYPE_F16) return FRSA_ERR_UNSUPPORTED_DTYPE;
  return FRSA_OK;
}

// Strides of a [.., n1, D] tensor: all zero = contiguous over the extents
// that follow each of them; otherwise positive multiples of 16 bytes.
template <int N>
bool serve_strides(int64_t (&st)[N], const int64_t (&inner)[N]) {
  bool zero = true;
  for (int i = 0; i < N; ++i) zero &= st[i] == 0;
  for (int i = 0; i < N; ++i) {
    if (zero) st[i] = inner[i];
    if (st[i] < 1 || st[i] % 8 != 0 || st[i] >= (int64_t(1) << 39)) return false;
  }
  return true;
}

int serve_cache(int64_t num_pages, int64_t page_size, int64_t max_pages, int64_t bt_stride) {
  if (num_pages < 1 || page_size < 1 || max_pages < 1 || bt_stride < 0 ||
      num_pages > 0x7FFFFFFFLL || page_size > (int64_t(1) << 30) ||
      max_pages > (int64_t(1) << 30) / page_size)
    return FRSA_ERR_BAD_SHAPE;
  return FRSA_OK;
}

// The kernels' exponentials are to the base 2: the scale times log2(e) has to be finite.
bool scale_ok(float s) { return s > 0.f && s * 1.4426950408889634f <= 3.402823466e38f; }

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

// 3-D map {D, heads, T} over packed tokens with (token, head) strides in
// elements; box {64, heads_box, tokens_box}, 128-byte swizzle, zero fill.
bool encode_map_tokens(CUtensorMap* m, const void* base, int64_t T, int64_t H, int64_t D,
                       const int64_t (&st)[2], int heads_box, int tokens_box, bool bf16) {
  auto fn = get_encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(H),
                              static_cast<cuuint64_t>(T)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(st[1]) * 2,
                                 static_cast<cuuint64_t>(st[0]) * 2};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(heads_box),
                             static_cast<cuuint32_t>(tokens_box)};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                        3, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) g_last_encode_result = static_cast<int>(r);
  return r == CUDA_SUCCESS;
}

}  // namespace

extern "C" {

int frsa_paged_append(const frsa_paged_append_args* args, void* stream) {
  if (!args) return FRSA_ERR_NULL_ARG;
  frsa_paged_append_args a = *args;
  if (!a.q || !a.k || !a.v || !a.q_out || !a.k_cache || !a.v_cache || !a.block_table ||
      !a.start_lens || !a.cosp || !a.sinp)
    return FRSA_ERR_NULL_ARG;
  int rc = serve_common(a.B, a.Hq, a.Hkv, a.D, a.dtype);
  if (rc == FRSA_OK) rc = serve_cache(a.num_pages, a.page_size, a.max_pages, a.block_table_stride);
  if (rc != FRSA_OK) return rc;
  if (a.T < 1 || a.T > (int64_t(1) << 30) || a.n_pos < 0 || (!a.cu_seqlens && a.T != a.B))
    return FRSA_ERR_BAD_SHAPE;
  if (!aligned16(a.q) || !aligned16(a.k) || !aligned16(a.v) || !aligned16(a.q_out) ||
      !aligned16(a.k_out) || !aligned16(a.k_cache) || !aligned16(a.v_cache) ||
      !aligned16(a.cosp) || !aligned16(a.sinp) || !aligned4(a.block_table) ||
      !aligned4(a.start_lens) || !aligned4(a.cu_seqlens) || !aligned4(a.positions) ||
      !serve_strides(a.q_strides, {a.Hq * a.D, a.D}) ||
      !serve_strides(a.k_strides, {a.Hkv * a.D, a.D}) ||
      !serve_strides(a.v_strides, {a.Hkv * a.D, a.D}) ||
      !serve_strides(a.cache_strides, {a.Hkv * a.page_size * a.D, a.page_size * a.D, a.D}))
    return FRSA_ERR_MISALIGNED;
  if (!device_is_sm100()) return FRSA_ERR_NO_DEVICE;
  if ((rc = pending_error("frsa_paged_append")) != FRSA_OK) return rc;
  const cudaError_t e = frsa::launch_paged_append(a, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? FRSA_OK : launch_error("frsa_paged_append", e);
}

size_t frsa_paged_decode_workspace_bytes(void) { return frsa::decode_workspace_bytes(); }

int frsa_paged_decode(const frsa_paged_decode_args* args, void* stream) {
  if (!args) return FRSA_ERR_NULL_ARG;
  frsa_paged_decode_args a = *args;
  if (!a.q || !a.k_cache || !a.v_cache || !a.o || !a.block_table || !a.seq_lens)
    return FRSA_ERR_NULL_ARG;
  int rc = serve_common(a.B, a.Hq, a.Hkv, a.D, a.dtype);
  if (rc == FRSA_OK) rc = serve_cache(a.num_pages, a.page_size, a.max_pages, a.block_table_stride);
  if (rc != FRSA_OK) return rc;
  if (!scale_ok(a.scale)) return FRSA_ERR_BAD_SHAPE;
  // The kernel numbers tiles of 64 keys over all (sequence, kv head, head
  // block) units in 31 bits, and page and slot strides in granules in 32.
  const int64_t tiles = (a.max_pages * a.page_size + 63) / 64;
  if (tiles > 0x7FFFFFFFLL / (a.B * a.Hkv * ((a.Hq / a.Hkv + 7) / 8)) ||
      a.cache_strides[0] >= (int64_t(1) << 35) || a.cache_strides[2] >= (int64_t(1) << 35))
    return FRSA_ERR_BAD_SHAPE;
  if (!aligned16(a.q) || !aligned16(a.k_cache) || !aligned16(a.v_cache) || !aligned16(a.o) ||
      !aligned4(a.lse) || !aligned4(a.block_table) || !aligned4(a.seq_lens) ||
      !serve_strides(a.q_strides, {a.Hq * a.D, a.D}) ||
      !serve_strides(a.cache_strides, {a.Hkv * a.page_size * a.D, a.page_size * a.D, a.D}))
    return FRSA_ERR_MISALIGNED;
  if (!a.workspace || a.workspace_bytes < frsa::decode_workspace_bytes()) return FRSA_ERR_WORKSPACE;
  if (!aligned16(a.workspace)) return FRSA_ERR_MISALIGNED;
  if (!device_is_sm100()) return FRSA_ERR_NO_DEVICE;
  if ((rc = pending_error("frsa_paged_decode")) != FRSA_OK) return rc;
  const cudaError_t e = frsa::launch_paged_decode(a, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? FRSA_OK : launch_error("frsa_paged_decode", e);
}

int frsa_prompt_fwd(const frsa_prompt_args* args, void* stream) {
  if (!args) return FRSA_ERR_NULL_ARG;
  frsa_prompt_args a = *args;
  if (!a.q || !a.k || !a.v || !a.o || !a.cu_seqlens) return FRSA_ERR_NULL_ARG;
  int rc = serve_common(a.B, a.Hq, a.Hkv, a.D, a.dtype);
  if (rc != FRSA_OK) return rc;
  const int64_t G = a.Hq / a.Hkv;
  if (!scale_ok(a.scale) || a.T < 1 || a.T > (int64_t(1) << 30) || G > 128 ||
      (a.T / (128 / G) + a.B) * a.Hkv > 0x7FFFFFFFLL)
    return FRSA_ERR_BAD_SHAPE;
  if (!aligned16(a.q) || !aligned16(a.k) || !aligned16(a.v) || !aligned16(a.o) ||
      !aligned4(a.lse) || !aligned4(a.cu_seqlens) ||
      !serve_strides(a.q_strides, {a.Hq * a.D, a.D}) ||
      !serve_strides(a.k_strides, {a.Hkv * a.D, a.D}) ||
      !serve_strides(a.v_strides, {a.Hkv * a.D, a.D}))
    return FRSA_ERR_MISALIGNED;
  if (!device_is_sm100()) return FRSA_ERR_NO_DEVICE;
  if ((rc = pending_error("frsa_prompt_fwd")) != FRSA_OK) return rc;
  const bool bf16 = a.dtype == FRSA_DTYPE_BF16;
  CUtensorMap tq, tk, tv;
  if (!encode_map_tokens(&tq, a.q, a.T, a.Hq, a.D, a.q_strides, static_cast<int>(G),
                         static_cast<int>(128 / G), bf16) ||
      !encode_map_tokens(&tk, a.k, a.T, a.Hkv, a.D, a.k_strides, 1, frsa::kTile, bf16) ||
      !encode_map_tokens(&tv, a.v, a.T, a.Hkv, a.D, a.v_strides, 1, frsa::kTile, bf16))
    return launch_error("frsa_prompt_fwd", cudaSuccess);
  const cudaError_t e = frsa::launch_prompt(a, tq, tk, tv, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? FRSA_OK : launch_error("frsa_prompt_fwd", e);
}

}  // extern "C"
