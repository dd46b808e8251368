// One attention row in f32, by one warp: for the rare row that the tensor
// products left with a NaN that its keys may not account for (an infinity in V
// times a probability that was split or rounded to zero, or times the 0 of a
// masked key), or whose scores are too large for their softmax base.
//
// K is any struct with `int n` (keys of the row), `int granules` (16-byte
// granules of a D) and `k(j)`, `v(j)`: key j's rows, or null for zeros. A half
// warp takes a key, lane & 15 its granule.
#pragma once

#include "frsa_ptx.cuh"

namespace frsa {

constexpr unsigned kWholeWarp = 0xffffffffu;

// Bits 2 i and 2 i + 1: the low and high half of word i is a NaN.
template <typename T>
__device__ __forceinline__ uint32_t nan_bits(uint4 x) {
  constexpr uint32_t kInf = Elt<T>::kBf16 ? 0x7f80u : 0x7c00u;
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((w[i] & 0x7fffu) > kInf) bits |= 1u << (2 * i);
    if ((w[i] >> 16 & 0x7fffu) > kInf) bits |= 2u << (2 * i);
  }
  return bits;
}

// Which of the columns `want` (8 bits per lane & 15) hold a NaN in the V of one
// of the first n keys.
template <typename T, typename K>
__device__ __forceinline__ uint32_t nan_columns(const K& keys, int n, uint32_t want) {
  constexpr int kBatch = 8;
  const int g = threadIdx.x & 15, half = threadIdx.x >> 4 & 1;
  uint32_t seen = 0;
#pragma unroll 1
  for (int j0 = 0; j0 < n; j0 += 2 * kBatch) {
    uint4 x[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int j = j0 + 2 * u + half;
      const uint4* row = j < n && g < keys.granules ? keys.v(j) : nullptr;
      x[u] = row == nullptr ? make_uint4(0u, 0u, 0u, 0u) : row[g];
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) seen |= nan_bits<T>(x[u]);
    seen |= __shfl_xor_sync(kWholeWarp, seen, 16);
    if (__all_sync(kWholeWarp, (want & ~seen) == 0)) break;
  }
  return seen & want;
}

// The row o = sum_j softmax_j(s_j) v_j, s_j = c2 q . k_j in base 2, over all
// keys, written as the type, and its natural-log LSE. The statistics are the
// row's own: those of the product kernels belong to sums in another order, which
// at scores of 2^20 and more is another value. About 30 instructions a key;
// their latency is hidden by four keys' loads per half warp.
template <typename T, typename K>
__device__ __forceinline__ float exact_row(const K& keys, const T* q, float c2, T* orow) {
  constexpr int kBatch = 4;
  const int g = threadIdx.x & 15, half = threadIdx.x >> 4 & 1;
  float qf[8], acc[8], m = -INFINITY, l = 0.f;
  auto unpack8 = [](uint4 x, float(&f)[8]) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = Elt<T>::unpack(w[i]);
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  };
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  unpack8(g < keys.granules ? reinterpret_cast<const uint4*>(q)[g] : zero, qf);
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
#pragma unroll 1
  for (int j0 = 0; j0 < keys.n; j0 += 2 * kBatch) {
    uint4 kx[kBatch], vx[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int j = j0 + 2 * u + half;
      const bool in = j < keys.n && g < keys.granules;
      const uint4* kr = in ? keys.k(j) : nullptr;
      const uint4* vr = in ? keys.v(j) : nullptr;
      kx[u] = kr == nullptr ? zero : kr[g];
      vx[u] = vr == nullptr ? zero : vr[g];
    }
    float x[kBatch], mn = m;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      float f[8], s = 0.f;
      unpack8(kx[u], f);
#pragma unroll
      for (int i = 0; i < 8; ++i) s = fmaf(qf[i], f[i], s);
#pragma unroll
      for (int d = 1; d < 16; d <<= 1) s += __shfl_xor_sync(kWholeWarp, s, d);
      x[u] = j0 + 2 * u + half < keys.n ? s * c2 : -INFINITY;
      mn = fmaxf(mn, x[u]);
    }
    mn = fmaxf(mn, __shfl_xor_sync(kWholeWarp, mn, 16));
    const float base = mn == -INFINITY ? 0.f : mn;
    if (__any_sync(kWholeWarp, mn > m)) {   // (alike in the whole warp)
      const float alpha = ex2(m - base);
      l *= alpha;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] *= alpha;
      m = mn;
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (j0 + 2 * u + half < keys.n) {
        float f[8];
        const float w = ex2(x[u] - base);
        unpack8(vx[u], f);
        l += w;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = fmaf(w, f[i], acc[i]);
      }
    }
  }
  uint32_t out[4];
  l += __shfl_xor_sync(kWholeWarp, l, 16);
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] += __shfl_xor_sync(kWholeWarp, acc[i], 16);
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = Elt<T>::pack(acc[2 * i] / l, acc[2 * i + 1] / l);
  if (half == 0 && g < keys.granules)
    reinterpret_cast<uint4*>(orow)[g] = make_uint4(out[0], out[1], out[2], out[3]);
  return (m + log2f(l)) * 0.69314718055994531f;
}

}  // namespace frsa
