// One attention row in f32, by one warp: for the rare row that the tensor
// products left with a NaN that its keys may not account for (an infinity in V
// times a probability that was split or rounded to zero, or times the 0 of a
// masked key), or whose scores are too large for their softmax base.
//
// K is any struct with `int n` (keys of the row), `int granules` (16-byte
// granules of a D), `place(j)`, where key j lies, and `k(place)`, `v(place)`, its
// rows there, or null for zeros. A half warp takes a key, lane & 15 its granule;
// the places of several keys, and then their rows, are read together.
#pragma once

#include "frsa_ptx.cuh"

namespace frsa {

constexpr unsigned kWholeWarp = 0xffffffffu;

// The elements of a granule (bit i: element i) that are at least `from`, without
// their sign: kInf those that are not finite, kInf + 1 the NaN.
template <typename T>
constexpr uint32_t kInf = Elt<T>::kBf16 ? 0x7f80u : 0x7c00u;
__device__ __forceinline__ uint32_t bits_from(uint4 x, uint32_t from) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((w[i] & 0x7fffu) >= from) bits |= 1u << (2 * i);
    if ((w[i] >> 16 & 0x7fffu) >= from) bits |= 2u << (2 * i);
  }
  return bits;
}
template <typename T>
__device__ __forceinline__ uint32_t nan_bits(uint4 x) {
  return bits_from(x, kInf<T> + 1);
}
// NaN in the low 8 bits, infinities in the next 8, negative ones in the next 8.
template <typename T>
__device__ __forceinline__ uint32_t special_bits(uint4 x) {
  const uint32_t all = bits_from(x, kInf<T>), nan = nan_bits<T>(x), inf = all & ~nan;
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t minus = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    minus |= (w[i] >> 15 & 1u) << (2 * i) | (w[i] >> 31) << (2 * i + 1);
  return nan | (inf & ~minus) << 8 | (inf & minus) << 16;
}
// Of such bits over several keys: the columns whose sum they make NaN.
__device__ __forceinline__ uint32_t explained(uint32_t seen) {
  return (seen | (seen >> 8 & seen >> 16)) & 0xffu;
}

// What the V of the first n keys holds in the columns `want` (8 bits per lane &
// 15): NaN, +inf and -inf as in special_bits, and in the high 8 bits infinities
// whose probability may be zero (a K near them is not finite). A column is done
// with when it holds a NaN or both infinities. The keys from `hint` on are looked
// at first (those where the last search found something: mostly it is the same
// token), then all in order. kBatch: keys in flight per half warp.
template <typename T, int kBatch, typename K>
__device__ __forceinline__ uint32_t special_columns(const K& keys, int n, uint32_t want,
                                                    int& hint) {
  const int g = threadIdx.x & 15, half = threadIdx.x >> 4 & 1;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  uint32_t seen = 0, open = want;
  bool hinted = hint >= 0 && hint < n;
#pragma unroll 1
  for (int next = 0; hinted || next < n; hinted = false) {
    const int j0 = hinted ? hint : next;
    if (!hinted) next += 2 * kBatch;
    decltype(keys.place(0)) at[kBatch];
    uint4 x[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) at[u] = keys.place(min(j0 + 2 * u + half, n - 1));
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {   // (past the end: the last key again)
      const uint4* row = g < keys.granules ? keys.v(at[u]) : nullptr;
      x[u] = row == nullptr ? zero : row[g];
    }
    uint32_t any = 0;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) any |= bits_from(x[u], kInf<T>);
    if (!__any_sync(kWholeWarp, (any & open) != 0)) continue;
    uint32_t found = 0;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) found |= special_bits<T>(x[u]);
    uint32_t k_odd = 0;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const uint4* row = g < keys.granules ? keys.k(at[u]) : nullptr;
      k_odd |= bits_from(row == nullptr ? zero : row[g], kInf<T>);
    }
    if (__any_sync(kWholeWarp, k_odd != 0))
      found = (found & 0xffu) | ((found >> 8 | found >> 16) & 0xffu) << 24;
    found |= __shfl_xor_sync(kWholeWarp, found, 16);
    found &= want * 0x01010101u;
    if (__any_sync(kWholeWarp, (found & ~seen) != 0)) hint = j0;
    seen |= found;
    open = want & ~explained(seen);
    if (__all_sync(kWholeWarp, open == 0)) break;
  }
  return seen;
}

// Which NaN of a written row that search leaves unexplained, and which stand for
// an infinity: a probability times an infinity is one, however small it is.
struct Mended {
  uint32_t left, plus, minus;
};
__device__ __forceinline__ Mended explain(uint32_t nan, uint32_t seen) {
  const uint32_t stay = explained(seen), unsure = seen >> 24;
  Mended m;
  m.plus = nan & seen >> 8 & ~(stay | unsure);
  m.minus = nan & seen >> 16 & ~(stay | unsure);
  m.left = nan & ~(stay | m.plus | m.minus);
  return m;
}
template <typename T>
__device__ __forceinline__ void put_infinities(T* granule, Mended m) {
#pragma unroll 1
  for (uint32_t left = m.plus | m.minus; left != 0; left &= left - 1) {
    const int e = __ffs(left) - 1;
    reinterpret_cast<uint16_t*>(granule)[e] =
        static_cast<uint16_t>(kInf<T> | (m.minus >> e & 1u) << 15);
  }
}

// The row o = sum_j softmax_j(s_j) v_j, s_j = c2 q . k_j in base 2, over all
// keys, written as the type, and its natural-log LSE. The statistics are the
// row's own: those of the product kernels belong to sums in another order, which
// at scores of 2^20 and more is another value.
template <typename T, int kBatch, typename K>
__device__ __forceinline__ float exact_row(const K& keys, const T* q, float c2, T* orow) {
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
    decltype(keys.place(0)) at[kBatch];
    uint4 kx[kBatch], vx[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) at[u] = keys.place(min(j0 + 2 * u + half, keys.n - 1));
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {   // (past the end: the last key again, not counted below)
      const uint4* kr = g < keys.granules ? keys.k(at[u]) : nullptr;
      const uint4* vr = g < keys.granules ? keys.v(at[u]) : nullptr;
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
