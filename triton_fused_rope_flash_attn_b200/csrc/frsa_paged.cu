// The paged key-value cache of the serving path: appending rotated keys (and
// values) to it, and the attention of one new token per sequence over it.
//
// A cache is [pages, Hkv, page_size, D] (any page, head and slot strides, unit
// d stride); block_table[b][i] is the page that holds tokens
// [i * page_size, (i + 1) * page_size) of sequence b.
#include "frsa_internal.h"
#include "frsa_ptx.cuh"

namespace frsa {

namespace {

// ---------------------------------------------------------------- append
// Token t of sequence b has index i = start_lens[b] + t - cu_seqlens[b] and
// rotation row p (positions[t], or i): q' = R_p q, k' = R_p k in f32, rounded
// once; k' and v go to slot i % page_size of page block_table[b][i / page_size].
// One CTA per token. The rows of q, k and v do not depend on where the token
// goes, so their loads are issued before the lookups (sequence, page, table
// row), whose dependent loads they then overlap.
constexpr int kAppendThreads = 256;

struct AppendParams {
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  void* k_out;
  void* k_cache;
  void* v_cache;
  const int* block_table;
  const int* start_lens;
  const int* cu_seqlens;
  const int* positions;
  const float* cosp;
  const float* sinp;
  long long T, n_pos, num_pages, max_pages, bt_stride;
  long long qs[2], ks[2], vs[2];   // token and head strides
  long long cs[3];                 // cache page, head and slot strides
  int B, Hq, Hkv, D, page_size;
};

// Largest b in [0, B) with cu[b] <= t (B - 1 when t is past the end), by a
// search with 32 probes a level: every lane of the warp takes part.
__device__ __forceinline__ int find_sequence(const int* cu, int B, long long t, int lane) {
  int lo = 0, n = B;   // the answer lies in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int probe = lo + lane * step;
    const bool below = lane * step < n && __ldg(cu + probe) <= t;
    const unsigned mask = __ballot_sync(0xffffffffu, below);
    const int i = mask == 0 ? 0 : 31 - __clz(mask);
    n = min(step, n - i * step);
    lo += i * step;
  }
  return lo;
}

template <typename T>
__device__ __forceinline__ uint4 rotate8(uint4 x, float4 c, float4 s) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = Elt<T>::unpack(w[i]);
    r[i] = Elt<T>::pack(v.x * cc[i] - v.y * ss[i], v.y * cc[i] + v.x * ss[i]);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

template <typename T>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const AppendParams p) {
  const long long t = blockIdx.x;
  const int G = p.D >> 3;                     // 16-byte granules per row
  const int rows = p.Hq + 2 * p.Hkv;          // q heads, k heads, v heads
  const int per = kAppendThreads / G;         // rows per pass
  const int g = threadIdx.x % G, r0 = threadIdx.x / G;
  const int lane = threadIdx.x & 31;
  constexpr int kAhead = 4;

  auto source = [&](int r) -> const uint4* {
    const void* base;
    long long off;
    if (r < p.Hq) {
      base = p.q;
      off = t * p.qs[0] + r * p.qs[1];
    } else if (r < p.Hq + p.Hkv) {
      base = p.k;
      off = t * p.ks[0] + (r - p.Hq) * p.ks[1];
    } else {
      base = p.v;
      off = t * p.vs[0] + (r - p.Hq - p.Hkv) * p.vs[1];
    }
    return reinterpret_cast<const uint4*>(static_cast<const T*>(base) + off) + g;
  };
  uint4 x[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int r = r0 + i * per;
    if (r0 < per && r < rows) x[i] = *source(r);
  }

  // Where the token goes and how it is turned.
  int b = static_cast<int>(t);
  long long index = 0;
  if (p.cu_seqlens != nullptr) {
    b = find_sequence(p.cu_seqlens, p.B, t, lane);
    index = t - __ldg(p.cu_seqlens + b);
  }
  const bool held = p.cu_seqlens == nullptr || (index >= 0 && t < __ldg(p.cu_seqlens + b + 1));
  index += __ldg(p.start_lens + b);
  const long long pos = p.positions != nullptr ? __ldg(p.positions + t) : index;
  const bool turn = pos >= 0 && pos < p.n_pos;
  float4 c = make_float4(1.f, 1.f, 1.f, 1.f), s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (turn) {
    c = __ldg(reinterpret_cast<const float4*>(p.cosp + pos * (p.D >> 1)) + g);
    s = __ldg(reinterpret_cast<const float4*>(p.sinp + pos * (p.D >> 1)) + g);
  }
  const long long page_no = index / p.page_size;
  bool stored = held && index >= 0 && page_no < p.max_pages;
  long long page = 0;
  if (stored) page = __ldg(p.block_table + b * p.bt_stride + page_no);
  const bool bad = (held && !stored) || page < 0 || page >= p.num_pages || pos < -1 ||
                   (held && pos >= p.n_pos);
  stored = stored && page >= 0 && page < p.num_pages;
  if (bad && threadIdx.x == 0) atomicCAS(&g_dev_status, 0, FRSA_DEV_INDEX);
  const long long slot = page * p.cs[0] + (index % p.page_size) * p.cs[2];

  auto finish = [&](int r, uint4 w) {
    if (r < p.Hq) {
      reinterpret_cast<uint4*>(static_cast<T*>(p.q_out) + (t * p.Hq + r) * p.D)[g] =
          rotate8<T>(w, c, s);
    } else if (r < p.Hq + p.Hkv) {
      const int h = r - p.Hq;
      w = rotate8<T>(w, c, s);
      if (p.k_out != nullptr)
        reinterpret_cast<uint4*>(static_cast<T*>(p.k_out) + (t * p.Hkv + h) * p.D)[g] = w;
      if (stored)
        reinterpret_cast<uint4*>(static_cast<T*>(p.k_cache) + slot + h * p.cs[1])[g] = w;
    } else if (stored) {
      const int h = r - p.Hq - p.Hkv;
      reinterpret_cast<uint4*>(static_cast<T*>(p.v_cache) + slot + h * p.cs[1])[g] = w;
    }
  };
  if (r0 >= per) return;
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int r = r0 + i * per;
    if (r < rows) finish(r, x[i]);
  }
  for (int r = r0 + kAhead * per; r < rows; r += per) finish(r, *source(r));
}

// ---------------------------------------------------------------- decode
// o[b, h] = sum_j softmax_j(scale q[b, h] . K_j) V_j over the cached tokens
// j < seq_lens[b] of kv head h / (Hq / Hkv).
//
// A unit is (sequence, kv head, block of up to 16 of the query heads that
// share it); its keys go in tiles of 64. The tiles of all units form one
// sequence that is cut evenly over the CTAs, whatever the lengths are, so a
// CTA works on the end of one unit, some whole units and the start of another.
// In a tile each of the CTA's four warps takes 16 keys and runs the softmax on
// its own (running maximum, sum and output): nothing is exchanged per tile.
// A warp reads its K and V rows with 16-byte asynchronous copies into its own
// ring in shared memory, several tiles ahead and across unit boundaries, so
// only the warp's own wait stands between the copies and the products. Rows
// past the sequence's end are filled with zeros by the copy itself: what the
// cache holds there (uninitialised memory too) never enters a product.
//
// Products: mma m16n8k16, the (padded) 16 query heads as rows. Reading the
// cache bounds this kernel (one multiply-add per element and query head), so
// the padding rows cost nothing that counts. The probabilities enter the
// second product as the sum of two 16-bit values (their rounding and what
// that left), which keeps them at f32's accuracy to 2^-17 for bf16.
//
// A unit within one CTA is written at once. For the others each CTA leaves
// its (m, l, o) in the workspace; the last of a unit's CTAs to arrive (a
// counter that it then sets back to zero) joins them in key order: the result
// does not depend on who comes last.
constexpr int kDecWarps = 4;
constexpr int kDecThreads = 32 * kDecWarps;
constexpr int kDecKeys = 16;                        // keys of a warp in a tile
constexpr int kDecTile = kDecWarps * kDecKeys;      // keys of a tile
constexpr int kDecCtasPerSm = 2;
constexpr int kDecRows = 16;
constexpr int kDecMaxD = 128;

struct DecodeParams {
  const void* q;
  const void* k_cache;
  const void* v_cache;
  void* o;
  float* lse;
  const int* block_table;
  const int* seq_lens;
  int* counters;       // [grid]
  float* part_o;       // [2 * grid][16][128]
  float* part_ml;      // [2 * grid][16][2]
  long long num_pages, max_pages, bt_stride;
  long long qs[2];     // sequence and head strides
  long long cs[3];     // cache page, head and slot strides
  int B, Hq, Hkv, D, page_size, group, blocks;   // blocks: 16-head blocks per kv head
  float c2;            // scale * log2(e)
};

template <int NK>
struct DecSmem {
  static constexpr int kStride = (2 * NK + 1) * 16;   // bytes of a row: an odd number of granules
  static constexpr int kRing = kDecKeys * kStride;    // one K or V part of a stage
  static constexpr int kStages = NK > 5 ? 3 : NK > 2 ? 4 : 6;
  uint8_t ring[kDecWarps][kStages][2][kRing];
  float merge[NK * 8][32];
  float merge_ml[2][2][32];
  long long scan[kDecWarps];
  long long find_rem;
  int find_b;
  int last;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool fill) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(fill ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  if constexpr (Elt<T>::kBf16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Cached tokens of sequence b, held within what its block table can name.
__device__ __forceinline__ int dec_len(const DecodeParams& p, int b) {
  const int n = __ldg(p.seq_lens + b);
  const long long most = p.max_pages * p.page_size;
  return n < 0 ? 0 : n > most ? static_cast<int>(most) : n;
}

// A place in the sequence of tiles: tile `tile` of unit (b, u).
struct DecCursor {
  int b, u, tile, ntiles, len;
  long long first;   // number of the unit's tile 0
};

__device__ __forceinline__ void dec_advance(const DecodeParams& p, DecCursor& c) {
  if (++c.tile < c.ntiles) return;
  c.tile = 0;
  c.first += c.ntiles;
  if (++c.u < p.Hkv * p.blocks) return;
  c.u = 0;
  do {
    ++c.b;
    c.len = c.b < p.B ? dec_len(p, c.b) : 1;
    c.ntiles = (c.len + kDecTile - 1) / kDecTile;
  } while (c.ntiles == 0);
}

template <typename T, int NK>
__global__ void __launch_bounds__(kDecThreads, kDecCtasPerSm)
    paged_decode_kernel(const DecodeParams p) {
  using Sm = DecSmem<NK>;
  constexpr int S = Sm::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Sm& sm = *reinterpret_cast<Sm*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quad = lane >> 2, ql = lane & 3;
  const int U = p.Hkv * p.blocks;

  // Sequences with nothing cached: zero output, lse -inf.
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    const int n = __ldg(p.seq_lens + b);
    if (n > 0 && n <= p.max_pages * p.page_size) continue;
    if (n != 0 && threadIdx.x == 0) atomicCAS(&g_dev_status, 0, FRSA_DEV_INDEX);
    if (n > 0) continue;
    for (int i = threadIdx.x; i < p.Hq * (p.D >> 3); i += kDecThreads)
      reinterpret_cast<uint4*>(static_cast<T*>(p.o) + static_cast<long long>(b) * p.Hq * p.D)[i] =
          make_uint4(0u, 0u, 0u, 0u);
    if (p.lse != nullptr)
      for (int h = threadIdx.x; h < p.Hq; h += kDecThreads)
        p.lse[static_cast<long long>(b) * p.Hq + h] = -INFINITY;
  }

  // Tiles before each thread's run of sequences, and in all.
  const int run = (p.B + kDecThreads - 1) / kDecThreads;
  const int b0 = min(p.B, static_cast<int>(threadIdx.x) * run), b1 = min(p.B, b0 + run);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) mine += (dec_len(p, b) + kDecTile - 1) / kDecTile;
  long long incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += o;
  }
  if (lane == 31) sm.scan[warp] = incl;
  __syncthreads();
  long long before = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kDecWarps; ++w) {
    if (w < warp) before += sm.scan[w];
    total += sm.scan[w];
  }
  total *= U;
  const long long ncta = min(static_cast<long long>(gridDim.x), total);
  const long long cta = blockIdx.x;
  if (cta >= ncta) return;
  auto range_begin = [&](long long c) { return c * total / ncta; };
  auto cta_of = [&](long long x) { return ((x + 1) * ncta - 1) / total; };
  const long long begin = range_begin(cta), end = range_begin(cta + 1);

  // The sequence in which this CTA's first tile lies.
  if (mine > 0 && before * U <= begin && begin < (before + mine) * U) {
    long long at = before * U;
    for (int b = b0; b < b1; ++b) {
      const long long n = static_cast<long long>((dec_len(p, b) + kDecTile - 1) / kDecTile) * U;
      if (begin < at + n) {
        sm.find_b = b;
        sm.find_rem = begin - at;
        break;
      }
      at += n;
    }
  }
  // Columns past D of the ring are never copied to: zero them once.
  for (int i = lane; i < S * 2 * kDecKeys * (2 * NK - (p.D >> 3)); i += 32) {
    const int pad = 2 * NK - (p.D >> 3);
    const int row = i / pad, gcol = (p.D >> 3) + i % pad;
    *reinterpret_cast<uint4*>(&sm.ring[warp][0][0][0] + row * Sm::kStride + gcol * 16) =
        make_uint4(0u, 0u, 0u, 0u);
  }
  __syncthreads();
  DecCursor cur;
  cur.b = sm.find_b;
  cur.len = dec_len(p, cur.b);
  cur.ntiles = (cur.len + kDecTile - 1) / kDecTile;
  cur.u = static_cast<int>(sm.find_rem / cur.ntiles);
  cur.tile = static_cast<int>(sm.find_rem % cur.ntiles);
  cur.first = begin - cur.tile;

  // The copying side runs ahead with a cursor of its own. Lane l (and l + 16)
  // looks up the page of the warp's key row l & 15, one tile before its copies.
  DecCursor ahead = cur;
  const uint32_t ring0 = smem_u32(&sm.ring[warp][0][0][0]);
  int page = 0;              // of the lane's key row
  long long in_page = -1;    // element offset within the page; < 0: no such key
  auto look_up = [&]() {
    const int key = ahead.tile * kDecTile + warp * kDecKeys + (lane & 15);
    in_page = -1;
    if (key < ahead.len) {
      const int pi = key / p.page_size;
      page = __ldg(p.block_table + ahead.b * p.bt_stride + pi);
      in_page = (ahead.u / p.blocks) * p.cs[1] +
                static_cast<long long>(key - pi * p.page_size) * p.cs[2];
    }
  };
  auto copy_tile = [&](int stage) {
    long long row_off = -1;
    if (in_page >= 0) {
      if (page >= 0 && page < p.num_pages) row_off = page * p.cs[0] + in_page;
      else atomicCAS(&g_dev_status, 0, FRSA_DEV_INDEX);
    }
    const uint32_t dk = ring0 + stage * 2 * Sm::kRing, dv = dk + Sm::kRing;
#pragma unroll
    for (int i = 0; i < NK; ++i) {   // 16 rows of 2 NK granules over 32 lanes
      const int idx = i * 32 + lane;
      const int row = idx / (2 * NK), gcol = idx % (2 * NK);
      const long long off = __shfl_sync(0xffffffffu, row_off, row);
      if (gcol * 8 < p.D) {
        const long long e = off < 0 ? 0 : off + gcol * 8;
        const uint32_t d = row * Sm::kStride + gcol * 16;
        cp_async16(dk + d, static_cast<const T*>(p.k_cache) + e, off >= 0);
        cp_async16(dv + d, static_cast<const T*>(p.v_cache) + e, off >= 0);
      }
    }
  };
  const int steps = static_cast<int>(end - begin);
  int copied = 0;
  look_up();
  auto copy_next = [&]() {
    if (copied < steps) {
      copy_tile(copied % S);
      ++copied;
      if (copied < steps) {
        dec_advance(p, ahead);
        look_up();
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i) copy_next();

  uint32_t qa[NK][4];
  float o[2 * NK][4];
  float m[2], l[2];
  bool fresh = true;
  const T* qp = static_cast<const T*>(p.q);

  for (int step = 0; step < steps; ++step) {
    if (fresh) {   // a unit begins: its query rows (16-byte aligned rows of 2-element pairs)
      const int h0 = (cur.u / p.blocks) * p.group + (cur.u % p.blocks) * kDecRows;
      const int rows = min(kDecRows, p.group - (cur.u % p.blocks) * kDecRows);
#pragma unroll
      for (int ks = 0; ks < NK; ++ks)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = quad + (i & 1) * 8, col = ks * 16 + (i >> 1) * 8 + ql * 2;
          qa[ks][i] = (r < rows && col < p.D)
                          ? __ldg(reinterpret_cast<const uint32_t*>(
                                qp + cur.b * p.qs[0] + (h0 + r) * p.qs[1] + col))
                          : 0u;
        }
#pragma unroll
      for (int n = 0; n < 2 * NK; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.f;
      fresh = false;
    }
    cp_async_wait<S - 2>();
    __syncwarp();
    copy_next();
    const int key0 = cur.tile * kDecTile + warp * kDecKeys;
    if (key0 < cur.len) {
      const uint32_t ks0 = ring0 + (step % S) * 2 * Sm::kRing, vs0 = ks0 + Sm::kRing;
      // Scores of 16 rows against 16 keys, in two chains over the head dim.
      float s[2][2][4];
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i >> 3][(i >> 2) & 1][i & 3] = 0.f;
      const uint32_t ka = ks0 + ((lane >> 4) * 8 + (lane & 7)) * Sm::kStride + ((lane >> 3) & 1) * 16;
#pragma unroll
      for (int ks = 0; ks < NK; ++ks) {
        uint32_t kb[4];
        ldsm4(ka + ks * 32, kb);
        mma16816<T>(s[ks & 1][0], qa[ks], kb[0], kb[1]);
        mma16816<T>(s[ks & 1][1], qa[ks], kb[2], kb[3]);
      }
      float x[2][4];   // [8-key half][row quad: c0, c1, row quad + 8: c2, c3]
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = key0 + n * 8 + ql * 2 + (i & 1);
          x[n][i] = key < cur.len ? (s[0][n][i] + s[1][n][i]) * p.c2 : -INFINITY;
        }
      float base[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float mx = fmaxf(fmaxf(x[0][2 * r], x[0][2 * r + 1]), fmaxf(x[1][2 * r], x[1][2 * r + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m[r], mx);
        base[r] = mn == -INFINITY ? 0.f : mn;
        if (mn > m[r]) {   // per row: earlier sums move to the new base
          const float alpha = ex2(m[r] - base[r]);
          l[r] *= alpha;
#pragma unroll
          for (int n = 0; n < 2 * NK; ++n) {
            o[n][2 * r] *= alpha;
            o[n][2 * r + 1] *= alpha;
          }
          m[r] = mn;
        }
      }
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float p0 = ex2(x[n][2 * r] - base[r]), p1 = ex2(x[n][2 * r + 1] - base[r]);
          l[r] += p0 + p1;
          const uint32_t h = Elt<T>::pack(p0, p1);
          const float2 back = Elt<T>::unpack(h);
          hi[n * 2 + r] = h;
          lo[n * 2 + r] = Elt<T>::pack(p0 - back.x, p1 - back.y);
        }
      const uint32_t va = vs0 + ((lane >> 3 & 1) * 8 + (lane & 7)) * Sm::kStride + (lane >> 4) * 16;
#pragma unroll
      for (int ks = 0; ks < NK; ++ks) {
        uint32_t vb[4];
        ldsm4_t(va + ks * 32, vb);
        mma16816<T>(o[2 * ks], hi, vb[0], vb[1]);
        mma16816<T>(o[2 * ks + 1], hi, vb[2], vb[3]);
        mma16816<T>(o[2 * ks], lo, vb[0], vb[1]);
        mma16816<T>(o[2 * ks + 1], lo, vb[2], vb[3]);
      }
    }
    __syncwarp();   // the stage's rows are read before a later copy replaces them

    if (cur.tile + 1 < cur.ntiles && step + 1 < steps) {
      dec_advance(p, cur);
      continue;
    }
    // The unit, or this CTA's part of it, ends: the four warps' states go into
    // warp 0's, one after another.
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
#pragma unroll 1
    for (int w = kDecWarps - 1; w > 0; --w) {
      if (warp == w) {
#pragma unroll
        for (int n = 0; n < 2 * NK; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) sm.merge[n * 4 + i][lane] = o[n][i];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          sm.merge_ml[0][r][lane] = m[r];
          sm.merge_ml[1][r][lane] = l[r];
        }
      }
      __syncthreads();
      if (warp == w - 1) {
        float fa[2], fb[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float mo = sm.merge_ml[0][r][lane], lo_ = sm.merge_ml[1][r][lane];
          const float mn = fmaxf(m[r], mo);
          const float bs = mn == -INFINITY ? 0.f : mn;
          fa[r] = ex2(m[r] - bs);
          fb[r] = ex2(mo - bs);
          l[r] = l[r] * fa[r] + lo_ * fb[r];
          m[r] = mn;
        }
#pragma unroll
        for (int n = 0; n < 2 * NK; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            o[n][i] = o[n][i] * fa[i >> 1] + sm.merge[n * 4 + i][lane] * fb[i >> 1];
      }
      __syncthreads();
    }
    const int kvh = cur.u / p.blocks, hb = cur.u % p.blocks;
    const int rows = min(kDecRows, p.group - hb * kDecRows);
    const long long row0 = static_cast<long long>(cur.b) * p.Hq + kvh * p.group + hb * kDecRows;
    const long long unit_end = cur.first + cur.ntiles;
    if (cur.first >= begin && unit_end <= end) {   // the whole unit is this CTA's
      if (warp == 0) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int row = quad + 8 * r;
          if (row < rows) {
            const float inv = 1.f / l[r];
            T* orow = static_cast<T*>(p.o) + (row0 + row) * p.D;
#pragma unroll
            for (int n = 0; n < 2 * NK; ++n)
              if (n * 8 < p.D)
                *reinterpret_cast<uint32_t*>(orow + n * 8 + ql * 2) =
                    Elt<T>::pack(o[n][2 * r] * inv, o[n][2 * r + 1] * inv);
            if (p.lse != nullptr && ql == 0)
              p.lse[row0 + row] = (m[r] + log2f(l[r])) * 0.69314718055994531f;
          }
        }
      }
    } else {
      const long long cf = cta_of(cur.first), cl = cta_of(unit_end - 1);
      const long long slot = cta == cf && cur.first > begin ? 2 * cta + 1 : 2 * cta;
      if (warp == 0) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int row = quad + 8 * r;
          if (row < rows) {
            float* po = p.part_o + (slot * kDecRows + row) * kDecMaxD;
#pragma unroll
            for (int n = 0; n < 2 * NK; ++n)
              *reinterpret_cast<float2*>(po + n * 8 + ql * 2) =
                  make_float2(o[n][2 * r], o[n][2 * r + 1]);
            if (ql == 0)
              *reinterpret_cast<float2*>(p.part_ml + (slot * kDecRows + row) * 2) =
                  make_float2(m[r], l[r]);
          }
        }
        __threadfence();
        __syncwarp();
        if (lane == 0) {
          const int n = static_cast<int>(cl - cf + 1);
          const int was = atomicAdd(p.counters + cf, 1);
          sm.last = was == n - 1;
          if (was == n - 1) p.counters[cf] = 0;   // as it was, for the next call
          __threadfence();
        }
      }
      __syncthreads();
      if (sm.last) {
        const long long s0 = range_begin(cf) == cur.first ? 2 * cf : 2 * cf + 1;
        for (int idx = threadIdx.x; idx < rows * (p.D >> 2); idx += kDecThreads) {
          const int row = idx / (p.D >> 2), c4 = idx % (p.D >> 2);
          float mx = -INFINITY;
#pragma unroll 8
          for (long long c = cf; c <= cl; ++c) {
            const long long sl = c == cf ? s0 : 2 * c;
            mx = fmaxf(mx, __ldcg(p.part_ml + (sl * kDecRows + row) * 2));
          }
          const float bs = mx == -INFINITY ? 0.f : mx;
          float lt = 0.f;
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
          for (long long c = cf; c <= cl; ++c) {
            const long long sl = c == cf ? s0 : 2 * c;
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(
                p.part_ml + (sl * kDecRows + row) * 2));
            const float4 v = __ldcg(reinterpret_cast<const float4*>(
                p.part_o + (sl * kDecRows + row) * kDecMaxD) + c4);
            const float f = ex2(ml.x - bs);
            lt += ml.y * f;
            acc.x += v.x * f;
            acc.y += v.y * f;
            acc.z += v.z * f;
            acc.w += v.w * f;
          }
          const float inv = 1.f / lt;
          *reinterpret_cast<uint2*>(static_cast<T*>(p.o) + (row0 + row) * p.D + c4 * 4) =
              make_uint2(Elt<T>::pack(acc.x * inv, acc.y * inv),
                         Elt<T>::pack(acc.z * inv, acc.w * inv));
          if (p.lse != nullptr && c4 == 0)
            p.lse[row0 + row] = (mx + log2f(lt)) * 0.69314718055994531f;
        }
      }
      __syncthreads();
    }
    fresh = true;
    if (step + 1 < steps) dec_advance(p, cur);
  }
}

template <typename T, int NK>
cudaError_t launch_decode_t(const DecodeParams& p, int grid, cudaStream_t stream) {
  auto kern = paged_decode_kernel<T, NK>;
  const size_t smem = sizeof(DecSmem<NK>);
  const cudaError_t e = set_max_dynamic_smem_once(kern, smem);
  if (e != cudaSuccess) return e;
  kern<<<grid, kDecThreads, smem, stream>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_decode_nk(const DecodeParams& p, int grid, cudaStream_t stream) {
  if (p.D <= 32) return launch_decode_t<T, 2>(p, grid, stream);
  if (p.D <= 64) return launch_decode_t<T, 4>(p, grid, stream);
  if (p.D <= 80) return launch_decode_t<T, 5>(p, grid, stream);
  if (p.D <= 96) return launch_decode_t<T, 6>(p, grid, stream);
  return launch_decode_t<T, 8>(p, grid, stream);
}

}  // namespace

int decode_grid() { return device_sm_count() * kDecCtasPerSm; }

size_t decode_counter_bytes() { return (static_cast<size_t>(decode_grid()) * 4 + 255) & ~size_t(255); }

size_t decode_workspace_bytes() {
  return decode_counter_bytes() +
         static_cast<size_t>(2) * decode_grid() * kDecRows * (kDecMaxD + 2) * sizeof(float);
}

cudaError_t launch_paged_append(const frsa_paged_append_args& a, cudaStream_t stream) {
  AppendParams p;
  p.q = a.q;
  p.k = a.k;
  p.v = a.v;
  p.q_out = a.q_out;
  p.k_out = a.k_out;
  p.k_cache = a.k_cache;
  p.v_cache = a.v_cache;
  p.block_table = a.block_table;
  p.start_lens = a.start_lens;
  p.cu_seqlens = a.cu_seqlens;
  p.positions = a.positions;
  p.cosp = a.cosp;
  p.sinp = a.sinp;
  p.T = a.T;
  p.n_pos = a.n_pos;
  p.num_pages = a.num_pages;
  p.max_pages = a.max_pages;
  p.bt_stride = a.block_table_stride;
  for (int i = 0; i < 2; ++i) {
    p.qs[i] = a.q_strides[i];
    p.ks[i] = a.k_strides[i];
    p.vs[i] = a.v_strides[i];
  }
  for (int i = 0; i < 3; ++i) p.cs[i] = a.cache_strides[i];
  p.B = static_cast<int>(a.B);
  p.Hq = static_cast<int>(a.Hq);
  p.Hkv = static_cast<int>(a.Hkv);
  p.D = static_cast<int>(a.D);
  p.page_size = static_cast<int>(a.page_size);
  const unsigned grid = static_cast<unsigned>(a.T);
  if (a.dtype == FRSA_DTYPE_BF16)
    paged_append_kernel<__nv_bfloat16><<<grid, kAppendThreads, 0, stream>>>(p);
  else
    paged_append_kernel<__half><<<grid, kAppendThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_paged_decode(const frsa_paged_decode_args& a, cudaStream_t stream) {
  DecodeParams p;
  p.q = a.q;
  p.k_cache = a.k_cache;
  p.v_cache = a.v_cache;
  p.o = a.o;
  p.lse = a.lse;
  p.block_table = a.block_table;
  p.seq_lens = a.seq_lens;
  const int grid = decode_grid();
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  p.counters = reinterpret_cast<int*>(ws);
  p.part_o = reinterpret_cast<float*>(ws + decode_counter_bytes());
  p.part_ml = p.part_o + static_cast<size_t>(2) * grid * kDecRows * kDecMaxD;
  p.num_pages = a.num_pages;
  p.max_pages = a.max_pages;
  p.bt_stride = a.block_table_stride;
  for (int i = 0; i < 2; ++i) p.qs[i] = a.q_strides[i];
  for (int i = 0; i < 3; ++i) p.cs[i] = a.cache_strides[i];
  p.B = static_cast<int>(a.B);
  p.Hq = static_cast<int>(a.Hq);
  p.Hkv = static_cast<int>(a.Hkv);
  p.D = static_cast<int>(a.D);
  p.page_size = static_cast<int>(a.page_size);
  p.group = p.Hq / p.Hkv;
  p.blocks = (p.group + kDecRows - 1) / kDecRows;
  p.c2 = a.scale * 1.4426950408889634f;
  return a.dtype == FRSA_DTYPE_BF16 ? launch_decode_nk<__nv_bfloat16>(p, grid, stream)
                                    : launch_decode_nk<__half>(p, grid, stream);
}

}  // namespace frsa
