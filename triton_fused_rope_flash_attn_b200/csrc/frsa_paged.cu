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
// A unit is (sequence, kv head, block of up to 8 NT of the query heads that
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
// Products: mma m16n8k16 with the keys (S^T = K Q^T) and then the head dim
// (O^T = V^T P^T) as the 16 rows and 8 query heads as columns, so groups of up
// to 8 heads fill the columns and the softmax has no padding rows beyond them
// (against the heads as rows: 521 -> about 200 instructions per warp and
// tile). P^T moves from the first product's result layout to the second's
// operand layout with movmatrix. The probabilities enter the second product
// as the sum of two 16-bit values (their rounding and what that left), which
// keeps them to 2^-16 for bf16.
//
// Little work (all units cut into pieces of up to 4 tiles give no more pieces
// than CTAs) is not shared out evenly: a CTA then has one piece, so short
// units need no joining.
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
constexpr int kDecPiece = 4;                        // tiles of a piece at most
constexpr int kDecMaxHeads = 16;                    // query heads of a unit at most
constexpr int kDecMaxD = 128;
constexpr int kDecSlot = kDecMaxHeads * kDecMaxD;   // floats of a partial o

struct DecodeParams {
  const void* q;
  const void* k_cache;
  const void* v_cache;
  void* o;
  float* lse;
  const int* block_table;
  const int* seq_lens;
  int* counters;       // [grid]
  float* part_o;       // [2 * grid][kDecSlot], in the layout of the warps' registers
  float* part_ml;      // [2 * grid][16][2]
  long long bt_stride;
  long long qs[2];     // sequence and head strides (elements)
  long long head_g;    // cache head stride in 16-byte granules
  uint32_t page_g, slot_g;   // cache page and slot strides in granules
  int num_pages, max_len;    // max_len: tokens that a row of the block table can name
  int B, Hq, Hkv, D, page_size, group, blocks;   // blocks: head blocks per kv head
  int page_shift;      // log2(page_size), or -1
  int rows16;          // 16 keys from a multiple of 16 lie in one page
  float c2;            // scale * log2(e)
};

template <int NK, int NT>
struct DecSmem {
  static constexpr int kStride = (2 * NK + 1) * 16;   // bytes of a row: an odd number of granules
  static constexpr int kRing = kDecKeys * kStride;    // one K or V part of a stage
  static constexpr int kStages = NK > 5 ? 3 : NK > 2 ? 4 : 6;
  uint8_t ring[kDecWarps][kStages][2][kRing];
  float ml[kDecWarps][2][2 * NT][32];
  int scan[2][kDecWarps];
  int find[3];
  int last;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// Copies 16 bytes, or fills them with zeros.
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool copy) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(copy ? 16 : 0)
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
// Transposes an 8 x 8 matrix of 16-bit values held as row lane / 4, columns
// 2 (lane % 4) and + 1.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
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
  return min(max(__ldg(p.seq_lens + b), 0), p.max_len);
}
__device__ __forceinline__ int dec_tiles(int len) { return (len + kDecTile - 1) / kDecTile; }
__device__ __forceinline__ int dec_pieces(int tiles) { return (tiles + kDecPiece - 1) / kDecPiece; }

// A place in the sequence of tiles: tile `tile` of unit (b, h, blk).
struct DecCursor {
  int b, h, blk, tile, ntiles, len;
  int first;   // number of the unit's tile 0
};

__device__ __forceinline__ bool dec_advance(const DecodeParams& p, DecCursor& c) {
  if (++c.tile < c.ntiles) return false;
  c.tile = 0;
  c.first += c.ntiles;
  if (++c.blk < p.blocks) return true;
  c.blk = 0;
  if (++c.h < p.Hkv) return true;
  c.h = 0;
  do {
    ++c.b;
    c.len = c.b < p.B ? dec_len(p, c.b) : 1;
    c.ntiles = dec_tiles(c.len);
  } while (c.ntiles == 0);
  return true;
}

// exp2 base of a running maximum (a row whose scores are all -inf has none).
__device__ __forceinline__ float dec_base(float m) { return m == -INFINITY ? 0.f : m; }

template <typename T, int NK, int NT>
__global__ void __launch_bounds__(kDecThreads, kDecCtasPerSm)
    paged_decode_kernel(const DecodeParams p) {
  using Sm = DecSmem<NK, NT>;
  constexpr int S = Sm::kStages;
  constexpr int kPer = (NK + kDecWarps - 1) / kDecWarps;   // 16-column steps of a warp in a join
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Sm& sm = *reinterpret_cast<Sm*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quad = lane >> 2, ql = lane & 3;
  const int U = p.Hkv * p.blocks;
  const int grid = gridDim.x, cta = blockIdx.x;

  // Tiles and pieces before each thread's run of sequences, and in all.
  const int run = (p.B + kDecThreads - 1) / kDecThreads;
  const int b0 = min(p.B, static_cast<int>(threadIdx.x) * run), b1 = min(p.B, b0 + run);
  int tiles = 0, pieces = 0;
  for (int b = b0; b < b1; ++b) {
    const int n = dec_tiles(dec_len(p, b));
    tiles += n;
    pieces += dec_pieces(n);
  }
  int tiles_in = tiles, pieces_in = pieces;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, tiles_in, d);
    const int y = __shfl_up_sync(0xffffffffu, pieces_in, d);
    if (lane >= d) {
      tiles_in += x;
      pieces_in += y;
    }
  }
  if (lane == 31) {
    sm.scan[0][warp] = tiles_in;
    sm.scan[1][warp] = pieces_in;
  }
  // Columns past D of the ring are never copied to: zero them.
  const int pad = 2 * NK - (p.D >> 3);
  auto zero_pad = [&](int row0, int rows) {
    for (int i = lane; i < rows * pad; i += 32)
      *reinterpret_cast<uint4*>(&sm.ring[warp][0][0][0] + (row0 + i / pad) * Sm::kStride +
                                ((p.D >> 3) + i % pad) * 16) = make_uint4(0u, 0u, 0u, 0u);
  };
  if (pad != 0) zero_pad(0, S * 2 * kDecKeys);
  __syncthreads();
  int tiles_before = tiles_in - tiles, pieces_before = pieces_in - pieces;
  int total = 0, total_pieces = 0;
#pragma unroll
  for (int w = 0; w < kDecWarps; ++w) {
    if (w < warp) {
      tiles_before += sm.scan[0][w];
      pieces_before += sm.scan[1][w];
    }
    total += sm.scan[0][w];
    total_pieces += sm.scan[1][w];
  }
  total *= U;
  total_pieces *= U;

  // Sequences with nothing cached: zero output, lse -inf.
  for (int b = cta; b < p.B; b += grid) {
    const int n = __ldg(p.seq_lens + b);
    if (n > 0 && n <= p.max_len) continue;
    if (n != 0 && threadIdx.x == 0) atomicCAS(&g_dev_status, 0, FRSA_DEV_INDEX);
    if (n > 0) continue;
    for (int i = threadIdx.x; i < p.Hq * (p.D >> 3); i += kDecThreads)
      reinterpret_cast<uint4*>(static_cast<T*>(p.o) + static_cast<long long>(b) * p.Hq * p.D)[i] =
          make_uint4(0u, 0u, 0u, 0u);
    if (p.lse != nullptr)
      for (int h = threadIdx.x; h < p.Hq; h += kDecThreads)
        p.lse[static_cast<long long>(b) * p.Hq + h] = -INFINITY;
  }

  // This CTA's tiles [begin, end). With few pieces: one piece of one unit.
  // Else an even share of all tiles: share c begins at c q + min(c, r).
  const bool by_piece = total_pieces <= grid;
  const int ncta = by_piece ? total_pieces : min(grid, total);
  if (cta >= ncta) return;
  const int q = total / ncta, r = total - q * ncta;
  auto share_begin = [&](int c) { return c * q + min(c, r); };
  auto share_of = [&](int x) {
    return x < r * (q + 1) ? x / (q + 1) : r + (x - r * (q + 1)) / q;
  };
  const int at = by_piece ? cta : share_begin(cta);
  {   // the sequence in which they lie: one thread's run holds it
    int lo = (by_piece ? pieces_before : tiles_before) * U;
    if (lo <= at && at < lo + (by_piece ? pieces : tiles) * U) {
      int t0 = tiles_before * U;
      for (int b = b0; b < b1; ++b) {
        const int n = dec_tiles(dec_len(p, b));
        const int w = (by_piece ? dec_pieces(n) : n) * U;
        if (at < lo + w) {
          sm.find[0] = b;
          sm.find[1] = at - lo;
          sm.find[2] = t0;
          break;
        }
        lo += w;
        t0 += n * U;
      }
    }
  }
  __syncthreads();
  DecCursor cur;
  cur.b = sm.find[0];
  cur.len = dec_len(p, cur.b);
  cur.ntiles = dec_tiles(cur.len);
  int begin, end, piece = 0, npieces = 1;
  {
    npieces = dec_pieces(cur.ntiles);
    const int per = by_piece ? npieces : cur.ntiles;
    const int u = sm.find[1] / per, rem = sm.find[1] - u * per;
    cur.h = u / p.blocks;
    cur.blk = u - cur.h * p.blocks;
    cur.first = sm.find[2] + u * cur.ntiles;
    if (by_piece) {   // pieces of a unit differ by one tile at most
      const int pq = cur.ntiles / npieces, pr = cur.ntiles - pq * npieces;
      piece = rem;
      cur.tile = piece * pq + min(piece, pr);
      begin = cur.first + cur.tile;
      end = begin + pq + (piece < pr);
    } else {
      cur.tile = rem;
      begin = at;
      end = share_begin(cta + 1);
    }
  }

  // The copying side runs ahead with a cursor of its own. Pages are looked up
  // one tile before their copies: one page for the warp's 16 keys where these
  // cannot straddle two, else lane l (and l + 16) that of key row l & 15. Each
  // lane copies the same NK granules of the 16 rows of every tile.
  DecCursor ahead = cur;
  const uint32_t ring0 = smem_u32(&sm.ring[warp][0][0][0]);
  const uint4* const kc = static_cast<const uint4*>(p.k_cache);
  const uint4* const vc = static_cast<const uint4*>(p.v_cache);
  const int* table = p.block_table + ahead.b * p.bt_stride;
  long long head_off = ahead.h * p.head_g;
  int page = 0;              // of the lane's key row (of the warp's 16 keys)
  int slot = -1;             // in that page; < 0: no such key
  int held = 0;              // keys of the 16 that the sequence has
  auto look_up = [&]() {
    const int key0 = ahead.tile * kDecTile + warp * kDecKeys;
    const int key = p.rows16 ? key0 : key0 + (lane & 15);
    held = ahead.len - key0;
    slot = -1;
    if (key < ahead.len) {
      const int pi = p.page_shift >= 0 ? key >> p.page_shift : key / p.page_size;
      page = __ldg(table + pi);
      slot = key - pi * p.page_size;
    }
  };
  uint32_t goff[NK];   // granule i of the lane, from its row's (rows16: its tile's) first
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    const int idx = i * 32 + lane;
    goff[i] = idx % (2 * NK) + (p.rows16 ? idx / (2 * NK) * p.slot_g : 0);
  }
  auto copy_tile = [&](int stage) {
    long long off = -1;
    if (slot >= 0) {
      if (page >= 0 && page < p.num_pages)
        off = static_cast<long long>(static_cast<uint64_t>(static_cast<uint32_t>(page)) * p.page_g +
                                     static_cast<uint64_t>(static_cast<uint32_t>(slot)) * p.slot_g) +
              head_off;
      else
        atomicCAS(&g_dev_status, 0, FRSA_DEV_INDEX);
    }
    const uint32_t dk = ring0 + stage * 2 * Sm::kRing;
    if (p.rows16 && off >= 0 && held >= kDecKeys) {
      const uint4* ks = kc + off;
      const uint4* vs = vc + off;
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        const int idx = i * 32 + lane;
        const int row = idx / (2 * NK), gcol = idx % (2 * NK);
        if (gcol * 8 < p.D) {
          const uint32_t d = dk + row * Sm::kStride + gcol * 16;
          cp_async16(d, ks + goff[i]);
          cp_async16(d + Sm::kRing, vs + goff[i]);
        }
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < NK; ++i) {   // 16 rows of 2 NK granules over 32 lanes
      const int idx = i * 32 + lane;
      const int row = idx / (2 * NK), gcol = idx % (2 * NK);
      long long e = p.rows16 ? off : __shfl_sync(0xffffffffu, off, row);
      const bool copy = e >= 0 && row < held;
      if (gcol * 8 < p.D) {
        e = copy ? e + goff[i] : 0;
        const uint32_t d = dk + row * Sm::kStride + gcol * 16;
        cp_async16_or_zero(d, kc + e, copy);
        cp_async16_or_zero(d + Sm::kRing, vc + e, copy);
      }
    }
  };
  const int steps = end - begin;
  int copied = 0, copy_stage = 0;
  look_up();
  auto copy_next = [&]() {
    if (copied < steps) {
      copy_tile(copy_stage);
      copy_stage = copy_stage + 1 == S ? 0 : copy_stage + 1;
      if (++copied < steps) {
        if (dec_advance(p, ahead)) {
          table = p.block_table + ahead.b * p.bt_stride;
          head_off = ahead.h * p.head_g;
        }
        look_up();
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i) copy_next();

  uint32_t qb[NT][NK][2];
  float o[NT][NK][4];   // O^T: rows 16 ks + quad, + 8; columns (heads) 8 nt + 2 ql, + 1
  float m[NT][2], l[NT][2];
  bool fresh = true;
  const T* qp = static_cast<const T*>(p.q);
  const uint32_t ka = ring0 + ((lane >> 3 & 1) * 8 + (lane & 7)) * Sm::kStride + (lane >> 4) * 16;
  const uint32_t va = ring0 + Sm::kRing + ((lane >> 4) * 8 + (lane & 7)) * Sm::kStride +
                      (lane >> 3 & 1) * 16;
  int stage = 0;

  for (int step = 0; step < steps; ++step) {
    if (fresh) {   // a unit begins: its query heads
      const int h0 = cur.h * p.group + cur.blk * 8 * NT;
      const int rows = min(8 * NT, p.group - cur.blk * 8 * NT);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int ks = 0; ks < NK; ++ks)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int row = nt * 8 + quad, col = ks * 16 + i * 8 + ql * 2;
            qb[nt][ks][i] = (row < rows && col < p.D)
                                ? __ldg(reinterpret_cast<const uint32_t*>(
                                      qp + cur.b * p.qs[0] + (h0 + row) * p.qs[1] + col))
                                : 0u;
          }
#pragma unroll
        for (int ks = 0; ks < NK; ++ks)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[nt][ks][i] = 0.f;
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
      }
      fresh = false;
    }
    copy_next();   // into the stage that the previous step read
    cp_async_wait<S - 1>();
    __syncwarp();
    const int key0 = cur.tile * kDecTile + warp * kDecKeys;
    if (key0 < cur.len) {
      const uint32_t at_stage = stage * 2 * Sm::kRing;
      // S^T: 16 keys x 8 NT heads, in two chains over the head dim.
      float s[NT][2][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 8; ++i) s[nt][i >> 2][i & 3] = 0.f;
#pragma unroll
      for (int ks = 0; ks < NK; ++ks) {
        uint32_t a[4];
        ldsm4(ka + at_stage + ks * 32, a);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16816<T>(s[nt][ks & 1], a, qb[nt][ks][0], qb[nt][ks][1]);
      }
      uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float x[4];   // keys quad (0, 1), quad + 8 (2, 3); heads 2 ql, 2 ql + 1
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (s[nt][0][i] + s[nt][1][i]) * p.c2;
        if (key0 + kDecKeys > cur.len) {
          if (key0 + quad >= cur.len) x[0] = x[1] = -INFINITY;
          if (key0 + quad + 8 >= cur.len) x[2] = x[3] = -INFINITY;
        }
        float mx[2] = {fmaxf(x[0], x[2]), fmaxf(x[1], x[3])};
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], d));
          mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], d));
        }
        // Earlier sums move to the new base where a maximum rose.
        if (__any_sync(0xffffffffu, mx[0] > m[nt][0] || mx[1] > m[nt][1])) {
          float alpha[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float mn = fmaxf(m[nt][c], mx[c]);
            alpha[c] = ex2(m[nt][c] - dec_base(mn));
            l[nt][c] *= alpha[c];
            m[nt][c] = mn;
          }
#pragma unroll
          for (int ks = 0; ks < NK; ++ks)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[nt][ks][i] *= alpha[i & 1];
        }
        const float base[2] = {dec_base(m[nt][0]), dec_base(m[nt][1])};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float p0 = ex2(x[2 * i] - base[0]), p1 = ex2(x[2 * i + 1] - base[1]);
          l[nt][0] += p0;
          l[nt][1] += p1;
          const uint32_t h = Elt<T>::pack(p0, p1);
          const float2 back = Elt<T>::unpack(h);
          hi[nt][i] = transpose8x8(h);
          lo[nt][i] = transpose8x8(Elt<T>::pack(p0 - back.x, p1 - back.y));
        }
      }
#pragma unroll
      for (int ks = 0; ks < NK; ++ks) {
        uint32_t a[4];
        ldsm4_t(va + at_stage + ks * 32, a);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma16816<T>(o[nt][ks], a, hi[nt][0], hi[nt][1]);
          mma16816<T>(o[nt][ks], a, lo[nt][0], lo[nt][1]);
        }
      }
    }
    const int used = stage;
    stage = stage + 1 == S ? 0 : stage + 1;
    __syncwarp();   // the stage's rows are read before a later copy replaces them

    if (cur.tile + 1 < cur.ntiles && step + 1 < steps) {
      ++cur.tile;
      continue;
    }
    // The unit, or this CTA's part of it, ends: the four warps' states meet in
    // the ring stage that each has just read (the next copy into it comes
    // after this), and warp w goes on with the 16-column steps w, w + 4, ...
    float* dump = reinterpret_cast<float*>(&sm.ring[warp][used][0][0]) + lane;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int ks = 0; ks < NK; ++ks)
#pragma unroll
        for (int i = 0; i < 4; ++i) dump[((nt * NK + ks) * 4 + i) * 32] = o[nt][ks][i];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        sm.ml[warp][0][nt * 2 + c][lane] = m[nt][c];
        sm.ml[warp][1][nt * 2 + c][lane] = l[nt][c];
      }
    }
    __syncthreads();
    float acc[NT][kPer][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float f[2][kDecWarps];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float mw[kDecWarps], mn = -INFINITY;
#pragma unroll
        for (int w = 0; w < kDecWarps; ++w) {
          mw[w] = sm.ml[w][0][nt * 2 + c][lane];
          mn = fmaxf(mn, mw[w]);
        }
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kDecWarps; ++w) {
          f[c][w] = ex2(mw[w] - dec_base(mn));
          sum += sm.ml[w][1][nt * 2 + c][lane] * f[c][w];
        }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        m[nt][c] = mn;
        l[nt][c] = sum;
      }
#pragma unroll
      for (int j = 0; j < kPer; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int ks = warp + j * kDecWarps;
          acc[nt][j][i] = 0.f;
          if (ks < NK)
#pragma unroll
            for (int w = 0; w < kDecWarps; ++w)
              acc[nt][j][i] += reinterpret_cast<const float*>(
                                   &sm.ring[w][used][0][0])[((nt * NK + ks) * 4 + i) * 32 + lane] *
                               f[i & 1][w];
        }
    }
    const int rows = min(8 * NT, p.group - cur.blk * 8 * NT);
    const long long row0 =
        static_cast<long long>(cur.b) * p.Hq + cur.h * p.group + cur.blk * 8 * NT;
    const int unit_end = cur.first + cur.ntiles;
    const bool whole = cur.first >= begin && unit_end <= end;
    int parts = 1, part0 = cta;   // the CTAs that share the unit
    if (!whole) {
      if (by_piece) {
        parts = npieces;
        part0 = cta - piece;
      } else {
        part0 = share_of(cur.first);
        parts = share_of(unit_end - 1) - part0 + 1;
      }
      // Partial o: value i of (nt, ks) at ((nt NK + ks) 4 + i) 32 + 8 ql + quad,
      // so a head pair's values are whole 32-byte sectors and only those of
      // heads that exist are written and read. A CTA leaves two partials at
      // most: of the unit that it ends and of the unit that it begins.
      const int mine = 2 * cta + (cta == part0 && cur.first > begin);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (nt * 8 + ql * 2 < rows) {
          float* po = p.part_o + static_cast<size_t>(mine) * kDecSlot + nt * NK * 128 + 8 * ql + quad;
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            const int ks = warp + j * kDecWarps;
            if (ks < NK)
#pragma unroll
              for (int i = 0; i < 4; ++i) po[(ks * 4 + i) * 32] = acc[nt][j][i];
          }
          if (warp == 0 && quad < 2)
            *reinterpret_cast<float2*>(p.part_ml +
                                       (mine * kDecMaxHeads + nt * 8 + ql * 2 + quad) * 2) =
                quad == 0 ? make_float2(m[nt][0], l[nt][0]) : make_float2(m[nt][1], l[nt][1]);
        }
      }
      __threadfence();
    }
    __syncthreads();   // (also: the dumped states are read before the next copies)
    if (pad != 0) zero_pad(used * 2 * kDecKeys, 2 * kDecKeys);
    bool write = whole;
    if (!whole) {
      if (threadIdx.x == 0) {
        const int was = atomicAdd(p.counters + part0, 1);
        sm.last = was == parts - 1;
        if (was == parts - 1) p.counters[part0] = 0;   // as it was, for the next call
        __threadfence();
      }
      __syncthreads();
      write = sm.last != 0;
      if (write) {
        const int s0 = 2 * part0 + (!by_piece && share_begin(part0) != cur.first);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (nt * 8 + ql * 2 >= rows) continue;
          auto ml_of = [&](int c) {
            return __ldcg(reinterpret_cast<const float4*>(
                p.part_ml +
                ((c == 0 ? s0 : 2 * (part0 + c)) * kDecMaxHeads + nt * 8 + ql * 2) * 2));
          };
          float mt[2] = {-INFINITY, -INFINITY}, lt[2] = {0.f, 0.f};
#pragma unroll 8
          for (int c = 0; c < parts; ++c) {
            const float4 x = ml_of(c);
            mt[0] = fmaxf(mt[0], x.x);
            mt[1] = fmaxf(mt[1], x.z);
          }
#pragma unroll
          for (int j = 0; j < kPer; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[nt][j][i] = 0.f;
#pragma unroll 4
          for (int c = 0; c < parts; ++c) {
            const float4 x = ml_of(c);
            const float f[2] = {ex2(x.x - dec_base(mt[0])), ex2(x.z - dec_base(mt[1]))};
            lt[0] += x.y * f[0];
            lt[1] += x.w * f[1];
            const float* po = p.part_o +
                              static_cast<size_t>(c == 0 ? s0 : 2 * (part0 + c)) * kDecSlot +
                              nt * NK * 128 + 8 * ql + quad;
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
              const int ks = warp + j * kDecWarps;
              if (ks < NK)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  acc[nt][j][i] += __ldcg(po + (ks * 4 + i) * 32) * f[i & 1];
            }
          }
          m[nt][0] = mt[0];
          m[nt][1] = mt[1];
          l[nt][0] = lt[0];
          l[nt][1] = lt[1];
        }
      }
    }
    if (write) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float inv[2] = {1.f / l[nt][0], 1.f / l[nt][1]};
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const int ks = warp + j * kDecWarps;
          if (ks >= NK) continue;
          const float(&v)[4] = acc[nt][j];
          // Back from O^T: head quad, columns 2 ql, + 1 (and + 8).
          const uint32_t w0 = transpose8x8(Elt<T>::pack(v[0] * inv[0], v[1] * inv[1]));
          const uint32_t w1 = transpose8x8(Elt<T>::pack(v[2] * inv[0], v[3] * inv[1]));
          const int row = nt * 8 + quad, col = ks * 16 + ql * 2;
          if (row < rows) {
            T* orow = static_cast<T*>(p.o) + (row0 + row) * p.D + col;
            if (col < p.D) *reinterpret_cast<uint32_t*>(orow) = w0;
            if (col + 8 < p.D) *reinterpret_cast<uint32_t*>(orow + 8) = w1;
          }
        }
        if (p.lse != nullptr && warp == 0 && quad < 2 && nt * 8 + ql * 2 + quad < rows)
          p.lse[row0 + nt * 8 + ql * 2 + quad] =
              ((quad == 0 ? m[nt][0] : m[nt][1]) + log2f(quad == 0 ? l[nt][0] : l[nt][1])) *
              0.69314718055994531f;
      }
    }
    fresh = true;
    if (step + 1 < steps) dec_advance(p, cur);
  }
}

template <typename T, int NK, int NT>
cudaError_t launch_decode_t(const DecodeParams& p, int grid, cudaStream_t stream) {
  auto kern = paged_decode_kernel<T, NK, NT>;
  const size_t smem = sizeof(DecSmem<NK, NT>);
  const cudaError_t e = set_max_dynamic_smem_once(kern, smem);
  if (e != cudaSuccess) return e;
  kern<<<grid, kDecThreads, smem, stream>>>(p);
  return cudaGetLastError();
}

template <typename T, int NT>
cudaError_t launch_decode_nk(const DecodeParams& p, int grid, cudaStream_t stream) {
  if (p.D <= 32) return launch_decode_t<T, 2, NT>(p, grid, stream);
  if (p.D <= 64) return launch_decode_t<T, 4, NT>(p, grid, stream);
  if (p.D <= 80) return launch_decode_t<T, 5, NT>(p, grid, stream);
  if (p.D <= 96) return launch_decode_t<T, 6, NT>(p, grid, stream);
  return launch_decode_t<T, 8, NT>(p, grid, stream);
}

// Groups of up to 8 query heads take 8 columns, larger ones blocks of 16.
template <typename T>
cudaError_t launch_decode_heads(DecodeParams& p, int grid, cudaStream_t stream) {
  const int heads = p.group <= 8 ? 8 : 16;
  p.blocks = (p.group + heads - 1) / heads;
  return heads == 8 ? launch_decode_nk<T, 1>(p, grid, stream)
                    : launch_decode_nk<T, 2>(p, grid, stream);
}

}  // namespace

int decode_grid() { return device_sm_count() * kDecCtasPerSm; }

size_t decode_counter_bytes() { return (static_cast<size_t>(decode_grid()) * 4 + 255) & ~size_t(255); }

size_t decode_workspace_bytes() {
  return decode_counter_bytes() +
         static_cast<size_t>(2) * decode_grid() * (kDecSlot + 2 * kDecMaxHeads) * sizeof(float);
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
  p.part_ml = p.part_o + static_cast<size_t>(2) * grid * kDecSlot;
  p.num_pages = static_cast<int>(a.num_pages);
  p.max_len = static_cast<int>(a.max_pages * a.page_size);
  p.bt_stride = a.block_table_stride;
  for (int i = 0; i < 2; ++i) p.qs[i] = a.q_strides[i];
  p.page_g = static_cast<uint32_t>(a.cache_strides[0] / 8);
  p.head_g = a.cache_strides[1] / 8;
  p.slot_g = static_cast<uint32_t>(a.cache_strides[2] / 8);
  p.B = static_cast<int>(a.B);
  p.Hq = static_cast<int>(a.Hq);
  p.Hkv = static_cast<int>(a.Hkv);
  p.D = static_cast<int>(a.D);
  p.page_size = static_cast<int>(a.page_size);
  p.group = p.Hq / p.Hkv;
  p.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (p.page_size == 1 << i) p.page_shift = i;
  p.rows16 = p.page_size % kDecKeys == 0 && p.slot_g < (1u << 27);   // 16 rows in 32 bits
  p.c2 = a.scale * 1.4426950408889634f;
  return a.dtype == FRSA_DTYPE_BF16 ? launch_decode_heads<__nv_bfloat16>(p, grid, stream)
                                    : launch_decode_heads<__half>(p, grid, stream);
}

}  // namespace frsa
