// The paged key-value cache of the serving path: appending rotated keys (and
// values) to it, and the attention of one new token per sequence over it.
//
// A cache is [pages, Hkv, page_size, D] (any page, head and slot strides, unit
// d stride); block_table[b][i] is the page that holds tokens
// [i * page_size, (i + 1) * page_size) of sequence b.
#include "frsa_internal.h"
#include "frsa_ptx.cuh"
#include "frsa_row.cuh"

namespace frsa {

namespace {

// ---------------------------------------------------------------- append
// Token t of sequence b has index i = start_lens[b] + t - cu_seqlens[b] and
// rotation row p (positions[t], or i): q' = R_p q, k' = R_p k in f32, rounded
// once; k' and v go to slot i % page_size of page block_table[b][i / page_size].
// A CTA takes one token, or four where there are many. The rows of q, k and v
// do not depend on where a token goes, so the first two rows' loads of a
// thread are issued before the look-ups (sequence, page, table row), a
// warp's for a token each, whose dependent loads they then overlap. What
// bounds it: memory for many tokens (8985 tokens of 16 + 32 heads of 80, 161
// MB: 36 us, 4.5 TB/s, with one token per CTA 48; 8192 tokens of 32 + 16 heads
// of 128, 222 MB: 44 us, 5.1 TB/s), the launch for few.
constexpr int kAppendThreads = 256;
constexpr int kAppendMost = 4;    // tokens of a CTA at most

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
  int tokens;                      // of a CTA
};

// Largest b in [0, B) with cu[b] <= t (B - 1 when t is past the end), by a
// search with 32 probes a level: every lane of the warp takes part.
__device__ __forceinline__ int find_sequence(const int* cu, int B, long long t, int lane) {
  int lo = 0, n = B;   // the answer lies in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int probe = lo + lane * step;
    const bool below = lane * step < n && ld_int(cu + probe) <= t;
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
__global__ void __launch_bounds__(kAppendThreads, 3) paged_append_kernel(const AppendParams p) {
  __shared__ long long slots[kAppendMost];   // offset of the token's slot in granules; < 0: nowhere
  __shared__ float4 turns[kAppendMost][2][16];   // its cosines and sines
  const int G = p.D >> 3;                     // 16-byte granules per row
  const int rows = p.Hq + 2 * p.Hkv;          // q heads, k heads, v heads
  const int per = kAppendThreads / G;         // rows per pass
  const int g = threadIdx.x % G, r0 = threadIdx.x / G;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  wait_previous();
  allow_next();
  const long long t0 = static_cast<long long>(blockIdx.x) * p.tokens;
  const int tokens = static_cast<int>(min(static_cast<long long>(p.tokens), p.T - t0));

  // Granule g of one row over the CTA's tokens: where it is read and written.
  // (Row by row with the tokens inside: all but a token's slot is found once
  // per row, 145 -> about 70 instructions per 16 bytes.)
  struct Row {
    const uint4* src;
    uint4* out;          // rotated copy (q_out, k_out), or null
    uint4* cache;        // slot 0 of page 0, or null for q
    long long src_step;  // granules from token to token
    int out_step;
    bool turn;
  };
  auto row_of = [&](int r) {
    Row w;
    const bool q = r < p.Hq, key = !q && r < p.Hq + p.Hkv;
    const int h = q ? r : key ? r - p.Hq : r - p.Hq - p.Hkv;
    const T* src = static_cast<const T*>(q ? p.q : key ? p.k : p.v);
    const long long* st = q ? p.qs : key ? p.ks : p.vs;
    w.src = reinterpret_cast<const uint4*>(src + t0 * st[0] + h * st[1]) + g;
    w.src_step = st[0] >> 3;
    w.out_step = (q ? p.Hq : p.Hkv) * G;
    T* out = static_cast<T*>(q ? p.q_out : key ? p.k_out : nullptr);
    w.out = out == nullptr ? nullptr
                           : reinterpret_cast<uint4*>(out) + t0 * w.out_step + h * G + g;
    w.cache = q ? nullptr
                : reinterpret_cast<uint4*>(static_cast<T*>(key ? p.k_cache : p.v_cache) +
                                           h * p.cs[1]) + g;
    w.turn = q || key;
    return w;
  };
  auto load = [&](const Row& w, uint4(&x)[kAppendMost]) {
#pragma unroll
    for (int i = 0; i < kAppendMost; ++i)
      if (i < tokens) x[i] = ld_stream16(w.src + i * w.src_step);
  };
  // Two rows' loads are in flight.
  const bool works = r0 < per;
  Row ra, rb;
  uint4 xa[kAppendMost], xb[kAppendMost];
  if (works && r0 < rows) {
    ra = row_of(r0);
    load(ra, xa);
  }
  if (works && r0 + per < rows) {
    rb = row_of(r0 + per);
    load(rb, xb);
  }

  // Where a token goes and how it is turned.
  if (warp < tokens) {
    const long long t = t0 + warp;
    int b = static_cast<int>(t);
    long long index = 0;
    bool held = true;
    if (p.cu_seqlens != nullptr) {
      b = find_sequence(p.cu_seqlens, p.B, t, lane);
      const int first = ld_int(p.cu_seqlens + b);
      index = t - first;
      held = first >= 0 && index >= 0 && t < ld_int(p.cu_seqlens + b + 1);
    }
    index += ld_int(p.start_lens + b);
    const long long pos = !held ? -1 : p.positions != nullptr ? ld_int(p.positions + t) : index;
    // (in 32 bits: an index past them lies outside every block table)
    const unsigned at = held && index >= 0 && index < (1LL << 31) ? static_cast<unsigned>(index)
                                                                  : 0xffffffffu;
    const unsigned page_no = at / static_cast<unsigned>(p.page_size);
    bool stored = at != 0xffffffffu && page_no < p.max_pages;
    long long page = 0;
    if (stored) page = ld_int(p.block_table + b * p.bt_stride + page_no);
    const bool bad = (held && !stored) || page < 0 || page >= p.num_pages || pos < -1 ||
                     pos >= p.n_pos;
    stored = stored && page >= 0 && page < p.num_pages;
    if (lane == 0) {
      if (bad) atomicCAS(&g_dev_status, 0, FRSA_DEV_INDEX);
      slots[warp] = stored ? (page * p.cs[0] +
                              static_cast<long long>(at - page_no * p.page_size) * p.cs[2]) >> 3
                           : -1;
    }
    const int pairs4 = p.D >> 3;   // float4s of a table row
    float4 f = lane < 16 ? make_float4(1.f, 1.f, 1.f, 1.f) : make_float4(0.f, 0.f, 0.f, 0.f);
    if (pos >= 0 && pos < p.n_pos && (lane & 15) < pairs4)
      f = ld_f4((lane < 16 ? p.cosp : p.sinp) + pos * (p.D >> 1) + (lane & 15) * 4);
    turns[warp][lane >> 4][lane & 15] = f;
  } else if (blockIdx.x == 0 && warp == kAppendMost && p.cu_seqlens != nullptr) {
    bool bad = false;   // boundaries outside the tokens, or out of order
    for (int b = lane; b <= p.B; b += 32) {
      const int c = ld_int(p.cu_seqlens + b);
      bad |= c < 0 || c > p.T || (b < p.B && ld_int(p.cu_seqlens + b + 1) < c);
    }
    if (bad) atomicCAS(&g_dev_status, 0, FRSA_DEV_INDEX);
  }
  __syncthreads();

  if (!works) return;
  auto finish = [&](const Row& w, const uint4(&x)[kAppendMost]) {
#pragma unroll
    for (int i = 0; i < kAppendMost; ++i)
      if (i < tokens) {
        const uint4 y = w.turn ? rotate8<T>(x[i], turns[i][0][g], turns[i][1][g]) : x[i];
        if (w.out != nullptr) w.out[i * w.out_step] = y;
        if (w.cache != nullptr && slots[i] >= 0) w.cache[slots[i]] = y;
      }
  };
  for (int r = r0; r < rows; r += 2 * per) {
    finish(ra, xa);
    if (r + 2 * per < rows) {
      ra = row_of(r + 2 * per);
      load(ra, xa);
    }
    if (r + per < rows) finish(rb, xb);
    if (r + 3 * per < rows) {
      rb = row_of(r + 3 * per);
      load(rb, xb);
    }
  }
}

// ---------------------------------------------------------------- decode
// o[b, h] = sum_j softmax_j(scale q[b, h] . K_j) V_j over the cached tokens
// j < seq_lens[b] of kv head h / (Hq / Hkv).
//
// A unit is (sequence, kv head, block of up to 8 NT of the query heads that
// share it); its keys go in tiles of 64, and the tiles of all units, in order,
// are the work, whatever the lengths are. It is cut into one share per CTA (the
// same number of tiles, give or take one); a share is the end of one unit, some
// whole units and the start of another, and its part of a unit is a segment.
// In a tile each of the CTA's four warps takes 16 keys and runs the softmax on
// its own (running maximum, sum and output): nothing is exchanged per tile.
// A warp reads its K and V rows with 16-byte asynchronous copies into its own
// ring in shared memory, several tiles ahead and across units, so
// only the warp's own wait stands between the copies and the products. Rows
// past the sequence's end are filled with zeros by the copy itself: what the
// cache holds there (uninitialised memory too) never enters a product.
//
// Little work goes otherwise: where all units cut into pieces of up to 4 tiles
// give no more pieces than CTAs, a CTA has one piece, so short units need no
// joining. (Pieces of up to 2: three sequences of up to 12987 tokens 22.1
// against 16.7 us, with more to join; of up to 8: eight sequences of up to
// 1370 tokens 16.5 against 12.4.)
//
// Products: mma m16n8k16 with the keys (S^T = K Q^T) and then the head dim
// (O^T = V^T P^T) as the 16 rows and 8 query heads as columns, so groups of up
// to 8 heads fill the columns and the softmax has no padding rows beyond them
// (with the heads as rows 64 sequences of up to 8000 tokens took 214 us against
// 194). P^T moves from the first product's result layout to the second's
// operand layout with movmatrix. The probabilities enter the second product
// as the sum of two 16-bit values (their rounding and what that left), which
// keeps them to 2^-16 for bf16 and 2^-22 for f16. f16's smallest step, 2^-24,
// would be coarse beside probabilities far below the largest one (an attention
// sink: with the tail 17 nats below it 44 % of the output), so there the
// softmax base lies kDecLift below the maximum and the largest probability is
// 2^15; a part's rounding is then at most 2^-40 of it. What was left is zero or negative for some, so
// an infinity in V, which by the definition makes its column infinite, comes
// out of that product as NaN. A row that is written with a NaN is therefore held
// against its V (dec_mend).
//
// A unit within one share is written at once. For the others each share leaves
// its (m, l, o) in the workspace, and the last of the unit's CTAs to arrive (a
// counter that it then sets back to zero) joins them in key order: the result
// does not depend on who comes last.
//
// What bounds it: memory. SMs do not read at the same speed: of 296 equal
// shares of one 131072-token sequence (8 kv heads, 537 MB) the first has computed
// its tiles after 67 to 71 us, half after 78 and the last after 83 to 87; the last
// join ends at 91 to 95 (time stamps in three launches). Tried against that and not
// faster: further, smaller shares claimed from a ticket counter (all done
// between 80 and 94 us, but with four times the partials, whose joining took
// the gain back, in the kernel or in a second one); a fifth warp that copies
// for all four (a 16-row TMA box takes about 100 cycles: 122 us in all for
// pages of 16, though 177 against 187 for 64 sequences with pages of 64) or
// that only schedules. Now 98 us of a call for 131072 tokens (5.5 TB/s), 178 for
// 64 sequences of up to 8000 tokens (5.8 TB/s, 90 % of the measured copy rate);
// of 5.9 us for 197 tokens, 2.1 pass before the first copies (lengths, pages), the
// four tiles are computed after 4.3, the row is written after 4.8.
constexpr int kDecWarps = 4;
constexpr int kDecThreads = 32 * kDecWarps;
constexpr int kDecKeys = 16;                        // keys of a warp in a tile
constexpr int kDecTile = kDecWarps * kDecKeys;      // keys of a tile
constexpr int kDecCtasPerSm = 2;
constexpr int kDecPiece = 4;                        // tiles of a piece at most
constexpr int kDecBatch = 8;                        // partials whose loads are in flight in a join
constexpr int kDecMaxHeads = 16;                    // query heads of a unit at most
constexpr int kDecMaxD = 128;

struct DecodeParams {
  const void* q;
  const void* k_cache;
  const void* v_cache;
  void* o;
  float* lse;
  const int* block_table;
  const int* seq_lens;
  int* counters;       // [grid] arrivals at a unit's shares, by its first one
  float* part_o;       // [2 * grid][slot_floats], in the layout of the warps' registers
  float* part_ml;      // [2 * grid][16][2]
  int slot_floats;
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
  // About 17 KB in flight per warp. More spreads the CTAs' speeds further apart
  // (three stages at D = 128: 131072 tokens 100 against 96 us in the kernel, 64
  // sequences of up to 8000 tokens 182 against 177).
  static constexpr int kStages = NK > 5 ? 2 : NK > 2 ? 3 : 5;
  uint8_t ring[kDecWarps][kStages][2][kRing];
  float ml[kDecWarps][2][2 * NT][32];
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
  return min(max(ld_int(p.seq_lens + b), 0), p.max_len);
}
__device__ __forceinline__ int dec_tiles(int len) { return (len + kDecTile - 1) / kDecTile; }
__device__ __forceinline__ int dec_pieces(int tiles) { return (tiles + kDecPiece - 1) / kDecPiece; }

// A place in the sequence of tiles: tile `tile` of unit (b, h, blk).
struct DecCursor {
  int b, h, blk, tile, ntiles, len;
  int first;   // number of the unit's tile 0
};

__device__ __forceinline__ void dec_advance(const DecodeParams& p, DecCursor& c) {
  if (++c.tile < c.ntiles) return;
  c.tile = 0;
  c.first += c.ntiles;
  if (++c.blk < p.blocks) return;
  c.blk = 0;
  if (++c.h < p.Hkv) return;
  c.h = 0;
  do {
    ++c.b;
    c.len = c.b < p.B ? dec_len(p, c.b) : 1;
    c.ntiles = dec_tiles(c.len);
  } while (c.ntiles == 0);
}

// The sequence that holds item x, an item being a tile or (by_piece) a piece
// of one of its U units: by a whole warp, 32 runs of sequences a level. x
// becomes the item's number in the sequence, `first` the number of the
// sequence's first tile.
__device__ __forceinline__ int dec_find(const DecodeParams& p, bool by_piece, int U, int& x,
                                        int& first, int lane) {
  int lo = 0, n = p.B;
  first = 0;
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int i0 = lo + min(n, lane * step), i1 = lo + min(n, (lane + 1) * step);
    int tiles = 0, items = 0;
    for (int i = i0; i < i1; ++i) {
      const int t = dec_tiles(dec_len(p, i));
      tiles += t * U;
      items += (by_piece ? dec_pieces(t) : t) * U;
    }
    int tiles_in = tiles, items_in = items;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, tiles_in, d);
      const int z = __shfl_up_sync(0xffffffffu, items_in, d);
      if (lane >= d) {
        tiles_in += y;
        items_in += z;
      }
    }
    const int i = __ffs(__ballot_sync(0xffffffffu, x < items_in)) - 1;
    x -= __shfl_sync(0xffffffffu, items_in - items, i);
    first += __shfl_sync(0xffffffffu, tiles_in - tiles, i);
    lo = __shfl_sync(0xffffffffu, i0, i);
    n = __shfl_sync(0xffffffffu, i1, i) - lo;
  }
  return lo;
}

// log2 of the largest probability that a warp forms: f16's largest power of two.
template <typename T>
constexpr float kDecLift = Elt<T>::kBf16 ? 0.f : 15.f;

// exp2 base of a running maximum (a row whose scores are all -inf has none).
__device__ __forceinline__ float dec_base(float m) { return m == -INFINITY ? 0.f : m; }

// Waits until at most `pending` (<= N) of the warp's copy groups are in flight.
template <int N>
__device__ __forceinline__ void cp_async_wait_to(int pending) {
  if constexpr (N == 0) {
    cp_async_wait<0>();
  } else {
    if (pending == N) cp_async_wait<N>();
    else cp_async_wait_to<N - 1>(pending);
  }
}

// The keys of one (sequence, kv head) for frsa_row.cuh.
struct DecKeys {
  const uint4* kc;
  const uint4* vc;
  const int* table;    // the sequence's row of the block table
  long long head_off;
  uint32_t page_g, slot_g;
  int page_size, num_pages;
  int n, granules;
  __device__ long long place(int j) const {
    const int pi = j / page_size, page = table[pi];
    const uint64_t off = static_cast<uint64_t>(static_cast<uint32_t>(page)) * page_g +
                         static_cast<uint64_t>(static_cast<uint32_t>(j - pi * page_size)) * slot_g;
    return page >= 0 && page < num_pages ? static_cast<long long>(off) + head_off : -1;
  }
  __device__ const uint4* k(long long at) const { return at < 0 ? nullptr : kc + at; }
  __device__ const uint4* v(long long at) const { return at < 0 ? nullptr : vc + at; }
};

// Row (cur.b, head) as it was written, by a whole warp: NaN that V does not
// explain become the infinity that it holds, or the row is computed again. A
// unit's rows go to the warps of the CTA that writes it: one sequence of 131072
// tokens takes 19 ms with an infinity in V (all of it is searched, for one of the
// other sign), 0.15 with a NaN near its start, where 0.1 is normal.
template <typename T>
__device__ __noinline__ void dec_mend(const DecKeys& keys, const T* q, float c2, T* orow) {
  const int lane = threadIdx.x & 31, g = lane & 15;
  uint32_t want = 0;
  if (g < keys.granules) want = nan_bits<T>(reinterpret_cast<const uint4*>(orow)[g]);
  if (!__any_sync(kWholeWarp, want != 0)) return;
  int hint = -1;
  const uint32_t seen = special_columns<T, 4>(keys, keys.n, want, hint);
  Mended m = explain(want, seen);
  if (__any_sync(kWholeWarp, m.left != 0)) {
    exact_row<T, 2>(keys, q, c2, orow);
    __syncwarp();
    // (an infinity whose weight is 0 in f32 makes NaN there too)
    if (g < keys.granules) m = explain(nan_bits<T>(reinterpret_cast<const uint4*>(orow)[g]), seen);
    __syncwarp();
  }
  if (lane < 16) put_infinities(orow + g * 8, m);
}

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

  // Columns past D of the ring are never copied to: zero them.
  const int pad = 2 * NK - (p.D >> 3);
  auto zero_pad = [&](int row0, int rows) {
    for (int i = lane; i < rows * pad; i += 32)
      *reinterpret_cast<uint4*>(&sm.ring[warp][0][0][0] + (row0 + i / pad) * Sm::kStride +
                                ((p.D >> 3) + i % pad) * 16) = make_uint4(0u, 0u, 0u, 0u);
  };
  if (pad != 0) zero_pad(0, S * 2 * kDecKeys);
  wait_previous();
  allow_next();

  // Tiles and pieces in all (every warp for itself).
  int total = 0, total_pieces = 0;
  for (int b = lane; b < p.B; b += 32) {
    const int n = dec_tiles(dec_len(p, b));
    total += n;
    total_pieces += dec_pieces(n);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, d);
    total_pieces += __shfl_xor_sync(0xffffffffu, total_pieces, d);
  }
  total *= U;
  total_pieces *= U;

  // Sequences with nothing cached: zero output, lse -inf.
  auto empty_sequences = [&]() {
    for (int b = cta; b < p.B; b += grid) {
      const int n = ld_int(p.seq_lens + b);
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
  };

  // This CTA's tiles [begin, end): one piece of one unit, or share number cta.
  const bool by_piece = total_pieces <= grid;
  const int ncta = by_piece ? total_pieces : min(grid, total);
  if (cta >= ncta) {
    empty_sequences();
    return;
  }
  const int per_share = total / ncta, longer = total - per_share * ncta;
  auto share_begin = [&](int c) { return c * per_share + min(c, longer); };
  auto share_of = [&](int x) {
    return x < longer * (per_share + 1) ? x / (per_share + 1)
                                        : longer + (x - longer * (per_share + 1)) / per_share;
  };
  auto locate = [&](int x, int& rem) {   // cursor at the unit of item x, `rem` its item there
    DecCursor c;
    int first;
    c.b = dec_find(p, by_piece, U, x, first, lane);
    c.len = dec_len(p, c.b);
    c.ntiles = dec_tiles(c.len);
    const int per = by_piece ? dec_pieces(c.ntiles) : c.ntiles;
    const int u = x / per;
    rem = x - u * per;
    c.h = u / p.blocks;
    c.blk = u - c.h * p.blocks;
    c.first = first + u * c.ntiles;
    c.tile = rem;
    return c;
  };
  int begin, end, piece = 0, npieces = 1;
  DecCursor cur;
  if (by_piece) {   // pieces of a unit differ by one tile at most
    cur = locate(cta, piece);
    npieces = dec_pieces(cur.ntiles);
    const int pq = cur.ntiles / npieces, pr = cur.ntiles - pq * npieces;
    cur.tile = piece * pq + min(piece, pr);
    begin = cur.first + cur.tile;
    end = begin + pq + (piece < pr);
  } else {
    begin = share_begin(cta);
    end = share_begin(cta + 1);
    cur = locate(begin, cur.tile);
  }
  // The copying side runs ahead with a cursor of its own. Pages are looked up
  // one tile before their copies: one page for the warp's 16 keys where these
  // cannot straddle two, else lane l (and l + 16) that of key row l & 15. Each
  // lane copies the same NK granules of the 16 rows of every tile.
  DecCursor ahead = cur;
  const uint32_t ring0 = smem_u32(&sm.ring[warp][0][0][0]);
  const uint4* const kc = static_cast<const uint4*>(p.k_cache);
  const uint4* const vc = static_cast<const uint4*>(p.v_cache);
  struct Rows {
    int page;             // of the lane's key row (rows16: of the warp's 16 keys)
    int slot;             // in that page; < 0: no such key
    int held;             // keys of the 16 that the sequence has
    long long head_off;   // of the kv head, in granules
  };
  auto look_up = [&]() {
    Rows w;
    const int key0 = ahead.tile * kDecTile + warp * kDecKeys;
    const int key = p.rows16 ? key0 : key0 + (lane & 15);
    w.page = 0;
    w.slot = -1;
    w.held = ahead.len - key0;
    w.head_off = ahead.h * p.head_g;
    if (key < ahead.len) {
      const int pi = p.page_shift >= 0 ? key >> p.page_shift : key / p.page_size;
      w.page = ld_int(p.block_table + ahead.b * p.bt_stride + pi);
      w.slot = key - pi * p.page_size;
    }
    return w;
  };
  uint32_t goff[NK];   // granule i of the lane, from its row's (rows16: its tile's) first
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    const int idx = i * 32 + lane;
    goff[i] = idx % (2 * NK) + (p.rows16 ? idx / (2 * NK) * p.slot_g : 0);
  }
  auto copy_tile = [&](int stage, const Rows& w) {
    long long off = -1;
    if (w.slot >= 0) {
      if (w.page >= 0 && w.page < p.num_pages)
        off = static_cast<long long>(static_cast<uint64_t>(static_cast<uint32_t>(w.page)) * p.page_g +
                                     static_cast<uint64_t>(static_cast<uint32_t>(w.slot)) * p.slot_g) +
              w.head_off;
      else
        atomicCAS(&g_dev_status, 0, FRSA_DEV_INDEX);
    }
    const uint32_t dk = ring0 + stage * 2 * Sm::kRing;
    if (p.rows16 && off >= 0 && w.held >= kDecKeys) {
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
      const bool copy = e >= 0 && row < w.held;
      if (gcol * 8 < p.D) {
        e = copy ? e + goff[i] : 0;
        const uint32_t d = dk + row * Sm::kStride + gcol * 16;
        cp_async16_or_zero(d, kc + e, copy);
        cp_async16_or_zero(d + Sm::kRing, vc + e, copy);
      }
    }
  };
  int left = end - begin;         // tiles of the share that are not computed
  int ahead_left = left;          // ... not copied
  int ahead_of = 0, copy_stage = 0;   // tiles copied and not computed
  Rows rows_next;
  {   // the first tiles: their pages are looked up together
    Rows w[S - 1];
    const int n = min(S - 1, left);
#pragma unroll
    for (int i = 0; i < S - 1; ++i)
      if (i < n) {
        if (i > 0) dec_advance(p, ahead);
        w[i] = look_up();
      }
    ahead_left -= n;
    if (ahead_left > 0) {
      dec_advance(p, ahead);
      rows_next = look_up();
    }
#pragma unroll
    for (int i = 0; i < S - 1; ++i)
      if (i < n) {
        copy_tile(i, w[i]);
        cp_async_commit();
      }
    ahead_of = copy_stage = n;
    if (copy_stage == S) copy_stage = 0;
  }
  auto copy_next = [&]() {
    if (ahead_left == 0) return;
    copy_tile(copy_stage, rows_next);
    cp_async_commit();
    copy_stage = copy_stage + 1 == S ? 0 : copy_stage + 1;
    ++ahead_of;
    if (--ahead_left > 0) {
      dec_advance(p, ahead);
      rows_next = look_up();
    }
  };

  uint32_t qb[NT][NK][2];
  float o[NT][NK][4];   // O^T: rows 16 ks + quad, + 8; columns (heads) 8 nt + 2 ql, + 1
  float m[NT][2], l[NT][2];   // m: the base, kDecLift below the maximum
  bool fresh = true;
  const T* qp = static_cast<const T*>(p.q);
  const uint32_t ka = ring0 + ((lane >> 3 & 1) * 8 + (lane & 7)) * Sm::kStride + (lane >> 4) * 16;
  const uint32_t va = ring0 + Sm::kRing + ((lane >> 4) * 8 + (lane & 7)) * Sm::kStride +
                      (lane >> 3 & 1) * 16;
  int stage = 0;

  for (;;) {
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
                                ? ld_u32(qp + cur.b * p.qs[0] + (h0 + row) * p.qs[1] + col)
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
    cp_async_wait_to<S - 1>(ahead_of - 1);
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
        if constexpr (!Elt<T>::kBf16) {   // rounded up: no probability passes 2^15
          mx[0] = __fsub_ru(mx[0], kDecLift<T>);
          mx[1] = __fsub_ru(mx[1], kDecLift<T>);
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
    --ahead_of;
    --left;
    __syncwarp();   // the stage's rows are read before a later copy replaces them

    if (cur.tile + 1 < cur.ntiles && left > 0) {
      ++cur.tile;
      continue;
    }
    // The unit, or this share's part of it, ends: the four warps' states meet
    // in the ring stage that each has just read (the next copy into it comes
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
    // A share leaves two partials at most: of the unit that it ends (slot 2 c)
    // and of the unit that it begins (2 c + 1, unless that is all of it).
    // The four values of (nt, ks) of head pair nt 4 + ql lie at (((nt 4 + ql) NK
    // + ks) 8 + quad) 4: 16 bytes a lane, those of heads that exist alone.
    int parts = 1, part0 = 0;
    bool odd0 = false;
    if (!whole) {
      if (by_piece) {
        parts = npieces;
        part0 = cta - piece;
      } else {
        part0 = share_of(cur.first);
        parts = share_of(unit_end - 1) - part0 + 1;
        odd0 = share_begin(part0) != cur.first;
      }
    }
    auto slot_of = [&](int i) { return 2 * (part0 + i) + (i == 0 && odd0); };
    auto part_o = [&](int slot, int nt) {
      return reinterpret_cast<float4*>(p.part_o + static_cast<size_t>(slot) * p.slot_floats) +
             (nt * 4 + ql) * (NK * 8) + quad;
    };
    auto part_ml = [&](int slot, int nt) {
      return reinterpret_cast<float4*>(p.part_ml + (slot * kDecMaxHeads + nt * 8 + ql * 2) * 2);
    };
    if (!whole) {
      const int mine = slot_of(cta - part0);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        if (nt * 8 + ql * 2 < rows) {
          float4* po = part_o(mine, nt);
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            const int ks = warp + j * kDecWarps;
            if (ks < NK)
              __stcg(po + ks * 8, make_float4(acc[nt][j][0], acc[nt][j][1], acc[nt][j][2],
                                              acc[nt][j][3]));
          }
          if (warp == 0 && quad == 0)
            __stcg(part_ml(mine, nt), make_float4(m[nt][0], l[nt][0], m[nt][1], l[nt][1]));
        }
    }
    __syncthreads();   // the dumped states are read, the partial is written
    if (pad != 0) zero_pad(used * 2 * kDecKeys, 2 * kDecKeys);
    bool write = whole;
    if (!whole) {
      if (threadIdx.x == 0) {
        __threadfence();   // (the barrier ordered the CTA's writes before it)
        const int was = atomicAdd(p.counters + part0, 1);
        sm.last = was == parts - 1;
        if (was == parts - 1) p.counters[part0] = 0;   // as it was, for the next call
        __threadfence();
      }
      __syncthreads();
      write = sm.last != 0;
      if (write) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (nt * 8 + ql * 2 >= rows) continue;
          float mt[2] = {-INFINITY, -INFINITY}, lt[2] = {0.f, 0.f};
#pragma unroll
          for (int j = 0; j < kPer; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[nt][j][i] = 0.f;
#pragma unroll 1
          for (int c0 = 0; c0 < parts; c0 += kDecBatch) {
            float4 ml[kDecBatch];   // (m, l) of two heads
            float4 v[kDecBatch][kPer];
#pragma unroll
            for (int c = 0; c < kDecBatch; ++c) {
              const int slot = slot_of(min(c0 + c, parts - 1));
              const float4* po = part_o(slot, nt);
              ml[c] = __ldcg(part_ml(slot, nt));
#pragma unroll
              for (int j = 0; j < kPer; ++j)
                v[c][j] = __ldcg(po + min(warp + j * kDecWarps, NK - 1) * 8);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              float mn = mt[k];
#pragma unroll
              for (int c = 0; c < kDecBatch; ++c)   // (past the end: the last one again)
                mn = fmaxf(mn, k == 0 ? ml[c].x : ml[c].z);
              const float f = ex2(mt[k] - dec_base(mn));
              mt[k] = mn;
              lt[k] *= f;
#pragma unroll
              for (int j = 0; j < kPer; ++j) {
                acc[nt][j][k] *= f;
                acc[nt][j][2 + k] *= f;
              }
            }
#pragma unroll
            for (int c = 0; c < kDecBatch; ++c)
              if (c0 + c < parts) {
                const float f[2] = {ex2(ml[c].x - dec_base(mt[0])), ex2(ml[c].z - dec_base(mt[1]))};
                lt[0] += ml[c].y * f[0];
                lt[1] += ml[c].w * f[1];
#pragma unroll
                for (int j = 0; j < kPer; ++j) {
                  acc[nt][j][0] += v[c][j].x * f[0];
                  acc[nt][j][1] += v[c][j].y * f[1];
                  acc[nt][j][2] += v[c][j].z * f[0];
                  acc[nt][j][3] += v[c][j].w * f[1];
                }
              }
          }
          m[nt][0] = mt[0];
          m[nt][1] = mt[1];
          l[nt][0] = lt[0];
          l[nt][1] = lt[1];
        }
      }
      __syncthreads();   // sm.last is read
    }
    if (write) {
      bool odd = false;   // a NaN that does not come from the row's scores
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float inv[2] = {1.f / l[nt][0], 1.f / l[nt][1]};
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const int ks = warp + j * kDecWarps;
          if (ks >= NK) continue;
          const float(&v)[4] = acc[nt][j];
#pragma unroll
          for (int i = 0; i < 4; ++i) odd |= isnan(v[i]) && l[nt][i & 1] > 0.f;
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
      if (__syncthreads_or(odd)) {   // (the barrier orders the rows' writes before their reads)
        const DecKeys keys = {kc, vc, p.block_table + cur.b * p.bt_stride, cur.h * p.head_g,
                              p.page_g, p.slot_g, p.page_size, p.num_pages, cur.len, p.D >> 3};
#pragma unroll 1
        for (int r = warp; r < rows; r += kDecWarps) {
          bool sound = false;   // l of head r: lane (r & 7) / 2, column r & 1 of part r / 8
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c)
              if (__shfl_sync(kWholeWarp, l[nt][c], (r & 7) >> 1) > 0.f && nt == r >> 3 &&
                  c == (r & 1))
                sound = true;
          if (sound)
            dec_mend<T>(keys,
                        qp + cur.b * p.qs[0] +
                            (cur.h * p.group + cur.blk * 8 * NT + r) * p.qs[1],
                        p.c2, static_cast<T*>(p.o) + (row0 + r) * p.D);
        }
      }
    }
    fresh = true;
    if (left > 0) {
      dec_advance(p, cur);
      continue;
    }
    break;
  }
  empty_sequences();
}

template <typename T, int NK, int NT>
cudaError_t launch_decode_t(DecodeParams& p, int grid, cudaStream_t stream) {
  p.slot_floats = ((p.group < 8 * NT ? p.group : 8 * NT) + 1) / 2 * NK * 32;
  auto kern = paged_decode_kernel<T, NK, NT>;
  const size_t smem = sizeof(DecSmem<NK, NT>);
  const cudaError_t e = set_max_dynamic_smem_once(kern, smem);
  if (e != cudaSuccess) return e;
  return launch_after(kern, grid, kDecThreads, smem, stream, p);
}

template <typename T, int NT>
cudaError_t launch_decode_nk(DecodeParams& p, int grid, cudaStream_t stream) {
  if (p.D <= 32) return launch_decode_t<T, 2, NT>(p, grid, stream);
  if (p.D <= 64) return launch_decode_t<T, 4, NT>(p, grid, stream);
  if (p.D <= 80) return launch_decode_t<T, 5, NT>(p, grid, stream);
  if (p.D <= 96) return launch_decode_t<T, 6, NT>(p, grid, stream);
  return launch_decode_t<T, 8, NT>(p, grid, stream);
}

// Groups of up to 8 query heads take 8 columns, larger ones blocks of 16, each of
// which reads the keys again, mostly from L2 (4 sequences of 16384 tokens, 2 kv
// heads of 128: groups of 8 take 22 us, of 16 32, of 17 36, of 32 37, of 64 54).
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
size_t decode_workspace_bytes() {   // two partials per share
  return decode_counter_bytes() + static_cast<size_t>(2) * decode_grid() * kDecMaxHeads *
                                      (kDecMaxD + 2) * sizeof(float);
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
  // Few tokens: a CTA each, for the shortest chain.
  p.tokens = a.T > 4 * device_sm_count() ? kAppendMost : 1;
  const unsigned grid = static_cast<unsigned>((a.T + p.tokens - 1) / p.tokens);
  return launch_after(a.dtype == FRSA_DTYPE_BF16 ? paged_append_kernel<__nv_bfloat16>
                                                 : paged_append_kernel<__half>,
                      grid, kAppendThreads, 0, stream, p);
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
  p.part_ml = p.part_o + static_cast<size_t>(2) * grid * kDecMaxHeads * kDecMaxD;
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
