// Causal attention over whole packed prompts with grouped heads:
//   o[t, h] = sum_{j <= t, same sequence} softmax_j(scale q[t, h] . k[j, h']) v[j, h'],
// h' = h / (Hq / Hkv), q [T, Hq, D], k and v [T, Hkv, D], sequence b = tokens
// [cu_seqlens[b], cu_seqlens[b + 1]). q and k arrive rotated.
//
// A query tile has 128 rows: TT = 128 / G tokens (rounded down) times the G
// query heads that share a kv head, row = token * G + head. One tile of
// products then serves all heads of the group, short prompts fill the rows,
// and the causal edge wastes at most TT tokens' worth of scores per row
// block. A unit is one or two consecutive query tiles of one (sequence, kv
// head); a persistent CTA walks its units, both tiles of a unit share each
// K / V load.
//
//   warp 0       TMA producer: the unit's query tiles, then K and V tiles of
//                128 keys into rings of KS stages
//   warp 1       TMEM allocator + tcgen05.mma issuer (the whole warp runs it, one
//                elected lane issues): P V and the next scores of one query tile,
//                then of the other, so that one is in its softmax while the
//                other's products run (with an issuer per query tile both came
//                into step: 673 against 637 us for one prompt of 8192 tokens, in
//                an earlier state)
//   warp 2       scheduler: turns unit numbers into units, one ahead. The grid
//                has one CTA per unit number; a running CTA takes over the
//                next one that has not started (clusterlaunchcontrol), so the
//                longest units, which come first, are shared out as SMs get
//                free
//   warp 3       mender: rows that hold a NaN (below). It has a warp of its own
//                because the same code in the softmax warps, inlined or called,
//                costs them 3 % where there is nothing to mend (one prompt of 8192
//                tokens 507 against 484 us)
//   warps 4..11  two softmax warpgroups, one per query tile (thread = row =
//                TMEM lane)
//
// TMEM columns: warpgroup g uses [256 g, 256 g + 128) for the scores and the
// columns from 256 g + 128 on for O, which accumulates there over the unit's
// key tiles. P is written as packed 16-bit pairs: for D <= 64 into columns of
// its own (256 g + 192 on), so that the next scores are computed as soon as
// these have been read; for larger D over the scores: with key tiles of 128, P
// takes 64 columns and O leaves 128 - D of them. The
// softmax base is raised (and O rescaled) only when a tile's maximum leaves
// the range above it (PrBase). P of a tile's first 64 keys is published before the
// rest is computed. The products of a tile's last keys are cut to the 16-key steps
// that some row can see.
//
// What bounds it: for one prompt of 8192 tokens (32 and 8 heads, D = 128) 509
// us over repeated calls, 1080 TFLOP/s, 65 % of the card's measured rate (479
// in a single one, before the card lowers its clocks under the power limit). Per
// 128 keys of a query tile 1.5 us of softmax (0.3 of them waits for TMEM, the
// rest about 600 instructions on a chain per row) and 0.4 us of products before
// the next scores; the two tiles share the SM's exponentials and its tensor core,
// of each of which they use 60 %. Tried and not faster: two threads per row; a
// fourth or an eighth of the exponentials by a polynomial on the FMA pipe; a
// thread of its own for each tile's products. Not kept: for bf16, whose range
// would allow it, no maximum per tile but a base raised when the sum has grown
// (478 against then 491 us, but a row that rises by more than 2^95 within a tile
// overflows; with a guard against that 486 us and slower on short prompts).
//
// Masked places: keys past a row's position get P = 0, but 0 times an infinity
// or NaN in V (a later token's, or another sequence's in the same tile) would
// still reach O. It makes NaN, so a row that holds a NaN is looked at again
// (pr_mend): where the V of keys that it sees explains it, by a NaN or infinities
// of both signs, the NaN stands; by one infinity, that is put in its place;
// otherwise the row is computed once more in f32, from its keys alone. One NaN in
// a sequence thus costs the rows behind it a search, which looks first where the
// last one ended (8192 tokens of 8 and 2 heads of 128: 0.16 ms; with a NaN in the
// first token's V 0.23, in the middle one's 0.36, with one element of V in a
// thousand infinite, where most rows see masked ones beside it, 65). The limit of
// the waits applies to the time between two rows then.
#include "frsa_internal.h"
#include "frsa_ptx.cuh"
#include "frsa_row.cuh"

namespace frsa {

namespace {

constexpr int kPrThreads = 384;
// Registers per thread after the split (launch: 168 each; 88 + 2 x 208 = 3 x 168).
constexpr uint32_t kPrRegsCtl = 88, kPrRegsSoftmax = 208;
// Softmax base (log2): set kLift below a maximum, raised when a tile's maximum
// lies more than kRange above it. The sums and O, in f32, do not mind; P is
// rounded to the type and has to stay in its range. bf16 has f32's: P between
// 2^-8 and 1 for a row's largest score, so that O stays in range where the result
// does. f16, whose smallest step is 2^-24: P of a row's largest
// score lies between 2^11 and 2^15, so that what lies 2^-25 below it (17 nats)
// is still normal and the rounding of smaller ones at most 2^-36 of it. (With
// the base at the maximum a tail 17 nats below one large score was 40 % off.)
template <typename T>
struct PrBase {
  static constexpr float kLift = Elt<T>::kBf16 ? -8.f : 11.f;
  static constexpr float kRange = Elt<T>::kBf16 ? 0.f : 15.f;
  // From here on the base's own step, by which it may lie above the scores, takes
  // P out of the range (f16: 16 at 2^27; bf16: 64 at 2^29): such a row is computed
  // again in f32.
  static constexpr float kCoarse = Elt<T>::kBf16 ? 536870912.f : 134217728.f;
};

// Base of a row with no score above -inf so far: finite, so that such scores give
// P = 0, and below every other.
constexpr float kPrNone = -3e38f;

struct PromptUnit {
  int valid;       // 0: no more units
  int start, len;  // the sequence's first token and length
  int tok0;        // first token (in the sequence) of query tile 0; tile 1 follows at + TT
  int kvh;
  int n[2];        // key tiles of each query tile (0: the tile has no tokens)
};

// What a softmax warp asks the mender to look at: rows (bits) of a query tile that
// begins at token t0 of the sequence from token `start` on; odd: the row holds a
// NaN, redo: it is computed again in any case.
struct Mend {
  int start, kvh, t0;
  unsigned odd, redo;
};

template <int NCH>
struct PromptSmem {
  static constexpr int KS = NCH == 1 ? 4 : 2;
  uint8_t q[2][NCH][kChunkBytes];
  uint8_t k[KS][NCH][kChunkBytes];
  uint8_t v[KS][NCH][kChunkBytes];
  uint64_t q_full[2], q_empty[2];
  uint64_t k_full[KS], k_empty[KS], v_full[KS], v_empty[KS];
  // s_free, pv_done at every key tile: NCH == 1 only (else pv_done at a unit's end).
  uint64_t s_full[2], s_free[2], p_full[2][2], pv_done[2];   // p_full: [tile][64-key half]
  uint64_t unit_full[2], unit_empty[2];
  uint64_t next_full, drained;
  uint64_t mend_full[2], mend_empty[2];
  alignas(16) uint32_t next[4];   // answer to the request for another unit number
  PromptUnit unit[2];
  Mend mend[2][8];
  int mend_end[2];
  uint32_t tmem_base;
  int abort_flag;
  uint32_t beat;   // rows that the mender has looked at
};

struct PromptParams {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  float* lse;
  const int* cu;
  long long qs[2], ks[2], vs[2];   // token and head strides
  int T, B, Hq, Hkv, D;
  int G, TT, ntile;   // heads per kv head, tokens per query tile, query tiles per unit
  int nids;           // unit numbers: an upper bound of the units
  float c2;
};

// Tokens [start, end) of sequence b, held within [0, T).
__device__ __forceinline__ void pr_sequence(const PromptParams& p, int b, int& start, int& len) {
  const int s = ld_int(p.cu + b), e = ld_int(p.cu + b + 1);
  start = min(max(s, 0), p.T);
  len = max(min(e, p.T) - start, 0);
  if (s < 0 || e < s || e > p.T) atomicCAS(&g_dev_status, 0, FRSA_DEV_INDEX);
}
__device__ __forceinline__ int pr_units_of(const PromptParams& p, int b) {
  int start, len;
  pr_sequence(p, b, start, len);
  const int per = p.TT * p.ntile;
  return (len + per - 1) / per;
}

// Unit number -> unit, by a whole warp. Up to 32 sequences the longest units
// come first over all sequences (a unit of query block t reads about t key
// blocks, so: by descending t); beyond that, where a lane would hold several
// sequences, sequence after sequence, each with its longest units first. What the
// order is worth (32 and 8 heads of 128): one of 2048 tokens before 40 of 64 takes
// 53 us, behind them 62; before or behind 31 of them, 53. The search reads about
// B / 32 pairs of boundaries for each unit, so many tiny sequences cost more than
// their work: 1000 of 16 tokens 0.59 ms, 2000 of them 2.1.
__device__ __forceinline__ PromptUnit pr_find_unit(const PromptParams& p, int id, int lane) {
  PromptUnit x;
  x.valid = 0;
  x.kvh = id % p.Hkv;
  int rank = id / p.Hkv;
  int b, t;
  if (p.B <= 32) {
    const int nb = lane < p.B ? pr_units_of(p, lane) : 0;
    auto at_least = [&](int lvl) {   // units with query block >= lvl (each lane its own lvl)
      int sum = 0;
      for (int i = 0; i < p.B; ++i) sum += max(0, __shfl_sync(0xffffffffu, nb, i) - lvl);
      return sum;
    };
    int n = nb;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) n = max(n, __shfl_xor_sync(0xffffffffu, n, d));
    if (rank >= at_least(0)) return x;
    int lo = 0;   // the largest t with at_least(t) > rank lies in [lo, lo + n)
    while (n > 1) {
      const int step = (n + 31) / 32;
      const int c = at_least(lo + lane * step);
      const unsigned mask = __ballot_sync(0xffffffffu, lane * step < n && c > rank);
      const int i = 31 - __clz(mask);
      n = min(step, n - i * step);
      lo += i * step;
    }
    t = lo;
    rank -= at_least(t + 1);
    const unsigned mask = __ballot_sync(0xffffffffu, nb > t);
    b = static_cast<int>(__fns(mask, 0, rank + 1));
  } else {
    int lo = 0, n = p.B;
    while (n > 1) {   // the sequence that holds `rank`, 32 runs of sequences a level
      const int step = (n + 31) / 32;
      const int i0 = lo + min(n, lane * step), i1 = lo + min(n, (lane + 1) * step);
      int sum = 0;
      for (int i = i0; i < i1; ++i) sum += pr_units_of(p, i);
      int incl = sum;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += o;
      }
      const unsigned mask = __ballot_sync(0xffffffffu, incl > rank);
      if (mask == 0) return x;
      const int i = __ffs(mask) - 1;
      rank -= __shfl_sync(0xffffffffu, incl - sum, i);
      lo = __shfl_sync(0xffffffffu, i0, i);
      n = __shfl_sync(0xffffffffu, i1 - i0, i);
    }
    b = lo;
    const int nb = pr_units_of(p, b);
    t = nb - 1 - rank;
  }
  pr_sequence(p, b, x.start, x.len);
  x.tok0 = t * p.TT * p.ntile;
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const int t0 = x.tok0 + g * p.TT;
    x.n[g] = g < p.ntile && t0 < x.len ? (min(x.len, t0 + p.TT) + kTile - 1) / kTile : 0;
  }
  x.valid = 1;
  return x;
}

// Keys of tile j that a query tile ending at token `last` (exclusive) can
// see, rounded up to the products' 16-key step.
__device__ __forceinline__ int pr_keys(int last, int j) {
  return min(kTile, (last - j * kTile + 15) & ~15);
}

// Asks for the next CTA of the grid that has not started, to run its work in
// its place; the 16-byte answer lands in `answer`, counted on `bar`.
__device__ __forceinline__ void request_next(uint32_t* answer, uint64_t* bar) {
  mbar_arrive_expect_tx(bar, 16);
  asm volatile(
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::
          "r"(smem_u32(answer)), "r"(smem_u32(bar))
      : "memory");
}
// The taken CTA's blockIdx.x, or -1 when none was left.
__device__ __forceinline__ int next_id(const uint32_t* answer) {
  uint32_t ok, x;
  asm volatile(
      "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\t"
      "ld.shared.b128 h, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "mov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}"
      : "=r"(ok), "=r"(x)
      : "r"(smem_u32(answer))
      : "memory");
  return ok ? static_cast<int>(x) : -1;
}

// Pairs of f32 in one 64-bit register.
__device__ __forceinline__ uint64_t f2_make(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 f2_get(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The keys of one (sequence, kv head) for frsa_row.cuh.
struct PrKeys {
  const uint4* k0;
  const uint4* v0;
  long long ks, vs;   // token strides in granules
  int n, granules;
  __device__ int place(int j) const { return j; }
  __device__ const uint4* k(int j) const { return k0 + j * ks; }
  __device__ const uint4* v(int j) const { return v0 + j * vs; }
};

// The 32 rows from `row0` on of a query tile, as they were written, by a whole warp.
// `hint`: the token where the last call found a NaN, or -1.
template <typename T>
__device__ __forceinline__ void pr_mend(const PromptParams& p, const Mend& a, int row0, int& hint,
                                        volatile uint32_t* beat) {
  const int lane = threadIdx.x & 31;
  const bool odd = a.odd >> lane & 1;
  PrKeys keys;
  keys.k0 = reinterpret_cast<const uint4*>(static_cast<const T*>(p.k) + a.start * p.ks[0] +
                                           a.kvh * p.ks[1]);
  keys.v0 = reinterpret_cast<const uint4*>(static_cast<const T*>(p.v) + a.start * p.vs[0] +
                                           a.kvh * p.vs[1]);
  keys.ks = p.ks[0] >> 3;
  keys.vs = p.vs[0] >> 3;
  keys.granules = p.D >> 3;
  auto token = [&](int r) { return a.t0 + r / p.G; };
  auto head = [&](int r) { return a.kvh * p.G + r % p.G; };
  auto out = [&](int r) {
    return static_cast<T*>(p.o) + (static_cast<long long>(a.start + token(r)) * p.Hq + head(r)) * p.D;
  };
  if (lane == 0) *beat = *beat + 1;
  const uint4* mine = reinterpret_cast<const uint4*>(out(row0 + lane));
  const int tok0 = __shfl_sync(kWholeWarp, token(row0), 0), tok = token(row0 + lane);
  uint32_t want = 0, seen = 0;   // 8 columns at lane & 15 = granule
  if (a.odd != 0) {
    // The NaN columns of all rows, and what the keys hold there that the first row
    // sees, and with it all rows ...
#pragma unroll 1
    for (int g = 0; g < keys.granules; ++g) {
      const uint32_t all = __reduce_or_sync(kWholeWarp, odd ? nan_bits<T>(mine[g]) : 0u);
      if ((lane & 15) == g) want = all;
    }
    int at = hint - a.start;
    seen = special_columns<T, 8>(keys, tok0 + 1, want, at);
    hint = a.start + at;
  }
  bool again = a.redo >> lane & 1;
  const bool search = __any_sync(kWholeWarp, (want & ~explained(seen)) != 0);
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    if (search) {
      // ... and those up to the row itself (fewer than 32; lane i looks at K of the
      // i-th of them).
      const int more = token(row0 + 31 - __clz(a.odd)) - tok0;
      uint32_t k_odd = 0;
      if (lane < more)
#pragma unroll 1
        for (int g = 0; g < keys.granules; ++g)
          k_odd |= bits_from(keys.k(tok0 + 1 + lane)[g], kInf<T>);
      const unsigned unsure = __ballot_sync(kWholeWarp, k_odd != 0);
#pragma unroll 1
      for (int g = 0; g < keys.granules; ++g) {
        const uint32_t nan = odd ? nan_bits<T>(mine[g]) : 0u;
        uint32_t holds = __shfl_sync(kWholeWarp, seen, g);
        if (!__any_sync(kWholeWarp, (nan & ~explained(holds)) != 0)) continue;
#pragma unroll 1
        for (int i = 0; i < more; ++i) {
          uint32_t x = special_bits<T>(keys.v(tok0 + 1 + i)[g]);
          if (unsure >> i & 1) x = (x & 0xffu) | ((x >> 8 | x >> 16) & 0xffu) << 24;
          if (tok0 + 1 + i <= tok) holds |= x;
        }
        const Mended m = explain(nan, holds);
        again |= m.left != 0;
        put_infinities(out(row0 + lane) + g * 8, m);
      }
      __syncwarp();
    }
    // (The second time only for rows that were computed again: an infinity whose
    // weight is 0 in f32 makes NaN there too.)
    if (pass == 1) break;
    unsigned todo = __ballot_sync(kWholeWarp, again);
    if (todo == 0) break;
    while (todo != 0) {
      const int i = __ffs(todo) - 1, r = row0 + i;
      todo &= todo - 1;
      if (lane == 0) *beat = *beat + 1;
      keys.n = __shfl_sync(kWholeWarp, token(r) + 1, 0);
      const float lse = exact_row<T, 4>(
          keys, static_cast<const T*>(p.q) + (a.start + token(r)) * p.qs[0] + head(r) * p.qs[1],
          p.c2, out(r));
      if (p.lse != nullptr && lane == i)
        p.lse[static_cast<long long>(head(r)) * p.T + a.start + token(r)] = lse;
    }
    __syncwarp();
  }
}

template <typename T, int NCH>
__global__ void __launch_bounds__(kPrThreads, 1)
    prompt_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                  const __grid_constant__ CUtensorMap tm_v, const PromptParams p) {
  using Sm = PromptSmem<NCH>;
  constexpr int KS = Sm::KS;
  constexpr bool kOwnP = NCH == 1;         // P has TMEM columns of its own
  constexpr uint32_t kPCol = kOwnP ? 192 : 0;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Sm* smp = aligned_smem<Sm>(smem_raw);
  if (smp == nullptr) return;
  Sm& sm = *smp;
  // (through a shuffle: the compiler then knows that it is the same in the warp)
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int DP = (p.D + 15) & ~15;
  volatile int* abort_flag = &sm.abort_flag;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return mbar_wait(bar, parity, abort_flag, &sm.beat);
  };

  if (threadIdx.x == 0) {
    sm.abort_flag = 0;
    sm.beat = 0;
    for (int s = 0; s < 2; ++s) {
      mbar_init(&sm.q_full[s], 1);
      mbar_init(&sm.q_empty[s], 1);
      mbar_init(&sm.s_full[s], 1);
      mbar_init(&sm.p_full[s][0], 4);
      mbar_init(&sm.p_full[s][1], 4);
      mbar_init(&sm.s_free[s], 4);
      mbar_init(&sm.pv_done[s], 1);
      mbar_init(&sm.unit_full[s], 1);
      mbar_init(&sm.unit_empty[s], 10);   // producer, issuer, eight softmax warps
      mbar_init(&sm.mend_full[s], 8);
      mbar_init(&sm.mend_empty[s], 1);
    }
    for (int s = 0; s < KS; ++s) {
      mbar_init(&sm.k_full[s], 1);
      mbar_init(&sm.k_empty[s], 1);
      mbar_init(&sm.v_full[s], 1);
      mbar_init(&sm.v_empty[s], 1);
    }
    mbar_init(&sm.next_full, 1);
    mbar_init(&sm.drained, 1);
    sm.mend_end[0] = sm.mend_end[1] = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&sm.tmem_base, 512);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  wait_previous();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;

  // Unit i of this CTA: slot i & 1 of the unit ring, parity (i >> 1) & 1.
  // On a wait that gave up the unit counts as the end, for all lanes of a warp
  // alike (take_unit); the producer is a single lane (take_unit_alone).
  auto take_unit_alone = [&](int i) {
    PromptUnit x;
    x.valid = 0;
    if (wait(&sm.unit_full[i & 1], (i >> 1) & 1)) x = sm.unit[i & 1];
    return x;
  };
  auto take_unit = [&](int i) {
    PromptUnit x;
    x.valid = 0;
    if (__all_sync(0xffffffffu, wait(&sm.unit_full[i & 1], (i >> 1) & 1)))
      x = sm.unit[i & 1];
    return x;
  };

  if (warp < 4) {
    setmaxnreg_dec<kPrRegsCtl>();
    if (warp == 2) {
      // ---------------------------------------------------------- scheduler
      int id = blockIdx.x, i = 0;
      for (int asked = 0;; ++asked) {
        const PromptUnit x = pr_find_unit(p, id, lane);
        // Tokens before the first sequence and after the last belong to none:
        // zero output.
        const int past = min(max(ld_int(p.cu + p.B), 0), p.T);
        const int early = min(max(ld_int(p.cu), 0), past);
        for (long long n = id; n < early + p.T - past; n += p.nids) {
          const long long t = n < early ? n : past + n - early;
          uint4* row = reinterpret_cast<uint4*>(static_cast<T*>(p.o) + t * p.Hq * p.D);
          for (int e = lane; e < p.Hq * (p.D >> 3); e += 32) row[e] = make_uint4(0u, 0u, 0u, 0u);
          if (p.lse != nullptr)
            for (int h = lane; h < p.Hq; h += 32)
              p.lse[static_cast<long long>(h) * p.T + t] = -INFINITY;
        }
        if (x.valid) {   // (its slot is free: the unit before it has been taken by all)
          if (lane == 0) {
            sm.unit[i & 1] = x;
            mbar_arrive(&sm.unit_full[i & 1]);
          }
          __syncwarp();
          // Another unit is asked for when this one's softmax begins. (Three
          // ahead, CTAs were done between 391 and 439 us of one prompt of 8192
          // tokens.)
          wait(&sm.unit_empty[i & 1], (i >> 1) & 1);
          ++i;
        }
        if (__any_sync(0xffffffffu, *abort_flag != 0)) break;
        if (lane == 0) request_next(sm.next, &sm.next_full);
        if (!__all_sync(0xffffffffu, wait(&sm.next_full, asked & 1))) {
          mbar_wait_limit(&sm.next_full, asked & 1);   // the answer lands before the CTA ends
          break;
        }
        id = next_id(sm.next);
        fence_proxy_async_smem();   // read before the next answer is written
        __syncwarp();
        if (id < 0) break;
      }
      if (lane == 0) {
        sm.unit[i & 1].valid = 0;
        mbar_arrive(&sm.unit_full[i & 1]);
      }
    } else if (warp == 0) {
      // ---------------------------------------------------------- producer
      if (lane == 0) {
        const uint32_t qbytes = static_cast<uint32_t>(NCH * p.G * p.TT * 128);
        int qf[2] = {0, 0}, kf = 0, vf = 0;   // fills issued
        bool ok = true;
        for (int i = 0; ok; ++i) {
          const PromptUnit x = take_unit_alone(i);
          if (!x.valid) break;
          mbar_arrive(&sm.unit_empty[i & 1]);
          for (int g = 0; g < 2 && ok; ++g) {
            if (x.n[g] == 0) continue;
            if (!(ok = wait(&sm.q_empty[g], (qf[g] & 1) ^ 1))) break;
            mbar_arrive_expect_tx(&sm.q_full[g], qbytes);
            for (int c = 0; c < NCH; ++c)
              tma_load_3d(sm.q[g][c], &tm_q, &sm.q_full[g], c * kChunkCols, x.kvh * p.G,
                          x.start + x.tok0 + g * p.TT);
            ++qf[g];
          }
          const int nmax = max(x.n[0], x.n[1]);
          for (int j = 0; j < nmax && ok; ++j) {
            int s = kf % KS;
            if (!(ok = wait(&sm.k_empty[s], ((kf / KS) & 1) ^ 1))) break;
            mbar_arrive_expect_tx(&sm.k_full[s], NCH * kChunkBytes);
            for (int c = 0; c < NCH; ++c)
              tma_load_3d(sm.k[s][c], &tm_k, &sm.k_full[s], c * kChunkCols, x.kvh,
                          x.start + j * kTile);
            ++kf;
            s = vf % KS;
            if (!(ok = wait(&sm.v_empty[s], ((vf / KS) & 1) ^ 1))) break;
            mbar_arrive_expect_tx(&sm.v_full[s], NCH * kChunkBytes);
            for (int c = 0; c < NCH; ++c)
              tma_load_3d(sm.v[s][c], &tm_v, &sm.v_full[s], c * kChunkCols, x.kvh,
                          x.start + j * kTile);
            ++vf;
          }
        }
        // Every load that was issued lands before the CTA may end (a wait
        // only where some other wait gave up).
        for (int g = 0; g < 2; ++g)
          if (qf[g] > 0) mbar_wait_limit(&sm.q_full[g], (qf[g] - 1) & 1);
        for (int b = 1; b <= KS; ++b) {
          if (kf >= b) mbar_wait_limit(&sm.k_full[(kf - b) % KS], ((kf - b) / KS) & 1);
          if (vf >= b) mbar_wait_limit(&sm.v_full[(vf - b) % KS], ((vf - b) / KS) & 1);
        }
      }
    } else if (warp == 3) {
      // ------------------------------------------------------------ mender
      int hint = -1;
      for (int i = 0;; ++i) {
        const int s = i & 1;
        if (!__all_sync(kWholeWarp, wait(&sm.mend_full[s], (i >> 1) & 1))) break;
        if (sm.mend_end[s]) break;
#pragma unroll 1
        for (int w = 0; w < 8; ++w) {
          const Mend a = sm.mend[s][w];
          if ((a.odd | a.redo) != 0)
            pr_mend<T>(p, a, (w & 3) * 32, hint, &sm.beat);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.mend_empty[s]);
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------- MMA issuer
      // The whole warp runs this; one elected lane issues. Descriptors stay in
      // uniform registers that way: with the loop inside `lane == 0` a product
      // was issued every 110 clocks, where it takes 64.
      {
        constexpr bool kBf = Elt<T>::kBf16;
        const int ksteps = DP >> 4;
        const uint32_t idO = idesc_f16(kBf, 128, DP, false, true);
        const uint64_t q_desc = sw128_desc(smem_u32(sm.q[0][0]), 16, 1024);
        const uint64_t k_desc = sw128_desc(smem_u32(sm.k[0][0]), 16, 1024);
        const uint64_t v_desc = sw128_desc(smem_u32(sm.v[0][0]), kChunkBytes, 1024);
        constexpr uint64_t kTileStep = NCH * kChunkBytes >> 4;   // of the next tile in a ring
        auto issue_s = [&](int g, int s, int keys) {
          const uint32_t tS = tmem + 256 * g;
          const uint32_t idS = idesc_f16(kBf, 128, keys, false, false);
          const uint64_t qd = q_desc + g * kTileStep, kd = k_desc + s * kTileStep;
#pragma unroll
          for (int ks = 0; ks < 4 * NCH; ++ks) {
            const uint64_t off = (ks >> 2) * (kChunkBytes >> 4) + (ks & 3) * 2;
            if (ks < ksteps) mma_ss_elect(tS, qd + off, kd + off, idS, ks > 0);
          }
          mma_commit_elect(&sm.s_full[g]);
        };
        auto issue_pv = [&](int g, int s, bool acc, int ks0, int ks1) {
          const uint32_t tS = tmem + 256 * g, tO = tS + 128;
          const uint64_t vd = v_desc + s * kTileStep;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int ks = ks0 + k;
            if (ks < ks1) mma_ts_elect(tO, tS + kPCol + 8 * ks, vd + ks * 128, idO, acc || ks > 0);
          }
        };
        auto last_of = [&](const PromptUnit& y, int g) {
          return min(y.len, y.tok0 + (g + 1) * p.TT);
        };
        int qf[2] = {0, 0}, tg[2] = {0, 0};
        int t = 0, i = 0;
        // A unit's scores against its first key tile (tile number `tile`).
        auto first_scores = [&](const PromptUnit& y, int tile) {
          const int s = tile % KS;
          wait(&sm.k_full[s], (tile / KS) & 1);
          for (int g = 0; g < 2; ++g) {
            if (y.n[g] == 0) continue;
            wait(&sm.q_full[g], qf[g] & 1);
            ++qf[g];
            tc_fence_after();
            issue_s(g, s, pr_keys(last_of(y, g), 0));
            if (y.n[g] == 1) mma_commit_elect(&sm.q_empty[g]);
          }
          mma_commit_elect(&sm.k_empty[s]);
        };
        PromptUnit x = take_unit(0);
        if (x.valid) {
          if (lane == 0) mbar_arrive(&sm.unit_empty[0]);
          first_scores(x, 0);
        }
        while (x.valid) {
          const int nmax = max(x.n[0], x.n[1]);
          PromptUnit y;
          y.valid = 0;
          for (int j = 0; j < nmax; ++j, ++t) {
            const int s = t % KS, s1 = (t + 1) % KS;
            wait(&sm.v_full[s], (t / KS) & 1);
            if (j + 1 < nmax) wait(&sm.k_full[s1], ((t + 1) / KS) & 1);
            for (int g = 0; g < 2; ++g) {
              if (j >= x.n[g]) continue;
              const int steps = pr_keys(last_of(x, g), j) / 16;
              const bool more = j + 1 < x.n[g];
              if (kOwnP && more) {   // the next scores, as soon as these are read
                wait(&sm.s_free[g], tg[g] & 1);
                tc_fence_after();
                issue_s(g, s1, pr_keys(last_of(x, g), j + 1));
              }
              wait(&sm.p_full[g][0], tg[g] & 1);
              tc_fence_after();
              issue_pv(g, s, j > 0, 0, min(steps, 4));
              wait(&sm.p_full[g][1], tg[g] & 1);
              tc_fence_after();
              issue_pv(g, s, true, 4, steps);
              ++tg[g];
              if (kOwnP || !more) mma_commit_elect(&sm.pv_done[g]);
              // (in order after the products that read P from the same columns)
              if (!kOwnP && more) issue_s(g, s1, pr_keys(last_of(x, g), j + 1));
              if (j + 2 == x.n[g]) mma_commit_elect(&sm.q_empty[g]);
            }
            mma_commit_elect(&sm.v_empty[s]);
            if (j + 1 < nmax) {
              mma_commit_elect(&sm.k_empty[s1]);
            } else {
              y = take_unit(i + 1);
              if (y.valid) {
                if (lane == 0) mbar_arrive(&sm.unit_empty[(i + 1) & 1]);
                first_scores(y, t + 1);
              }
            }
          }
          x = y;
          ++i;
        }
        // The products complete before the CTA frees the tensor memory and ends,
        // also where a softmax warp's wait for them gave up.
        mma_commit_elect(&sm.drained);
        mbar_wait_limit(&sm.drained, 0);
      }
    }
  } else {
    // ------------------------------------------------------------ softmax
    setmaxnreg_inc<kPrRegsSoftmax>();
    const int g = (warp - 4) >> 2;
    const int wq = warp & 3;
    const int r = wq * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(wq * 32) << 16;
    using Base = PrBase<T>;
    const float c2 = p.c2;
    auto base_of = [&](float mx) { return __fmaf_ru(mx, c2, -Base::kLift); };
    const uint32_t tS = tmem + 256 * g + lane_off, tO = tS + 128, tP = tS + kPCol;
    const int rtok = r / p.G, head = r - rtok * p.G;
    int tg = 0, uo = 0;
    // What the mender has to look at in unit i (of every unit: it waits for all
    // eight warps).
    auto tell = [&](int i, const Mend& a, int end) {
      wait(&sm.mend_empty[i & 1], ((i >> 1) & 1) ^ 1);
      if (lane == 0) {
        sm.mend[i & 1][warp - 4] = a;
        if (end) sm.mend_end[i & 1] = 1;
      }
      __syncwarp();   // (orders the warp's rows before the mender's reads)
      if (lane == 0) mbar_arrive(&sm.mend_full[i & 1]);
    };
    for (int i = 0;; ++i) {
      const PromptUnit x = take_unit(i);
      if (!x.valid) {
        tell(i, Mend{0, 0, 0, 0u, 0u}, 1);
        break;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.unit_empty[i & 1]);
      if (x.n[g] == 0) {
        tell(i, Mend{0, 0, 0, 0u, 0u}, 0);
        continue;
      }
      const int t0 = x.tok0 + g * p.TT;
      const int tok = t0 + rtok;
      const int last = min(x.len, t0 + p.TT);
      const int see = min(tok, last - 1);   // the last key this row sees
      float m2 = kPrNone, l = 0.f;
      for (int j = 0; j < x.n[g]; ++j, ++tg) {
        const int keys = pr_keys(last, j);
        const bool edge = j * kTile + kTile - 1 > t0;   // some row does not see all keys
        wait(&sm.s_full[g], tg & 1);
        tc_fence_after();
        const int lim = see - j * kTile;   // the last key of the tile that this row sees
        // 64 scores at a time: with 96 or 128 in registers the compiler has none
        // left to overlap the exponentials (526 and 557 against 513 us for one
        // prompt of 8192 tokens).
        float sv[2][32];
        auto load = [&](int h) {
          if (h * 64 < keys) tmem_ld32(tS + h * 64, sv[0]);
          if (h * 64 + 32 < keys) tmem_ld32(tS + h * 64 + 32, sv[1]);
          tmem_wait_ld();
          if (edge) {   // (columns that were not loaded lie past lim)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (h * 64 + c * 32 + e > lim) sv[c][e] = -INFINITY;
          }
        };
        auto half_max = [&]() {
          float a[4] = {sv[0][0], sv[0][1], sv[0][2], sv[0][3]};
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 32; e += 8)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                a[k] = max3(a[k], sv[c][e + 2 * k], sv[c][e + 2 * k + 1]);
          return fmaxf(max3(a[0], a[1], a[2]), a[3]);
        };
        // P of 32 keys as packed pairs.
        uint64_t sp[2];
        auto exps = [&](int c, uint32_t(&pk)[16]) {
          const uint64_t cc = f2_make(c2, c2), mm = f2_make(-m2, -m2);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const uint64_t x = f2_fma(f2_make(sv[c][2 * e], sv[c][2 * e + 1]), cc, mm);
            const float2 z = f2_get(x);
            const float y0 = ex2(z.x), y1 = ex2(z.y);
            sp[e & 1] = f2_add(sp[e & 1], f2_make(y0, y1));
            pk[e] = Elt<T>::pack(y0, y1);
          }
        };
        auto publish = [&](int h) {
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.p_full[g][h]);
        };
        // The first 64 keys' P with the base so far, then the maximum of the rest;
        // rarely, a new base, and those keys again.
        uint32_t pk0[16], pk1[16];
        bool pv_waited = j == 0;
#pragma unroll 1
        for (;;) {
          load(0);
          float mx = half_max();
          // (Bases are rounded up, so that no exponent passes kRange.)
          if (m2 == kPrNone) m2 = fmaxf(base_of(mx), kPrNone);   // (the unit's first tile)
          sp[0] = sp[1] = f2_make(0.f, 0.f);
          exps(0, pk0);
          exps(1, pk1);
          if (64 < keys) {
            load(1);
            mx = fmaxf(mx, half_max());
          }
          if (kOwnP && !pv_waited) {   // the products before this tile have read P and written O
            pv_waited = true;
            wait(&sm.pv_done[g], uo & 1);
            ++uo;
            tc_fence_after();
          }
          const bool up = __fmaf_ru(mx, c2, -m2) > Base::kRange;
          if (!__any_sync(0xffffffffu, up)) break;
          const float mn = up ? base_of(mx) : m2;
          const float alpha = ex2(m2 - mn);
          l *= alpha;
          m2 = mn;
          if (j == 0) continue;
#pragma unroll 1
          for (int c16 = 0; c16 * 16 < DP; ++c16) {
            float ov[16];
            tmem_ld16(tO + c16 * 16, ov);
            tmem_wait_ld();
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(ov[e] * alpha);
            tmem_st16(tO + c16 * 16, w);
          }
        }
        if (kOwnP) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.s_free[g]);
        }
        tmem_st16(tP, pk0);
        if (32 < keys) tmem_st16(tP + 16, pk1);
        if (64 < keys) exps(0, pk0);   // while the stores complete
        publish(0);
        if (64 < keys) tmem_st16(tP + 32, pk0);
        if (96 < keys) {
          exps(1, pk1);
          tmem_st16(tP + 48, pk1);
        }
        publish(1);
        const float2 s0 = f2_get(f2_add(sp[0], sp[1]));
        l += s0.x + s0.y;
      }
      // O / l once the unit's last P V has completed.
      wait(&sm.pv_done[g], uo & 1);
      ++uo;
      tc_fence_after();
      const bool stored = rtok < p.TT && tok < x.len;
      const int h = x.kvh * p.G + head;
      const long long tq = x.start + tok;
      T* orow = static_cast<T*>(p.o) + (tq * p.Hq + h) * p.D;
      const float inv = 1.f / l;
      bool odd = false;   // a NaN in O
#pragma unroll 1
      for (int c = 0; c < DP; c += 32) {   // (the last 16 may be past DP: not stored)
        float v[32];
        tmem_ld32(tO + c, v);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          if (c + e < p.D) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float y0 = v[e + 2 * k] * inv, y1 = v[e + 2 * k + 1] * inv;
              odd |= isnan(v[e + 2 * k]) || isnan(v[e + 2 * k + 1]);
              w[k] = Elt<T>::pack(y0, y1);
            }
            if (stored)
              reinterpret_cast<uint4*>(orow + c + e)[0] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      tc_fence_before();   // O is read before this group's next arrival lets a product overwrite it
      if (stored && p.lse != nullptr)
        p.lse[static_cast<long long>(h) * p.T + tq] = (m2 + log2f(l)) * 0.69314718055994531f;
      // (l is NaN where a score is, and there is no base where all scores are -inf:
      // the row is NaN then.)
      const bool redo = stored && l >= 0.f && m2 > kPrNone && fabsf(m2) >= Base::kCoarse;
      const bool look = stored && l > 0.f && odd;
      tell(i, Mend{x.start, x.kvh, t0, __ballot_sync(kWholeWarp, look),
                   __ballot_sync(kWholeWarp, redo)}, 0);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T, int NCH>
cudaError_t launch_prompt_t(const PromptParams& p, const CUtensorMap& tq, const CUtensorMap& tk,
                            const CUtensorMap& tv, cudaStream_t stream) {
  const size_t smem = sizeof(PromptSmem<NCH>) + 1024;
  auto kern = prompt_kernel<T, NCH>;
  const cudaError_t e = set_max_dynamic_smem_once(kern, smem);
  if (e != cudaSuccess) return e;
  return launch_after(kern, p.nids, kPrThreads, smem, stream, tq, tk, tv, p);
}

}  // namespace

cudaError_t launch_prompt(const frsa_prompt_args& a, const CUtensorMap& tq, const CUtensorMap& tk,
                          const CUtensorMap& tv, cudaStream_t stream) {
  PromptParams p;
  p.q = a.q;
  p.k = a.k;
  p.v = a.v;
  p.o = a.o;
  p.lse = a.lse;
  p.cu = a.cu_seqlens;
  for (int i = 0; i < 2; ++i) {
    p.qs[i] = a.q_strides[i];
    p.ks[i] = a.k_strides[i];
    p.vs[i] = a.v_strides[i];
  }
  p.T = static_cast<int>(a.T);
  p.B = static_cast<int>(a.B);
  p.Hq = static_cast<int>(a.Hq);
  p.Hkv = static_cast<int>(a.Hkv);
  p.D = static_cast<int>(a.D);
  p.G = p.Hq / p.Hkv;
  p.TT = kTile / p.G;
  p.c2 = a.scale * 1.4426950408889634f;
  // Two query tiles per unit share its K and V loads and keep the tensor core
  // busy during one another's softmax; one, when two would leave SMs idle.
  auto ids = [&](int ntile) {
    return (static_cast<long long>(p.T) / (p.TT * ntile) + p.B) * p.Hkv;
  };
  p.ntile = ids(2) < device_sm_count() ? 1 : 2;
  p.nids = static_cast<int>(ids(p.ntile));
  const bool two = p.D > 64;
  if (a.dtype == FRSA_DTYPE_BF16)
    return two ? launch_prompt_t<__nv_bfloat16, 2>(p, tq, tk, tv, stream)
               : launch_prompt_t<__nv_bfloat16, 1>(p, tq, tk, tv, stream);
  return two ? launch_prompt_t<__half, 2>(p, tq, tk, tv, stream)
             : launch_prompt_t<__half, 1>(p, tq, tk, tv, stream);
}

}  // namespace frsa
