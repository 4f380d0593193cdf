// Attention over the 8-bit cache for many query rows, on SM pairs (tcgen05
// cta_group::2).  The query rows of the heads that share a cache head are one
// list of rows (row r: token r / group, head r % group); a cluster of two CTAs
// takes them in rounds of two 256-row tiles, each CTA 128 rows of a tile.
//
//   S = Q K^T            bf16 (e4m3 codes are exact in bf16)
//   x = S ks c           ks: the key block's scale, c = log2(e) / sqrt(D)
//   P = 2^(x - m + d)    m: running maximum of x, raised when x exceeds it by 8;
//                        d = lv - R, lv: log2 of the value block's scale
//   l += P 2^-d,  O += P V8       P and the value codes in f16
//   out = 2^R O / l
//
// so the cache's bytes enter the products as they are and its scales cost one
// fused multiply-add that the exponent needs anyway.  The reference R is one
// for all rows and keeps d in [0, 7], P within f16: P has every bit there that
// p = 2^(x - m) has.  Blocks outside the window move R, and O with it.  Where a
// step's two blocks lie further apart than the window, its P.V runs in two
// parts, the other block's probabilities zero and R moved in between.  (With
// the scale in the maximum instead, m the largest x + lv, a block of zeros,
// whose scale is 1, takes the bits of the small values beside it.)
//
// Per step of 128 keys each CTA converts its half of the pair's operands from
// the cache (64 keys x D, and D / 2 features x 128 tokens; the cache keeps
// the tokens of a value block innermost, so both halves are whole contiguous
// pieces and both operands are K-major) into a ring of stages.  Both tiles of
// a round use a stage, and where all steps fit the ring (D = 128: 512 keys)
// the stages stay for all rounds of a cache head.  With one tile per head the
// tiles' accumulators take the even and the odd steps instead.
//
// TMEM (512 columns per CTA): S at [0, 128); P of slot s at 128 + 64 s (f16
// pairs, the A operand); O of slot s at 256 + 128 s.  S(i + 1) may overwrite
// S(i) as soon as the softmax has copied it to registers, so the tensor core
// runs S of one slot while the other slot's softmax works.
//
// Work is dealt to the clusters in step space by the lengths on the device:
// equal numbers of steps each, whole rounds where all steps fit the ring,
// else rounds cut at the cluster boundaries, whose parts (2^R O / l, m,
// l) a second kernel joins in a fixed order.
//
// Roles per CTA (512 threads):
//   warps 0-3 / 4-7   softmax of slot 0 / 1 (thread <-> TMEM lane <-> row)
//   warps 8-11        cache conversion, epilogue
//   warps 12, 14      in the leader, the issuers of S and of P.V; TMEM allocation (12)
//   warp 13           query loads (TMA, or copies where a box cannot hold whole tokens)
//   warp 15           the scales: R, d and the factors of each step, for the softmax
// Every wait is bounded (about one second).
//
// 2 x 40 heads, D = 128: 32760 queries over 512 keys 635 to 680 us with the
// clock (1.0 PFLOP/s; the bf16 rate would be 426 us), 256 over 32000 540 us, of
// which filling the stages is the larger part.  In whole rounds a unit (a step of one tile)
// takes 1930 clk against 1049 of its products and 1024 of its exponentials:
// with the softmax's arithmetic left out it still takes 1500, the round trip
// of the one S buffer (product, read, next product), and a softmax warpgroup
// is busy for 3400 of the 3860 clk between its steps.  S in two halves with
// barriers of their own shortened the one and lengthened the other: 741 us.
#include "icsa_attn_common.cuh"
#include "icsa_lowp.cuh"
#include "icsa_pair.cuh"

#include <cuda_fp16.h>

#include <algorithm>
#include <utility>

namespace icsa {

namespace {

using namespace attn;

constexpr int kThreads = 512;
constexpr int kIssuerWarp = 12, kQueryWarp = 13, kPvWarp = 14, kScaleWarp = 15;
constexpr int kPairRows = 256, kCtaRows = 128;
constexpr int kStepKeys = 128;
constexpr int kMaxBatch = kKv8TcMaxBatch;
constexpr uint32_t kTmP = 128, kTmO = 256, kTmemCols = 512;

enum : int {
  kErrKvFull = 0x501, kErrKvEmpty = 0x502, kErrQFull = 0x503, kErrQEmpty = 0x504, kErrSFull = 0x505, kErrSFree = 0x506,
  kErrPFull = 0x507, kErrPvDone = 0x508, kErrOFull = 0x509, kErrOFree = 0x50A, kErrMlFull = 0x50B, kErrMlFree = 0x50C,
  kErrUnitFull = 0x50D, kErrUnitEmpty = 0x50E, kErrXFull = 0x50F, kErrXDone = 0x510
};

template <int D>
struct Cfg {
  static constexpr int kQBytes = kCtaRows * D * 2;
  static constexpr int kKBytes = 64 * D * 2;              // 64 keys, chunks of 8 KB
  static constexpr int kVRows = D / 2;                    // value features of this CTA
  static constexpr int kVChunk = kVRows * 128;            // 64 tokens of them
  static constexpr int kVBytes = 2 * kVChunk;
  static constexpr int kStages = D == 128 ? 4 : 8;
};

// A cluster's rounds of one batch element: [i, end), of which the first may
// start and the last may end inside a round.
struct Range {
  int i, end;
  int first, last;  // steps cut off the first and the last round
};

// What the softmax needs of a step's scales, in chunks of kChunk units of a slot.
constexpr int kChunk = 32;
struct __align__(16) Unit {
  float c0, c1;          // base-2 score of a product, for the step's first and second block
  float d0, d1;          // lv - R
  float w0, w1;          // 2^-d
  float ref0, ref1;      // R; where the two differ the step's P.V runs in two parts
  uint32_t stage, pad[3];  // the step's place in the ring of stages, counted on
};

template <int D>
struct __align__(1024) Smem {
  using C = Cfg<D>;
  uint8_t q[2][C::kQBytes];
  uint8_t kv[C::kStages][C::kKBytes + C::kVBytes];  // [keys | values]
  uint8_t out[4][32 * 128];                         // output box of each helper warp
  Range ranges[kMaxBatch];
  float ml[2][3][kCtaRows];                         // [slot][m, 2^-R l, 2^R] of a finished tile
  Unit units[2][2][kChunk];                         // [slot][buffer]
  uint32_t any_two[2][2];                         // whether a chunk has units that run in two parts
  uint64_t unit_full[2][2], unit_empty[2][2], x_full[2], x_done[2];
  uint64_t kv_full[C::kStages], kv_empty[C::kStages];
  uint64_t q_full[2], q_empty[2], s_full[2], s_free[2], p_full[2], pv_done[2], o_full[2], o_free[2];
  uint64_t ml_full[2], ml_free[2];
  uint64_t fin[2];
  uint32_t tmem_base;
  int abort_flag;
};

// ------------------------------------------------------------------- work --
struct Round {
  int b, h, r;       // batch, cache head, pair of tiles
  int len, n0, n1;   // valid keys; steps [n0, n1) of this cluster
  int part;          // -1: the whole round; else the cluster's partial buffer
  ICSA_DEV int steps() const { return n1 - n0; }
};

ICSA_DEV int cache_length(const Kv8Cache& c, int b) {
  return c.lengths == nullptr ? c.L : min(max(c.lengths[b], 0), c.L);
}
ICSA_DEV int steps_of(int len) { return (len + kStepKeys - 1) / kStepKeys; }

// Work space: the rounds of batch element 0, 1, .. one behind the other, heads
// outermost, a step of a round of two tiles weighing 12 and of one tile 10: the
// latter is bound by the filling of its stage.  (1 x 12 heads, 700 rows over
// 6000 keys, three tiles a head: 12 to 10 61.7 us, 12 to 9 63.6, 12 to 8, the
// ratio of the times that plan_attention fits over all sizes, 66.8.)  A round
// without keys, and in whole rounds its epilogue, count as a step.
constexpr int kWeightTwo = 12, kWeightOne = 10;
struct Extent {
  int n;             // steps that a round counts for
  int64_t head;      // of all rounds of a cache head
};
ICSA_DEV Extent extent(const Kv8TcParams& p, int len) {
  Extent e;
  e.n = p.whole ? steps_of(len) + 1 : max(1, steps_of(len));
  e.head = int64_t(e.n) * ((p.tiles >> 1) * kWeightTwo + (p.tiles & 1) * kWeightOne);
  return e;
}
// A point of a batch element's work space as a round and a step in it; points
// inside a step belong to it, and in whole rounds points inside a round to the
// next one.
struct Point {
  int round, step;
};
ICSA_DEV Point locate(const Kv8TcParams& p, const Kv8Cache& c, const Extent& e, int64_t x) {
  if (x <= 0) return {0, 0};
  if (x >= e.head * c.H) return {c.H * p.rounds, 0};
  const int h = int(x / e.head);
  int64_t in = x - int64_t(h) * e.head;
  const int two = p.tiles >> 1;
  const int r = min(int(in / (int64_t(e.n) * kWeightTwo)), two);
  in -= int64_t(r) * e.n * kWeightTwo;
  Point q = {h * p.rounds + r, int(in / (r < two ? kWeightTwo : kWeightOne))};
  if (p.whole && in > 0) {
    ++q.round;
    q.step = 0;
  }
  return q;
}

// (Computed once per CTA, a thread per batch element: inlined into every role
// its 64-bit divisions would be half of the kernel's code.)
// The batch element, round and step at which a cluster's range starts.
ICSA_DEV int4 cluster_start(const Kv8TcParams& p, const Kv8Cache& c, int cluster, int clusters) {
  int64_t total = 0;
  for (int i = 0; i < c.B; ++i) total += extent(p, cache_length(c, i)).head * c.H;
  int64_t x = total * cluster / clusters;
  int b = 0;
  Extent e = extent(p, cache_length(c, 0));
  while (x >= e.head * c.H && b + 1 < c.B) {
    x -= e.head * c.H;
    e = extent(p, cache_length(c, ++b));
  }
  const Point q = locate(p, c, e, x);
  return make_int4(b, q.round, q.step, 0);
}
ICSA_DEV Range cluster_range(const Kv8TcParams& p, const Kv8Cache& c, int b, int cluster, int clusters) {
  int64_t total = 0, base = 0;
#pragma unroll 1
  for (int k = 0; k < c.B; ++k) {
    if (k == b) base = total;
    total += extent(p, cache_length(c, k)).head * c.H;
  }
  const Extent e = extent(p, cache_length(c, b));
  const Point lo = locate(p, c, e, total * cluster / clusters - base);
  const Point hi = locate(p, c, e, total * (cluster + 1) / clusters - base);
  Range r;
  r.i = lo.round;
  r.first = lo.step;
  r.end = hi.round + (hi.step > 0 ? 1 : 0);
  r.last = hi.step > 0 ? e.n - hi.step : 0;
  if (lo.round == hi.round && lo.step == hi.step) r.end = r.i;
  return r;
}

// The rounds of one cluster, in order.
struct Walk {
  const Range* ranges;  // shared memory, one per batch element
  int b = -1, i = 0, end = 0;
  ICSA_DEV explicit Walk(const Range* r) : ranges(r) {}
  ICSA_DEV bool next(const Kv8TcParams& p, const Kv8Cache& c, Round& out) {
    while (i == end) {
      if (++b >= c.B) return false;
      i = ranges[b].i;
      end = ranges[b].end;
    }
    const Range r = ranges[b];
    out.b = b;
    out.h = i / p.rounds;
    out.r = i - out.h * p.rounds;
    out.len = cache_length(c, b);
    out.n0 = i == r.i ? r.first : 0;
    const int cut = i + 1 == end ? r.last : 0;
    out.n1 = steps_of(out.len) - cut;
    out.part = out.n0 > 0 ? 0 : cut > 0 ? 1 : -1;
    ++i;
    return true;
  }
};

// Whether a round's stages are not those of the round before it.
ICSA_DEV bool new_kv(const Kv8TcParams& p, const Round& a, const Round& before) {
  return !p.whole || a.b != before.b || a.h != before.h;
}

// Steps of slot s in a round: every step of its own tile, or every second
// step of the round's only tile.
ICSA_DEV bool has_tile(const Kv8TcParams& p, const Round& w, int s) { return 2 * w.r + s < p.tiles; }
ICSA_DEV bool alternate(const Kv8TcParams& p, const Round& w) { return !has_tile(p, w, 1); }
// What a slot's chunk of units in whole rounds depends on: rounds of the same
// kind follow each other and share it.
ICSA_DEV int unit_kind(const Kv8TcParams& p, const Kv8Cache& c, const Round& w) {
  return 2 * (w.b * c.H + w.h) + int(alternate(p, w));
}
ICSA_DEV int slot_steps(const Kv8TcParams& p, const Round& w, int s) {
  return alternate(p, w) ? (w.steps() + 1 - s) >> 1 : w.steps();
}

// ----------------------------------------------------------------- helper --
ICSA_DEV uint4 load_bytes16(const uint8_t* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

// Two e4m3 codes (bytes 0, 1 or 2, 3 of w) as bf16: the code's bits moved to
// bf16's places are the value times 2^-120 (also below e4m3's normal range).
// NaN codes come out as 480 (see has_nan).
template <int PAIR>
ICSA_DEV uint32_t e4m3_bf16x2(uint32_t w) {
  const uint32_t t = __byte_perm(w, 0u, PAIR ? 0x3424 : 0x1404);  // codes in the high bytes of the halves
  const uint32_t bits = (t & 0x80008000u) | ((t >> 4) & 0x07F007F0u);
  const __nv_bfloat162 up = __nv_bfloat162(__float2bfloat16_rn(0x1p120f), __float2bfloat16_rn(0x1p120f));
  const __nv_bfloat162 v = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&bits), up);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// nonzero where one of four codes is a NaN (all magnitude bits set)
ICSA_DEV uint32_t has_nan(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }
ICSA_DEV uint32_t nan_halves(uint32_t w, int pair) {
  const uint32_t lo = (w >> (16 * pair)) & 0x7Fu, hi = (w >> (16 * pair + 8)) & 0x7Fu;
  return (lo == 0x7Fu ? 0x7FC0u : 0u) | (hi == 0x7Fu ? 0x7FC00000u : 0u);
}
ICSA_DEV uint32_t e4m3_f16x2(uint16_t pair) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(pair));
  return r;
}
// bytes [0, n) of a word, the others zero
ICSA_DEV uint32_t keep(uint32_t w, int n) { return n >= 4 ? w : n <= 0 ? 0u : w & (0xFFFFFFFFu >> (8 * (4 - n))); }

// 16 codes as 32 bytes at two 16-byte units (2 c, 2 c + 1) of a swizzled row
template <bool BF16, bool NANS = false>
ICSA_DEV void put16(uint8_t* row_base, int row, int c, const uint4& u) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF16) {
      o[2 * i] = e4m3_bf16x2<0>(w[i]);
      o[2 * i + 1] = e4m3_bf16x2<1>(w[i]);
      if constexpr (NANS) {
        o[2 * i] |= nan_halves(w[i], 0);
        o[2 * i + 1] |= nan_halves(w[i], 1);
      }
    } else {
      o[2 * i] = e4m3_f16x2(uint16_t(w[i]));
      o[2 * i + 1] = e4m3_f16x2(uint16_t(w[i] >> 16));
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k)
    *reinterpret_cast<uint4*>(row_base + row * 128 + ((uint32_t(2 * c + k) ^ uint32_t(row & 7)) << 4)) =
        make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
}

// Signals the leader's barrier once per warp after this warp's shared-memory
// writes are visible to the tensor core.
ICSA_DEV void publish(uint64_t* bar) {
  fence_proxy_async_smem();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) pair::arrive_cluster(pair::mapa(bar, 0));
}

constexpr int kFillThreads = 128;  // the helper warps
ICSA_DEV int fill_thread() { return int(threadIdx.x & (kFillThreads - 1)); }

// Step j of a round: this CTA's 64 keys and its D / 2 features of 128 tokens,
// in 16-byte pieces (kUnits of each per thread).
template <int D>
struct Pieces {
  using C = Cfg<D>;
  static constexpr int kUnits = 64 * D / 16 / kFillThreads;
  static_assert(kUnits == C::kVRows * 8 / kFillThreads, "as many pieces of values as of keys");

  ICSA_DEV static void load_keys(const Kv8Cache& c, const Round& w, int j, uint32_t rank, uint4 (&x)[kUnits]) {
    const int kb = 2 * j + int(rank), nbl = (w.len + 63) >> 6;
    const uint8_t* src = c.k + ((size_t(w.b) * c.H + w.h) * c.nb + min(kb, nbl - 1)) * 64 * D + fill_thread() * 16;
#pragma unroll
    for (int i = 0; i < kUnits; ++i) x[i] = kb < nbl ? load_bytes16(src + i * (kFillThreads * 16)) : make_uint4(0u, 0u, 0u, 0u);
  }
  template <bool NANS>
  ICSA_DEV static void put_keys_as(const uint4 (&x)[kUnits], uint8_t* stage) {
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int u = i * kFillThreads + fill_thread(), row = u / (D / 16), c16 = u % (D / 16);
      put16<true, NANS>(stage + (c16 >> 2) * 8192, row, c16 & 3, x[i]);
    }
  }
  ICSA_DEV static void put_keys(const uint4 (&x)[kUnits], uint8_t* stage) {
    uint32_t nans = 0;
#pragma unroll
    for (int i = 0; i < kUnits; ++i) nans |= has_nan(x[i].x) | has_nan(x[i].y) | has_nan(x[i].z) | has_nan(x[i].w);
    if (nans == 0) put_keys_as<false>(x, stage);
    else put_keys_as<true>(x, stage);
  }
  // a later step's 128-byte lines to L2
  ICSA_DEV static void prefetch(const Kv8Cache& c, const Round& w, int j, uint32_t rank) {
    constexpr int kLines = 64 * D / 128;  // lines of each tensor's piece
    const int nbl = (w.len + 63) >> 6;
    const size_t block0 = (size_t(w.b) * c.H + w.h) * c.nb + 2 * j;
    for (int t = fill_thread(); t < 2 * kLines; t += kFillThreads) {
      const uint8_t* src;
      if (t < kLines) {
        if (2 * j + int(rank) >= nbl) continue;
        src = c.k + (block0 + rank) * 64 * D + t * 128;
      } else {
        const int u = t - kLines, kc = u / (kLines / 2);
        if (2 * j + kc >= nbl) continue;
        src = c.v + (block0 + kc) * 64 * D + size_t(rank) * C::kVRows * 64 + (u % (kLines / 2)) * 128;
      }
      asm volatile("prefetch.global.L2 [%0];" ::"l"(src));
    }
  }
  ICSA_DEV static void load_values(const Kv8Cache& c, const Round& w, int j, uint32_t rank, uint4 (&x)[kUnits]) {
    const int nbl = (w.len + 63) >> 6;
    const uint8_t* src = c.v + ((size_t(w.b) * c.H + w.h) * c.nb + 2 * j) * 64 * D + size_t(rank) * C::kVRows * 64;
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int u = i * kFillThreads + fill_thread(), kc = u / (C::kVRows * 4), rem = u % (C::kVRows * 4);
      x[i] = 2 * j + kc < nbl ? load_bytes16(src + kc * 64 * D + rem * 16) : make_uint4(0u, 0u, 0u, 0u);
    }
  }
  ICSA_DEV static void put_values(const Round& w, int j, uint4 (&x)[kUnits], uint8_t* dst) {
    const bool cut = w.len < (j + 1) * kStepKeys;
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int u = i * kFillThreads + fill_thread(), kc = u / (C::kVRows * 4), rem = u % (C::kVRows * 4);
      const int row = rem >> 2, c16 = rem & 3;
      if (cut) {
        // tokens behind the length: a probability of zero does not hide a NaN code
        const int left = w.len - ((2 * j + kc) * 64 + c16 * 16);
        x[i] = make_uint4(keep(x[i].x, left), keep(x[i].y, left - 4), keep(x[i].z, left - 8), keep(x[i].w, left - 12));
      }
      put16<false>(dst + kc * C::kVChunk, row, c16, x[i]);
    }
  }
};

// This CTA's 128 rows of a tile of queries, by TMA (a box holds whole tokens
// of the group's heads); completes the leader's barrier.  `fetch` brings a
// tile to L2 ahead of that.
template <int D, bool FETCH>
ICSA_DEV void tma_queries(const Kv8TcParams& p, const Kv8TcMaps& maps, const Round& w, int tile, uint32_t rank,
                          uint8_t* q, uint32_t q_full) {
  const int token0 = (tile * kPairRows + int(rank) * kCtaRows) / p.group;
#pragma unroll
  for (int c = 0; c < D / 64; ++c) {
    if constexpr (FETCH) {
      asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %3, %4}];" ::"l"(
                       reinterpret_cast<uint64_t>(&maps.q)),
                   "r"(c * 64), "r"(w.h * p.group), "r"(token0), "r"(w.b)
                   : "memory");
    } else {
      pair::tma_load_4d(q + c * (kCtaRows * 128), &maps.q, q_full, c * 64, w.h * p.group, token0, w.b);
    }
  }
}

// The same with 16-byte copies of one warp, for groups that do not divide a box.
template <int D>
ICSA_DEV void copy_queries(const Kv8TcParams& p, const Round& w, int tile, uint32_t rank, uint8_t* q) {
  constexpr int kUnits = D / 8;                 // 16-byte units of a row
  constexpr int kRowStep = 32 / kUnits;         // rows between a thread's copies
  const int tid = threadIdx.x & 31, c = tid % kUnits;
  const int r0 = tile * kPairRows + int(rank) * kCtaRows + tid / kUnits;
  int token = r0 / p.group, head = r0 % p.group;
  const int dt = kRowStep / p.group, dh = kRowStep % p.group;
  const __nv_bfloat16* base = p.q + int64_t(w.b) * p.q_sb + int64_t(w.h * p.group) * p.q_sh + c * 8;
#pragma unroll 4
  for (int i = 0; i < kCtaRows / kRowStep; ++i) {
    const int row = i * kRowStep + tid / kUnits;
    const bool ok = r0 + i * kRowStep < p.rows;
    const __nv_bfloat16* src = ok ? base + int64_t(token) * p.q_st + int64_t(head) * p.q_sh : base;
    const uint32_t dst = smem_u32(q + (c >> 3) * (kCtaRows * 128) + row * 128 + ((uint32_t(c & 7) ^ uint32_t(row & 7)) << 4));
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16u : 0u) : "memory");
    token += dt;
    head += dh;
    if (head >= p.group) {
      head -= p.group;
      ++token;
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// A tile's partial result, [D + 2][256 rows] (2^R O / l, then m and l): the
// rows, which lie across the lanes, are innermost.
ICSA_DEV float* partial_tile(const Kv8TcParams& p, int cluster, int part, int slot, int D) {
  return p.partial + (size_t(cluster * 2 + part) * 2 + slot) * kPairRows * (D + 2);
}
// behind the parts: where each cluster's range starts
ICSA_DEV int4* cluster_starts(const Kv8TcParams& p, int clusters, int D) {
  return reinterpret_cast<int4*>(p.partial + size_t(clusters) * 4 * kPairRows * (D + 2));
}

ICSA_DEV float reciprocal(float x) {
  float y;
  asm("rcp.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// O of a tile (of both slots where they took the steps in turn) to the
// output, or to this cluster's partial buffer.
template <int D>
ICSA_DEV void epilogue(const Kv8TcParams& p, const Kv8TcMaps& maps, const Round& w, int slot, bool two, uint32_t rank, Smem<D>& sm,
                       uint32_t tmem) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = warp & 3;
  const int row = quad * 32 + lane;
  const uint32_t o0 = tmem + (uint32_t(quad * 32) << 16) + kTmO + 128u * uint32_t(slot), o1 = o0 + 128u;
  const float ma = sm.ml[slot][0][row], la = sm.ml[slot][1][row];
  float m = ma, l = 1.f, fa = reciprocal(la), fb = 0.f;
  if (two) {
    // each slot's part of the row sum
    const float mb = sm.ml[1][0][row], lb = sm.ml[1][1][row];
    m = fmaxf(ma, mb);
    const float ref = m == -INFINITY ? 0.f : m;
    const float wa = la * sm.ml[slot][2][row] * ex2(ma - ref), wb = lb * sm.ml[1][2][row] * ex2(mb - ref);
    l = wa + wb;
    const float inv = reciprocal(l);
    fa *= wa * inv;
    fb = wb * inv * reciprocal(lb);
  } else if (w.part >= 0) {
    l = la * sm.ml[slot][2][row];
  }
  const int tile = 2 * w.r + slot;
  const int tile_row = int(rank) * kCtaRows + row, r = tile * kPairRows + tile_row;
  const bool ok = r < p.rows;
  const int token = r / p.group;
  uint8_t* box = sm.out[quad];
  // where a thread's row goes: the warp's box, the output, or the partial buffer
  float* part = nullptr;
  __nv_bfloat16* out = nullptr;
  if (w.part >= 0) part = partial_tile(p, blockIdx.x >> 1, w.part, slot, D) + tile_row;
  else if (!p.o_tma) out = p.out + ((size_t(w.b) * p.Lq + token) * p.Hq + w.h * p.group + (r - token * p.group)) * D;
#pragma unroll 1
  for (int c = 0; c < D / 32; ++c) {
    uint32_t x[32];
    tc::tmem_ld32(o0 + 32u * uint32_t(c), x);
    if (two) {
      uint32_t y[32];
      tc::tmem_ld32(o1 + 32u * uint32_t(c), y);
      tc::tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 32; ++e)
        x[e] = __float_as_uint(__uint_as_float(x[e]) * fa + __uint_as_float(y[e]) * fb);
    } else {
      tc::tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * fa);
    }
    if (c == D / 32 - 1) {
      // O has been read: its slot's next tile may start
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        pair::arrive_cluster_relaxed(pair::mapa(&sm.o_free[slot], 0));
        if (two) pair::arrive_cluster_relaxed(pair::mapa(&sm.o_free[1], 0));
      }
      __syncwarp();
    }
    if (part != nullptr) {
      if (ok) {
#pragma unroll
        for (int e = 0; e < 32; ++e) part[(32 * c + e) * kPairRows] = __uint_as_float(x[e]);
      }
      continue;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = pack_bf16x2(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1]));
    if (out == nullptr) {
      if ((c & 1) == 0) {
        // the box's previous contents have been read by their store
        if (lane == 0) bulk_wait_read();
        __syncwarp();
      }
#pragma unroll
      for (int v = 0; v < 4; ++v)
        *reinterpret_cast<uint4*>(box + lane * 128 + ((uint32_t((c & 1) * 4 + v) ^ uint32_t(lane & 7)) << 4)) =
            make_uint4(x[4 * v], x[4 * v + 1], x[4 * v + 2], x[4 * v + 3]);
      if ((c & 1) == 1) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && ok) {  // (lane 0 holds the box's first row)
          tma_store_4d(&maps.o, box, (c >> 1) * 64, w.h * p.group, token, w.b);
          bulk_commit();
        }
      }
    } else if (ok) {
#pragma unroll
      for (int v = 0; v < 4; ++v)
        *reinterpret_cast<uint4*>(out + 32 * c + 8 * v) = make_uint4(x[4 * v], x[4 * v + 1], x[4 * v + 2], x[4 * v + 3]);
    }
  }
  if (ok && part != nullptr) {
    part[D * kPairRows] = m;
    part[(D + 1) * kPairRows] = l;
  }
}

// rows of a tile without keys (never a cut round)
template <int D>
ICSA_DEV void empty_tile(const Kv8TcParams& p, const Round& w, int slot, uint32_t rank) {
  const int row = int(rank) * kCtaRows + int(threadIdx.x & 127), r = (2 * w.r + slot) * kPairRows + row;
  if (r >= p.rows) return;
  uint4* out = reinterpret_cast<uint4*>(
      p.out + ((size_t(w.b) * p.Lq + r / p.group) * p.Hq + w.h * p.group + r % p.group) * D);
  for (int i = 0; i < D / 8; ++i) out[i] = make_uint4(0u, 0u, 0u, 0u);
}

template <int D>
struct Helper {
  using C = Cfg<D>;
  using P = Pieces<D>;
  const Kv8TcParams& p;
  const Kv8TcMaps& maps;
  const Kv8Cache& c;
  Smem<D>& sm;
  uint32_t tmem, rank;
  uint32_t kv_next = 0;                 // stage count behind the newest round
  uint32_t o_phase = 0;                 // bit s: phase of slot s's finished tiles
  static constexpr int kAhead = 6;      // steps between a prefetch to L2 and its use

  // Steps [j0, j1) of a round, the first of them stage count `count`.  The
  // loads of a step are issued as soon as the registers of the step before it
  // are free, ahead of that step's hand-over.  (Two warps a stage, even and
  // odd stages in turn, overlap more of the latency but take the softmax's
  // issue slots in bursts: 860 us against 640 us for 2 x 40 heads, 512 rows,
  // 32760 keys.)
  ICSA_DEV bool fill(const Round& w, int j0, int j1, uint32_t count) {
    if (j0 >= j1) return true;
    uint4 k[P::kUnits], v[P::kUnits];
    P::load_keys(c, w, j0, rank, k);
    P::load_values(c, w, j0, rank, v);
    for (int j = j0; j < j1; ++j, ++count) {
      const int st = int(count % C::kStages);
      if (!warp_mbar_wait(&sm.kv_empty[st], ((count / C::kStages) & 1u) ^ 1u, nullptr, kErrKvEmpty, &sm.abort_flag))
        return false;
      if (j + kAhead < w.n1) P::prefetch(c, w, j + kAhead, rank);
      P::put_keys(k, sm.kv[st]);
      if (j + 1 < j1) P::load_keys(c, w, j + 1, rank, k);
      P::put_values(w, j, v, sm.kv[st] + C::kKBytes);
      if (j + 1 < j1) P::load_values(c, w, j + 1, rank, v);
      publish(&sm.kv_full[st]);
    }
    return true;
  }
  ICSA_DEV bool wait_tile(int s) {
    const uint32_t par = (o_phase >> s) & 1u;
    o_phase ^= 1u << s;
    const bool ok = warp_mbar_wait(&sm.ml_full[s], par, nullptr, kErrMlFull, &sm.abort_flag) &&
                    warp_mbar_wait(&sm.o_full[s], par, nullptr, kErrOFull, &sm.abort_flag);
    tc::fence_after_sync();
    return ok;
  }
  ICSA_DEV void release_ml(int s) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&sm.ml_free[s]);
    __syncwarp();
  }
  ICSA_DEV bool end(const Round& w) {
    const bool two = alternate(p, w) && w.steps() > 1;
#pragma unroll 1
    for (int s = 0; s < 2; ++s) {
      if (!has_tile(p, w, s)) continue;
      if (w.steps() == 0) {
        empty_tile<D>(p, w, s, rank);
        continue;
      }
      if (!wait_tile(s) || (two && !wait_tile(1))) return false;
      epilogue<D>(p, maps, w, s, two, rank, sm, tmem);
      release_ml(s);
      if (two) release_ml(1);
    }
    return true;
  }
  // The stages beyond the ring of the round at hand, the first stages of the
  // next round (which wait for nothing that the epilogue at hand releases),
  // then the epilogue.  (Written so that the conversion and the epilogue
  // exist once: the kernel's code has to stay in the instruction cache.)
  ICSA_DEV void run() {
    Walk walk(sm.ranges);
    Round cur, nxt;
    bool have = false, more = walk.next(p, c, nxt), fresh = more, beyond = false;
    cur = nxt;
    while (have || more) {
#pragma unroll 1
      for (int part = 0; part < 2; ++part) {
        if (!(part ? fresh : beyond)) continue;
        const Round& w = part ? nxt : cur;
        const int j0 = w.n0 + (part ? 0 : C::kStages), j1 = part ? min(w.n1, w.n0 + C::kStages) : w.n1;
        if (!fill(w, j0, j1, part ? kv_next : kv_next - uint32_t(w.steps() - C::kStages))) return;
        if (part) kv_next += uint32_t(w.steps());
      }
      if (have && !end(cur)) return;
      beyond = fresh && nxt.steps() > C::kStages;
      cur = nxt;
      have = more;
      more = more && walk.next(p, c, nxt);
      fresh = more && new_kv(p, nxt, cur);
    }
    if ((threadIdx.x & 31) == 0) bulk_wait_read();
  }
};

// -------------------------------------------------------- query loads (warp) --
// Returns the number of tiles that were requested for each slot.
template <int D>
ICSA_DEV void load_queries(const Kv8TcParams& p, const Kv8TcMaps& maps, const Kv8Cache& c, uint32_t rank, Smem<D>& sm,
                           uint32_t& count0, uint32_t& count1) {
  using C = Cfg<D>;
  const int lane = threadIdx.x & 31;
  Walk walk(sm.ranges);
  Round w;
  while (walk.next(p, c, w)) {
    if (w.steps() == 0) continue;
    if (p.q_tma && lane < 2 && has_tile(p, w, lane))
      tma_queries<D, true>(p, maps, w, 2 * w.r + lane, rank, nullptr, 0u);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (!has_tile(p, w, s)) continue;
      uint32_t& count = s ? count1 : count0;
      if (!warp_mbar_wait(&sm.q_empty[s], (count & 1u) ^ 1u, nullptr, kErrQEmpty, &sm.abort_flag)) return;
      ++count;
      if (p.q_tma) {
        if (lane == 0) {
          if (rank == 0) mbar_arrive_expect_tx(&sm.q_full[s], 2 * C::kQBytes);
          tma_queries<D, false>(p, maps, w, 2 * w.r + s, rank, sm.q[s], pair::mapa(&sm.q_full[s], 0));
        }
        __syncwarp();
      } else {
        copy_queries<D>(p, w, 2 * w.r + s, rank, sm.q[s]);
        publish(&sm.q_full[s]);
      }
    }
  }
}

// ------------------------------------------------------------ scales (warp) --
// exponent of a power of two; NaN stays NaN
ICSA_DEV float exponent(float s) { return s != s ? s : float(int(__float_as_uint(s) >> 23) - 127); }
constexpr float kWindow = 7.f;  // most of d = lv - R: P up to 2^15 with the 2^8 of the lazy maximum

// R of a slot, moved as little as the window allows.
struct Reference {
  float r = 0.f, top = -1000.f;  // R, and the largest lv of the round so far
  // scales lo to hi, no further apart than the window
  ICSA_DEV void cover(float lo, float hi, float spread) {
    top = fmaxf(top, hi);
    if (lo < r || hi > r + kWindow) r = fmaxf(lo - floorf(0.5f * (kWindow - (hi - lo))), top - spread);
  }
};

// The units of every slot, a unit for each lane: where a chunk's scales fit the
// window one R serves it (nearly always), else R goes from unit to unit, and
// where it has to move between the blocks of a step, that step runs in two
// parts.  Both CTAs of a pair come to the same R, as they read the same scales.
// (A NaN scale moves nothing and makes its row NaN.)  Done by the softmax and
// the issuer themselves it took 606 us instead of 545 for 2 x 40 heads, 256 over
// 32000, and 738 instead of 635 for the text.
template <int D>
ICSA_DEV void prepare_units(const Kv8TcParams& p, const Kv8Cache& c, Smem<D>& sm) {
  const int lane = threadIdx.x & 31;
  uint32_t count0 = 0, count1 = 0;  // chunks of each slot
  uint32_t kv_base = 0, kv_next = 0;  // stages, as the issuers count them
  int kind0 = -1, kind1 = -1;
  Reference ref0, ref1;
  Walk walk(sm.ranges);
  Round w, before;
  before.b = -1;
  while (walk.next(p, c, w)) {
    if (new_kv(p, w, before)) {
      kv_base = kv_next;
      kv_next += uint32_t(w.steps());
    }
    before = w;
    const size_t slot0 = (size_t(w.b) * c.H + w.h) * c.nb;
    const float spread = value_spread(w.len);
    const bool alt = alternate(p, w);
    const int nbl = (w.len + 63) >> 6, most = slot_steps(p, w, 0);  // (slot 1 has no more)
    ref0.top = ref1.top = -1000.f;
#pragma unroll 1
    for (int q = 0; q < 2 * most; ++q) {
      // chunk q / 2 of slot q & 1
      const int s = q & 1, k0 = (q >> 1) * kChunk, n = slot_steps(p, w, s);
      if (k0 >= most) break;
      if (k0 >= n) continue;
      if (p.whole) {
        const int kind = unit_kind(p, c, w);
        if (kind == (s ? kind1 : kind0)) continue;
        if (s) kind1 = kind;
        else kind0 = kind;
      }
      const int k = k0 + lane, j = w.n0 + (alt ? s + 2 * k : k);
      float ks0 = 0.f, ks1 = 0.f, e0 = __uint_as_float(0x7FC00000u), e1 = e0;
      if (k < n) {
        const int b0 = 2 * j, b1 = min(2 * j + 1, nbl - 1);  // (a block behind the length has no key)
        ks0 = __ldg(c.k_scale + slot0 + b0);
        ks1 = __ldg(c.k_scale + slot0 + b1);
        e0 = exponent(__ldg(c.v_scale + slot0 + b0));
        e1 = exponent(__ldg(c.v_scale + slot0 + b1));
      }
      // (fminf and fmaxf pass over a NaN)
      const float lo = float(__reduce_min_sync(0xffffffffu, int(fminf(fminf(e0, e1), 1000.f))));
      const float hi = float(__reduce_max_sync(0xffffffffu, int(fmaxf(fmaxf(e0, e1), -1000.f))));
      Reference ref = s ? ref1 : ref0;
      float r0, r1;
      const bool calm = hi - lo <= kWindow;
      if (calm) {
        ref.cover(lo, hi, spread);
        r0 = r1 = ref.r;
      } else {
        r0 = r1 = 0.f;
#pragma unroll 1
        for (int i = 0; i < min(kChunk, n - k0); ++i) {
          const float a0 = __shfl_sync(0xffffffffu, e0, i), a1 = __shfl_sync(0xffffffffu, e1, i);
          const float lo1 = fminf(a0, a1), hi1 = fmaxf(a0, a1);
          float first;
          if (hi1 - lo1 > kWindow) {
            ref.top = fmaxf(ref.top, hi1);
            first = fmaxf(a0 - 4.f, ref.top - spread);
            ref.r = fmaxf(a1 - 4.f, ref.top - spread);
          } else {
            ref.cover(lo1, hi1, spread);
            first = ref.r;
          }
          if (lane == i) {
            r0 = first;
            r1 = ref.r;
          }
        }
      }
      if (s) ref1 = ref;
      else ref0 = ref;
      const uint32_t count = s ? count1++ : count0++;
      const int buf = int(count & 1u);
      if (!warp_mbar_wait(&sm.unit_empty[s][buf], ((count >> 1) & 1u) ^ 1u, nullptr, kErrUnitEmpty, &sm.abort_flag)) return;
      const float d0 = e0 - r0, d1 = e1 - r1;
      float4* u = reinterpret_cast<float4*>(&sm.units[s][buf][lane]);
      u[0] = make_float4(p.scale_log2 * ks0, p.scale_log2 * ks1, d0, d1);
      u[1] = make_float4(ex2(-d0), ex2(-d1), r0, r1);
      if (lane == 0) sm.any_two[s][buf] = calm ? 0u : 1u;
      sm.units[s][buf][lane].stage = kv_base + uint32_t(j - w.n0);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.unit_full[s][buf]);
      __syncwarp();
    }
  }
}

// ----------------------------------------------------------------- issuer --
template <int D, int KK>
constexpr uint32_t kQOff = uint32_t(((KK >> 2) * (kCtaRows * 128) + (KK & 3) * 32) >> 4);
template <int D, int KK>
constexpr uint32_t kKOff = uint32_t(((KK >> 2) * 8192 + (KK & 3) * 32) >> 4);
template <int D, int KK>
constexpr uint32_t kVOff = uint32_t(((KK >> 2) * Cfg<D>::kVChunk + (KK & 3) * 32) >> 4);

// kind::f16 with f16 operands and a float32 accumulator, both K-major
__host__ __device__ constexpr uint32_t make_idesc_f16(int M, int N) {
  return (1u << 4) | (uint32_t(N >> 3) << 17) | (uint32_t(M >> 4) << 24);
}

template <int D, int... KK>
ICSA_DEV void issue_s(uint64_t q_desc, uint64_t k_desc, uint32_t d_tmem, std::integer_sequence<int, KK...>) {
  constexpr uint32_t idesc = tc::make_idesc_bf16(256, kStepKeys, false, false);
  (pair::mma_ss_elect<kQOff<D, KK>, kKOff<D, KK>>(d_tmem, q_desc, k_desc, idesc, KK > 0 ? 1u : 0u), ...);
}
template <int D, int... KK>
ICSA_DEV void issue_pv(uint64_t v_desc, uint32_t p_tmem, uint32_t o_tmem, uint32_t acc,
                       std::integer_sequence<int, KK...>) {
  constexpr uint32_t idesc = make_idesc_f16(256, D);
  (pair::mma_ts_elect<uint32_t(KK * 8), kVOff<D, KK>>(o_tmem, p_tmem, v_desc, idesc, (KK > 0) ? 1u : acc), ...);
}

// Two warps of the leader walk the units (step, slot) of all rounds: one
// issues the S of each, the other its P.V.  The tensor core's queue holds few
// instructions, so what an issuer spends between them on waits is lost unless
// the other one fills it (a single issuer, S of a unit and P.V of the unit
// two before it in turn: 2490 clk a unit; two: 1930, in whole rounds).
template <int D, bool PV>
struct Issuer {
  using C = Cfg<D>;
  static constexpr uint64_t kStageDesc = (C::kKBytes + C::kVBytes) >> 4;
  const Kv8TcParams& p;
  const Kv8Cache& c;
  Smem<D>& sm;
  uint32_t tmem;

  // The same value in every lane, in a form that lets the compiler keep what
  // follows from it in uniform registers.
  ICSA_DEV static int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }
  ICSA_DEV bool wait(uint64_t* bar, uint32_t phase, int code) {
    return warp_mbar_wait(bar, phase & 1u, nullptr, code, &sm.abort_flag);
  }

  ICSA_DEV void run() {
    const uint64_t qd = tc::make_sw128_desc(smem_u32(sm.q[0]), 16, 1024);
    const uint64_t kd = tc::make_sw128_desc(smem_u32(sm.kv[0]), 16, 1024);
    const uint64_t vd = tc::make_sw128_desc(smem_u32(sm.kv[0] + C::kKBytes), 16, 1024);
    // bit s: phase of the next wait on slot s's barrier
    uint32_t ph0 = 0, ph1 = PV ? 3u : 0u;  // S: queries, S read;  P.V: P written, O read
    int last_s = -1;                       // slot of the S that occupies the buffer
    Walk walk(sm.ranges);
    Round cur, nxt;
    bool have = walk.next(p, c, cur), fresh = true;
    uint32_t kv_base = 0, kv_next = 0;
    while (have) {
      const bool more = walk.next(p, c, nxt);
      const int n = cur.steps();
      if (fresh) {
        kv_base = kv_next;
        kv_next += uint32_t(n);
      }
      // the round is the last to read its stages
      const bool frees = !more || new_kv(p, nxt, cur);
      const bool both = has_tile(p, cur, 1), alt = !both;
      const int units = both ? 2 * n : n;
#pragma unroll 1
      for (int u = 0; u < units; ++u) {
        const int k = both ? u >> 1 : u, s = uniform(u & 1);
        const uint32_t count = kv_base + uint32_t(k);
        const int st = uniform(int(count % C::kStages));
        const bool first = alt ? u < 2 : k == 0, last = alt ? u + 2 >= n : k + 1 == n;
        if (fresh && !(both && s) && !wait(&sm.kv_full[st], count / C::kStages, kErrKvFull)) return;
        if constexpr (!PV) {
          const int qb = alt ? 0 : s;
          if (k == 0) {
            if (!wait(&sm.q_full[qb], ph0 >> qb, kErrQFull)) return;
            ph0 ^= 1u << qb;
          }
          // the softmax has read the S before this one
          if (last_s >= 0) {
            if (!wait(&sm.s_free[last_s], ph1 >> last_s, kErrSFree)) return;
            ph1 ^= 1u << last_s;
          }
          last_s = s;
          tc::fence_after_sync();
          issue_s<D>(qd + uint64_t(qb) * (C::kQBytes >> 4), kd + uint64_t(st) * kStageDesc, tmem,
                     std::make_integer_sequence<int, D / 16>{});
          pair::commit_both_elect(&sm.s_full[s]);
          if (alt ? u + 1 == n : last) pair::commit_both_elect(&sm.q_empty[qb]);
        } else {
          if (!wait(&sm.p_full[s], ph0 >> s, kErrPFull)) return;
          ph0 ^= 1u << s;
          if (first) {
            // the slot's last tile has been read
            if (!wait(&sm.o_free[s], ph1 >> s, kErrOFree)) return;
            ph1 ^= 1u << s;
          }
          tc::fence_after_sync();
          issue_pv<D>(vd + uint64_t(st) * kStageDesc, tmem + kTmP + 64u * uint32_t(s), tmem + kTmO + 128u * uint32_t(s),
                      first ? 0u : 1u, std::make_integer_sequence<int, 8>{});
          pair::commit_both_elect(&sm.pv_done[s]);
          if (last) pair::commit_both_elect(&sm.o_full[s]);
          if (frees && (!both || s)) pair::commit_both_elect(&sm.kv_empty[st]);
        }
      }
      fresh = frees;
      cur = nxt;
      have = more;
    }
  }
};

// ---------------------------------------------------------------- softmax --
// 64 scores x to 2^(x c + off), their sum added to l0 .. l3, as f16 pairs
ICSA_DEV void exp_half(float* s, float c, float off, float& l0, float& l1, float& l2, float& l3) {
#pragma unroll
  for (int e = 0; e < 64; e += 4) {
    ffma2(s[e], s[e + 1], s[e], s[e + 1], c, c, off, off);
    ffma2(s[e + 2], s[e + 3], s[e + 2], s[e + 3], c, c, off, off);
    s[e] = ex2(s[e]);
    s[e + 1] = ex2(s[e + 1]);
    s[e + 2] = ex2(s[e + 2]);
    s[e + 3] = ex2(s[e + 3]);
    fadd2(l0, l1, l0, l1, s[e], s[e + 1]);
    fadd2(l2, l3, l2, l3, s[e + 2], s[e + 3]);
  }
}
ICSA_DEV uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
ICSA_DEV void store_p(uint32_t taddr, const float* s) {
  uint32_t pk[32];
#pragma unroll
  for (int e = 0; e < 32; ++e) pk[e] = pack_f16x2(s[2 * e], s[2 * e + 1]);
  tc::tmem_st32(taddr, pk);
}
ICSA_DEV void store_zeros(uint32_t taddr) {
  uint32_t pk[32];
#pragma unroll
  for (int e = 0; e < 32; ++e) pk[e] = 0u;
  tc::tmem_st32(taddr, pk);
}
ICSA_DEV float max64(const float* s) {
  float t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = fmaxf(s[i], s[4 + i]);
#pragma unroll
  for (int e = 8; e < 64; e += 8)
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = fmax3(t[i], s[e + i], s[e + 4 + i]);
  return fmax3(fmaxf(t[0], t[1]), t[2], t[3]);
}
// O of this thread's row times 2^shift
template <int D>
ICSA_DEV void rescale(uint32_t o_base, float shift) {
  const float alpha = ex2(shift);
#pragma unroll 1
  for (int q = 0; q < D / 32; ++q) {
    uint32_t r[32];
    tc::tmem_ld32(o_base + 32u * uint32_t(q), r);
    tc::tmem_wait_ld();
#pragma unroll
    for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * alpha);
    tc::tmem_st32(o_base + 32u * uint32_t(q), r);
  }
}

// The softmax of one slot: a warpgroup, a thread for each row.
template <int D>
struct Softmax {
  Smem<D>& sm;
  uint32_t tmem, rank;
  int slot;
  uint32_t count = 0, extra = 0;  // units, and of them those in two parts
  uint32_t tiles = 0;
  float m = 0.f, l = 0.f;         // of this thread's row
  float ref_v = 0.f;              // R (the same in all rows)
  uint32_t s_free = pair::mapa(&sm.s_free[slot], 0), p_full = pair::mapa(&sm.p_full[slot], 0);

  ICSA_DEV uint32_t lanes() const { return uint32_t(((threadIdx.x >> 5) & 3) * 32) << 16; }
  ICSA_DEV uint32_t p_base() const { return tmem + lanes() + kTmP + 64u * uint32_t(slot); }
  ICSA_DEV uint32_t o_base() const { return tmem + lanes() + kTmO + 128u * uint32_t(slot); }
  ICSA_DEV bool wait(uint64_t* bar, uint32_t phase, int code) {
    return warp_mbar_wait(bar, phase & 1u, nullptr, code, &sm.abort_flag);
  }
  // P and O are written: tells the leader's barrier
  ICSA_DEV void give(uint32_t bar) {
    tc::tmem_wait_st();
    tc::fence_before_sync();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) pair::arrive_cluster_relaxed(bar);
    __syncwarp();
  }

  // Unit k of the round, of which `left` keys are valid.  TWO: its chunk has
  // units that run in two parts.
  template <bool TWO>
  ICSA_DEV void step(const Unit& unit, int k, int left, bool any_row) {
    const float4 cd = *reinterpret_cast<const float4*>(&unit.c0), wr = *reinterpret_cast<const float4*>(&unit.w0);
    wait(&sm.s_full[slot], count, kErrSFull);
    tc::fence_after_sync();
    float s[128];
    tmem_load_row128(tmem + lanes(), s);
    tc::fence_before_sync();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) pair::arrive_cluster_relaxed(s_free);
    __syncwarp();
    float shift = ref_v - wr.z;
    ref_v = wr.w;
    bool need = shift != 0.f;  // O is to be multiplied by 2^shift: R's move and the maximum's rise in one exponent
    if (any_row) {
      if (left < kStepKeys) {
#pragma unroll
        for (int e = 0; e < 128; ++e)
          if (e >= left) s[e] = -INFINITY;
      }
      const float top = fmaxf(max64(s) * cd.x, max64(s + 64) * cd.y);
      if (top - m > kRescaleThreshold) {
        if (m > -INFINITY) {
          l *= ex2(m - top);
          shift += m - top;
        }
        m = top;
        need = true;
      }
      float a0 = 0.f, a1 = 0.f, a2 = 0.f, a3 = 0.f;
      exp_half(s, cd.x, cd.z - m, a0, a1, a2, a3);
      l += ((a0 + a1) + (a2 + a3)) * wr.x;
      a0 = a1 = a2 = a3 = 0.f;
      exp_half(s + 64, cd.y, cd.w - m, a0, a1, a2, a3);
      l += ((a0 + a1) + (a2 + a3)) * wr.y;
    }
    // P and O of this slot were last used by its previous P.V
    if constexpr (!TWO) {
      wait_pv();
      if (any_row) {
        store_p(p_base(), s);
        store_p(p_base() + 32u, s + 64);
      }
      if (k > 0 && __any_sync(0xffffffffu, need)) rescale<D>(o_base(), shift);
      give(p_full);
    } else {
      uint32_t pk[64];
#pragma unroll
      for (int e = 0; e < 64; ++e) pk[e] = pack_f16x2(s[2 * e], s[2 * e + 1]);
      wait_pv();
      const bool two = unit.ref0 != unit.ref1;
      if (two) {
        first_part(pk, unit, k, any_row, k > 0 && __any_sync(0xffffffffu, need), shift);
        shift = unit.ref0 - unit.ref1;
        need = true;
        if (any_row) store_zeros(p_base());
      } else if (any_row) {
        tc::tmem_st32(p_base(), reinterpret_cast<const uint32_t(&)[32]>(pk[0]));
      }
      if (any_row) tc::tmem_st32(p_base() + 32u, reinterpret_cast<const uint32_t(&)[32]>(pk[32]));
      if (k > 0 && __any_sync(0xffffffffu, need)) rescale<D>(o_base(), shift);
      if (two && k == 0) join_first(shift);
      else give(p_full);
    }
    ++count;
  }
  ICSA_DEV void wait_pv() {
    if (count > 0) {
      wait(&sm.pv_done[slot], count - 1, kErrPvDone);
      tc::fence_after_sync();
    }
  }
  // A step in two parts: P.V of its first block alone.  A warp of the leader's
  // softmax issues it: the issuer, whose every instruction counts, knows
  // nothing of it.
  ICSA_DEV void first_part(const uint32_t (&pk)[64], const Unit& unit, int k, bool any_row, bool need, float shift) {
    if (any_row) {
      tc::tmem_st32(p_base(), reinterpret_cast<const uint32_t(&)[32]>(pk[0]));
      store_zeros(p_base() + 32u);
    }
    if (need) rescale<D>(o_base(), shift);
    give(pair::mapa(&sm.x_full[slot], 0));
    if (rank == 0 && ((threadIdx.x >> 5) & 3) == 0) {
      using C = Cfg<D>;
      const uint32_t st = unit.stage % C::kStages;
      bool ok = wait(&sm.x_full[slot], extra, kErrXFull) && wait(&sm.kv_full[st], unit.stage / C::kStages, kErrKvFull);
      // (a tile's first unit: the slot's last tile has been read)
      if (k == 0) ok = ok && wait(&sm.o_free[slot], tiles ^ 1u, kErrOFree);
      if (ok) {
        tc::fence_after_sync();
        issue_pv<D>(tc::make_sw128_desc(smem_u32(sm.kv[st] + C::kKBytes), 16, 1024),
                    tmem + kTmP + 64u * uint32_t(slot), tmem + kTmO + 128u * uint32_t(slot), k == 0 ? 0u : 1u,
                    std::make_integer_sequence<int, 8>{});
        pair::commit_both_elect(&sm.x_done[slot]);
        // whatever becomes of the other waits, these products are over before the CTA ends
        if ((threadIdx.x & 31) == 0) drain_wait(&sm.x_done[slot], extra & 1u, nullptr);
        __syncwarp();
      }
    }
    wait(&sm.x_done[slot], extra, kErrXDone);
    tc::fence_after_sync();
    ++extra;
  }
  // The issuer's P.V of a tile's first unit starts O anew: the first part is
  // kept meanwhile (in local memory, this is rare and registers are not to be
  // had) and added to it.
  ICSA_DEV void join_first(float shift) {
    uint32_t kept[D];
#pragma unroll 1
    for (int q = 0; q < D; q += 32) {
      uint32_t r[32];
      tc::tmem_ld32(o_base() + uint32_t(q), r);
      tc::tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 32; ++e) kept[q + e] = r[e];
    }
    give(p_full);
    wait(&sm.pv_done[slot], count, kErrPvDone);
    tc::fence_after_sync();
    const float alpha = ex2(shift);
#pragma unroll 1
    for (int q = 0; q < D; q += 32) {
      uint32_t r[32];
      tc::tmem_ld32(o_base() + uint32_t(q), r);
      tc::tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 32; ++e)
        r[e] = __float_as_uint(__uint_as_float(r[e]) + __uint_as_float(kept[q + e]) * alpha);
      tc::tmem_st32(o_base() + uint32_t(q), r);
    }
    tc::tmem_wait_st();
    tc::fence_before_sync();
  }

  ICSA_DEV void run(const Kv8TcParams& p, const Kv8Cache& c) {
    const int row = threadIdx.x & 127, lane = threadIdx.x & 31;
    uint32_t chunks = 0;
    int kind = -1;
    Walk walk(sm.ranges);
    Round w;
    while (walk.next(p, c, w)) {
      const int n = slot_steps(p, w, slot);
      if (n == 0) continue;
      const bool fresh = !p.whole || unit_kind(p, c, w) != kind;
      kind = unit_kind(p, c, w);
      const bool alt = alternate(p, w);
      const int keys = alt ? 2 * kStepKeys : kStepKeys;  // between the slot's steps
      int left = w.len - (w.n0 + (alt ? slot : 0)) * kStepKeys;
      // rows of this warp behind the last one need no exponentials
      const int tile = 2 * w.r + (alt ? 0 : slot);
      const bool any_row = tile * kPairRows + int(rank) * kCtaRows + (row & ~31) < p.rows;
      m = -INFINITY;
      l = 0.f;
      for (int k0 = 0; k0 < n; k0 += kChunk) {
        if (fresh) {
          // the next chunk, and the one before it is free
          wait(&sm.unit_full[slot][chunks & 1u], chunks >> 1, kErrUnitFull);
          __syncwarp();
          if (chunks > 0 && lane == 0) mbar_arrive(&sm.unit_empty[slot][(chunks - 1) & 1u]);
          __syncwarp();
          ++chunks;
        }
        const int buf = int((chunks - 1) & 1u), kn = min(n - k0, kChunk);
        const Unit* units = sm.units[slot][buf];
        if (sm.any_two[slot][buf] == 0) {
          for (int k = 0; k < kn; ++k) step<false>(units[k], k0 + k, left - k * keys, any_row);
        } else {
#pragma unroll 1
          for (int k = 0; k < kn; ++k) step<true>(units[k], k0 + k, left - k * keys, any_row);
        }
        left -= kn * keys;
      }
      // the helper has read the last tile's statistics
      wait(&sm.ml_free[slot], tiles ^ 1u, kErrMlFree);
      ++tiles;
      sm.ml[slot][0][row] = m;
      sm.ml[slot][1][row] = l * ex2(-ref_v);  // (O over this is the result)
      sm.ml[slot][2][row] = ex2(ref_v);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.ml_full[slot]);
      __syncwarp();
    }
  }
};

template <int D>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    kv8_tc_kernel(const Kv8TcParams p, const Kv8Cache c, const __grid_constant__ Kv8TcMaps maps) {
  extern __shared__ uint8_t smem_raw[];
  Smem<D>& sm = *reinterpret_cast<Smem<D>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  using C = Cfg<D>;
  const int warp = threadIdx.x >> 5;
  const uint32_t rank = pair::cluster_rank();
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&sm.kv_full[i], 8);   // helper warps of both CTAs
      mbar_init(&sm.kv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.q_full[i], p.q_tma ? 1 : 2);  // expected bytes, or the query warps of both CTAs
      mbar_init(&sm.q_empty[i], 1);
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.s_free[i], 8);    // softmax warps of both CTAs
      mbar_init(&sm.p_full[i], 8);
      mbar_init(&sm.pv_done[i], 1);
      mbar_init(&sm.o_full[i], 1);
      mbar_init(&sm.o_free[i], 8);
      mbar_init(&sm.ml_full[i], 4);
      mbar_init(&sm.ml_free[i], 4);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&sm.fin[i], 1);
    for (int i = 0; i < 4; ++i) {
      mbar_init(&sm.unit_full[i >> 1][i & 1], 1);
      mbar_init(&sm.unit_empty[i >> 1][i & 1], 4);  // a slot's softmax warps
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.x_full[i], 8);
      mbar_init(&sm.x_done[i], 1);
    }
    sm.abort_flag = 0;
    fence_mbarrier_init();
  }
  if (threadIdx.x >= 256 && threadIdx.x - 256 < c.B)
    sm.ranges[threadIdx.x - 256] = cluster_range(p, c, threadIdx.x - 256, blockIdx.x >> 1, gridDim.x >> 1);
  if (warp == kIssuerWarp) {
    pair::tmem_alloc(&sm.tmem_base, kTmemCols);
    pair::tmem_relinquish();
  }
  tc::fence_before_sync();
  pair::cluster_sync();
  tc::fence_after_sync();
  const uint32_t tmem = sm.tmem_base;
  // Register split: 512 threads launch with 128 registers each;
  // 256 x 176 + 128 x 104 + 128 x 56 = 512 x 128.
  if (warp < 8) {
    tc::reg_alloc<176>();
    Softmax<D>{sm, tmem, rank, warp >> 2}.run(p, c);
  } else if (warp < kIssuerWarp) {
    tc::reg_dealloc<104>();
    Helper<D> h{p, maps, c, sm, tmem, rank};
    h.run();
  } else {
    tc::reg_dealloc<56>();
    if (warp == kIssuerWarp && rank == 0) {
      Issuer<D, false>{p, c, sm, tmem}.run();
      pair::commit_both_elect(&sm.fin[0]);
      if ((threadIdx.x & 31) == 0) drain_wait(&sm.fin[0], 0, nullptr);
    } else if (warp == kPvWarp && rank == 0) {
      Issuer<D, true>{p, c, sm, tmem}.run();
      pair::commit_both_elect(&sm.fin[1]);
      if ((threadIdx.x & 31) == 0) drain_wait(&sm.fin[1], 0, nullptr);
    } else if (warp == kQueryWarp) {
      uint32_t q0 = 0, q1 = 0;
      load_queries<D>(p, maps, c, rank, sm, q0, q1);
      if (sm.abort_flag && p.q_tma && rank == 0 && (threadIdx.x & 31) == 0) {
        // the leader's barriers count the bytes of both CTAs: let every copy
        // still in flight land before either CTA releases its memory
        if (q0) drain_wait(&sm.q_full[0], (q0 - 1) & 1u, nullptr);
        if (q1) drain_wait(&sm.q_full[1], (q1 - 1) & 1u, nullptr);
      }
    } else if (warp == kScaleWarp) {
      prepare_units<D>(p, c, sm);
      // for the kernel that joins the parts
      if (!p.whole && rank == 0 && (threadIdx.x & 31) == 0)
        cluster_starts(p, gridDim.x >> 1, D)[blockIdx.x >> 1] = cluster_start(p, c, blockIdx.x >> 1, gridDim.x >> 1);
    }
  }
  __syncwarp();
  tc::fence_before_sync();
  pair::cluster_sync();
  if (warp == kIssuerWarp) {
    tc::fence_after_sync();
    pair::tmem_dealloc(tmem, kTmemCols);
  }
}

// Joins the parts of the rounds that were cut at cluster boundaries, in the
// order of the clusters.  blockIdx.x + 1 is a cluster: its CTAs join the round
// that its range starts inside of, if the round starts in the range just
// before.  A CTA takes 32 rows.  (Rows behind the last one join whatever the
// buffer holds and are not stored.)
template <int D>
__global__ void __launch_bounds__(256) kv8_tc_join_kernel(const Kv8TcParams p, const Kv8Cache c, int clusters) {
  const int k = int(blockIdx.x) + 1;
  wait_prior_grid();
  extern __shared__ int4 at[];  // where the clusters' ranges start
  for (int j = threadIdx.x; j <= clusters; j += 256)
    at[j] = j < clusters ? cluster_starts(p, clusters, D)[j] : make_int4(-1, 0, 0, 0);
  __syncthreads();
  const auto same_round = [&](int i, int j) { return at[i].x == at[j].x && at[i].y == at[j].y; };
  const int4 q0 = at[k];
  if (q0.z == 0 || (same_round(k - 1, k) && at[k - 1].z > 0)) return;
  const int k0 = k - 1, b = q0.x;
  int k1 = k;
  while (same_round(k1 + 1, k)) ++k1;
  const int h = q0.y / p.rounds, r = q0.y - h * p.rounds;
  // the round starts in cluster k0's range (its last partial buffer) and
  // before those of the clusters behind it; lanes are rows
  const int tr = blockIdx.y * 32 + (threadIdx.x & 31), slot = tr / kPairRows, row = tr % kPairRows;
  const int row0 = 2 * r * kPairRows + blockIdx.y * 32;
  constexpr int kPer = D / 8;  // features of a thread
  const int d0 = (threadIdx.x >> 5) * kPer;
  float mm = -INFINITY, l = 0.f, acc[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = 0.f;
  constexpr int kAhead = 4;  // parts whose loads are on their way together
  for (int j = k0; j <= k1; j += kAhead) {
    float x[kAhead][kPer], m[kAhead], lk[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      m[i] = -INFINITY;
      lk[i] = 0.f;
#pragma unroll
      for (int e = 0; e < kPer; ++e) x[i][e] = 0.f;
      const int n = j + i;
      // (a cluster without a step between two others has no part)
      if (n > k1 || (same_round(n, n + 1) && at[n].z == at[n + 1].z)) continue;
      const float* src = partial_tile(p, n, n == k0 ? 1 : 0, slot, D) + row;
      m[i] = src[D * kPairRows];
      lk[i] = src[(D + 1) * kPairRows];
#pragma unroll
      for (int e = 0; e < kPer; ++e) x[i][e] = src[(d0 + e) * kPairRows];
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      // a weighted mean, which no value overflows
      const float top = fmaxf(mm, m[i]), ref = top == -INFINITY ? 0.f : top;
      const float f = l * ex2(mm - ref), g = lk[i] * ex2(m[i] - ref);
      l = f + g;
      mm = top;
      const float inv = l == 0.f ? 0.f : __frcp_rn(l);
#pragma unroll
      for (int e = 0; e < kPer; ++e) acc[e] = acc[e] * (f * inv) + x[i][e] * (g * inv);
    }
  }
  __shared__ float tile[32][D + 1];
#pragma unroll
  for (int e = 0; e < kPer; ++e) tile[threadIdx.x & 31][d0 + e] = acc[e];
  __syncthreads();
  for (int e = threadIdx.x; e < 32 * D; e += 256) {
    const int q = row0 + e / D;
    if (q >= p.rows) break;
    p.out[((size_t(b) * p.Lq + q / p.group) * p.Hq + h * p.group + q % p.group) * D + e % D] =
        __float2bfloat16_rn(tile[e / D][e % D]);
  }
}

template <int D>
cudaError_t launch_as(const Kv8TcParams& p, const Kv8TcMaps& maps, const Kv8Cache& c, int clusters,
                      cudaStream_t stream) {
  const size_t smem = sizeof(Smem<D>) + 1024;
  static_assert(kMaxBatch <= 256 && sizeof(Smem<D>) + 1024 <= 232448, "shared memory exceeds 227 KB");
  cudaError_t e = cudaFuncSetAttribute(kv8_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
  if (e != cudaSuccess) return e;
  kv8_tc_kernel<D><<<2 * clusters, kThreads, smem, stream>>>(p, c, maps);
  if ((e = cudaGetLastError()) != cudaSuccess || p.whole || clusters == 1) return e;
  const int rows = std::min(p.rows, 2 * kPairRows);
  return launch_chained(kv8_tc_join_kernel<D>, dim3(clusters - 1, (rows + 31) / 32), dim3(256),
                        (clusters + 1) * sizeof(int4), stream, p, c, clusters);
}

}  // namespace

Kv8TcPlan kv8_tc_plan(const Kv8Cache& c, int rows, int num_sms) {
  Kv8TcPlan t;
  t.tiles = (rows + kPairRows - 1) / kPairRows;
  t.rounds = (t.tiles + 1) / 2;
  const int64_t steps = (int64_t(c.L) + kStepKeys - 1) / kStepKeys;
  t.whole = steps <= (c.D == 128 ? Cfg<128>::kStages : Cfg<64>::kStages);
  const int64_t work = int64_t(c.B) * c.H * t.rounds * (t.whole ? 1 : steps);
  t.clusters = int(std::max<int64_t>(1, std::min<int64_t>(num_sms / 2, work)));
  t.bytes = t.whole ? 0 : size_t(t.clusters) * (4 * kPairRows * (c.D + 2) * sizeof(float) + sizeof(int4));
  return t;
}

cudaError_t launch_kv8_tc(Kv8TcParams p, const Kv8TcMaps& maps, const Kv8TcPlan& plan, const Kv8Cache& c,
                          cudaStream_t stream) {
  p.tiles = plan.tiles;
  p.rounds = plan.rounds;
  p.whole = plan.whole;
  return c.D == 128 ? launch_as<128>(p, maps, c, plan.clusters, stream)
                    : launch_as<64>(p, maps, c, plan.clusters, stream);
}

ICSA_DEFINE_STICKY_ACCESSOR(sticky_status_kv8_tc)

}  // namespace icsa
