// Key/value cache in e4m3 with a power-of-two scale for each block of 64
// tokens and head (storage form in icsa_lowp.h), and the attention of a few
// query tokens over it.
//
// Scales are powers of two, so scaling is exact both ways: a code times its
// scale is an exact bf16 number, and the only rounding of the cache is the one
// to e4m3.  Floating-point codes lose nothing by it, as their relative step
// does not depend on the scale.
//
// Attention of few queries (kv8_decode_kernel) is a read of the cache, so it
// is built around that read: every warp takes whole 64-token blocks by itself
// and loads their bytes from global memory straight into the registers in
// which the tensor core wants them, without shared memory or barriers in the
// loop.  It computes transposed products, S^T = K Q^T and O^T = V^T P^T, so
// the bytes are the 16-row operand and the queries the 8-column one
// (mma m16n8k16), and the order of the summed index is free:
//   * S: the head features are split so that thread t of a quad owns the 16
//     consecutive bytes 16 t .. 16 t + 15 of each 64-byte half of a key row;
//   * P.V: V is stored with the tokens of a block innermost, and the keys are
//     dealt to the rows of S such that thread t needs tokens 16 t .. 16 t + 15,
//     again 16 consecutive bytes;
// so a block is read in 16-byte loads of which each covers whole sectors.
// P^T reaches its operand form with one 8 x 8 transpose (movmatrix) per 8 keys.
//
// Both products run in f16 with float32 accumulation: e4m3 codes are exact in
// f16, a query row is scaled by a power of two to [2^14, 2^15) (bf16 has 8
// significant bits, f16 11; only elements 2^-28 below the row's largest lose
// bits), and the probabilities have 11 bits (those below 2^-14 of the row's
// largest at least are multiples of 2^-24 of it).  With s the base-2 scores, m
// their running maximum and v the log2 of a value block's scale,
//   P = 2^(s - m + d),  d = v - R,  O = 2^R sum P code,  l = sum 2^-d P:
// the block's scale enters P against the reference R, and d in [0, 15] keeps P
// within f16 and every bit that p = 2^(s - m) has there.  A block outside that
// window moves R and rescales O (see value_spread); O is float32, so what one
// block's values are does not cost another block bits.  (With the scale in the
// maximum instead, m the largest s + v, a block of zeros, whose scale is 1,
// takes the bits of the small values beside it.)
//
// Long caches are split over CTAs (and over the warps of a CTA); partial
// results (O / l, m, l) are joined in a fixed order.
//
// A CTA takes one group of 8 query rows, or two, which share the conversion
// of the codes (16 a clock and SM, which bounds anything beyond 8 rows).
// One query, 2 x 40 heads x 32760 keys, D = 128: 103 us (587 MB, 5.7 TB/s);
// 16 rows 130 us, 48 rows 361 us.  Joining in order with one
// part loaded after the other cost 5 us of 16 for 1 x 8 heads x 8000 keys;
// eight at a time, and launched while the parts are computed, 11 us in all.
//
// Filling and expanding are bound by memory: 1 x 32760 x 40 x 128, keys and
// values, from bfloat16 164 us (6.1 TB/s), float32 248 us (6.8 TB/s), to
// bfloat16 166 us (6.1 TB/s).
#include "icsa_attn_common.cuh"
#include "icsa_lowp.cuh"

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

namespace icsa {

namespace {

constexpr int kTokens = 64;
constexpr int kDWarps = 4;           // warps of a decode CTA
constexpr int kMaxSplits = 32;       // of the keys over CTAs
// CTAs of NQ groups of 8 rows that fit an SM, by their registers
constexpr int decode_ctas(int D, int NQ) { return D == 128 || NQ == 2 ? 2 : 3; }
constexpr float kNegInf = -INFINITY;
constexpr float kWindow = 15.f;      // most of d = v - R: P up to 2^15 is in f16's range

ICSA_DEV int valid_tokens(const Kv8Cache& c, int b) {
  return c.lengths == nullptr ? c.L : min(max(c.lengths[b], 0), c.L);
}

// two e4m3 bytes (low 16 bits of `pair`) to f16x2
ICSA_DEV uint32_t e4m3x2_f16x2(uint16_t pair) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(pair));
  return r;
}
ICSA_DEV float2 f16x2_floats(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }

// two floats to e4m3 bytes (nearest even, saturating), the first in the low byte
ICSA_DEV uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// ---------------------------------------------------------------- filling --
// One CTA per (block, head, batch): keys and values together in bfloat16, so
// that 32 KB are on their way before the first is needed, one tensor a CTA in
// float32 (as many bytes).  Thread: 8 consecutive features of tokens
// 4 i .. 4 i + 3, so that the four tokens' bytes of one feature make a word
// of the transposed value block.
template <typename T>
constexpr int fill_tensors() { return sizeof(T) == 2 ? 2 : 1; }

template <typename T>
struct Raw8 {  // 8 elements as loaded
  uint32_t w[2 * sizeof(T)];
};

template <typename T>
ICSA_DEV void load_raw(const T* p, bool vec, Raw8<T>& x) {
  if (vec) {
#pragma unroll
    for (int h = 0; h < int(sizeof(T)) / 2; ++h) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(p) + h);
      x.w[4 * h] = u.x;
      x.w[4 * h + 1] = u.y;
      x.w[4 * h + 2] = u.z;
      x.w[4 * h + 3] = u.w;
    }
    return;
  }
  if constexpr (sizeof(T) == 2) {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) x.w[i] = uint32_t(q[2 * i]) | (uint32_t(q[2 * i + 1]) << 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x.w[i] = __float_as_uint(p[i]);
  }
}

template <typename T>
ICSA_DEV float raw_float(const Raw8<T>& x, int i) {
  if constexpr (sizeof(T) == 2) return __uint_as_float(i & 1 ? x.w[i >> 1] & 0xFFFF0000u : x.w[i >> 1] << 16);
  else return __uint_as_float(x.w[i]);
}

// largest magnitude of four rows as float bits: NaN and infinity stay above every number
template <typename T>
ICSA_DEV uint32_t raw_top(const Raw8<T> (&x)[4]) {
  uint32_t top = 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < int(2 * sizeof(T)); ++j) {
      if constexpr (sizeof(T) == 2) top = __vmaxu2(top, x[i].w[j] & 0x7FFF7FFFu);
      else top = max(top, x[i].w[j] & 0x7FFFFFFFu);
    }
  if constexpr (sizeof(T) == 2) top = max(top & 0xFFFF0000u, top << 16);
  return top;
}

template <int D>
struct FillShape {
  static constexpr int kPerRow = D / 8;                   // threads over the features of a token
  static constexpr int kThreads = 16 * kPerRow;           // 16 groups of 4 tokens
};

template <typename T, int D>
__global__ void __launch_bounds__(FillShape<D>::kThreads) kv8_quantize_kernel(const Kv8Rows x, const Kv8Cache c) {
  constexpr int kPerRow = FillShape<D>::kPerRow, kThreads = FillShape<D>::kThreads;
  constexpr int kTensors = fill_tensors<T>();
  // heads run fastest: the CTAs of one time read whole rows of x
  const int h = blockIdx.x % c.H, bk = blockIdx.x / c.H;
  const int blk = bk % c.nb, b = bk / c.nb, bh = b * c.H + h;
  const int len = valid_tokens(c, b);
  const int f0 = (threadIdx.x % kPerRow) * 8, g = threadIdx.x / kPerRow;
  Raw8<T> raw[kTensors][4];
  __shared__ uint32_t tops[kTensors][kThreads / 32];
#pragma unroll
  for (int t = 0; t < kTensors; ++t) {
    const bool values = kTensors == 2 ? t == 1 : blockIdx.y == 1;
    const void* from = values ? x.x[1] : x.x[0];
    const int64_t sb = values ? x.sb[1] : x.sb[0], st = values ? x.st[1] : x.st[0], sh = values ? x.sh[1] : x.sh[0];
    // 16-byte accesses: every row start and stride aligned
    const bool vec = (reinterpret_cast<uintptr_t>(from) & 15u) == 0 && ((sb | st | sh) * int64_t(sizeof(T))) % 16 == 0;
    const T* src = static_cast<const T*>(from) + b * sb + h * sh + int64_t(blk * kTokens + 4 * g) * st + f0;
#pragma unroll
    for (int i = 0; i < 4; ++i, src += st) {
      if (blk * kTokens + 4 * g + i < len) {
        load_raw<T>(src, vec, raw[t][i]);
      } else {
#pragma unroll
        for (uint32_t& w : raw[t][i].w) w = 0u;
      }
    }
  }
#pragma unroll
  for (int t = 0; t < kTensors; ++t) {
    const uint32_t top = __reduce_max_sync(0xffffffffu, raw_top(raw[t]));
    if ((threadIdx.x & 31) == 0) tops[t][threadIdx.x >> 5] = top;
  }
  __syncthreads();
  const size_t slot = size_t(bh) * c.nb + blk;
#pragma unroll
  for (int t = 0; t < kTensors; ++t) {
    const bool values = kTensors == 2 ? t == 1 : blockIdx.y == 1;
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) top = max(top, tops[t][i]);
    // smallest e with amax <= 448 2^e = 1.75 2^(8 + e); a subnormal amax is far
    // below the clamp at -96
    int e = int(top >> 23) - 127 - 8 + ((top & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    e = min(max(e, -96), 96);
    const bool bad = top >= 0x7F800000u;
    if (top == 0u || bad) e = 0;
    const float inv = __uint_as_float(uint32_t(127 - e) << 23);
    if (threadIdx.x == 0)
      (values ? c.v_scale : c.k_scale)[slot] =
          bad ? __uint_as_float(0x7FC00000u) : __uint_as_float(uint32_t(127 + e) << 23);
    uint32_t code[2][4] = {};  // [features 0-3 | 4-7][token], 4 code bytes each
    if (!bad) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < 2; ++q)
          code[q][i] = e4m3x2(raw_float(raw[t][i], 4 * q) * inv, raw_float(raw[t][i], 4 * q + 1) * inv) |
                       (e4m3x2(raw_float(raw[t][i], 4 * q + 2) * inv, raw_float(raw[t][i], 4 * q + 3) * inv) << 16);
    }
    if (!values) {
      uint8_t* dst = c.k + (slot * kTokens + 4 * g) * D + f0;
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<uint2*>(dst + i * D) = make_uint2(code[0][i], code[1][i]);
      continue;
    }
    // values: words of four tokens, [feature][token / 4], the words of two
    // features in an order that keeps stores and loads off each other's banks
    __shared__ uint32_t tile[D * 16];
    auto word = [](int f, int q) { return (f >> 1) * 32 + ((f ^ q) & 1) * 16 + (q ^ ((f >> 3) & 15)); };
#pragma unroll
    for (int e8 = 0; e8 < 8; ++e8) {
      const uint32_t sel = uint32_t(e8 & 3) | (uint32_t((e8 & 3) + 4) << 4);
      const uint32_t p01 = __byte_perm(code[e8 >> 2][0], code[e8 >> 2][1], sel);
      const uint32_t p23 = __byte_perm(code[e8 >> 2][2], code[e8 >> 2][3], sel);
      tile[word(f0 + e8, g)] = __byte_perm(p01, p23, 0x5410);
    }
    __syncthreads();
    // four words of one feature a thread: 16-byte stores
    uint4* out = reinterpret_cast<uint4*>(c.v + slot * kTokens * D);
#pragma unroll
    for (int i = 0; i < D * 4 / kThreads; ++i) {
      const int wd = i * kThreads + threadIdx.x, f = wd >> 2, q = (wd & 3) * 4;
      out[wd] = make_uint4(tile[word(f, q)], tile[word(f, q + 1)], tile[word(f, q + 2)], tile[word(f, q + 3)]);
    }
  }
}

// ------------------------------------------------------------- expansion --
// [B, L, H, D] of T from the cache; rows behind a length are zero whatever
// the cache holds there.
template <typename T, int D>
ICSA_DEV void store8(T* dst, const float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    uint4 u;
    u.x = pack_bf16x2(v[0], v[1]);
    u.y = pack_bf16x2(v[2], v[3]);
    u.z = pack_bf16x2(v[4], v[5]);
    u.w = pack_bf16x2(v[6], v[7]);
    *reinterpret_cast<uint4*>(dst) = u;
  } else {
    reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}

ICSA_DEV uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// exponent of a power of two as a float; NaN stays NaN
ICSA_DEV float scale_log2(float s) { return s != s ? s : float(int(__float_as_uint(s) >> 23) - 127); }

// R of a head for launch_kv8_copy, a CTA each: codes are exact in f16 from
// 2^-15 to 2^7 of themselves, so where the scales lie within 22 binades
// R = (log2 of the largest) - 7.  (A NaN scale goes with any R.)
constexpr int kRefThreads = 256;
__global__ void __launch_bounds__(kRefThreads) kv8_reference_kernel(const Kv8Cache c, float* v_ref) {
  const int len = valid_tokens(c, blockIdx.x / c.H), nb = (len + kTokens - 1) / kTokens;
  const float* scale = c.v_scale + size_t(blockIdx.x) * c.nb;
  int lo = 1000, hi = -1000;
  for (int i = threadIdx.x; i < nb; i += kRefThreads) {
    const float e = scale_log2(scale[i]);
    if (e == e) {
      lo = min(lo, int(e));
      hi = max(hi, int(e));
    }
  }
  __shared__ int part[2][kRefThreads / 32];
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if ((threadIdx.x & 31) == 0) {
    part[0][threadIdx.x >> 5] = lo;
    part[1][threadIdx.x >> 5] = hi;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < kRefThreads / 32; ++i) {
    lo = min(lo, part[0][i]);
    hi = max(hi, part[1][i]);
  }
  v_ref[blockIdx.x] = hi < lo ? 0.f : hi - lo <= 22 ? float(hi - 7) : __uint_as_float(0x7FC00000u);
}

// V_REF: the operands of launch_kv8_copy.
template <typename T, int D, bool V_REF>
__global__ void __launch_bounds__(FillShape<D>::kThreads)
    kv8_dequantize_kernel(const Kv8Cache c, T* k_out, T* v_out, const float* v_ref) {
  constexpr int kPerRow = FillShape<D>::kPerRow, kThreads = FillShape<D>::kThreads;
  const int which = k_out == nullptr ? 1 : int(blockIdx.y);
  T* out = which ? v_out : k_out;
  const int blk = blockIdx.x % c.nb, bh = blockIdx.x / c.nb;
  const int b = bh / c.H, h = bh % c.H;
  const int len = valid_tokens(c, b);
  const int f0 = (threadIdx.x % kPerRow) * 8, g = threadIdx.x / kPerRow;
  const size_t slot = size_t(bh) * c.nb + blk;
  const bool any = blk * kTokens < len;
  float scale = any ? (which ? c.v_scale : c.k_scale)[slot] : 0.f;
  bool f16 = false;
  if constexpr (V_REF) {
    wait_prior_grid();
    const float r = which ? v_ref[bh] : __uint_as_float(0x7FC00000u);
    f16 = r == r;
    if (f16) scale *= __uint_as_float(uint32_t(127 - int(r)) << 23);
  }
  uint32_t code[2][4] = {};  // [features 0-3 | 4-7][token]
  __shared__ uint32_t tile[D][17];
  if (any) {
    if (which == 0) {
      const uint8_t* src = c.k + (slot * kTokens + 4 * g) * D + f0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(src + i * D));
        code[0][i] = u.x;
        code[1][i] = u.y;
      }
    } else {
      const uint32_t* src = reinterpret_cast<const uint32_t*>(c.v + slot * kTokens * D);
#pragma unroll
      for (int i = 0; i < D * 16 / kThreads; ++i) {
        const int wd = i * kThreads + threadIdx.x;
        tile[wd >> 4][wd & 15] = __ldg(src + wd);
      }
      __syncthreads();
      // four tokens' bytes of a feature back to one token's bytes of four features
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = tile[f0 + 4 * half + e][g];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t sel = uint32_t(i) | (uint32_t(i + 4) << 4);
          code[half][i] = (__byte_perm(w[0], w[1], sel) & 0xFFFFu) | (__byte_perm(w[2], w[3], sel) << 16);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int tok = blk * kTokens + 4 * g + i;
    if (tok >= c.L) break;
    float v[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = f16x2_floats(e4m3x2_f16x2(uint16_t(code[e >> 1][i] >> (16 * (e & 1)))));
      v[2 * e] = f.x * scale;
      v[2 * e + 1] = f.y * scale;
    }
    if (tok >= len) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
    }
    T* dst = out + ((size_t(b) * c.L + tok) * c.H + h) * D + f0;
    if (V_REF && f16)
      *reinterpret_cast<uint4*>(dst) = make_uint4(pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]),
                                                  pack_f16x2(v[4], v[5]), pack_f16x2(v[6], v[7]));
    else store8<T, D>(dst, v);
  }
}

// ---------------------------------------------------- attention, few rows --
ICSA_DEV void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
ICSA_DEV uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
ICSA_DEV uint4 load_stream16(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}
ICSA_DEV uint32_t word(const uint4& u, int i) { return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w; }

// the bytes of tokens [0, n) of the 16 in `u` (n <= 0: none)
ICSA_DEV uint4 keep_bytes(uint4 u, int n) {
  uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int k = n - 4 * i;
    w[i] = k >= 4 ? w[i] : k <= 0 ? 0u : w[i] & (0xFFFFFFFFu >> (8 * (4 - k)));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The 8 NQ rows blockIdx.z of (b, cache head): row r is query token r / group,
// head h * group + r % group.
template <int D, int NQ>
__global__ void __launch_bounds__(kDWarps * 32, decode_ctas(D, NQ)) kv8_decode_kernel(const Kv8AttnParams p, const Kv8Cache c) {
  constexpr int kHalves = D / 64;            // 64-byte halves of a key row
  constexpr int kSteps = D / 16;             // 16-feature steps of S
  constexpr int kOTiles = D / 16;            // 16-feature tiles of O^T
  release_next_grid();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x, bh = blockIdx.y, b = bh / c.H, h = bh % c.H;
  const int rows = p.Lq * p.group, row0 = blockIdx.z * 8 * NQ;
  const int len = valid_tokens(c, b);
  const int nb = (len + kTokens - 1) / kTokens;
  const int blk0 = int(int64_t(nb) * split / p.splits), blk1 = int(int64_t(nb) * (split + 1) / p.splits);

  auto q_row = [&](int r) {
    return p.q + int64_t(b) * p.q_sb + int64_t(r / p.group) * p.q_st + int64_t(h * p.group + r % p.group) * p.q_sh;
  };
  // Q^T operand: query row g, features 64 hf + 16 t + 4 j + {0,1 | 2,3} for step 4 hf + j
  uint32_t qf[NQ][kSteps][2];
  float q_scale[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    uint32_t raw[kHalves][8];
    const bool ok = row0 + 8 * n + g < rows;
    uint32_t top = 0;
#pragma unroll
    for (int hf = 0; hf < kHalves; ++hf) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint4 u = make_uint4(0u, 0u, 0u, 0u);
        if (ok) u = __ldg(reinterpret_cast<const uint4*>(q_row(row0 + 8 * n + g) + 64 * hf + 16 * t) + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) raw[hf][4 * i + k] = word(u, k);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k)
        top = max(top, max(raw[hf][k] & 0x7FFFu, (raw[hf][k] >> 16) & 0x7FFFu));
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // scale the row's largest magnitude into [2^14, 2^15); a row with a NaN or
    // an infinity makes all its scores NaN
    const int e = min(max(int(top >> 7) - 127 - 14, -126), 126);
    const float inv = __uint_as_float(uint32_t(127 - e) << 23);
    q_scale[n] = top >= 0x7F80u ? __uint_as_float(0x7FC00000u) : __uint_as_float(uint32_t(127 + e) << 23);
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t w = raw[s >> 2][2 * (s & 3) + i];
        qf[n][s][i] = pack_f16x2(__uint_as_float(w << 16) * inv, __uint_as_float(w & 0xFFFF0000u) * inv);
      }
  }
  // columns 2 t, 2 t + 1 of this thread's accumulators
  float qs[NQ][2], o[NQ][kOTiles][4], m[NQ][2], l[NQ][2];
  // R (the same in all lanes; below any v, so that the first block sets it), and
  // for the rare moves an upper bound of the v so far
  float ref_v = -1000.f;
  __shared__ float top_v[kDWarps];
  if (lane == 0) top_v[warp] = -1000.f;
  __syncwarp();
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      qs[n][i] = __shfl_sync(0xffffffffu, q_scale[n], (2 * t + i) * 4) * p.scale_log2;
      m[n][i] = kNegInf;
      l[n][i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < kOTiles; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
  }

  const size_t slot0 = size_t(bh) * c.nb;
  // key row of S row (tile i, row r): 16 (r' / 2) + 4 i + r' % 2, + 2 for rows r = r' + 8
  const int key_g = 16 * (g >> 1) + (g & 1);
  const uint8_t* kbase = c.k + slot0 * kTokens * D + key_g * D + 16 * t;
  const uint8_t* vbase = c.v + slot0 * kTokens * D + g * kTokens + 16 * t;

  const auto move_reference = [&](float lv) {
    if (lv < ref_v || lv > ref_v + kWindow) {
      // (8 binades more than the spread: p is at most 1 here)
      const float top = fmaxf(fmaxf(top_v[warp], ref_v + kWindow), lv);
      const float r = fmaxf(lv - 8.f, top - value_spread(len) - 8.f), f = attn::ex2(ref_v - r);
      __syncwarp();
      if (lane == 0) top_v[warp] = top;
      __syncwarp();
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int i = 0; i < kOTiles; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][i][e] *= f;
      ref_v = r;
    }
  };
  // two groups: the scale comes a block ahead, and R moves before the loads
  // (after the scores it cost 8 us of 131 for 2 x 40 heads, 16 rows); one
  // group: after the scores, where the loads hide it
  float vs = NQ > 1 && blk0 + warp < blk1 ? c.v_scale[slot0 + blk0 + warp] : 1.f;
  for (int blk = blk0 + warp; blk < blk1; blk += kDWarps) {
    float lv = 0.f;
    if constexpr (NQ > 1) {
      lv = scale_log2(vs);
      if (blk + kDWarps < blk1) vs = c.v_scale[slot0 + blk + kDWarps];
      move_reference(lv);
    }
    const uint8_t* kp = kbase + size_t(blk) * kTokens * D;
    const uint8_t* vp = vbase + size_t(blk) * kTokens * D;
    uint4 kr[4][2][kHalves];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int hf = 0; hf < kHalves; ++hf) kr[i][r][hf] = load_stream16(kp + (4 * i + 2 * r) * D + 64 * hf);
    const float ks = c.k_scale[slot0 + blk];
    if constexpr (NQ == 1) lv = scale_log2(c.v_scale[slot0 + blk]);
    uint4 vr[kOTiles][2];
    const auto load_values = [&]() {
#pragma unroll
      for (int i = 0; i < kOTiles; ++i)
#pragma unroll
        for (int r = 0; r < 2; ++r) vr[i][r] = load_stream16(vp + (16 * i + 8 * r) * kTokens);
    };
    // one group of rows: the read is what counts, both loads at once; two
    // groups leave no registers for that
    if (NQ == 1) load_values();

    float s[NQ][4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) s[n][i][0] = s[n][i][1] = s[n][i][2] = s[n][i][3] = 0.f;
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        const uint32_t w0 = word(kr[i][0][st >> 2], st & 3), w1 = word(kr[i][1][st >> 2], st & 3);
        const uint32_t a0 = e4m3x2_f16x2(uint16_t(w0)), a1 = e4m3x2_f16x2(uint16_t(w1));
        const uint32_t a2 = e4m3x2_f16x2(uint16_t(w0 >> 16)), a3 = e4m3x2_f16x2(uint16_t(w1 >> 16));
#pragma unroll
        for (int n = 0; n < NQ; ++n) mma_f16(s[n][i], a0, a1, a2, a3, qf[n][st][0], qf[n][st][1]);
      }
    }
    if (NQ > 1) load_values();
    const int left = len - blk * kTokens;  // valid tokens of this block
    if constexpr (NQ == 1) move_reference(lv);
    const float dv = lv - ref_v, wl = attn::ex2(-dv);
    uint32_t pb[NQ][4][2];  // P^T operands
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float mx[2] = {kNegInf, kNegInf};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // rows g (e < 2) and g + 8, columns 2 t + (e & 1)
          float x = s[n][i][e] * (qs[n][e & 1] * ks);
          if (left < kTokens && key_g + 4 * i + 2 * (e >> 1) >= left) x = kNegInf;
          s[n][i][e] = x;
          mx[e & 1] = fmaxf(mx[e & 1], x);
        }
      float neg[2], a[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int d = 4; d < 32; d *= 2) mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], d));
        const float mn = fmaxf(m[n][i], mx[i]);
        const float ref = mn == kNegInf ? 0.f : mn;
        a[i] = attn::ex2(m[n][i] - ref);
        m[n][i] = mn;
        neg[i] = dv - ref;
      }
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[n][i][e] = attn::ex2(s[n][i][e] + neg[e & 1]);
          sum[e & 1] += s[n][i][e];
        }
#pragma unroll
      for (int i = 0; i < 2; ++i) l[n][i] = l[n][i] * a[i] + sum[i] * wl;
#pragma unroll
      for (int i = 0; i < kOTiles; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][i][e] *= a[e & 1];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        pb[n][i][0] = transpose8x8(pack_f16x2(s[n][i][0], s[n][i][1]));
        pb[n][i][1] = transpose8x8(pack_f16x2(s[n][i][2], s[n][i][3]));
      }
    }
    if (left < kTokens) {
      // a probability of zero does not hide a NaN code
#pragma unroll
      for (int i = 0; i < kOTiles; ++i)
#pragma unroll
        for (int r = 0; r < 2; ++r) vr[i][r] = keep_bytes(vr[i][r], left - 16 * t);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int d = 0; d < kOTiles; ++d) {
        const uint32_t w0 = word(vr[d][0], i), w1 = word(vr[d][1], i);
        const uint32_t a0 = e4m3x2_f16x2(uint16_t(w0)), a1 = e4m3x2_f16x2(uint16_t(w1));
        const uint32_t a2 = e4m3x2_f16x2(uint16_t(w0 >> 16)), a3 = e4m3x2_f16x2(uint16_t(w1 >> 16));
#pragma unroll
        for (int n = 0; n < NQ; ++n) mma_f16(o[n][d], a0, a1, a2, a3, pb[n][i][0], pb[n][i][1]);
      }
    }
  }
  // the threads of a column hold different keys: join their sums (m is equal)
#pragma unroll
  for (int n = 0; n < NQ; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int d = 4; d < 32; d *= 2) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], d);

  // join the warps: O / l in the values' own unit, [warp][column][feature] (a
  // warp without a key has l = 0 and O = 0)
  const float unit = attn::ex2(ref_v);
  __shared__ float so[kDWarps][8 * NQ][D + 4];
  __shared__ float sm[kDWarps][8 * NQ], sl[kDWarps][8 * NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    float inv[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) inv[i] = l[n][i] == 0.f ? 0.f : 1.0f / l[n][i];
#pragma unroll
    for (int d = 0; d < kOTiles; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        so[warp][8 * n + 2 * t + (e & 1)][16 * d + g + 8 * (e >> 1)] = o[n][d][e] * inv[e & 1] * unit;
    if (g == 0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        sm[warp][8 * n + 2 * t + i] = m[n][i];
        sl[warp][8 * n + 2 * t + i] = l[n][i];
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 8 * NQ * D; i += kDWarps * 32) {
    const int col = i / D, d = i % D, r = row0 + col;
    if (r >= rows) break;
    float mm = kNegInf;
#pragma unroll
    for (int w = 0; w < kDWarps; ++w) mm = fmaxf(mm, sm[w][col]);
    const float ref = mm == kNegInf ? 0.f : mm;
    float f[kDWarps], lt = 0.f;
#pragma unroll
    for (int w = 0; w < kDWarps; ++w) {
      f[w] = sl[w][col] * attn::ex2(sm[w][col] - ref);
      lt += f[w];
    }
    // the warps' shares of the sum: a weighted mean, which no value overflows
    const float inv = lt == 0.f && blk0 == blk1 ? 0.f : 1.0f / lt;
    float y = 0.f;
#pragma unroll
    for (int w = 0; w < kDWarps; ++w) y += so[w][col][d] * (f[w] * inv);
    if (p.splits == 1) {
      p.out[((size_t(b) * p.Lq + r / p.group) * p.Hq + h * p.group + r % p.group) * D + d] = __float2bfloat16_rn(y);
    } else {
      float* dst = p.partial + ((size_t(bh) * rows + r) * p.splits + split) * (D + 2);
      dst[d] = y;
      if (d == 0) {
        dst[D] = mm;
        dst[D + 1] = lt;
      }
    }
  }
}

// joins the splits of one query row, at most kMaxSplits; one CTA per (b, cache
// head, row).  Every lane takes one split's weight l 2^(m - max m).
template <int D>
__global__ void __launch_bounds__(D) kv8_join_kernel(const Kv8AttnParams p, const Kv8Cache c) {
  static_assert(kMaxSplits == 32, "a lane for each split");
  const int rows = p.Lq * p.group;
  const int r = blockIdx.x, bh = blockIdx.y, b = bh / c.H, h = bh % c.H, d = threadIdx.x, lane = threadIdx.x & 31;
  wait_prior_grid();
  const float* src = p.partial + (size_t(bh) * rows + r) * p.splits * (D + 2);
  constexpr int kAhead = 8;  // splits whose loads are on their way together
  float x[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) x[i] = i < p.splits ? src[i * (D + 2) + d] : 0.f;
  const float m = lane < p.splits ? src[lane * (D + 2) + D] : kNegInf;
  float w = lane < p.splits ? src[lane * (D + 2) + D + 1] : 0.f;
  float top = m;
#pragma unroll
  for (int i = 16; i > 0; i /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
  w *= attn::ex2(m - (top == kNegInf ? 0.f : top));
  float total = w;
#pragma unroll
  for (int i = 16; i > 0; i /= 2) total += __shfl_xor_sync(0xffffffffu, total, i);
  w *= valid_tokens(c, b) == 0 ? 0.f : 1.0f / total;
  float y = 0.f;
  for (int s0 = 0; s0 < p.splits; s0 += kAhead) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) y += x[i] * __shfl_sync(0xffffffffu, w, s0 + i);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) x[i] = s0 + kAhead + i < p.splits ? src[(s0 + kAhead + i) * (D + 2) + d] : 0.f;
  }
  p.out[((size_t(b) * p.Lq + r / p.group) * p.Hq + h * p.group + r % p.group) * D + d] = __float2bfloat16_rn(y);
}

template <typename T>
cudaError_t quantize_as(const Kv8Rows& x, const Kv8Cache& c, cudaStream_t stream) {
  const dim3 grid(unsigned(c.B) * c.H * c.nb, 2 / fill_tensors<T>());
  if (c.D == 128) kv8_quantize_kernel<T, 128><<<grid, FillShape<128>::kThreads, 0, stream>>>(x, c);
  else kv8_quantize_kernel<T, 64><<<grid, FillShape<64>::kThreads, 0, stream>>>(x, c);
  return cudaGetLastError();
}

template <typename T>
cudaError_t dequantize_as(const Kv8Cache& c, void* const out[2], cudaStream_t stream) {
  const dim3 grid(unsigned(c.B) * c.H * c.nb, (out[0] != nullptr) + (out[1] != nullptr));
  T *k = static_cast<T*>(out[0]), *v = static_cast<T*>(out[1]);
  if (c.D == 128) kv8_dequantize_kernel<T, 128, false><<<grid, FillShape<128>::kThreads, 0, stream>>>(c, k, v, nullptr);
  else kv8_dequantize_kernel<T, 64, false><<<grid, FillShape<64>::kThreads, 0, stream>>>(c, k, v, nullptr);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv8_quantize(const Kv8Rows& x, int dtype, const Kv8Cache& c, cudaStream_t stream) {
  return dtype == ICSA_BF16 ? quantize_as<__nv_bfloat16>(x, c, stream) : quantize_as<float>(x, c, stream);
}

cudaError_t launch_kv8_dequantize(const Kv8Cache& c, void* const out[2], int out_dtype, cudaStream_t stream) {
  return out_dtype == ICSA_BF16 ? dequantize_as<__nv_bfloat16>(c, out, stream) : dequantize_as<float>(c, out, stream);
}

cudaError_t launch_kv8_copy(const Kv8Cache& c, void* k, void* v, float* v_ref, cudaStream_t stream) {
  kv8_reference_kernel<<<c.B * c.H, kRefThreads, 0, stream>>>(c, v_ref);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const dim3 grid(unsigned(c.B) * c.H * c.nb, 2);
  __nv_bfloat16 *kb = static_cast<__nv_bfloat16*>(k), *vb = static_cast<__nv_bfloat16*>(v);
  const float* ref = v_ref;
  return c.D == 128 ? launch_chained(kv8_dequantize_kernel<__nv_bfloat16, 128, true>, grid,
                                     dim3(FillShape<128>::kThreads), 0, stream, c, kb, vb, ref)
                    : launch_chained(kv8_dequantize_kernel<__nv_bfloat16, 64, true>, grid,
                                     dim3(FillShape<64>::kThreads), 0, stream, c, kb, vb, ref);
}

Kv8DecodePlan kv8_decode_plan(int B, int H, int rows, int L, int D, int num_sms) {
  const int64_t nb = (int64_t(L) + kTokens - 1) / kTokens;
  // Waves of CTAs times the steps of a warp, two steps' time for a CTA's start
  // and its part of the join; a split keeps at least one block for each warp.
  // 2 x 40 heads x 32760 tokens, D = 64, one row: three splits (two CTAs to an
  // SM) 83 us, eleven 69 us.  One or two groups of 8 rows a CTA, us: D = 128, 2 x
  // 40 x 32000, 16 rows 208 / 130, 48 rows 569 / 361; 1 x 8 x 2000, 64 rows
  // 15 / 17; D = 64, 2 x 40 x 32000, 48 rows 300 / 224.
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(nb / kDWarps, kMaxSplits));
  Kv8DecodePlan best = {1, 1, 0.0};
  for (int groups = 1; groups <= (rows > 8 ? 2 : 1); ++groups) {
    const int64_t ctas = int64_t(B) * H * ((rows + 8 * groups - 1) / (8 * groups));
    const int64_t slots = int64_t(num_sms) * decode_ctas(D, groups);
    const double step = groups == 1 ? (D == 128 ? 2.4 : 1.5) : (D == 128 ? 3.2 : 1.8);
    for (int64_t s = 1; s <= most; ++s) {
      const double us = double((ctas * s + slots - 1) / slots) * (double(nb) / double(s * kDWarps) + 2.0) * step +
                        (s > 1 ? 6.0 : 4.0);
      if (best.us == 0.0 || us < best.us) best = {int(s), groups, us};
    }
  }
  return best;
}

cudaError_t launch_kv8_decode(const Kv8AttnParams& p, const Kv8Cache& c, cudaStream_t stream) {
  const int rows = p.Lq * p.group;
  const dim3 grid(p.splits, c.B * c.H, (rows + 8 * p.groups - 1) / (8 * p.groups));
  const auto kernel = c.D == 128 ? (p.groups == 2 ? kv8_decode_kernel<128, 2> : kv8_decode_kernel<128, 1>)
                                 : (p.groups == 2 ? kv8_decode_kernel<64, 2> : kv8_decode_kernel<64, 1>);
  kernel<<<grid, kDWarps * 32, 0, stream>>>(p, c);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || p.splits == 1) return e;
  const dim3 jgrid(rows, c.B * c.H);
  return c.D == 128 ? launch_chained(kv8_join_kernel<128>, jgrid, dim3(128), 0, stream, p, c)
                    : launch_chained(kv8_join_kernel<64>, jgrid, dim3(64), 0, stream, p, c);
}

}  // namespace icsa
