// Microscaled 4-bit floating point: quantisation of rows into the storage form
// of icsa_lowp.cuh, and back.
//
// Quantisation of one block of n elements (n = 16: nvfp4, n = 32: mxfp4):
//   amax = max |x|
//   nvfp4: s = e4m3(amax / (6 g)), step d = s g    (g: the tensor's global scale)
//   mxfp4: s = 2^(floor(log2 amax) - 2) (exponent in [-127, 127]), d = s
//   code = e2m1(x / d), rounded to nearest even, largest magnitude 6; 0 where d = 0
// or, for the rows of a linear layer, with g a power of two for each row: the
// smallest with which the row's largest magnitude is in range (448 x 6 g), so
// that rows of any magnitude keep the format's bits.
// Quotients are those of IEEE float32 division, so a host computation in
// float32 gives the same bytes.  A block that holds a NaN or an infinity gets
// the format's NaN scale (0x7f / 0xff).
//
// One pass over memory: a thread owns 16 elements of a row (32 bytes of bf16:
// one 256-bit load), writes their 8 code bytes, and each group of four scales
// is gathered by shuffles into one 32-bit store.  The eight warps of a CTA
// take eight rows of one scale tile whose scale words share 32-byte sectors
// (rows r, r + 1 and those 32, 64, 96 further), so that the scattered words
// reach memory as whole sectors.
//
// Bound by memory: 65536 x 5120, quantised and back, float32 233 and 236 us
// (6.5 TB/s), bfloat16 mxfp4 145 and 150 us (5.7 TB/s); bfloat16 nvfp4, with
// twice the scales and quotients by steps that are no powers of two, 168 us
// (5.1 TB/s, bound by issue; 178 us without the two-lane float instructions).
// Loading a chunk ahead changed none of them.
#include "icsa_attn_common.cuh"
#include "icsa_lowp.cuh"

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cstring>

namespace icsa {

namespace {

constexpr int kQThreads = 256;
constexpr int kQChunk = 512;  // elements of a row that one warp takes at a time

struct alignas(32) Words8 {
  uint32_t w[8];
};

// 32-byte global accesses (the address is a multiple of 32)
ICSA_DEV Words8 load32(const void* p) {
  Words8 r;
  asm volatile("ld.global.nc.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]),
                 "=r"(r.w[7])
               : "l"(p));
  return r;
}
ICSA_DEV void store32(void* p, const Words8& r) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r.w[0]), "r"(r.w[1]), "r"(r.w[2]),
               "r"(r.w[3]), "r"(r.w[4]), "r"(r.w[5]), "r"(r.w[6]), "r"(r.w[7])
               : "memory");
}

template <typename T>
ICSA_DEV float to_float(T v);
template <>
ICSA_DEV float to_float<float>(float v) {
  return v;
}
template <>
ICSA_DEV float to_float<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <typename T>
ICSA_DEV T from_float(float v);
template <>
ICSA_DEV float from_float<float>(float v) {
  return v;
}
template <>
ICSA_DEV __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// Bytes by which every row start is aligned: 32 (one access per 8 words), 16,
// or 0 (any alignment: the warp moves its 512 elements through shared memory,
// so that global accesses stay contiguous).
constexpr int kStage = kQChunk / 16 * 17;  // floats of one warp's stage, a pad word behind each lane's 16

ICSA_DEV Words8 load16x2(const void* p) {
  const uint4 a = __ldg(static_cast<const uint4*>(p)), b = __ldg(static_cast<const uint4*>(p) + 1);
  return Words8{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}
ICSA_DEV void store16x2(void* p, const Words8& r) {
  static_cast<uint4*>(p)[0] = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
  static_cast<uint4*>(p)[1] = make_uint4(r.w[4], r.w[5], r.w[6], r.w[7]);
}

// Elements [c0 + 16 lane, + 16) of a row of K (zeros from column K on); called
// by whole warps.  Returns their largest magnitude as float32 bits: NaN and
// infinity stay above every number.  (Elements of 16 bits are compared in pairs.)
template <typename T, int ALIGN>
ICSA_DEV uint32_t load16(const T* row, int c0, int lane, int K, float* stage, float (&v)[16]) {
  const int k0 = c0 + 16 * lane;
  uint32_t top = 0u;
  if constexpr (ALIGN > 0) {
    if (k0 + 16 <= K) {
#pragma unroll
      for (int h = 0; h < int(sizeof(T)) / 2; ++h) {
        const T* src = row + k0 + 8 * h;
        const Words8 r = ALIGN == 32 ? load32(src) : load16x2(src);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if constexpr (sizeof(T) == 2) {
            v[2 * i] = __uint_as_float(r.w[i] << 16);
            v[2 * i + 1] = __uint_as_float(r.w[i] & 0xFFFF0000u);
            top = __vmaxu2(top, r.w[i] & 0x7FFF7FFFu);
          } else {
            v[8 * h + i] = __uint_as_float(r.w[i]);
            top = max(top, r.w[i] & 0x7FFFFFFFu);
          }
        }
      }
      return sizeof(T) == 2 ? max(top << 16, top & 0xFFFF0000u) : top;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = k0 + i < K ? to_float<T>(row[k0 + i]) : 0.f;
  } else {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int k = 32 * i + lane;
      stage[k + (k >> 4)] = c0 + k < K ? to_float<T>(row[c0 + k]) : 0.f;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = stage[17 * lane + i];
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  return top;
}

template <typename T, int ALIGN>
ICSA_DEV void store16(T* row, int c0, int lane, int K, float* stage, const float (&v)[16]) {
  const int k0 = c0 + 16 * lane;
  if constexpr (ALIGN > 0) {
    if (k0 + 16 <= K) {
#pragma unroll
      for (int h = 0; h < int(sizeof(T)) / 2; ++h) {
        Words8 o;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if constexpr (sizeof(T) == 2) o.w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
          else o.w[i] = __float_as_uint(v[8 * h + i]);
        }
        if constexpr (ALIGN == 32) store32(row + k0 + 8 * h, o);
        else store16x2(row + k0 + 8 * h, o);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (k0 + i < K) row[k0 + i] = from_float<T>(v[i]);
    }
  } else {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i) stage[17 * lane + i] = v[i];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int k = 32 * i + lane;
      if (c0 + k < K) row[c0 + k] = from_float<T>(stage[k + (k >> 4)]);
    }
  }
}

// eight floats to e2m1 (nearest even, saturating), the first in the low half of byte 0
ICSA_DEV uint32_t e2m1x8(const float* v) {
  uint32_t o;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(o)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return o;
}

// four code bytes to eight floats
ICSA_DEV void e2m1x8_floats(uint32_t w, float (&v)[8]) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

ICSA_DEV float e4m3_float(uint32_t byte) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3);
  return __half2float(__half(h));
}

// byte offset of the scale tile row of row r, and of K tile / scale c in it
ICSA_DEV size_t scale_row(int r, int k_tiles, int atoms) {
  return size_t(r >> 7) * k_tiles * atoms * kScaleAtomBytes + (r & 31) * 16 + ((r >> 5) & 3) * 4;
}

// rows of CTA blockIdx.x: warp w of pair-group i
ICSA_DEV int tile_row(int cta, int warp) {
  return (cta >> 4) * kFp4TileRows + (cta & 15) * 2 + (warp & 1) + 32 * (warp >> 1);
}

// The 16 codes of x / d, those of the correctly rounded float32 quotient:
// with 1 / d as the sum of two floats, rh + rl, the sum x rh + x rl is within
// a relative 2^-42 of the quotient before its one rounding (both parts are
// positive, so that an x of -0 stays -0).  That rounding is
// the quotient's own unless a midpoint m of two floats (25 bits) lies between
// the two, and with d of at most 8 significant bits m d has at most 33, so a
// float x is no closer to it than a relative 2^-33.  Such steps are those of
// a global scale that is a power of two; others divide, as do blocks beyond
// the largest scale, whose quotients might overflow.  Two operations an
// element instead of a division: 65536 x 5120 bfloat16 168 us, with the
// divisions (a global scale of 0.9) 258 us.
ICSA_DEV bool short_step(float d) { return (__float_as_uint(d) & 0xFFFFu) == 0u; }
ICSA_DEV void quotient_codes(const float (&v)[16], float amax, float d, uint32_t (&code)[2]) {
  float q[16];
  if (d > 0x1p-100f && d < 0x1p100f && amax <= 8.f * d && short_step(d)) {
    float rh;
    asm("rcp.approx.f32 %0, %1;" : "=f"(rh) : "f"(d));  // within one unit in the last place of 1 / d
    rh = __uint_as_float(__float_as_uint(rh) - 2u);       // below it: rl > 0
    const float rl = fmaf(-d, rh, 1.0f) * rh;
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      float a, b;
      attn::fmul2(a, b, v[i], v[i + 1], rl, rl);
      attn::ffma2(q[i], q[i + 1], v[i], v[i + 1], rh, rh, a, b);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) q[i] = __fdiv_rn(v[i], d);
  }
  code[0] = e2m1x8(q);
  code[1] = e2m1x8(q + 8);
}

// The global scale of a row whose largest magnitude has these float32 bits:
// 2^e, e the smallest with top <= 2688 2^e = 1.3125 2^(11 + e), in [-90, 90] (as
// quotient_codes takes them); 1 for a row of zeros, and for one with a NaN or an
// infinity, of which the blocks without them count nothing.
ICSA_DEV float row_scale(uint32_t top) {
  if (top == 0u || top >= 0x7F800000u) return 1.f;
  const int e = int(top >> 23) - 127 - 11 + ((top & 0x7FFFFFu) > 0x280000u ? 1 : 0);
  return __uint_as_float(uint32_t(127 + min(max(e, -90), 90)) << 23);
}

// ROWS: nvfp4 with a global scale for each row.  Every warp reads its whole row
// for the maximum first (the second time from L2, where the rows at hand fit
// it).  A linear layer's call, us, with one scale / with the rows' own: 1 x 5120
// -> 30720 18.6 / 22.3, 1024 x 5120 -> 10240 34.5 / 38.6, 65536 x 5120 -> 5120
// 818 / 844, 65536 x 13824 -> 5120 2237 / 2621.
template <typename T, int FMT, int ALIGN, bool ROWS>
__global__ void __launch_bounds__(kQThreads) fp4_quantize_kernel(const Fp4QuantParams p, int chunks_per_cta) {
  constexpr int kAtoms = FMT == ICSA_NVFP4 ? 4 : 2;
  release_next_grid();  // a linear layer sets itself up meanwhile
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = tile_row(blockIdx.x, warp);
  const int k_tiles = (p.K + kFp4TileK - 1) / kFp4TileK;
  const int k_end = k_tiles * kFp4TileK;
  const int row_bytes = (p.K + 31) / 32 * 16;
  uint8_t* srow = p.scales + scale_row(r, k_tiles, kAtoms);
  const T* xrow = static_cast<const T*>(p.x) + int64_t(r) * p.ldx;
  uint8_t* drow = p.data + int64_t(r) * row_bytes;
  const bool row_ok = r < p.rows;
  __shared__ float stages[ALIGN > 0 ? 1 : kQThreads / 32 * kStage];
  float* stage = stages + (ALIGN > 0 ? 0 : warp * kStage);
  const int c0 = blockIdx.y * chunks_per_cta;
  float g = p.global_scale, inv_hi = p.inv_hi, inv_lo = p.inv_lo;
  if constexpr (ROWS) {
    uint32_t top = 0u;
    if (row_ok) {
#pragma unroll 4
      for (int c = 0; c < (p.K + kQChunk - 1) / kQChunk; ++c) {
        float v[16];
        top = max(top, load16<T, ALIGN>(xrow, c * kQChunk, lane, p.K, stage, v));
      }
    }
    g = row_scale(__reduce_max_sync(0xffffffffu, top));
    if (row_ok && blockIdx.y == 0 && lane == 0) p.row_scales[r] = g;
    const float inv = __uint_as_float((254u << 23) - __float_as_uint(g));  // 1 / g, an exact factor
    inv_hi *= inv;
    inv_lo *= inv;
  }
  for (int c = c0; c < c0 + chunks_per_cta; ++c) {
    const int k0 = c * kQChunk + lane * 16;
    if (c * kQChunk >= k_end) break;
    float v[16];
    uint32_t top = 0u;
    if (row_ok) {
      top = load16<T, ALIGN>(xrow, c * kQChunk, lane, p.K, stage, v);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = 0.f;
    }
    uint32_t code[2] = {0u, 0u};
    uint32_t sbyte;
    if (FMT == ICSA_NVFP4) {
      const float amax = __uint_as_float(top);
      // (beyond 597 x 6 g the scale is 448 in any case: no product overflows)
      const float capped = fminf(amax, 3584.f * g);
      const float t = inv_hi != 0.f ? fmaf(capped, inv_hi, capped * inv_lo) : __fdiv_rn(amax, 6.0f * g);
      sbyte = top >= 0x7F800000u ? 0x7Fu : uint32_t(__nv_cvt_float_to_fp8(t, __NV_SATFINITE, __NV_E4M3));
      const float d = e4m3_float(sbyte) * g;
      if (d > 0.f && top < 0x7F800000u) quotient_codes(v, amax, d, code);
    } else {
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      // floor(log2 amax): the exponent field; subnormal magnitudes clamp to 2^-127
      const int e = min(max(int(top >> 23) - 127 - 2, -127), 127);
      sbyte = top >= 0x7F800000u ? 0xFFu : uint32_t(e + 127);
      if (top < 0x7F800000u) {
        const float inv = __uint_as_float(uint32_t(127 - e) << 23);  // 2^-e, exact products
        float q[16];
#pragma unroll
        for (int i = 0; i < 16; i += 2) attn::fmul2(q[i], q[i + 1], v[i], v[i + 1], inv, inv);
        code[0] = e2m1x8(q);
        code[1] = e2m1x8(q + 8);
      }
    }
    if (row_ok && k0 / 2 < row_bytes) *reinterpret_cast<uint2*>(drow + k0 / 2) = make_uint2(code[0], code[1]);
    // four scales to one word
    if (FMT == ICSA_NVFP4) {
      uint32_t w = sbyte << (8 * (lane & 3));
      w |= __shfl_xor_sync(0xffffffffu, w, 1);
      w |= __shfl_xor_sync(0xffffffffu, w, 2);
      if ((lane & 3) == 0 && k0 < k_end) *reinterpret_cast<uint32_t*>(srow + size_t(k0 / 64) * kScaleAtomBytes) = w;
    } else {
      uint32_t w = (lane & 1) ? 0u : sbyte << (8 * ((lane >> 1) & 3));
      w |= __shfl_xor_sync(0xffffffffu, w, 2);
      w |= __shfl_xor_sync(0xffffffffu, w, 4);
      if ((lane & 7) == 0 && k0 < k_end) *reinterpret_cast<uint32_t*>(srow + size_t(k0 / 128) * kScaleAtomBytes) = w;
    }
  }
}

template <typename T, int FMT, int ALIGN>
__global__ void __launch_bounds__(kQThreads) fp4_dequantize_kernel(const Fp4DequantParams p, int chunks_per_cta) {
  constexpr int kAtoms = FMT == ICSA_NVFP4 ? 4 : 2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = tile_row(blockIdx.x, warp);
  if (r >= p.rows) return;
  const int k_tiles = (p.K + kFp4TileK - 1) / kFp4TileK;
  const int row_bytes = (p.K + 31) / 32 * 16;
  const uint8_t* srow = p.scales + scale_row(r, k_tiles, kAtoms);
  const uint8_t* drow = p.data + int64_t(r) * row_bytes;
  T* orow = static_cast<T*>(p.out) + int64_t(r) * p.ldo;
  __shared__ float stages[ALIGN > 0 ? 1 : kQThreads / 32 * kStage];
  float* stage = stages + (ALIGN > 0 ? 0 : warp * kStage);
  const int c0 = blockIdx.y * chunks_per_cta;
  for (int c = c0; c < c0 + chunks_per_cta; ++c) {
    if (c * kQChunk >= p.K) break;
    const int k0 = min(c * kQChunk + lane * 16, (p.K - 1) & ~15);  // lanes behind the row repeat its last block
    const uint2 code = __ldg(reinterpret_cast<const uint2*>(drow + k0 / 2));
    float d;
    if (FMT == ICSA_NVFP4) {
      d = e4m3_float(__ldg(srow + size_t(k0 / 64) * kScaleAtomBytes + (k0 / 16) % 4)) * p.global_scale;
    } else {
      const uint32_t e = __ldg(srow + size_t(k0 / 128) * kScaleAtomBytes + (k0 / 32) % 4);
      // 2^(e - 127): the subnormal 2^-127 for 0, NaN for 255
      d = __uint_as_float(e == 255u ? 0x7FC00000u : e == 0u ? 0x00400000u : e << 23);
    }
    float v[16];
    float h[8];
    e2m1x8_floats(code.x, h);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = h[i] * d;
    e2m1x8_floats(code.y, h);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[8 + i] = h[i] * d;
    store16<T, ALIGN>(orow, c * kQChunk, lane, p.K, stage, v);
  }
}

// alignment of every row start: 32, 16 or 0
int row_alignment(const void* base, int64_t ld, int elem) {
  const uint64_t bits = reinterpret_cast<uintptr_t>(base) | uint64_t(ld * elem);
  return bits % 32 == 0 ? 32 : bits % 16 == 0 ? 16 : 0;
}

// CTAs cover `chunks` row chunks in grid.y; four chunks per CTA once there are
// plenty of rows, one where there are not (latency).  K = 5120, bfloat16 to
// nvfp4, one / four chunks a CTA: 64 rows 1.7 / 3.0 us, 1024 rows 5.0 / 6.1,
// 4096 rows 13.2 / 11.8, 8192 rows 25.4 / 22.4.
void quant_grid(int rows, int k_elems, dim3* grid, int* chunks_per_cta, bool row_scales = false) {
  const int row_ctas = (rows + kFp4TileRows - 1) / kFp4TileRows * 16;
  const int chunks = (k_elems + kQChunk - 1) / kQChunk;
  if (row_scales) *chunks_per_cta = row_ctas >= 512 ? chunks : std::min(chunks, 4);
  else *chunks_per_cta = row_ctas >= 512 ? std::min(chunks, 4) : 1;
  *grid = dim3(row_ctas, (chunks + *chunks_per_cta - 1) / *chunks_per_cta);
}

template <typename T, int FMT>
cudaError_t quantize_as(Fp4QuantParams p, cudaStream_t stream) {
  const float c = 6.0f * p.global_scale;
  p.inv_hi = p.inv_lo = 0.f;
  uint32_t bits;
  std::memcpy(&bits, &c, sizeof(bits));
  if (c > 0x1p-100f && c < 0x1p100f && (bits & 0xFFFFu) == 0u) {  // as in quotient_codes
    p.inv_hi = float(1.0 / double(c));
    p.inv_lo = float(1.0 / double(c) - double(p.inv_hi));
  }
  dim3 grid;
  int per;
  const int al = row_alignment(p.x, p.ldx, sizeof(T));
  if constexpr (FMT == ICSA_NVFP4) {
    if (p.row_scales != nullptr) {
      // every CTA reads whole rows first: with plenty of them it quantises
      // whole rows too, else four chunks
      quant_grid(p.rows, (p.K + kFp4TileK - 1) / kFp4TileK * kFp4TileK, &grid, &per, true);
      const auto kernel = al == 32   ? fp4_quantize_kernel<T, FMT, 32, true>
                          : al == 16 ? fp4_quantize_kernel<T, FMT, 16, true>
                                     : fp4_quantize_kernel<T, FMT, 0, true>;
      kernel<<<grid, kQThreads, 0, stream>>>(p, per);
      return cudaGetLastError();
    }
  }
  quant_grid(p.rows, (p.K + kFp4TileK - 1) / kFp4TileK * kFp4TileK, &grid, &per);
  const auto kernel = al == 32   ? fp4_quantize_kernel<T, FMT, 32, false>
                      : al == 16 ? fp4_quantize_kernel<T, FMT, 16, false>
                                 : fp4_quantize_kernel<T, FMT, 0, false>;
  kernel<<<grid, kQThreads, 0, stream>>>(p, per);
  return cudaGetLastError();
}

template <typename T, int FMT>
cudaError_t dequantize_as(const Fp4DequantParams& p, cudaStream_t stream) {
  dim3 grid;
  int per;
  quant_grid(p.rows, p.K, &grid, &per);
  const int al = row_alignment(p.out, p.ldo, sizeof(T));
  const auto kernel = al == 32   ? fp4_dequantize_kernel<T, FMT, 32>
                      : al == 16 ? fp4_dequantize_kernel<T, FMT, 16>
                                 : fp4_dequantize_kernel<T, FMT, 0>;
  kernel<<<grid, kQThreads, 0, stream>>>(p, per);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_fp4_quantize(const Fp4QuantParams& p, int x_dtype, int format, cudaStream_t stream) {
  if (x_dtype == ICSA_BF16)
    return format == ICSA_NVFP4 ? quantize_as<__nv_bfloat16, ICSA_NVFP4>(p, stream)
                                : quantize_as<__nv_bfloat16, ICSA_MXFP4>(p, stream);
  return format == ICSA_NVFP4 ? quantize_as<float, ICSA_NVFP4>(p, stream) : quantize_as<float, ICSA_MXFP4>(p, stream);
}

cudaError_t launch_fp4_dequantize(const Fp4DequantParams& p, int out_dtype, int format, cudaStream_t stream) {
  if (out_dtype == ICSA_BF16)
    return format == ICSA_NVFP4 ? dequantize_as<__nv_bfloat16, ICSA_NVFP4>(p, stream)
                                : dequantize_as<__nv_bfloat16, ICSA_MXFP4>(p, stream);
  return format == ICSA_NVFP4 ? dequantize_as<float, ICSA_NVFP4>(p, stream)
                              : dequantize_as<float, ICSA_MXFP4>(p, stream);
}

}  // namespace icsa
