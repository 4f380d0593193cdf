// What the kernels of the 4-bit linear layer share: descriptors of the
// block-scaled MMA kinds and the output function.
#pragma once

#include "icsa_attn_common.cuh"
#include "icsa_lowp.cuh"

namespace icsa {

// Descriptor of scale tiles in shared memory: 16-byte rows without swizzle,
// 8-row groups 128 bytes apart.
ICSA_DEV uint64_t scale_desc(uint32_t saddr) {
  uint64_t d = 0;
  d |= uint64_t((saddr >> 4) & 0x3FFFu);
  d |= uint64_t(1) << 16;
  d |= uint64_t(128 >> 4) << 32;
  d |= uint64_t(1) << 46;  // descriptor version for sm_100
  return d;
}

// Instruction descriptor of the block-scaled kinds with e2m1 operands.
template <int FMT>
__host__ __device__ constexpr uint32_t make_idesc_fp4(int M, int N, uint32_t scale_id) {
  return (scale_id << 4)                                  // which scale byte pair of w
         | (1u << 7)                                      // A format: e2m1
         | (1u << 10)                                     // B format: e2m1
         | (uint32_t(N >> 3) << 17)                       // N / 8
         | ((FMT == ICSA_MXFP4 ? 1u : 0u) << 23)          // scale format: e4m3 or e8m0
         | (uint32_t(M >> 4) << 24)                       // M / 16
         | (scale_id << 29);                              // which scale byte pair of a
}

// The tanh form of GELU, 0.5 x (1 + tanh u), u = sqrt(2/pi) (x + 0.044715 x^3),
// as x / (1 + 2^(-2 u log2 e)): no cancellation at negative x, two
// multi-function operations.
ICSA_DEV float gelu_tanh(float x) {
  constexpr float c1 = -2.0f * 0.7978845608028654f * 1.4426950408889634f;
  constexpr float c3 = c1 * 0.044715f;
  return __fdividef(x, 1.0f + attn::ex2(x * fmaf(c3 * x, x, c1)));
}

// both global scales of an output row
ICSA_DEV float row_alpha(const Fp4GemmParams& p, int row) {
  return p.row_scales != nullptr ? p.alpha * p.row_scales[row] : p.alpha;
}

ICSA_DEV float finish(const Fp4GemmParams& p, float acc, float alpha, float bias) {
  const float y = fmaf(acc, alpha, bias);
  return p.activation == ICSA_ACT_GELU_TANH ? gelu_tanh(y) : y;
}

}  // namespace icsa
