// Parameter blocks and launchers of the low-precision operators: microscaled
// 4-bit quantisation and linear layers (icsa_fp4.cu, icsa_fp4_gemm.cu,
// icsa_fp4_rows.cu) and the 8-bit key/value cache with the attention that
// reads it (icsa_kv8.cu, icsa_kv8_tc.cu).
#pragma once

#include "icsa_kernels.cuh"
#include "icsa_lowp.h"

namespace icsa {

// ------------------------------------------------------ 4-bit storage form --
// Rows of K e2m1 codes, two in a byte, rows padded to 32 elements; one scale
// byte for each block of 16 (nvfp4, e4m3) or 32 (mxfp4, e8m0) elements, in
// tiles of 128 rows x 4 scales of 512 bytes: row r of a tile, scale c at
// (r % 32) * 16 + (r / 32) * 4 + c, which is the order in which the tensor
// core's scale columns are filled from shared memory.  Tiles run along K
// first; K is padded to 256 elements, rows to 128, with zero bytes.
constexpr int kFp4TileK = 256;
constexpr int kFp4TileRows = 128;
constexpr int kScaleAtomBytes = 512;

inline int64_t fp4_row_bytes(int64_t K) { return (K + 31) / 32 * 16; }
inline int fp4_block(int format) { return format == ICSA_NVFP4 ? 16 : 32; }
// scale tiles (of 4 scales) in one K tile of 256 elements
inline int fp4_atoms(int format) { return kFp4TileK / (4 * fp4_block(format)); }
inline int64_t fp4_scale_bytes(int format, int64_t rows, int64_t K) {
  return (rows + kFp4TileRows - 1) / kFp4TileRows * ((K + kFp4TileK - 1) / kFp4TileK) * fp4_atoms(format) *
         kScaleAtomBytes;
}

struct Fp4QuantParams {
  const void* x;  // [rows, ldx], K columns used
  int64_t ldx;
  int rows, K;
  float global_scale;
  uint8_t* data;
  uint8_t* scales;
  float inv_hi, inv_lo;  // 1 / (6 global_scale) as a sum of two floats (0: divide instead); set by the launcher
  float* row_scales;     // nvfp4, [rows] or nullptr: a power of two for each row in place of global_scale, written here
};
cudaError_t launch_fp4_quantize(const Fp4QuantParams& p, int x_dtype, int format, cudaStream_t stream);

struct Fp4DequantParams {
  const uint8_t* data;
  const uint8_t* scales;
  int rows, K;
  float global_scale;
  void* out;  // [rows, ldo]
  int64_t ldo;
};
cudaError_t launch_fp4_dequantize(const Fp4DequantParams& p, int out_dtype, int format, cudaStream_t stream);

// ------------------------------------------------------ 4-bit linear layer --
struct Fp4GemmMaps {
  CUtensorMap a, w;      // uint8 [rows, row bytes], box {128 bytes, 128 rows}, 128-byte swizzle
  CUtensorMap sa, sw;    // uint32 [scale tiles, 128], box {128, scale tiles of one K tile}
  CUtensorMap out;       // bf16 [M, ldo], box {64, 32}, 128-byte swizzle (when tma_out)
};
struct Fp4GemmParams {
  int M, N, K;
  float alpha;                 // product of the two global scales
  const float* row_scales;     // [M] or nullptr: a's global scales by row, on top of alpha
  const __nv_bfloat16* bias;   // [N] or nullptr
  int activation;
  __nv_bfloat16* out;          // [M, ldo]
  int64_t ldo;
  float* partial;              // [splits, M, n_pad] when splits > 1 (launch_fp4_rows: parts of tiles)
  int n_pad;
  int splits;                  // of K (launch_fp4_rows: 1 whole tiles, 2 cut ones)
  int m_tiles, n_tiles, units, k_steps;
  int tma_out;                 // the output's rows are 16-byte aligned: written by TMA (launch_fp4_gemm)
  int w_ready;                 // the kernel before this one in the stream did not write w (launch_fp4_rows)
};
// Splits of K for an M x N x K product on `num_sms` SMs (1: none).
int fp4_gemm_splits(int M, int N, int K, int num_sms);
cudaError_t launch_fp4_gemm(Fp4GemmParams p, const Fp4GemmMaps& maps, int format, int num_sms, cudaStream_t stream);
cudaError_t sticky_status_fp4(int** out);

// At most kFp4MaxRows rows: see icsa_fp4_rows.cu.  maps.a has boxes of
// fp4_rows_box(M) rows; partial: plan.bytes of workspace.
constexpr int kFp4MaxRows = 64;
struct Fp4RowsPlan {
  int ctas;
  bool join;     // tiles are cut between CTAs
  size_t bytes;
};
Fp4RowsPlan fp4_rows_plan(int M, int N, int K, int num_sms);
int fp4_rows_box(int M);
cudaError_t launch_fp4_rows(Fp4GemmParams p, const Fp4GemmMaps& maps, int format, const Fp4RowsPlan& plan,
                            cudaStream_t stream);
cudaError_t sticky_status_fp4_rows(int** out);

// ------------------------------------------------------------- 8-bit cache --
struct Kv8Cache {
  uint8_t* k;      // e4m3 [B, H, nb, 64, D]
  uint8_t* v;      // e4m3 [B, H, nb, D, 64]
  float* k_scale;  // [B, H, nb] powers of two
  float* v_scale;
  const int* lengths;  // [B] or nullptr (all L)
  int B, H, L, D, nb;
};
struct Kv8Rows {
  const void* x[2];    // k, v: [B, L, H, D], features contiguous
  int64_t sb[2], st[2], sh[2];
};
// The attention kernels hold O in units of 2^R, R a reference that follows the
// scales of the value blocks.  It stays within 2^-value_spread of the largest
// scale so far, so that O < keys x 2^8 x 448 x 2^spread stays below 2^127;
// blocks whose scale lies further below (95 binades at 16384 keys) lose bits of
// their probabilities.
__device__ __forceinline__ float value_spread(int keys) { return float(78 + __clz(keys)); }
cudaError_t launch_kv8_quantize(const Kv8Rows& x, int dtype, const Kv8Cache& c, cudaStream_t stream);
// out[i]: [B, L, H, D] contiguous of out_dtype; rows behind a length are zero
cudaError_t launch_kv8_dequantize(const Kv8Cache& c, void* const out[2], int out_dtype, cudaStream_t stream);
// The same as operands of the dense kernels: keys in bf16, the values of a head
// in f16 as 2^-R of themselves where its scales allow that exactly (R to
// v_ref[b, h]), else in bf16 (v_ref NaN).
cudaError_t launch_kv8_copy(const Kv8Cache& c, void* k, void* v, float* v_ref, cudaStream_t stream);

struct Kv8AttnParams {
  const __nv_bfloat16* q;  // [B, Lq, Hq, D]
  int64_t q_sb, q_st, q_sh;
  __nv_bfloat16* out;      // [B, Lq, Hq, D] contiguous
  int Lq, Hq, group;       // group = Hq / H
  float scale_log2;
  int splits, groups;
  float* partial;          // [rows, splits, D + 2] when splits > 1
};
struct Kv8DecodePlan {
  int splits;
  int groups;              // of 8 rows a CTA
  double us;               // estimated time
};
Kv8DecodePlan kv8_decode_plan(int B, int H, int rows, int L, int D, int num_sms);
cudaError_t launch_kv8_decode(const Kv8AttnParams& p, const Kv8Cache& c, cudaStream_t stream);

// The same for many query rows, on the tensor cores of SM pairs, for at most
// kKv8TcMaxBatch sequences.
constexpr int kKv8TcMaxBatch = 128;
struct Kv8TcParams {
  const __nv_bfloat16* q;  // [B, Lq, Hq, D]
  int64_t q_sb, q_st, q_sh;
  __nv_bfloat16* out;      // [B, Lq, Hq, D] contiguous
  int Lq, Hq, group;
  int rows;                // Lq * group query rows per cache head
  float scale_log2;
  float* partial;          // plan.bytes
  int tiles, rounds, whole;  // from the plan
  int q_tma, o_tma;          // queries loaded / output stored by TMA through the maps
};
struct Kv8TcMaps {
  CUtensorMap q;  // bf16 [B, Lq, Hq, D], box {64, group, 128 / group, 1}, 128-byte swizzle
  CUtensorMap o;  // the same of the output, box {64, group, 32 / group, 1}
};
struct Kv8TcPlan {
  int tiles, rounds;       // 256-row tiles and pairs of them per cache head
  bool whole;              // all key steps fit the ring of stages: rounds are not cut
  int clusters;
  size_t bytes;            // partial results
};
Kv8TcPlan kv8_tc_plan(const Kv8Cache& c, int rows, int num_sms);
cudaError_t launch_kv8_tc(Kv8TcParams p, const Kv8TcMaps& maps, const Kv8TcPlan& plan, const Kv8Cache& c,
                          cudaStream_t stream);
cudaError_t sticky_status_kv8_tc(int** out);

}  // namespace icsa
