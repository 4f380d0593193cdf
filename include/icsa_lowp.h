/*
 * icsa_lowp.h -- C ABI of the low-precision operators of libicsa.so: linear
 * layers on microscaled 4-bit operands, and a key/value cache held in 8 bits
 * with the attention that reads it.  They serve the DiT around the in-context
 * sparse attention: its projections (the reference's nn.Linear layers,
 * model.py:128-288) and its cross-attention, whose keys and values stay the
 * same over all denoising steps (model.py:180-188).  The reference runs both
 * in bf16 only.
 *
 * Conventions as in icsa.h: plain device pointers, strides in elements,
 * asynchronous on `stream`, no allocation, an icsa_status return and
 * icsa_last_error() for the message.  Device-side timeouts of the linear
 * layer and of the attention are reported by icsa_last_status().
 */
#ifndef ICSA_LOWP_H_
#define ICSA_LOWP_H_

#include "icsa.h"

#ifdef __cplusplus
extern "C" {
#endif

/* 4-bit formats: e2m1 elements {0, .5, 1, 1.5, 2, 3, 4, 6} with
 *   ICSA_NVFP4  one e4m3 scale for 16 elements and a global float scale
 *   ICSA_MXFP4  one power-of-two scale (e8m0) for 32 elements */
enum icsa_fp4_format { ICSA_NVFP4 = 0, ICSA_MXFP4 = 1 };
enum icsa_activation { ICSA_ACT_NONE = 0, ICSA_ACT_GELU_TANH = 1 };

/*
 * Storage of a [rows, K] tensor.
 *   data:   rows of (K rounded up to 32) / 2 bytes, the even element in the
 *           low half of a byte; elements from K on are zero codes
 *   scales: tiles of 128 rows x 4 scales, 512 bytes each: the scale of row r,
 *           block c of a tile at byte (r % 32) * 16 + (r / 32) * 4 + c; the
 *           tiles of a row band run along K, bands follow each other; K is
 *           padded to 256 elements and rows to 128 with zero bytes
 * Byte counts of the two buffers (0 for invalid arguments).
 */
ICSA_API size_t icsa_fp4_data_bytes(int rows, int K);
ICSA_API size_t icsa_fp4_scale_bytes(int format, int rows, int K);

/*
 * Quantises x (ICSA_BF16 or ICSA_F32, rows ldx elements apart), block by
 * block, amax being the block's largest magnitude:
 *   ICSA_NVFP4: s = e4m3(amax / (6 global_scale)), d = s * global_scale
 *   ICSA_MXFP4: s = 2^(floor(log2 amax) - 2) (exponent in [-127, 127]), d = s;
 *               global_scale must be 1
 *   code = e2m1(x / d), magnitudes above 6 become 6; 0 where d is 0
 * All roundings are to nearest, ties to even, of float32 quotients.  A block
 * with a NaN or an infinity gets the format's NaN scale.  data must be
 * 16-byte, scales 128-byte aligned; x has any alignment (32-byte aligned rows
 * are read in one access).
 */
ICSA_API int icsa_fp4_quantize(const void* x, int x_dtype, int64_t ldx, int rows, int K, int format,
                               float global_scale, void* data, void* scales, cudaStream_t stream);

/* out[r, k] = code * d, rounded once to out_dtype; rows ldo elements apart. */
ICSA_API int icsa_fp4_dequantize(const void* data, const void* scales, int rows, int K, int format,
                                 float global_scale, void* out, int out_dtype, int64_t ldo, cudaStream_t stream);

/*
 * out[r, c] = bf16( act( sum_k a[r, k] w[c, k] + bias[c] ) ), a: [M, K],
 * w: [N, K] (nn.Linear weight) in the same 4-bit format, products and scales
 * in the tensor core, float32 accumulation, one rounding.  The product of the
 * two global scales must be in float's range.
 *   bias: bf16 [N] or NULL;  activation: enum icsa_activation
 *   out:  bf16 [M, ldo]
 *   workspace: icsa_fp4_linear_workspace_size() bytes (0: none needed), 256-byte
 *   aligned; its contents do not matter before the call and mean nothing after it
 * The workspace size is that of the current device.
 */
ICSA_API size_t icsa_fp4_linear_workspace_size(int M, int N, int K);
ICSA_API int icsa_fp4_linear(int format, const void* a_data, const void* a_scales, float a_global_scale,
                             const void* w_data, const void* w_scales, float w_global_scale, const void* bias,
                             int activation, void* out, int64_t ldo, int M, int N, int K, void* workspace,
                             size_t workspace_bytes, cudaStream_t stream);

/*
 * The same for x of ICSA_BF16 or ICSA_F32 (rows ldx elements apart), which is
 * quantised to the weight's format in the workspace first: by
 * icsa_fp4_linear_rows with global scale 1, by icsa_fp4_linear_scaled_rows with
 * a global scale for each row of x, 2^e with e the smallest with which the
 * row's largest magnitude is at most 2688 x 2^e (in [-90, 90]; 1 for a row of
 * zeros and one with a NaN or an infinity).  ICSA_NVFP4 scales end at 2^-9 and
 * 448, so with scale 1 a block below 0.0059 becomes zero, below 0.09 it loses
 * bits, and above 2688 it saturates: rows of any magnitude want their own
 * scales.  ICSA_MXFP4 scales have the range of float; there the two are one.
 */
ICSA_API size_t icsa_fp4_linear_rows_workspace_size(int format, int M, int N, int K);
ICSA_API int icsa_fp4_linear_rows(int format, const void* x, int x_dtype, int64_t ldx, const void* w_data,
                                  const void* w_scales, float w_global_scale, const void* bias, int activation,
                                  void* out, int64_t ldo, int M, int N, int K, void* workspace,
                                  size_t workspace_bytes, cudaStream_t stream);

ICSA_API size_t icsa_fp4_linear_scaled_rows_workspace_size(int format, int M, int N, int K);
ICSA_API int icsa_fp4_linear_scaled_rows(int format, const void* x, int x_dtype, int64_t ldx, const void* w_data,
                                         const void* w_scales, float w_global_scale, const void* bias, int activation,
                                         void* out, int64_t ldo, int M, int N, int K, void* workspace,
                                         size_t workspace_bytes, cudaStream_t stream);

/*
 * Key/value cache in e4m3 with one power-of-two scale for each block of 64
 * tokens and head.  nb = ceil(L / 64).
 *   k: [B, H, nb, 64, D] bytes;  v: [B, H, nb, D, 64] bytes (a block's tokens
 *   innermost);  k_scale, v_scale: float [B, H, nb]
 *   lengths: int32 [B] on the device, the valid tokens of each sequence
 *   (values are taken into [0, L]), or NULL: all L
 * All cache buffers 16-byte aligned; D 64 or 128.
 */
typedef struct icsa_kv8_cache {
  int B, H, L, D;
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  const int* lengths;
} icsa_kv8_cache;

/*
 * Fills the cache from k, v (ICSA_BF16 or ICSA_F32) [B, L, H, D] with the
 * given batch, token and head strides and contiguous features:
 *   scale = 2^e, e the smallest with amax 2^-e <= 448 over the valid tokens of
 *   the block, taken into [-96, 96]; 1 where amax is 0; NaN where a valid
 *   element is NaN or infinite
 *   code = e4m3(x 2^-e), nearest even, saturating
 * Tokens behind a length are not read and become zero codes.
 */
ICSA_API int icsa_kv8_quantize(const icsa_kv8_cache* cache, const void* k, const void* v, int dtype,
                               const int64_t k_strides[3], const int64_t v_strides[3], cudaStream_t stream);

/* k_out, v_out [B, L, H, D] contiguous: code * scale (exact in bf16), zero
 * behind a length.  Either may be NULL. */
ICSA_API int icsa_kv8_dequantize(const icsa_kv8_cache* cache, void* k_out, void* v_out, int out_dtype,
                                 cudaStream_t stream);

/*
 * out[b, i, h] = softmax(q[b, i, h] . k[b, :len, h'] / sqrt(D)) . v[b, :len, h'],
 * h' = h / (Hq / H), len = lengths[b]; zero where len is 0.  Replaces the
 * reference's flash_attention call (wanx/attention.py:18-85, with its k_lens)
 * for keys and values that are kept over many calls.  float32 scores, softmax
 * and accumulation; the probabilities p enter the second product as fp16 (off
 * by 2^-11 of themselves, below 2^-14 of the row's largest by 2^-25 of that
 * one, whatever the scales of the value blocks, as long as these lie within
 * 2^80 of each other); one rounding of the result.  Many queries over a long
 * cache run on a 16-bit copy of it in the workspace (two bytes there for each
 * byte of the cache); in that case heads whose value scales lie more than 2^22
 * apart have their probabilities in bf16 (off by 2^-8 of themselves).
 *   q: bf16 [B, Lq, Hq, D] with batch, token, head strides (multiples of 8
 *   elements, 16-byte aligned), contiguous features; Hq a multiple of H.
 *   Many queries over a long cache read q as rows: contiguous heads, tokens
 *   that do not overlap, no gaps between batch elements.  A q of other strides
 *   takes another kernel then, for which the workspace has to be of
 *   icsa_kv8_attention_strided_workspace_size() bytes (ICSA_ERR_UNSUPPORTED
 *   where it is smaller); for every other size that is the same number.
 *   out: bf16 [B, Lq, Hq, D], contiguous
 *   workspace: icsa_kv8_attention_workspace_size() bytes, 256-byte aligned;
 *   its contents do not matter before the call and mean nothing after it
 */
ICSA_API size_t icsa_kv8_attention_workspace_size(const icsa_kv8_cache* cache, int Lq, int Hq);
ICSA_API size_t icsa_kv8_attention_strided_workspace_size(const icsa_kv8_cache* cache, int Lq, int Hq);
ICSA_API int icsa_kv8_attention(const icsa_kv8_cache* cache, const void* q, const int64_t q_strides[3], void* out,
                                int Lq, int Hq, void* workspace, size_t workspace_bytes, cudaStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* ICSA_LOWP_H_ */
