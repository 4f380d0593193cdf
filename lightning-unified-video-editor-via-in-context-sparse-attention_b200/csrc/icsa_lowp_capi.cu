// C ABI of the low-precision operators (include/icsa_lowp.h): argument
// checks, workspaces, TMA descriptors and launches.
#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>

#include "icsa_lowp.cuh"

namespace {

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  icsa_set_last_error(buf);
  return code;
}

int cuda_fail(cudaError_t e, const char* where) {
  return fail(ICSA_ERR_CUDA, "%s: %s (%s)", where, cudaGetErrorName(e), cudaGetErrorString(e));
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

bool dtype_ok(int d) { return d == ICSA_BF16 || d == ICSA_F32; }

// SMs of the current device; false with the message set on failure
bool sm_count(int* sms) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) cuda_fail(e, "device query");
  return e == cudaSuccess;
}

// ------------------------------------------------------------------ 4 bits --
constexpr int kMaxRows = 1 << 27, kMaxK = 1 << 20;

int check_fp4(const char* who, int format, int rows, int K) {
  if (format != ICSA_NVFP4 && format != ICSA_MXFP4)
    return fail(ICSA_ERR_INVALID, "%s: format %d is neither ICSA_NVFP4 nor ICSA_MXFP4", who, format);
  if (rows < 0 || K < 1) return fail(ICSA_ERR_INVALID, "%s: rows=%d must not be negative, K=%d must be positive", who, rows, K);
  if (rows > kMaxRows || K > kMaxK)
    return fail(ICSA_ERR_UNSUPPORTED, "%s: rows=%d / K=%d exceed this build's limits of %d and %d", who, rows, K, kMaxRows, kMaxK);
  if (icsa::fp4_scale_bytes(format, rows, K) / icsa::kScaleAtomBytes > 0x7FFFFFFFll)
    return fail(ICSA_ERR_UNSUPPORTED, "%s: %d x %d has more scale tiles than this build's limit", who, rows, K);
  return ICSA_OK;
}

int check_global_scale(const char* who, int format, float g) {
  if (!(g > 0.f) || std::isinf(g)) return fail(ICSA_ERR_INVALID, "%s: the global scale must be positive and finite", who);
  if (format == ICSA_MXFP4 && g != 1.f) return fail(ICSA_ERR_INVALID, "%s: mxfp4 has no global scale (must be 1)", who);
  return ICSA_OK;
}

int check_fp4_buffers(const char* who, const void* data, const void* scales) {
  if (data == nullptr || scales == nullptr) return fail(ICSA_ERR_INVALID, "%s: data and scales must be non-NULL", who);
  if (!aligned(data, 16) || !aligned(scales, 128))
    return fail(ICSA_ERR_INVALID, "%s: data must be 16-byte and scales 128-byte aligned", who);
  return ICSA_OK;
}

int encode_fp4_maps(CUtensorMap* data_map, CUtensorMap* scale_map, const void* data, const void* scales, int format,
                    int rows, int K, int box_rows) {
  const uint64_t row_bytes = uint64_t(icsa::fp4_row_bytes(K));
  int rc = icsa::encode_tensor_map_2d(data_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, data, row_bytes, uint64_t(rows),
                                      row_bytes, 128, uint32_t(box_rows), CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != ICSA_OK) return rc;
  const uint64_t atoms = uint64_t(icsa::fp4_scale_bytes(format, rows, K)) / icsa::kScaleAtomBytes;
  return icsa::encode_tensor_map_2d(scale_map, CU_TENSOR_MAP_DATA_TYPE_UINT32, scales, 128, atoms,
                                    icsa::kScaleAtomBytes, 128, uint32_t(icsa::fp4_atoms(format)),
                                    CU_TENSOR_MAP_SWIZZLE_NONE);
}

int fp4_n_pad(int N) { return (N + 255) / 256 * 256; }

// How an M x N x K product runs, and its workspace.
struct LinearPlan {
  bool rows;              // launch_fp4_rows, else launch_fp4_gemm
  icsa::Fp4RowsPlan few;
  int splits;
  size_t bytes;
};
LinearPlan plan_linear(int M, int N, int K, int sms) {
  LinearPlan l = {};
  l.rows = M <= icsa::kFp4MaxRows;
  l.splits = 1;
  if (l.rows) {
    l.few = icsa::fp4_rows_plan(M, N, K, sms);
    l.bytes = align256(l.few.bytes);
  } else {
    l.splits = icsa::fp4_gemm_splits(M, N, K, sms);
    l.bytes = l.splits == 1 ? 0 : align256(size_t(l.splits) * M * fp4_n_pad(N) * sizeof(float));
  }
  return l;
}

struct Fp4Call {
  icsa::Fp4GemmMaps maps;
  icsa::Fp4GemmParams p;
  LinearPlan plan;
  int sms;
};

// Checks of a linear layer, and its launch parameters (M = 0: nothing to launch).
int prepare_linear(Fp4Call* call, int format, const void* a_data, const void* a_scales, float a_global_scale,
                   const void* w_data, const void* w_scales, float w_global_scale, const void* bias, int activation,
                   void* out, int64_t ldo, int M, int N, int K, void* workspace, size_t workspace_bytes) {
  int rc;
  std::memset(call, 0, sizeof(*call));
  icsa::Fp4GemmParams& p = call->p;
  icsa::Fp4GemmMaps& maps = call->maps;
  int& sms = call->sms;
  if ((rc = check_fp4("fp4_linear", format, M, K)) != ICSA_OK) return rc;
  if ((rc = check_fp4("fp4_linear", format, N, K)) != ICSA_OK) return rc;
  if ((rc = check_global_scale("fp4_linear", format, a_global_scale)) != ICSA_OK) return rc;
  if ((rc = check_global_scale("fp4_linear", format, w_global_scale)) != ICSA_OK) return rc;
  const float alpha = a_global_scale * w_global_scale;
  if (!std::isnormal(alpha) && (std::isinf(alpha) || double(alpha) != double(a_global_scale) * double(w_global_scale)))
    return fail(ICSA_ERR_INVALID, "fp4_linear: the product of the global scales %g and %g is out of float's range",
                double(a_global_scale), double(w_global_scale));
  if (N < 1) return fail(ICSA_ERR_INVALID, "fp4_linear: N=%d must be positive", N);
  if (activation != ICSA_ACT_NONE && activation != ICSA_ACT_GELU_TANH)
    return fail(ICSA_ERR_INVALID, "fp4_linear: unknown activation %d", activation);
  if (ldo < N) return fail(ICSA_ERR_INVALID, "fp4_linear: ldo=%lld is smaller than N=%d", (long long)ldo, N);
  const int64_t tiles = ((int64_t(M) + 255) / 256) * ((int64_t(N) + 255) / 256);
  if (tiles > 0x3FFFFFFFll) return fail(ICSA_ERR_UNSUPPORTED, "fp4_linear: M=%d x N=%d exceeds this build's limits", M, N);
  if (M == 0) return ICSA_OK;
  if ((rc = check_fp4_buffers("fp4_linear", a_data, a_scales)) != ICSA_OK) return rc;
  if ((rc = check_fp4_buffers("fp4_linear", w_data, w_scales)) != ICSA_OK) return rc;
  if (out == nullptr || !aligned(out, 2) || !aligned(bias, 2))
    return fail(ICSA_ERR_INVALID, "fp4_linear: out must be non-NULL, out and bias aligned to their elements");
  if (!sm_count(&sms)) return ICSA_ERR_CUDA;
  p.M = M; p.N = N; p.K = K;
  p.alpha = alpha;
  p.bias = static_cast<const __nv_bfloat16*>(bias);
  p.activation = activation;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.ldo = ldo;
  p.tma_out = aligned(out, 16) && ldo % 8 == 0;
  const LinearPlan& plan = call->plan = plan_linear(M, N, K, sms);
  p.splits = plan.splits;
  p.n_pad = fp4_n_pad(N);
  if (plan.bytes > 0) {
    const size_t need = plan.bytes;
    if (workspace == nullptr || workspace_bytes < need)
      return fail(ICSA_ERR_WORKSPACE, "fp4_linear: workspace of %zu bytes is smaller than the %zu bytes required",
                  workspace == nullptr ? size_t(0) : workspace_bytes, need);
    if (!aligned(workspace, 256)) return fail(ICSA_ERR_INVALID, "fp4_linear: the workspace must be 256-byte aligned");
    p.partial = static_cast<float*>(workspace);
  }
  if ((rc = encode_fp4_maps(&maps.a, &maps.sa, a_data, a_scales, format, M, K,
                            plan.rows ? icsa::fp4_rows_box(M) : 128)) != ICSA_OK) return rc;
  if ((rc = encode_fp4_maps(&maps.w, &maps.sw, w_data, w_scales, format, N, K, 128)) != ICSA_OK) return rc;
  if (p.tma_out && !plan.rows && (rc = icsa::encode_tensor_map_2d(&maps.out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, out, uint64_t(N),
                                                    uint64_t(M), uint64_t(ldo) * 2, 64, 32,
                                                    CU_TENSOR_MAP_SWIZZLE_128B)) != ICSA_OK)
    return rc;
  return ICSA_OK;
}

int launch_linear(const Fp4Call& call, int format, cudaStream_t stream) {
  if (call.p.M == 0) return ICSA_OK;
  const cudaError_t e = call.plan.rows
                            ? icsa::launch_fp4_rows(call.p, call.maps, format, call.plan.few, stream)
                            : icsa::launch_fp4_gemm(call.p, call.maps, format, call.sms, stream);
  return e == cudaSuccess ? ICSA_OK : cuda_fail(e, "fp4_linear");
}

// icsa_fp4_quantize, with the rows' own scales where row_scales is not NULL
int quantize_rows(const void* x, int x_dtype, int64_t ldx, int rows, int K, int format, float global_scale, void* data,
                  void* scales, float* row_scales, cudaStream_t stream) {
  int rc;
  if ((rc = check_fp4("fp4_quantize", format, rows, K)) != ICSA_OK) return rc;
  if ((rc = check_global_scale("fp4_quantize", format, global_scale)) != ICSA_OK) return rc;
  if (!dtype_ok(x_dtype)) return fail(ICSA_ERR_INVALID, "fp4_quantize: x_dtype must be ICSA_BF16 or ICSA_F32");
  if (ldx < K) return fail(ICSA_ERR_INVALID, "fp4_quantize: ldx=%lld is smaller than K=%d", (long long)ldx, K);
  if (rows == 0) return ICSA_OK;
  if ((rc = check_fp4_buffers("fp4_quantize", data, scales)) != ICSA_OK) return rc;
  if (x == nullptr || !aligned(x, x_dtype == ICSA_F32 ? 4 : 2))
    return fail(ICSA_ERR_INVALID, "fp4_quantize: x must be non-NULL and aligned to its elements");
  icsa::Fp4QuantParams p = {x, ldx, rows, K, global_scale, static_cast<uint8_t*>(data), static_cast<uint8_t*>(scales),
                            0.f, 0.f, row_scales};
  cudaError_t e = icsa::launch_fp4_quantize(p, x_dtype, format, stream);
  return e == cudaSuccess ? ICSA_OK : cuda_fail(e, "fp4_quantize");
}

// Bytes of the quantised rows in a linear layer's workspace: data, scales, row scales.
size_t rows_bytes(int format, int M, int K, bool scaled) {
  return align256(size_t(M) * size_t(icsa::fp4_row_bytes(K))) + align256(size_t(icsa::fp4_scale_bytes(format, M, K))) +
         (scaled ? align256(size_t(M) * sizeof(float)) : 0);
}

// A linear layer on rows that are quantised in the workspace first; `scaled`:
// with a global scale for each row (nvfp4; mxfp4's own scales have the range).
int linear_rows(const char* who, bool scaled, int format, const void* x, int x_dtype, int64_t ldx, const void* w_data,
                const void* w_scales, float w_global_scale, const void* bias, int activation, void* out, int64_t ldo,
                int M, int N, int K, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  int rc;
  if ((rc = check_fp4(who, format, M, K)) != ICSA_OK) return rc;
  const size_t data = align256(size_t(M) * size_t(icsa::fp4_row_bytes(K)));
  const size_t scales = align256(size_t(icsa::fp4_scale_bytes(format, M, K)));
  const size_t need = rows_bytes(format, M, K, scaled);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (M > 0) {
    if (workspace == nullptr || workspace_bytes < need)
      return fail(ICSA_ERR_WORKSPACE, "%s: workspace of %zu bytes is smaller than the %zu bytes that the "
                  "quantised rows take", who, workspace == nullptr ? size_t(0) : workspace_bytes, need);
    if (!aligned(workspace, 256)) return fail(ICSA_ERR_INVALID, "%s: the workspace must be 256-byte aligned", who);
  }
  // the linear layer's own checks come before anything is launched
  Fp4Call call;
  if ((rc = prepare_linear(&call, format, ws, ws + data, 1.f, w_data, w_scales, w_global_scale, bias, activation, out,
                           ldo, M, N, K, M > 0 ? ws + need : nullptr, M > 0 ? workspace_bytes - need : 0)) != ICSA_OK)
    return rc;
  float* row_scales = scaled && format == ICSA_NVFP4 && M > 0 ? reinterpret_cast<float*>(ws + data + scales) : nullptr;
  if ((rc = quantize_rows(x, x_dtype, ldx, M, K, format, 1.f, ws, ws + data, row_scales, stream)) != ICSA_OK) return rc;
  call.p.row_scales = row_scales;
  call.p.w_ready = 1;  // that kernel is an ordinary launch, behind whatever wrote the weight
  return launch_linear(call, format, stream);
}

// ------------------------------------------------------------------ 8 bits --
int check_cache(const char* who, const icsa_kv8_cache* c, icsa::Kv8Cache* out) {
  if (c == nullptr) return fail(ICSA_ERR_INVALID, "%s: the cache is NULL", who);
  if (c->B < 1 || c->H < 1 || c->L < 1)
    return fail(ICSA_ERR_INVALID, "%s: B, H, L must be positive (got %d, %d, %d)", who, c->B, c->H, c->L);
  if (c->D != 64 && c->D != 128) return fail(ICSA_ERR_UNSUPPORTED, "%s: head dim D=%d (supported: 64, 128)", who, c->D);
  const int64_t nb = (int64_t(c->L) + 63) / 64;
  if (c->L > (1 << 30) || int64_t(c->B) * c->H > 65535 || int64_t(c->B) * c->H * nb > 0x7FFFFFFFll)
    return fail(ICSA_ERR_UNSUPPORTED, "%s: B=%d, H=%d, L=%d exceed this build's limits", who, c->B, c->H, c->L);
  out->B = c->B; out->H = c->H; out->L = c->L; out->D = c->D; out->nb = int(nb);
  out->k = static_cast<uint8_t*>(c->k);
  out->v = static_cast<uint8_t*>(c->v);
  out->k_scale = c->k_scale;
  out->v_scale = c->v_scale;
  out->lengths = c->lengths;
  return ICSA_OK;
}

int check_cache_buffers(const char* who, const icsa_kv8_cache* c, bool k, bool v) {
  if ((k && (c->k == nullptr || c->k_scale == nullptr)) || (v && (c->v == nullptr || c->v_scale == nullptr)))
    return fail(ICSA_ERR_INVALID, "%s: the cache's buffers must be non-NULL", who);
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4) ||
      !aligned(c->lengths, 4))
    return fail(ICSA_ERR_INVALID, "%s: cache bytes must be 16-byte aligned, scales and lengths 4-byte", who);
  return ICSA_OK;
}

enum AttnPath { kDecode, kPairs, kDense };

struct AttnPlan {
  AttnPath path;
  int splits, groups;            // kDecode
  icsa::Kv8TcPlan tc;    // kPairs
  size_t v_offset;       // kDense: 16-bit copy of the values, behind that of the keys; then a float for each head
  size_t bytes;          // workspace
};

// Estimated times of the three ways to attend, us.
//  * The register-fed kernel (decode) reads the cache once for every 8 or 16
//    rows (kv8_decode_plan).
//  * The pair kernel deals its steps evenly to all SM pairs, 2.7 us (2.0) for
//    a step of two 256-row tiles and 1.8 us (1.65) for one; where rounds are
//    cut their parts are joined, the more the fewer rounds there are.
//  * The dense kernels run a 256-row tile per SM pair (D = 128) or SM (D = 64)
//    at a time, 0.86 / 1.87 us a step of 128 keys, in waves of about 7 us
//    beside the steps, on a 16-bit copy that is written and read (6 bytes an
//    element).  The values of a head are f16 there, scaled by one power of
//    two, and so are its probabilities; only where the head's scales do not
//    let f16 hold the values exactly both are bf16, so few rows do without.
// Constants fitted to 324 sizes (1, 8 and 2 x 40 heads, D = 64 and 128, 100 to
// 32000 keys, 16 to 4096 rows): the choice is within 1 % of the best of the
// three on average, at worst a third slower.  Measured, us, decode / pairs /
// dense, D = 128: 1 x 8 heads, 8000 keys, 64 rows 21 / 37 / 67, 512 rows 72 /
// 47 / 67, 4096 rows - / 159 / 128; 2 x 40 heads, 600 keys, 48 rows 19 / 33 /
// 33, 256 rows 82 / 40 / 33; 32000 keys, 16 rows 130 / 569 / 740, 48 rows 361 /
// 555 / 734, 128 rows 909 / 550 / 749, 1024 rows - / 1559 / 1542, 2048 rows -
// / 2799 / 2387.
constexpr int kNoCopyRows = 48, kDecodeMost = 8 * 65535;
double dense_us(const icsa::Kv8Cache& c, int Lq, int Hq, int sms) {
  const bool wide = c.D == 128;
  const int64_t tiles = int64_t(c.B) * Hq * ((Lq + 255) / 256), units = std::max(1, wide ? sms / 2 : sms);
  const int64_t steps = (int64_t(c.L) + 127) / 128, waves = (tiles + units - 1) / units;
  return waves * (steps * (wide ? 0.86 : 1.87) + 7.0) + 6.0 * c.B * c.H * double(c.L) * c.D / 5.5e6 + 8.0;
}
double pairs_us(const icsa::Kv8Cache& c, const icsa::Kv8TcPlan& t, int sms) {
  const bool wide = c.D == 128;
  const double steps = double((int64_t(c.L) + 127) / 128), clusters = std::max(1, sms / 2);
  const double two = wide ? 2.74 : 2.02, one = wide ? 1.83 : 1.65;  // a step of two tiles, of one
  const double heads = double(c.B) * c.H;
  if (t.whole) {
    const double end = 1.76;  // of a round
    const double head = (t.tiles / 2) * (steps * two + end) + (t.tiles & 1) * (steps * one + end);
    const double round = steps * (t.tiles > 1 ? two : one) + end;
    return 9.1 + std::max(heads * head / clusters, t.tiles == 1 ? round * std::ceil(heads / clusters) : round);
  }
  const double head = (t.tiles / 2) * two + (t.tiles & 1) * one;
  return 27.4 + 0.19 * std::max(1.0, clusters / (heads * t.rounds)) + heads * steps * head / clusters;
}
AttnPlan plan_attention(const icsa::Kv8Cache& c, int Lq, int Hq, int sms) {
  AttnPlan a = {};
  const int64_t rows = int64_t(Lq) * (Hq / c.H);
  a.tc = icsa::kv8_tc_plan(c, int(rows), sms);
  a.path = kPairs;
  a.bytes = align256(a.tc.bytes);
  double us = pairs_us(c, a.tc, sms);
  if (rows <= kDecodeMost) {
    const icsa::Kv8DecodePlan d = icsa::kv8_decode_plan(c.B, c.H, int(rows), c.L, c.D, sms);
    if (d.us < us) {
      us = d.us;
      a.path = kDecode;
      a.splits = d.splits;
      a.groups = d.groups;
      a.bytes = a.splits == 1 ? 0 : align256(size_t(c.B) * c.H * rows * a.splits * (c.D + 2) * sizeof(float));
    }
  }
  if (rows > kNoCopyRows && c.nb <= 16384 && dense_us(c, Lq, Hq, sms) < us) {
    a.path = kDense;
    a.v_offset = align256(size_t(c.B) * c.L * c.H * c.D * 2);
    a.bytes = 2 * a.v_offset + align256(size_t(c.B) * c.H * sizeof(float));
  }
  return a;
}

int check_queries(const char* who, const icsa::Kv8Cache& c, int Lq, int Hq) {
  if (Lq < 1 || Hq < 1 || Hq % c.H != 0)
    return fail(ICSA_ERR_INVALID, "%s: Lq=%d must be positive and Hq=%d a multiple of H=%d", who, Lq, Hq, c.H);
  if (Lq > (1 << 28) || int64_t(Lq) * Hq > 0x7FFFFF00ll)  // rows are rounded up to tiles
    return fail(ICSA_ERR_UNSUPPORTED, "%s: Lq=%d, Hq=%d exceed this build's limits", who, Lq, Hq);
  return ICSA_OK;
}

// Whether q is rows of contiguous heads, as the dense kernels read it.
bool query_rows(const icsa::Kv8Cache& c, const int64_t q_strides[3], int Lq, int Hq) {
  return q_strides[2] == c.D && q_strides[1] >= int64_t(Hq) * c.D &&
         (c.B == 1 || q_strides[0] == Lq * q_strides[1]);
}

// The dense tensor core kernels on a 16-bit copy of the cache.
int dense_attention(const icsa::Kv8Cache& c, const AttnPlan& plan, const void* q, const int64_t q_strides[3], void* out,
                    int Lq, int Hq, float scale_log2, void* workspace, cudaStream_t stream) {
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  void* const copy[2] = {ws, ws + plan.v_offset};
  float* v_ref = reinterpret_cast<float*>(ws + 2 * plan.v_offset);
  cudaError_t e = icsa::launch_kv8_copy(c, copy[0], copy[1], v_ref, stream);
  if (e != cudaSuccess) return cuda_fail(e, "kv8_attention: 16-bit copy of the cache");
  const int nbq = (Lq + icsa::kBlock - 1) / icsa::kBlock;
  icsa::AttnMaps maps;
  std::memset(&maps, 0, sizeof(maps));
  int rc;
  if ((rc = icsa::encode_rows_tensor_map(&maps.q, q, c.B, Lq, Hq, c.D, q_strides[1])) != ICSA_OK) return rc;
  if ((rc = icsa::encode_rows_tensor_map(&maps.k, copy[0], c.B, c.L, c.H, c.D, 0)) != ICSA_OK) return rc;
  if ((rc = icsa::encode_rows_tensor_map(&maps.v, copy[1], c.B, c.L, c.H, c.D, 0)) != ICSA_OK) return rc;
  if ((rc = icsa::encode_rows_tensor_map(&maps.o, out, c.B, Lq, Hq, c.D, 0)) != ICSA_OK) return rc;
  icsa::AttnParams a;
  std::memset(&a, 0, sizeof(a));
  a.B = c.B; a.S = Lq; a.H = Hq; a.NB = nbq;
  a.num_flat = nbq;
  a.flat_tiles = (nbq + 1) / 2;
  a.nkv = c.nb; a.nkv_pad = (c.nb + 127) / 128 * 128; a.tkv = c.L;
  a.scale_log2 = scale_log2;
  a.alpha_mode = ICSA_ALPHA_SCALAR;
  a.out = out; a.out_dtype = ICSA_BF16; a.out_tma = 1;
  a.kv_lens = c.lengths;
  a.kv_group = Hq / c.H;
  a.v_ref = v_ref;
  e = icsa::launch_flat_attention(a, maps, c.D, stream);
  return e == cudaSuccess ? ICSA_OK : cuda_fail(e, "kv8_attention");
}

}  // namespace

extern "C" {

size_t icsa_fp4_data_bytes(int rows, int K) {
  if (check_fp4("fp4_data_bytes", ICSA_NVFP4, rows, K) != ICSA_OK) return 0;
  return size_t(rows) * size_t(icsa::fp4_row_bytes(K));
}

size_t icsa_fp4_scale_bytes(int format, int rows, int K) {
  if (check_fp4("fp4_scale_bytes", format, rows, K) != ICSA_OK) return 0;
  return size_t(icsa::fp4_scale_bytes(format, rows, K));
}

int icsa_fp4_quantize(const void* x, int x_dtype, int64_t ldx, int rows, int K, int format, float global_scale,
                      void* data, void* scales, cudaStream_t stream) {
  return quantize_rows(x, x_dtype, ldx, rows, K, format, global_scale, data, scales, nullptr, stream);
}

int icsa_fp4_dequantize(const void* data, const void* scales, int rows, int K, int format, float global_scale,
                        void* out, int out_dtype, int64_t ldo, cudaStream_t stream) {
  int rc;
  if ((rc = check_fp4("fp4_dequantize", format, rows, K)) != ICSA_OK) return rc;
  if ((rc = check_global_scale("fp4_dequantize", format, global_scale)) != ICSA_OK) return rc;
  if (!dtype_ok(out_dtype)) return fail(ICSA_ERR_INVALID, "fp4_dequantize: out_dtype must be ICSA_BF16 or ICSA_F32");
  if (ldo < K) return fail(ICSA_ERR_INVALID, "fp4_dequantize: ldo=%lld is smaller than K=%d", (long long)ldo, K);
  if (rows == 0) return ICSA_OK;
  if ((rc = check_fp4_buffers("fp4_dequantize", data, scales)) != ICSA_OK) return rc;
  if (out == nullptr || !aligned(out, out_dtype == ICSA_F32 ? 4 : 2))
    return fail(ICSA_ERR_INVALID, "fp4_dequantize: out must be non-NULL and aligned to its elements");
  icsa::Fp4DequantParams p = {static_cast<const uint8_t*>(data), static_cast<const uint8_t*>(scales), rows, K,
                              global_scale, out, ldo};
  cudaError_t e = icsa::launch_fp4_dequantize(p, out_dtype, format, stream);
  return e == cudaSuccess ? ICSA_OK : cuda_fail(e, "fp4_dequantize");
}

size_t icsa_fp4_linear_workspace_size(int M, int N, int K) {
  int sms = 0;
  if (M < 1 || N < 1 || K < 1 || M > kMaxRows || N > kMaxRows || K > kMaxK || !sm_count(&sms)) return 0;
  return plan_linear(M, N, K, sms).bytes;
}

int icsa_fp4_linear(int format, const void* a_data, const void* a_scales, float a_global_scale, const void* w_data,
                    const void* w_scales, float w_global_scale, const void* bias, int activation, void* out,
                    int64_t ldo, int M, int N, int K, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  Fp4Call call;
  const int rc = prepare_linear(&call, format, a_data, a_scales, a_global_scale, w_data, w_scales, w_global_scale, bias,
                                activation, out, ldo, M, N, K, workspace, workspace_bytes);
  return rc != ICSA_OK ? rc : launch_linear(call, format, stream);
}

size_t icsa_fp4_linear_rows_workspace_size(int format, int M, int N, int K) {
  if (check_fp4("fp4_linear_rows_workspace_size", format, M, K) != ICSA_OK || M < 1 || N < 1) return 0;
  return rows_bytes(format, M, K, false) + icsa_fp4_linear_workspace_size(M, N, K);
}

size_t icsa_fp4_linear_scaled_rows_workspace_size(int format, int M, int N, int K) {
  if (check_fp4("fp4_linear_scaled_rows_workspace_size", format, M, K) != ICSA_OK || M < 1 || N < 1) return 0;
  return rows_bytes(format, M, K, true) + icsa_fp4_linear_workspace_size(M, N, K);
}

int icsa_fp4_linear_rows(int format, const void* x, int x_dtype, int64_t ldx, const void* w_data,
                         const void* w_scales, float w_global_scale, const void* bias, int activation, void* out,
                         int64_t ldo, int M, int N, int K, void* workspace, size_t workspace_bytes,
                         cudaStream_t stream) {
  return linear_rows("fp4_linear_rows", false, format, x, x_dtype, ldx, w_data, w_scales, w_global_scale, bias,
                     activation, out, ldo, M, N, K, workspace, workspace_bytes, stream);
}

int icsa_fp4_linear_scaled_rows(int format, const void* x, int x_dtype, int64_t ldx, const void* w_data,
                                const void* w_scales, float w_global_scale, const void* bias, int activation,
                                void* out, int64_t ldo, int M, int N, int K, void* workspace, size_t workspace_bytes,
                                cudaStream_t stream) {
  return linear_rows("fp4_linear_scaled_rows", true, format, x, x_dtype, ldx, w_data, w_scales, w_global_scale, bias,
                     activation, out, ldo, M, N, K, workspace, workspace_bytes, stream);
}

int icsa_kv8_quantize(const icsa_kv8_cache* cache, const void* k, const void* v, int dtype, const int64_t k_strides[3],
                      const int64_t v_strides[3], cudaStream_t stream) {
  icsa::Kv8Cache c;
  int rc;
  if ((rc = check_cache("kv8_quantize", cache, &c)) != ICSA_OK) return rc;
  if ((rc = check_cache_buffers("kv8_quantize", cache, true, true)) != ICSA_OK) return rc;
  if (!dtype_ok(dtype)) return fail(ICSA_ERR_INVALID, "kv8_quantize: dtype must be ICSA_BF16 or ICSA_F32");
  const uintptr_t es = dtype == ICSA_F32 ? 4 : 2;
  if (k == nullptr || v == nullptr || k_strides == nullptr || v_strides == nullptr || !aligned(k, es) || !aligned(v, es))
    return fail(ICSA_ERR_INVALID, "kv8_quantize: k, v and their strides must be non-NULL, k and v aligned to their elements");
  icsa::Kv8Rows x = {{k, v}, {k_strides[0], v_strides[0]}, {k_strides[1], v_strides[1]}, {k_strides[2], v_strides[2]}};
  for (int i = 0; i < 3; ++i)
    if (k_strides[i] < 0 || v_strides[i] < 0) return fail(ICSA_ERR_INVALID, "kv8_quantize: strides must not be negative");
  cudaError_t e = icsa::launch_kv8_quantize(x, dtype, c, stream);
  return e == cudaSuccess ? ICSA_OK : cuda_fail(e, "kv8_quantize");
}

int icsa_kv8_dequantize(const icsa_kv8_cache* cache, void* k_out, void* v_out, int out_dtype, cudaStream_t stream) {
  icsa::Kv8Cache c;
  int rc;
  if ((rc = check_cache("kv8_dequantize", cache, &c)) != ICSA_OK) return rc;
  if ((rc = check_cache_buffers("kv8_dequantize", cache, k_out != nullptr, v_out != nullptr)) != ICSA_OK) return rc;
  if (!dtype_ok(out_dtype)) return fail(ICSA_ERR_INVALID, "kv8_dequantize: out_dtype must be ICSA_BF16 or ICSA_F32");
  if (!aligned(k_out, 16) || !aligned(v_out, 16))
    return fail(ICSA_ERR_INVALID, "kv8_dequantize: outputs must be 16-byte aligned");
  if (k_out == nullptr && v_out == nullptr) return ICSA_OK;
  void* const out[2] = {k_out, v_out};
  cudaError_t e = icsa::launch_kv8_dequantize(c, out, out_dtype, stream);
  return e == cudaSuccess ? ICSA_OK : cuda_fail(e, "kv8_dequantize");
}

size_t icsa_kv8_attention_workspace_size(const icsa_kv8_cache* cache, int Lq, int Hq) {
  icsa::Kv8Cache c;
  int sms = 0;
  if (check_cache("kv8_attention_workspace_size", cache, &c) != ICSA_OK ||
      check_queries("kv8_attention_workspace_size", c, Lq, Hq) != ICSA_OK || !sm_count(&sms))
    return 0;
  return plan_attention(c, Lq, Hq, sms).bytes;
}

size_t icsa_kv8_attention_strided_workspace_size(const icsa_kv8_cache* cache, int Lq, int Hq) {
  icsa::Kv8Cache c;
  int sms = 0;
  if (check_cache("kv8_attention_strided_workspace_size", cache, &c) != ICSA_OK ||
      check_queries("kv8_attention_strided_workspace_size", c, Lq, Hq) != ICSA_OK || !sm_count(&sms))
    return 0;
  const AttnPlan plan = plan_attention(c, Lq, Hq, sms);
  return plan.path == kDense ? align256(plan.tc.bytes) : plan.bytes;
}

int icsa_kv8_attention(const icsa_kv8_cache* cache, const void* q, const int64_t q_strides[3], void* out, int Lq,
                       int Hq, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  icsa::Kv8Cache c;
  int rc;
  if ((rc = check_cache("kv8_attention", cache, &c)) != ICSA_OK) return rc;
  if ((rc = check_cache_buffers("kv8_attention", cache, true, true)) != ICSA_OK) return rc;
  if ((rc = check_queries("kv8_attention", c, Lq, Hq)) != ICSA_OK) return rc;
  if (q == nullptr || out == nullptr || q_strides == nullptr)
    return fail(ICSA_ERR_INVALID, "kv8_attention: q, its strides and out must be non-NULL");
  if (!aligned(q, 16) || !aligned(out, 16)) return fail(ICSA_ERR_INVALID, "kv8_attention: q and out must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    if (q_strides[i] < 0 || q_strides[i] % 8 != 0)
      return fail(ICSA_ERR_INVALID, "kv8_attention: strides of q must be non-negative multiples of 8 elements");
  int sms = 0;
  if (!sm_count(&sms)) return ICSA_ERR_CUDA;
  AttnPlan plan = plan_attention(c, Lq, Hq, sms);
  if (plan.path == kDense && !query_rows(c, q_strides, Lq, Hq)) {
    // the copy path reads q as rows; the pair kernel takes any strides, in its own workspace
    plan.path = kPairs;
    plan.bytes = align256(plan.tc.bytes);
    if (plan.bytes > 0 && (workspace == nullptr || workspace_bytes < plan.bytes))
      return fail(ICSA_ERR_UNSUPPORTED, "kv8_attention: %d query tokens over a long cache need contiguous heads, token "
                  "strides of at least Hq * D and a batch stride of Lq tokens, or a workspace of "
                  "icsa_kv8_attention_strided_workspace_size() = %zu bytes", Lq, plan.bytes);
  }
  if (plan.bytes > 0) {
    if (workspace == nullptr || workspace_bytes < plan.bytes)
      return fail(ICSA_ERR_WORKSPACE, "kv8_attention: workspace of %zu bytes is smaller than the %zu bytes required",
                  workspace == nullptr ? size_t(0) : workspace_bytes, plan.bytes);
    if (!aligned(workspace, 256)) return fail(ICSA_ERR_INVALID, "kv8_attention: the workspace must be 256-byte aligned");
  }
  const float scale_log2 = float(std::sqrt(1.0 / c.D) * 1.44269504);
  if (plan.path == kDecode) {
    icsa::Kv8AttnParams p;
    p.q = static_cast<const __nv_bfloat16*>(q);
    p.q_sb = q_strides[0]; p.q_st = q_strides[1]; p.q_sh = q_strides[2];
    p.out = static_cast<__nv_bfloat16*>(out);
    p.Lq = Lq; p.Hq = Hq; p.group = Hq / c.H;
    p.scale_log2 = scale_log2;
    p.splits = plan.splits;
    p.groups = plan.groups;
    p.partial = static_cast<float*>(workspace);
    cudaError_t e = icsa::launch_kv8_decode(p, c, stream);
    return e == cudaSuccess ? ICSA_OK : cuda_fail(e, "kv8_attention");
  }
  if (plan.path == kDense) return dense_attention(c, plan, q, q_strides, out, Lq, Hq, scale_log2, workspace, stream);
  icsa::Kv8TcParams p;
  std::memset(&p, 0, sizeof(p));
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_sb = q_strides[0]; p.q_st = q_strides[1]; p.q_sh = q_strides[2];
  p.out = static_cast<__nv_bfloat16*>(out);
  p.Lq = Lq; p.Hq = Hq; p.group = Hq / c.H;
  p.rows = Lq * p.group;
  p.scale_log2 = scale_log2;
  p.partial = static_cast<float*>(workspace);
  // boxes of whole tokens of a group; strides of 0 are left to the copies
  p.q_tma = 128 % p.group == 0 && (c.B == 1 || q_strides[0] > 0) && (Lq == 1 || q_strides[1] > 0) &&
            (Hq == 1 || q_strides[2] > 0);
  p.o_tma = 32 % p.group == 0;
  const auto st = [&](int i, int n) { return uint64_t(n == 1 ? 8 : q_strides[i]) * 2; };  // an axis of one has any stride
  const uint64_t row = uint64_t(Hq) * c.D * 2;
  const size_t blocks = size_t(c.H) * c.nb;  // of one sequence
  for (int b0 = 0; b0 < c.B; b0 += icsa::kKv8TcMaxBatch) {
    icsa::Kv8Cache part = c;
    part.B = std::min(c.B - b0, icsa::kKv8TcMaxBatch);
    part.k += size_t(b0) * blocks * 64 * c.D;
    part.v += size_t(b0) * blocks * 64 * c.D;
    part.k_scale += size_t(b0) * blocks;
    part.v_scale += size_t(b0) * blocks;
    if (c.lengths != nullptr) part.lengths += b0;
    icsa::Kv8TcParams pp = p;
    pp.q += int64_t(b0) * p.q_sb;
    pp.out += int64_t(b0) * Lq * Hq * c.D;
    icsa::Kv8TcMaps maps;
    std::memset(&maps, 0, sizeof(maps));
    if (p.q_tma && (rc = icsa::encode_heads_tensor_map(&maps.q, pp.q, part.B, Lq, Hq, c.D, st(0, c.B), st(1, Lq),
                                                       st(2, Hq), p.group, 128 / p.group)) != ICSA_OK)
      return rc;
    if (p.o_tma && (rc = icsa::encode_heads_tensor_map(&maps.o, pp.out, part.B, Lq, Hq, c.D, Lq * row, row,
                                                       uint64_t(c.D) * 2, p.group, 32 / p.group)) != ICSA_OK)
      return rc;
    cudaError_t e = icsa::launch_kv8_tc(pp, maps, icsa::kv8_tc_plan(part, p.rows, sms), part, stream);
    if (e != cudaSuccess) return cuda_fail(e, "kv8_attention");
  }
  return ICSA_OK;
}

}  // extern "C"
