// Linear layer on microscaled 4-bit operands for few rows (M <= 64: a
// timestep's embedding, a token, a short prompt), where the product is a read
// of the weight:
//
//   out[m, n] = bf16( act( alpha * sum_k a[m, k] w[n, k] + bias[n] ) )
//
// The operands change places: a tile is 128 weight rows (the MMA's M) by all
// rows of a (its N, 16 or 64), so a CTA's shared memory is filled with weight
// bytes, 8 or 10 K steps of 256 columns (16 KB of codes, 2 KB of scales) on
// their way at a time, and accumulators are narrow enough for two in TMEM.
//
// Work: CTAs take whole tiles where that is fast enough.  Few tiles with a
// long K are cut into equal parts, and tiles that do not divide among the SMs
// may be dealt in K steps (T = tiles x steps, CTA c of C takes steps
// [T c / C, T (c + 1) / C)).  Parts of a tile go to the workspace as float32,
// at most two for a CTA, and a second kernel adds them in the order of K.
//
// Captured calls of one row, us (whole tiles / in steps over all SMs / as
// chosen): 5120 -> 30720 (88.6 MB, 13.5 us at the copy rate) 17.7 / 19.8 /
// 17.7, 5120 -> 5120 8.7 / 9.8 / 8.7, 13824 -> 1024 18.2 / 13.4 / 8.2, 13824 ->
// 5120 18.5 / 13.1 / 11.8.  With the row's quantisation 5120 -> 30720 takes
// 21.8 us a call, against 33.2 us in the 256 x 256 tiles of icsa_fp4_gemm.cu.
// A step of one CTA takes 0.29 us (0.37 where all of them share the memory),
// so what is left is the start and the end of each CTA's stream.
//
// Roles per CTA (192 threads): warps 0-3 epilogue (thread <-> TMEM lane <->
// weight row <-> output column), warp 4 TMA producer, warp 5 TMEM allocation
// and MMA issuer.  TMEM (256 columns): accumulators [0, 64) and [64, 128),
// scale buffers from 128, 32 columns each (w at 0, a at 16).
//
// Every wait is bounded (about one second); a wait that gives up records a
// status code (report_error) and the kernel winds down.
#include "icsa_fp4_mma.cuh"

#include <algorithm>

namespace icsa {

namespace {

constexpr int kThreads = 192;
constexpr int kProducerWarp = 4;
constexpr int kMmaWarp = 5;
constexpr int kTileN = 128;                 // weight rows of a tile
constexpr int kWBytes = kTileN * 128;       // their codes of one K step
constexpr int kScaleBytes = 4 * kScaleAtomBytes;
constexpr uint32_t kTmemCols = 256;
constexpr uint32_t kTmAccStep = 64, kTmScale = 128, kTmScaleStep = 32, kTmSfb = 16;

enum : int { kErrFull = 0x411, kErrEmpty = 0x412, kErrAccFull = 0x413, kErrAccEmpty = 0x414 };

template <int MP>
constexpr int stages() {
  return (232448 - 2048) / (kWBytes + MP * 128 + 2 * kScaleBytes);
}

template <int MP>
struct __align__(1024) Smem {
  uint8_t w[stages<MP>()][kWBytes];
  uint8_t a[stages<MP>()][MP * 128];
  uint8_t sw[stages<MP>()][kScaleBytes];
  uint8_t sa[stages<MP>()][kScaleBytes];
  uint64_t full[stages<MP>()], empty[stages<MP>()];
  uint64_t acc_full[2], acc_empty[2];
  uint32_t tmem_base;
  int abort_flag;
};

// first step of CTA c
__host__ __device__ __forceinline__ int64_t first_step(int64_t total, int c, int ctas) { return total * c / ctas; }

// A CTA's share of one tile: steps [k0, k1).
struct Segment {
  int tile, k0, k1;
};
ICSA_DEV Segment segment_at(int64_t x, int64_t end, int k_steps) {
  Segment s;
  s.tile = int(x / k_steps);
  s.k0 = int(x - int64_t(s.tile) * k_steps);
  s.k1 = int(min(int64_t(k_steps), s.k0 + (end - x)));
  return s;
}

// partial sums of a CTA: [first or last tile of its range][m][128]
ICSA_DEV float* partial_tile(const Fp4GemmParams& p, int cta, bool from_start) {
  return p.partial + size_t(2 * cta + (from_start ? 1 : 0)) * p.M * kTileN;
}

template <int ATOMS>
ICSA_DEV void copy_scales_elect(uint32_t sfa, uint64_t sw_desc, uint64_t sa_desc) {
#define ICSA_CP(D, OFF_T, OFF_D)                                        \
  "add.u32 t, %0, " #OFF_T ";\n\tadd.s64 d, " D ", " #OFF_D ";\n\t" \
  "@e tcgen05.cp.cta_group::1.32x128b.warpx4 [t], d;\n\t"
  if constexpr (ATOMS == 4) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t.reg .b32 t;\n\t.reg .b64 d;\n\telect.sync _|e, 0xffffffff;\n\t"
        ICSA_CP("%1", 0, 0) ICSA_CP("%2", 16, 0) ICSA_CP("%1", 4, 32) ICSA_CP("%2", 20, 32)
        ICSA_CP("%1", 8, 64) ICSA_CP("%2", 24, 64) ICSA_CP("%1", 12, 96) ICSA_CP("%2", 28, 96)
        "}" ::"r"(sfa), "l"(sw_desc), "l"(sa_desc) : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred e;\n\t.reg .b32 t;\n\t.reg .b64 d;\n\telect.sync _|e, 0xffffffff;\n\t"
        ICSA_CP("%1", 0, 0) ICSA_CP("%2", 16, 0) ICSA_CP("%1", 4, 32) ICSA_CP("%2", 20, 32)
        "}" ::"r"(sfa), "l"(sw_desc), "l"(sa_desc) : "memory");
  }
#undef ICSA_CP
}
static_assert(kScaleAtomBytes >> 4 == 32 && kTmSfb == 16, "offsets of copy_scales_elect");

template <int FMT>
ICSA_DEV void mma_elect(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sa, uint32_t sb,
                        uint32_t accumulate) {
  if constexpr (FMT == ICSA_NVFP4) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
            d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
            d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
        : "memory");
  }
}

template <int FMT, int MP>
__global__ void __launch_bounds__(kThreads, 1)
    fp4_rows_kernel(const Fp4GemmParams p, const __grid_constant__ Fp4GemmMaps maps) {
  constexpr int kAtoms = FMT == ICSA_NVFP4 ? 4 : 2;
  constexpr int kStages = stages<MP>();
  constexpr uint32_t kBytes = kWBytes + MP * 128 + 2 * kAtoms * kScaleAtomBytes;
  extern __shared__ uint8_t smem_raw[];
  Smem<MP>& sm = *reinterpret_cast<Smem<MP>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  static_assert(sizeof(Smem<MP>) + 1024 <= 232448, "fp4 rows shared memory exceeds 227 KB");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &sm.abort_flag;
  const int64_t total = int64_t(p.n_tiles) * p.k_steps;
  // cut tiles: equal numbers of steps; whole tiles: equal numbers of tiles
  const int64_t grain = p.splits > 1 ? 1 : p.k_steps;
  const int64_t x0 = first_step(total / grain, blockIdx.x, gridDim.x) * grain;
  const int64_t x1 = first_step(total / grain, blockIdx.x + 1, gridDim.x) * grain;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.acc_full[i], 1);
      mbar_init(&sm.acc_empty[i], 4);  // one arrival per epilogue warp
    }
    sm.abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == kMmaWarp) {
    tc::tmem_alloc(&sm.tmem_base, kTmemCols);
    tc::tmem_relinquish();
  }
  if (warp == kProducerWarp && lane == 0) {
    prefetch_tensormap(&maps.a);
    prefetch_tensormap(&maps.w);
    prefetch_tensormap(&maps.sa);
    prefetch_tensormap(&maps.sw);
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = sm.tmem_base;
  const auto load_w = [&](int s, int tile, int kb) {
    mbar_arrive_expect_tx(&sm.full[s], kBytes);
    tma_load_2d(sm.w[s], &maps.w, &sm.full[s], kb * 128, tile * kTileN);
    tma_load_2d(sm.sw[s], &maps.sw, &sm.full[s], 0, (tile * p.k_steps + kb) * kAtoms);
  };
  // the weight's first stages while the kernel before quantises a
  int early = 0;
  if (p.w_ready && warp == kProducerWarp && lane == 0)
    for (; early < kStages && x0 + early < x1; ++early)
      load_w(early, int((x0 + early) / p.k_steps), int((x0 + early) % p.k_steps));
  wait_prior_grid();  // the operands are the previous kernels' outputs
  release_next_grid();
  if (warp < 4) {
    int count = 0;
    for (int64_t x = x0; x < x1; ++count) {
      const Segment g = segment_at(x, x1, p.k_steps);
      x += g.k1 - g.k0;
      const int buf = count & 1;
      const int n = g.tile * kTileN + int(threadIdx.x);
      const bool ok = attn::warp_mbar_wait(&sm.acc_full[buf], uint32_t(count >> 1) & 1u, nullptr, kErrAccFull, abort_flag);
      tc::fence_after_sync();
      const uint32_t src = tmem + uint32_t(buf) * kTmAccStep + (uint32_t(warp * 32) << 16);
      uint32_t acc[MP];
      if constexpr (MP == 16) {
        tc::tmem_ld16(src, acc);
      } else {
        tc::tmem_ld32(src, reinterpret_cast<uint32_t(&)[32]>(acc[0]));
        tc::tmem_ld32(src + 32, reinterpret_cast<uint32_t(&)[32]>(acc[32]));
      }
      tc::tmem_wait_ld();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.acc_empty[buf]);
      __syncwarp();
      if (!ok) continue;
      if (g.k0 > 0 || g.k1 < p.k_steps) {
        float* dst = partial_tile(p, blockIdx.x, g.k0 == 0) + threadIdx.x;
#pragma unroll
        for (int m = 0; m < MP; ++m)
          if (m < p.M) dst[m * kTileN] = __uint_as_float(acc[m]);
      } else if (n < p.N) {
        const float bias = p.bias != nullptr ? __bfloat162float(p.bias[n]) : 0.f;
        const auto store = [&](auto alpha) {
#pragma unroll
          for (int m = 0; m < MP; ++m)
            if (m < p.M) p.out[size_t(m) * p.ldo + n] = __float2bfloat16_rn(finish(p, __uint_as_float(acc[m]), alpha(m), bias));
        };
        // (the choice outside the loop: 64 rows x 5120 -> 13824 14.3 us, inside it 15.3)
        if (p.row_scales == nullptr) store([&](int) { return p.alpha; });
        else store([&](int m) { return row_alpha(p, m); });
      }
    }
  } else if (warp == kProducerWarp) {
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (int64_t x = x0; x < x1 && ok;) {
        const Segment g = segment_at(x, x1, p.k_steps);
        x += g.k1 - g.k0;
        for (int kb = g.k0; kb < g.k1; ++kb, ++it) {
          const int s = it % kStages;
          if (it >= early) {
            ok = mbar_wait(&sm.empty[s], (uint32_t(it / kStages) & 1u) ^ 1u, nullptr, kErrEmpty, abort_flag);
            if (!ok) break;
            load_w(s, g.tile, kb);
          }
          tma_load_2d(sm.a[s], &maps.a, &sm.full[s], kb * 128, 0);
          tma_load_2d(sm.sa[s], &maps.sa, &sm.full[s], 0, kb * kAtoms);
        }
      }
      if (sm.abort_flag)  // let every copy still in flight land before the CTA releases its memory
        for (int j = max(0, it - kStages); j < it; ++j)
          attn::drain_wait(&sm.full[j % kStages], uint32_t(j / kStages) & 1u, nullptr);
    }
  } else {
    // MMA issuer: waits are warp-uniform, one elected lane issues each instruction
    const uint64_t wd0 = tc::make_sw128_desc(smem_u32(sm.w[0]), 16, 1024);
    const uint64_t ad0 = tc::make_sw128_desc(smem_u32(sm.a[0]), 16, 1024);
    const uint64_t swd0 = scale_desc(smem_u32(sm.sw[0])), sad0 = scale_desc(smem_u32(sm.sa[0]));
    int it = 0, count = 0;
    bool ok = true;
    for (int64_t x = x0; x < x1 && ok; ++count) {
      const Segment g = segment_at(x, x1, p.k_steps);
      x += g.k1 - g.k0;
      const int buf = count & 1;
      const uint32_t acc = tmem + uint32_t(buf) * kTmAccStep;
      // the epilogue has read this accumulator's last tile
      ok = attn::warp_mbar_wait(&sm.acc_empty[buf], (uint32_t(count >> 1) & 1u) ^ 1u, nullptr, kErrAccEmpty, abort_flag);
      if (!ok) break;
      tc::fence_after_sync();
      for (int kb = g.k0; kb < g.k1; ++kb, ++it) {
        const int s = it % kStages;
        ok = attn::warp_mbar_wait(&sm.full[s], uint32_t(it / kStages) & 1u, nullptr, kErrFull, abort_flag);
        if (!ok) break;
        tc::fence_after_sync();
        const uint32_t sfw = tmem + kTmScale + uint32_t(it & 1) * kTmScaleStep, sfa = sfw + kTmSfb;
        copy_scales_elect<kAtoms>(sfw, swd0 + uint64_t(s) * (kScaleBytes >> 4), sad0 + uint64_t(s) * (kScaleBytes >> 4));
        const uint64_t wd = wd0 + uint64_t(s) * (kWBytes >> 4), ad = ad0 + uint64_t(s) * (MP * 128 >> 4);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          // nvfp4: one scale tile a step; mxfp4: two steps share a tile, bytes 0-1 and 2-3
          const uint32_t at = FMT == ICSA_NVFP4 ? ks : ks >> 1;
          const uint32_t id = FMT == ICSA_NVFP4 ? 0u : uint32_t(ks & 1) * 2u;
          mma_elect<FMT>(acc, wd + uint64_t(ks * 2), ad + uint64_t(ks * 2), make_idesc_fp4<FMT>(kTileN, MP, id),
                         sfw + 4u * at, sfa + 4u * at, (kb > g.k0 || ks > 0) ? 1u : 0u);
        }
        tc::mma_commit_elect(&sm.empty[s]);
      }
      if (ok) tc::mma_commit_elect(&sm.acc_full[buf]);
    }
  }
  __syncwarp();
  tc::fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, kTmemCols);
  }
}

// out = bf16(act(alpha * (sum of a tile's parts, in the order of K) + bias));
// blockIdx.x: tile, blockIdx.y: four rows of a
constexpr int kJoinRows = 4;
__global__ void __launch_bounds__(kTileN) fp4_rows_join_kernel(const Fp4GemmParams p, int ctas) {
  wait_prior_grid();
  const int64_t total = int64_t(p.n_tiles) * p.k_steps;
  const int64_t t0 = int64_t(blockIdx.x) * p.k_steps, t1 = t0 + p.k_steps;
  // CTA of step x: the largest c with total c / ctas < x + 1
  const int c0 = int(((t0 + 1) * ctas - 1) / total), c1 = int((t1 * ctas - 1) / total);
  const int n = blockIdx.x * kTileN + threadIdx.x;
  if (c0 == c1 || n >= p.N) return;  // one CTA wrote the tile
  const int m0 = blockIdx.y * kJoinRows;
  float acc[kJoinRows] = {}, alpha[kJoinRows];
#pragma unroll
  for (int i = 0; i < kJoinRows; ++i) alpha[i] = m0 + i < p.M ? row_alpha(p, m0 + i) : 0.f;
  constexpr int kAhead = 4;  // parts whose loads are on their way together
  for (int c = c0; c <= c1; c += kAhead) {
    float x[kAhead][kJoinRows] = {};
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (c + j > c1) break;
      const float* src = partial_tile(p, c + j, first_step(total, c + j, ctas) <= t0) + threadIdx.x;
#pragma unroll
      for (int i = 0; i < kJoinRows; ++i)
        if (m0 + i < p.M) x[j][i] = src[(m0 + i) * kTileN];
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
#pragma unroll
      for (int i = 0; i < kJoinRows; ++i) acc[i] += x[j][i];
  }
  const float bias = p.bias != nullptr ? __bfloat162float(p.bias[n]) : 0.f;
#pragma unroll
  for (int i = 0; i < kJoinRows; ++i)
    if (m0 + i < p.M) p.out[size_t(m0 + i) * p.ldo + n] = __float2bfloat16_rn(finish(p, acc[i], alpha[i], bias));
}

template <int FMT, int MP>
cudaError_t launch_as(const Fp4GemmParams& p, const Fp4GemmMaps& maps, int ctas, cudaStream_t stream) {
  const size_t smem = sizeof(Smem<MP>) + 1024;
  const auto kernel = fp4_rows_kernel<FMT, MP>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
  if (e != cudaSuccess) return e;
  return launch_chained(kernel, dim3(ctas), dim3(kThreads), smem, stream, p, maps);
}

int tiles_of(int N) { return (N + kTileN - 1) / kTileN; }

}  // namespace

Fp4RowsPlan fp4_rows_plan(int M, int N, int K, int num_sms) {
  Fp4RowsPlan r = {};
  const int64_t k_steps = (K + kFp4TileK - 1) / kFp4TileK, tiles = tiles_of(N), total = tiles * k_steps;
  // A step takes 0.29 us, 0.37 where all SMs read the weight at once; joining
  // parts 3 us and a launch, and 0.15 us for each part of a tile.
  const auto step = [&](int64_t ctas) { return std::max(0.29, 0.37 * double(ctas) / num_sms); };
  r.ctas = int(std::min<int64_t>(num_sms, tiles));
  double best = double((tiles + r.ctas - 1) / r.ctas * k_steps) * step(r.ctas);
  const auto consider = [&](int64_t ctas, int64_t steps, double parts) {
    const double us = double(steps) * step(ctas) + 4.0 + 0.15 * parts;
    if (us >= best) return;
    best = us;
    r.ctas = int(ctas);
    r.join = true;
  };
  for (int64_t parts = 2; parts <= k_steps && tiles * parts <= num_sms; ++parts)
    consider(tiles * parts, (k_steps + parts - 1) / parts, double(parts));
  if (tiles * 2 > num_sms && tiles % num_sms != 0 && total > num_sms) consider(num_sms, (total + num_sms - 1) / num_sms, 2.0);
  r.bytes = r.join ? size_t(2) * r.ctas * M * kTileN * sizeof(float) : 0;
  return r;
}

int fp4_rows_box(int M) { return M <= 16 ? 16 : kFp4MaxRows; }

cudaError_t launch_fp4_rows(Fp4GemmParams p, const Fp4GemmMaps& maps, int format, const Fp4RowsPlan& plan,
                            cudaStream_t stream) {
  p.k_steps = (p.K + kFp4TileK - 1) / kFp4TileK;
  p.n_tiles = tiles_of(p.N);
  p.splits = plan.join ? 2 : 1;
  const bool nv = format == ICSA_NVFP4;
  cudaError_t e;
  if (fp4_rows_box(p.M) == 16)
    e = nv ? launch_as<ICSA_NVFP4, 16>(p, maps, plan.ctas, stream) : launch_as<ICSA_MXFP4, 16>(p, maps, plan.ctas, stream);
  else
    e = nv ? launch_as<ICSA_NVFP4, kFp4MaxRows>(p, maps, plan.ctas, stream)
           : launch_as<ICSA_MXFP4, kFp4MaxRows>(p, maps, plan.ctas, stream);
  if (e != cudaSuccess || !plan.join) return e;
  return launch_chained(fp4_rows_join_kernel, dim3(p.n_tiles, (p.M + kJoinRows - 1) / kJoinRows), dim3(kTileN), 0, stream,
                        p, plan.ctas);
}

ICSA_DEFINE_STICKY_ACCESSOR(sticky_status_fp4_rows)

}  // namespace icsa
