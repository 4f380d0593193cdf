// Linear layer on microscaled 4-bit operands, on SM pairs (tcgen05
// cta_group::2, block-scaled kinds):
//
//   out[r, c] = bf16( act( alpha * sum_k a[r, k] w[c, k] + bias[c] ) )
//
// with a and w in the storage form of icsa_lowp.cuh (e2m1 codes, e4m3 scales
// for 16 elements or e8m0 scales for 32); the tensor core multiplies codes and
// scales itself and accumulates in float32 in TMEM.  alpha is the product of
// the two global scales; act is the identity or the tanh form of GELU.
//
// Tiles: a cluster of two CTAs computes 256 x 256 outputs, each CTA 128 rows.
// A K step is 256 elements (128-byte rows, 128-byte swizzle): each CTA loads
// its 128 rows of a and 128 of the 256 weight rows (16 KB each), the scales
// of its own rows of a (2 KB nvfp4) and of all 256 weight rows (4 KB, since
// each SM scales all columns of its half of the tile).  The leader copies
// both CTAs' scales from shared memory to TMEM (tcgen05.cp, one 512-byte
// scale tile fills four columns, repeated in the four lane quadrants) and
// issues four M = 256, N = 256, K = 64 MMAs.  The scale columns are double
// buffered; copies and MMAs of one thread execute in issue order.
//
// TMEM (512 columns): accumulator [0, 256), scale buffers from 256, 48 each.
//
// Roles per CTA (320 threads): warps 0-7 epilogue (warpgroup w: columns
// [128 w, 128 w + 128), thread <-> TMEM lane <-> output row), warp 8 TMA
// producer, warp 9 TMEM allocation and, in the leader, the MMA issuer.  The
// epilogue first moves its whole 128-column row into registers, releases the
// accumulator, and then works from registers while the next tile's MMAs run.
//
// Few tiles (few rows, or few outputs): K is split over clusters, each
// writing float32 partial sums that a second kernel adds in a fixed order.
//
// 65536 x 5120 -> 13824: 1810 us (5.1 PFLOP/s; nvfp4 and mxfp4 alike), with
// GELU 1980; 18901 x 13824 -> 5120 517 us.  A K step takes about 700 clk
// against 512 of its MMAs: filling its 38 KB per SM takes about 600, and
// operands, fills and scale copies share the 128 B/clk of shared memory.
// Between tiles the accumulator is drained and refilled once, in about 3600
// clk of a K = 5120 tile's 17600.
//
// Every wait is bounded (about one second); a wait that gives up records a
// status code (report_error) and the kernel winds down.
#include "icsa_fp4_mma.cuh"
#include "icsa_pair.cuh"

#include <algorithm>
#include <utility>

namespace icsa {

namespace {

constexpr int kThreads = 320;
constexpr int kProducerWarp = 8;
constexpr int kMmaWarp = 9;
constexpr int kStages = 5;
constexpr int kRows = 128;                  // output rows per CTA
constexpr int kCols = 256;                  // output columns per pair
constexpr int kOpBytes = 128 * 128;         // 128 rows x 256 codes
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kTmScale = 256, kTmScaleStep = 48, kTmSfb = 16;  // scale buffer: a at 0, w at 16
constexpr int kGroupM = 8;                  // tile rows per raster group

enum : int { kErrFull = 0x401, kErrEmpty = 0x402, kErrAccFull = 0x403, kErrAccEmpty = 0x404 };

struct __align__(1024) Smem {
  uint8_t a[kStages][kOpBytes];
  uint8_t w[kStages][kOpBytes];
  uint8_t sa[kStages][4 * kScaleAtomBytes];
  uint8_t sw[kStages][8 * kScaleAtomBytes];
  uint8_t out[8][32 * 128];   // output box of each epilogue warp
  float bias[2][128];
  uint64_t full[kStages], empty[kStages];
  uint64_t acc_full, acc_empty;
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(Smem) + 1024 <= 232448, "fp4 gemm shared memory exceeds 227 KB");

struct Unit {
  int mt, nt, split, k0, k1;
};

// unit u: split (u / tiles) of a tile; tiles run in groups of kGroupM tile
// rows, rows fastest, so that the clusters running at one time share their
// rows of a and their columns of w in L2
ICSA_DEV Unit decode_unit(const Fp4GemmParams& p, int u) {
  const int tiles = p.m_tiles * p.n_tiles;
  Unit t;
  t.split = u / tiles;
  const int i = u - t.split * tiles;
  const int group = kGroupM * p.n_tiles;
  const int g = i / group, r = i - g * group;
  const int m0 = g * kGroupM;
  const int gm = min(kGroupM, p.m_tiles - m0);
  t.mt = m0 + r % gm;
  t.nt = r / gm;
  t.k0 = int(int64_t(p.k_steps) * t.split / p.splits);
  t.k1 = int(int64_t(p.k_steps) * (t.split + 1) / p.splits);
  return t;
}

template <int ATOMS>
ICSA_DEV void producer(const Fp4GemmParams& p, const Fp4GemmMaps& maps, Smem& sm, uint32_t rank, int* issued) {
  constexpr uint32_t kBytes = 2u * (2 * kOpBytes + 3 * ATOMS * kScaleAtomBytes);
  volatile int* abort_flag = &sm.abort_flag;
  const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;
  int it = 0;
  for (int u = cluster; u < p.units; u += clusters) {
    const Unit t = decode_unit(p, u);
    const int row0 = t.mt * (2 * kRows) + int(rank) * kRows;
    const int wrow0 = t.nt * kCols + int(rank) * kRows;
    const int sa0 = (t.mt * 2 + int(rank)) * p.k_steps * ATOMS;
    const int sw0 = t.nt * 2 * p.k_steps * ATOMS, sw1 = sw0 + p.k_steps * ATOMS;
    for (int kb = t.k0; kb < t.k1; ++kb, ++it) {
      const int s = it % kStages;
      if (!mbar_wait(&sm.empty[s], (uint32_t(it / kStages) & 1u) ^ 1u, nullptr, kErrEmpty, abort_flag)) {
        *issued = it;
        return;
      }
      if (rank == 0) mbar_arrive_expect_tx(&sm.full[s], kBytes);
      const uint32_t full = pair::mapa(&sm.full[s], 0);
      pair::tma_load_2d(sm.a[s], &maps.a, full, kb * 128, row0);
      pair::tma_load_2d(sm.w[s], &maps.w, full, kb * 128, wrow0);
      pair::tma_load_2d(sm.sa[s], &maps.sa, full, 0, sa0 + kb * ATOMS);
      pair::tma_load_2d(sm.sw[s], &maps.sw, full, 0, sw0 + kb * ATOMS);
      pair::tma_load_2d(sm.sw[s] + ATOMS * kScaleAtomBytes, &maps.sw, full, 0, sw1 + kb * ATOMS);
    }
  }
  *issued = it;
}

// The scales of one K step to TMEM, in both CTAs of the pair: a scale tile
// fills four columns (32 lanes x 16 bytes, repeated in the four lane
// quadrants); a's tiles go to sfa + 4 i, the weight's first and second 128
// rows to sfa + 16 + 8 i and + 4.  One election for all copies keeps the
// issuing warp short.
#define ICSA_CP(T, D, OFF_T, OFF_D)                                      \
  "add.u32 t, " T ", " #OFF_T ";\n\tadd.s64 d, " D ", " #OFF_D ";\n\t" \
  "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [t], d;\n\t"
template <int ATOMS>
ICSA_DEV void copy_scales_elect(uint32_t sfa, uint64_t sa_desc, uint64_t sw_desc) {
  if constexpr (ATOMS == 4) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t.reg .b32 t;\n\t.reg .b64 d;\n\telect.sync _|e, 0xffffffff;\n\t"
        ICSA_CP("%0", "%1", 0, 0) ICSA_CP("%0", "%2", 16, 0) ICSA_CP("%0", "%2", 20, 128)
        ICSA_CP("%0", "%1", 4, 32) ICSA_CP("%0", "%2", 24, 32) ICSA_CP("%0", "%2", 28, 160)
        ICSA_CP("%0", "%1", 8, 64) ICSA_CP("%0", "%2", 32, 64) ICSA_CP("%0", "%2", 36, 192)
        ICSA_CP("%0", "%1", 12, 96) ICSA_CP("%0", "%2", 40, 96) ICSA_CP("%0", "%2", 44, 224)
        "}" ::"r"(sfa), "l"(sa_desc), "l"(sw_desc) : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred e;\n\t.reg .b32 t;\n\t.reg .b64 d;\n\telect.sync _|e, 0xffffffff;\n\t"
        ICSA_CP("%0", "%1", 0, 0) ICSA_CP("%0", "%2", 16, 0) ICSA_CP("%0", "%2", 20, 64)
        ICSA_CP("%0", "%1", 4, 32) ICSA_CP("%0", "%2", 24, 32) ICSA_CP("%0", "%2", 28, 96)
        "}" ::"r"(sfa), "l"(sa_desc), "l"(sw_desc) : "memory");
  }
}
#undef ICSA_CP
static_assert(kScaleAtomBytes >> 4 == 32 && kTmSfb == 16, "offsets of copy_scales_elect");

template <int FMT>
ICSA_DEV void mma_fp4_elect(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sa,
                            uint32_t sb, uint32_t accumulate) {
  if constexpr (FMT == ICSA_NVFP4) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "@e tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
            d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "@e tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
            d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
        : "memory");
  }
}

// MMA issuer: all 32 lanes of warp 9 of the leader (waits are warp-uniform,
// one elected lane issues each instruction).
template <int FMT>
ICSA_DEV void issuer(const Fp4GemmParams& p, Smem& sm, uint32_t tmem) {
  constexpr int kAtoms = FMT == ICSA_NVFP4 ? 4 : 2;
  volatile int* abort_flag = &sm.abort_flag;
  const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;
  const uint64_t ad0 = tc::make_sw128_desc(smem_u32(sm.a[0]), 16, 1024);
  const uint64_t wd0 = tc::make_sw128_desc(smem_u32(sm.w[0]), 16, 1024);
  const uint64_t sad0 = scale_desc(smem_u32(sm.sa[0]));
  const uint64_t swd0 = scale_desc(smem_u32(sm.sw[0]));
  int it = 0, count = 0;
  for (int u = cluster; u < p.units; u += clusters, ++count) {
    const Unit t = decode_unit(p, u);
    // the epilogue has read the previous tile's accumulator
    if (!attn::warp_mbar_wait(&sm.acc_empty, (uint32_t(count) & 1u) ^ 1u, nullptr, kErrAccEmpty, abort_flag)) return;
    tc::fence_after_sync();
    for (int kb = t.k0; kb < t.k1; ++kb, ++it) {
      const int s = it % kStages;
      if (!attn::warp_mbar_wait(&sm.full[s], uint32_t(it / kStages) & 1u, nullptr, kErrFull, abort_flag)) return;
      tc::fence_after_sync();
      const uint32_t sfa = tmem + kTmScale + uint32_t(it & 1) * kTmScaleStep, sfb = sfa + kTmSfb;
      const uint64_t sad = sad0 + uint64_t(s) * (4 * kScaleAtomBytes >> 4);
      const uint64_t swd = swd0 + uint64_t(s) * (8 * kScaleAtomBytes >> 4);
      copy_scales_elect<kAtoms>(sfa, sad, swd);
      const uint64_t ad = ad0 + uint64_t(s) * (kOpBytes >> 4), wd = wd0 + uint64_t(s) * (kOpBytes >> 4);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        // nvfp4: one scale tile a step; mxfp4: two steps share a tile, bytes 0-1 and 2-3
        const int at = FMT == ICSA_NVFP4 ? ks : ks >> 1;
        const uint32_t id = FMT == ICSA_NVFP4 ? 0u : uint32_t(ks & 1) * 2u;
        mma_fp4_elect<FMT>(tmem, ad + uint64_t(ks * 2), wd + uint64_t(ks * 2), make_idesc_fp4<FMT>(256, kCols, id),
                           sfa + 4u * at, sfb + 8u * at, (kb > t.k0 || ks > 0) ? 1u : 0u);
      }
      pair::commit_both_elect(&sm.empty[s]);
    }
    pair::commit_both_elect(&sm.acc_full);
  }
}

// Epilogue warps: thread <-> TMEM lane <-> output row, warpgroup w columns
// [128 w, 128 w + 128) of the tile.  The row goes to registers in one piece,
// so the accumulator is free again after one TMEM read; the output leaves in
// 32-row x 64-column boxes staged in shared memory (one 4 KB box a warp,
// 128-byte swizzle) and written by TMA, which stores whole lines and clips
// the tile at M and N, or row by row where the output's rows are not aligned.  (Storing the rows straight from registers, 16 bytes
// a lane in 32 different lines, took 8600 clk a tile, more than half of a
// K = 5120 main loop.)
// SCALED: a's rows have their own global scales (read in the same instance by
// every call they cost 30 us of 1890 with GELU).
template <bool SCALED>
ICSA_DEV void epilogue(const Fp4GemmParams& p, const Fp4GemmMaps& maps, Smem& sm, uint32_t tmem, uint32_t rank) {
  volatile int* abort_flag = &sm.abort_flag;
  const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int w = warp >> 2;
  const uint32_t src = tmem + (uint32_t((warp & 3) * 32) << 16) + 128u * uint32_t(w);
  uint8_t* box = sm.out[warp];
  float* bias = sm.bias[w];
  const uint32_t acc_empty = pair::mapa(&sm.acc_empty, 0);
  int count = 0;
  for (int u = cluster; u < p.units; u += clusters, ++count) {
    const Unit t = decode_unit(p, u);
    const int row0 = t.mt * (2 * kRows) + int(rank) * kRows + 32 * (warp & 3);
    const int c0 = t.nt * kCols + 128 * w;
    {
      const int c = c0 + int(threadIdx.x & 127);
      const float bv = p.bias != nullptr && c < p.N ? __bfloat162float(p.bias[c]) : 0.f;
      pair::named_sync(1u + uint32_t(w), 128);  // the last tile's bias has been read
      bias[threadIdx.x & 127] = bv;
      pair::named_sync(1u + uint32_t(w), 128);
    }
    const float alpha = !SCALED ? p.alpha : row0 + lane < p.M ? row_alpha(p, row0 + lane) : 0.f;
    const bool ok = attn::warp_mbar_wait(&sm.acc_full, uint32_t(count) & 1u, nullptr, kErrAccFull, abort_flag);
    tc::fence_after_sync();
    float acc[128];
    attn::tmem_load_row128(src, acc);
    tc::fence_before_sync();
    __syncwarp();
    if (lane == 0) pair::arrive_cluster_relaxed(acc_empty);
    __syncwarp();
    if (!ok || row0 >= p.M) continue;
    if (p.splits > 1) {
      // through the box, so that a warp stores whole lines (rows straight from
      // registers, 32 lines an instruction, took 4 us a tile); n_pad is a
      // multiple of 256: whole rows of the tile are stored
      const int unit = lane & 7;
      float* dst = p.partial + (size_t(t.split) * p.M + row0) * p.n_pad + c0 + 4 * unit;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float* x = acc + 32 * q + 4 * i;
          *reinterpret_cast<float4*>(box + lane * 128 + ((uint32_t(i) ^ uint32_t(lane & 7)) << 4)) =
              make_float4(x[0], x[1], x[2], x[3]);
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = 4 * i + (lane >> 3);
          const float4 v =
              *reinterpret_cast<const float4*>(box + row * 128 + ((uint32_t(unit) ^ uint32_t(row & 7)) << 4));
          if (row0 + row < p.M) *reinterpret_cast<float4*>(dst + size_t(row) * p.n_pad + 32 * q) = v;
        }
      }
      continue;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int cols = p.N - (c0 + 64 * h);
      if (cols <= 0) break;
      // the box's previous contents have been read by their store
      if (p.tma_out && lane == 0) bulk_wait_read();
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 b0 = *reinterpret_cast<const float4*>(bias + 64 * h + 8 * i);
        const float4 b1 = *reinterpret_cast<const float4*>(bias + 64 * h + 8 * i + 4);
        const float* x = acc + 64 * h + 8 * i;
        uint4 o;
        o.x = pack_bf16x2(finish(p, x[0], alpha, b0.x), finish(p, x[1], alpha, b0.y));
        o.y = pack_bf16x2(finish(p, x[2], alpha, b0.z), finish(p, x[3], alpha, b0.w));
        o.z = pack_bf16x2(finish(p, x[4], alpha, b1.x), finish(p, x[5], alpha, b1.y));
        o.w = pack_bf16x2(finish(p, x[6], alpha, b1.z), finish(p, x[7], alpha, b1.w));
        *reinterpret_cast<uint4*>(box + lane * 128 + ((uint32_t(i) ^ uint32_t(lane & 7)) << 4)) = o;
      }
      if (p.tma_out) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&maps.out, box, c0 + 64 * h, row0);
          bulk_commit();
        }
        continue;
      }
      // an output whose rows are not 16-byte aligned: row by row, so that a
      // warp's stores still fill lines
      __syncwarp();
      const int rows = min(32, p.M - row0);
      __nv_bfloat16* dst = p.out + size_t(row0) * p.ldo + c0 + 64 * h;
#pragma unroll 4
      for (int q = 0; q < rows; ++q, dst += p.ldo) {
        const uint32_t w2 = *reinterpret_cast<const uint32_t*>(
            box + q * 128 + ((uint32_t(lane >> 2) ^ uint32_t(q & 7)) << 4) + (lane & 3) * 4);
        const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&w2);
        if (2 * lane < cols) dst[2 * lane] = v.x;
        if (2 * lane + 1 < cols) dst[2 * lane + 1] = v.y;
      }
    }
  }
  if (lane == 0) bulk_wait_read();
}

template <int FMT, bool SCALED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    fp4_gemm_kernel(const Fp4GemmParams p, const __grid_constant__ Fp4GemmMaps maps) {
  extern __shared__ uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = pair::cluster_rank();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], 1);
    }
    mbar_init(&sm.acc_full, 1);
    mbar_init(&sm.acc_empty, 16);  // one arrival per epilogue warp, both CTAs
    sm.abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == kMmaWarp) {
    pair::tmem_alloc(&sm.tmem_base, kTmemCols);
    pair::tmem_relinquish();
  }
  if (warp == kProducerWarp && lane == 0) {
    prefetch_tensormap(&maps.a);
    prefetch_tensormap(&maps.w);
    prefetch_tensormap(&maps.sa);
    prefetch_tensormap(&maps.sw);
  }
  tc::fence_before_sync();
  pair::cluster_sync();
  tc::fence_after_sync();
  const uint32_t tmem = sm.tmem_base;
  wait_prior_grid();  // the operands are the previous kernels' outputs
  if (warp < 8) {
    epilogue<SCALED>(p, maps, sm, tmem, rank);
  } else if (warp == kProducerWarp) {
    if (lane == 0) {
      int issued = 0;
      producer<FMT == ICSA_NVFP4 ? 4 : 2>(p, maps, sm, rank, &issued);
      if (sm.abort_flag && rank == 0) {
        // the leader's full barriers count the bytes of both CTAs: let every
        // copy still in flight land before either CTA releases its memory
        for (int j = max(0, issued - kStages); j < issued; ++j)
          attn::drain_wait(&sm.full[j % kStages], uint32_t(j / kStages) & 1u, nullptr);
      }
    }
  } else if (rank == 0) {
    issuer<FMT>(p, sm, tmem);
  }
  __syncwarp();
  tc::fence_before_sync();
  pair::cluster_sync();
  if (warp == kMmaWarp) {
    tc::fence_after_sync();
    pair::tmem_dealloc(tmem, kTmemCols);
  }
}

// out = bf16(act(alpha * (sum of the splits, in order) + bias)); a thread
// takes four columns of one row.
__global__ void __launch_bounds__(256) fp4_reduce_kernel(const Fp4GemmParams p) {
  const int quads = p.n_pad / 4;
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  const int r = int(i / quads), c = 4 * int(i - int64_t(r) * quads);
  wait_prior_grid();
  if (r >= p.M || c >= p.N) return;
  const float4* src = reinterpret_cast<const float4*>(p.partial + size_t(r) * p.n_pad + c);
  const size_t step = size_t(p.M) * quads;
  float4 a = *src;
#pragma unroll 4
  for (int s = 1; s < p.splits; ++s) {
    const float4 x = src[s * step];
    a.x += x.x;
    a.y += x.y;
    a.z += x.z;
    a.w += x.w;
  }
  const float v[4] = {a.x, a.y, a.z, a.w}, alpha = row_alpha(p, r);
  __nv_bfloat16* out = p.out + size_t(r) * p.ldo + c;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c + e < p.N)
      out[e] = __float2bfloat16_rn(finish(p, v[e], alpha, p.bias != nullptr ? __bfloat162float(p.bias[c + e]) : 0.f));
}

}  // namespace

int fp4_gemm_splits(int M, int N, int K, int num_sms) {
  const int64_t tiles = int64_t((M + 2 * kRows - 1) / (2 * kRows)) * ((N + kCols - 1) / kCols);
  const int k_steps = (K + kFp4TileK - 1) / kFp4TileK;
  const int clusters = std::max(1, num_sms / 2);
  if (tiles <= 0 || tiles * 2 > clusters) return 1;
  // A step takes 0.33 us; splitting costs a second kernel (2.5 us with its
  // launch) and the partial sums, written and read at 8 TB/s.  Captured calls,
  // us, one / two / three splits: 256 x 13824 -> 5120 24.9 / 19.8 / 18.3, 256 x
  // 5120 -> 5120 14.2 / 14.1 / 13.8, 1024 x 1024 -> 1024 8.4 / 9.9 / 10.4.
  const int most = int(std::min<int64_t>(clusters / tiles, k_steps));
  int best = 1;
  double best_us = k_steps * 0.33;
  for (int s = 2; s <= most; ++s) {
    const double us = (k_steps + s - 1) / s * 0.33 + 2.5 + 8.0 * s * M * double(N) / 8e6;
    if (us < best_us) {
      best_us = us;
      best = s;
    }
  }
  return best;
}

cudaError_t launch_fp4_gemm(Fp4GemmParams p, const Fp4GemmMaps& maps, int format, int num_sms, cudaStream_t stream) {
  p.m_tiles = (p.M + 2 * kRows - 1) / (2 * kRows);
  p.n_tiles = (p.N + kCols - 1) / kCols;
  p.k_steps = (p.K + kFp4TileK - 1) / kFp4TileK;
  p.units = p.m_tiles * p.n_tiles * p.splits;
  if (p.units == 0) return cudaSuccess;
  const int clusters = std::max(1, std::min(num_sms / 2, p.units));
  const size_t smem = sizeof(Smem) + 1024;
  const auto kernel = format == ICSA_MXFP4      ? fp4_gemm_kernel<ICSA_MXFP4, false>
                      : p.row_scales != nullptr ? fp4_gemm_kernel<ICSA_NVFP4, true>
                                                : fp4_gemm_kernel<ICSA_NVFP4, false>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
  if (e != cudaSuccess) return e;
  e = launch_chained(kernel, dim3(2 * clusters), dim3(kThreads), smem, stream, p, maps);
  if (e != cudaSuccess || p.splits == 1) return e;
  const int64_t threads = int64_t(p.M) * (p.n_pad / 4);
  return launch_chained(fp4_reduce_kernel, dim3(unsigned((threads + 255) / 256)), dim3(256), 0, stream, p);
}

ICSA_DEFINE_STICKY_ACCESSOR(sticky_status_fp4)

}  // namespace icsa
