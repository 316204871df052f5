// Product of two microscaled 4-bit matrices on the block-scaled tcgen05 kinds:
//
//   C[m, n] = ga gb sum_k (a[m, k] sa[m, k / B]) (b[n, k] sb[n, k / B]) (+ bias[n])
//
// kind::mxf4 (B = 32, E8M0) and kind::mxf4nvf4 (B = 16, E4M3) multiply the
// E2M1 codes with their scales inside the tensor core and accumulate in fp32,
// so no operand is ever expanded.  The 128 rows of an MMA are features (rows of
// B), its NT columns are tokens (rows of A): a single token costs an MMA of
// N = 16 instead of 128, and in the epilogue a warp holds 32 adjacent
// features of one token, which leave as one run.
//
// One CTA owns a 128 x NT tile, or with split K (few tiles) one of S K ranges
// of it; the S CTAs form a cluster, leave their partial tiles in shared memory
// and add them over distributed shared memory in rank order, so the result
// does not depend on timing and one launch does it all.
//   warp 0       TMA producer: codes of 128 features and NT tokens (256 K values
//                = 128 bytes a row, 128-byte swizzle) a stage;
//   warp 1       TMEM allocation, 4 MMAs of K = 64 a stage;
//   warps 2-9    epilogue: tcgen05.ld, factor, bias, rounding, store;
//   warps 10-13  scales: the stored order is the tensor core's, so they go by
//                cp.async into a ring and with one or two tcgen05.st a stage to
//                TMEM.  tcgen05.cp would stand in line with the MMAs (about 65
//                cycles a 512-byte tile measured, so 520 beside 256 of MMAs for
//                nvfp4), and bulk copies would cost the TMA unit as much as a
//                box of codes each (14 of 100 us at 4096 x 8192 x 8192).
// Two CTAs an SM: one alone draws 73 KB/us of operands through its ring, two
// 121, and each covers the other's start and epilogue.
//
// Few tokens are bound by the weight's bytes and the start of a launch (1 token,
// 4096 -> 11008: 8.0 us for 24 MB), many by the operands' way from L2 and then by
// power: 4096 tokens, 8192 -> 8192 138 us = 4.0 PFLOP/s in mxfp4, 160 us where the
// clock has fallen to 1.58 GHz at 986 W; 2048 tokens, 4096 -> 11008 in nvfp4 62 and
// 70 us.
#include "mxb_common.cuh"
#include "mxb_internal.h"

#include <cuda.h>

#define MXB_ERROR_WORD_BY_POINTER
#include "tc_ptx.cuh"

using namespace mxb;

namespace mxb {
namespace fp4g {

constexpr int BM = 128;       // features per tile
constexpr int BK = 256;       // K values per stage (128 bytes of codes)
constexpr int kEpiWarps = 8;
constexpr int kSfWarps = 4;
constexpr int kThreads = 64 + 32 * (kEpiWarps + kSfWarps);
constexpr int kMaxSplit = 8;  // portable cluster size

constexpr int kTileF = BM * BK / 2;  // 16 KB of feature codes

template <int FMT>
constexpr int groups() { return FMT == MXB_FP4_NV ? 4 : 2; }  // scale tiles per stage and 128 rows
template <int NT>
constexpr int tok_blocks() { return (NT + 127) / 128; }
template <int NT>
constexpr int stage_bytes() { return kTileF + NT * BK / 2; }
template <int NT>
constexpr int stages() { return NT >= 128 ? 3 : 4; }
template <int NT>
constexpr int acc_cols() { return NT < 32 ? 32 : NT; }
// scale tiles of a stage (features and tokens), their ring, and their two sets
// of TMEM columns, four a tile
template <int FMT, int NT>
constexpr int sf_tiles() { return groups<FMT>() * (1 + tok_blocks<NT>()); }
constexpr int kSfRing = 3;
template <int FMT, int NT>
constexpr int sf_cols() { return 4 * sf_tiles<FMT, NT>(); }
constexpr int pow2_cols(int c) { return c <= 64 ? 64 : c <= 128 ? 128 : c <= 256 ? 256 : 512; }
template <int FMT, int NT>
constexpr int tmem_cols() { return pow2_cols(acc_cols<NT>() + 2 * sf_cols<FMT, NT>()); }

constexpr int kBarBytes = 256;
template <int FMT, int NT>
constexpr size_t smem_bytes() {
  return 1024 + (size_t)stages<NT>() * stage_bytes<NT>() + kSfRing * sf_tiles<FMT, NT>() * 512 +
         kBarBytes;
}

struct Bars {
  uint64_t full[4];
  uint64_t empty[4];
  uint64_t sf_ready[2], sf_free[2];  // a stage's scales in TMEM
  uint64_t acc;
  uint32_t tmem_base;
};
static_assert(sizeof(Bars) <= kBarBytes, "barrier block overflows its slot");

struct Args {
  const uint8_t* fs;   // feature scales
  const uint8_t* ts;   // token scales
  const float* fg;     // nvfp4 factors
  const float* tg;
  const float* bias;
  void* out;
  int* err;
  int M, N;            // tokens, features
  int kbytes;          // row bytes of the codes (16 per 32 K values)
  int kgroups;         // scale tiles per 128 rows
  int ksteps;          // stages over the whole K
  int tok_rblocks;     // 128-row scale blocks of the tokens
  int splits;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t saddr, uint32_t rank) {
  uint32_t a;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(a));
  return v;
}

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <typename OutT>
__device__ __forceinline__ void store1(OutT* p, float v) {
  if constexpr (sizeof(OutT) == 2) *p = __float2bfloat16_rn(v);
  else *p = v;
}

template <int FMT, int NT, typename OutT>
__global__ void __launch_bounds__(kThreads, 2)
    fp4_gemm_kernel(const __grid_constant__ CUtensorMap tmap_f,
                    const __grid_constant__ CUtensorMap tmap_t, const Args a) {
  constexpr int S = stages<NT>(), G = groups<FMT>(), TB = tok_blocks<NT>();
  constexpr int kTileT = NT * BK / 2;
  constexpr int kAcc = acc_cols<NT>(), kCols = tmem_cols<FMT, NT>();
  constexpr int kSfTiles = sf_tiles<FMT, NT>(), kSfCols = sf_cols<FMT, NT>();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  // [S feature tiles][S token tiles][scale ring][barriers]
  uint8_t* sF = smem;
  uint8_t* sT = sF + S * kTileF;
  uint8_t* sS = sT + S * kTileT;
  Bars* bars = reinterpret_cast<Bars*>(sS + kSfRing * kSfTiles * 512);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = a.splits > 1 ? (int)(blockIdx.x % a.splits) : 0;
  const int n0 = (int)(blockIdx.x / a.splits) * BM;  // first feature
  const int m0 = (int)blockIdx.y * NT;               // first token
  const int per = (a.ksteps + a.splits - 1) / a.splits;
  const int k_lo = min(split * per, a.ksteps), k_hi = min(k_lo + per, a.ksteps);
  const int nk = k_hi - k_lo;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->sf_ready[i], kSfWarps);
      mbar_init(&bars->sf_free[i], 1);
    }
    mbar_init(&bars->acc, 1);
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tmap_f);
    prefetch_tmap(&tmap_t);
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = bars->tmem_base;
  pdl_trigger();
  pdl_wait();  // the setup above overlaps the end of the quantize kernel

  if (warp == 0) {
    if (lane == 0) {
      int i = 0;
      for (; i < nk; ++i) {
        const int s = i % S, round = i / S, ks = k_lo + i;
        if (round > 0 && !mbar_wait_to(&bars->empty[s], (round - 1) & 1, kErrTimeoutEmpty, a.err))
          break;
        mbar_expect_tx(&bars->full[s], kTileF + kTileT);
        tma_load_2d(sF + s * kTileF, &tmap_f, &bars->full[s], ks * (BK / 2), n0);
        tma_load_2d(sT + s * kTileT, &tmap_t, &bars->full[s], ks * (BK / 2), m0);
      }
      // the last copies land before the CTA may end, also where a wait gave up
      for (int j = max(i - S, 0); j < i; ++j)
        mbar_wait_to(&bars->full[j % S], (j / S) & 1, kErrTimeoutFull, a.err);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t i0 = make_idesc_fp4(FMT == MXB_FP4_MX, BM, NT, 0);
      constexpr uint32_t i2 = make_idesc_fp4(FMT == MXB_FP4_MX, BM, NT, 2);
      for (int i = 0; i < nk; ++i) {
        const int s = i % S, round = i / S, ks = k_lo + i;
        const uint32_t sf0 = tbase + kAcc + (i & 1) * kSfCols;
        if (!mbar_wait_to(&bars->sf_ready[i & 1], (i >> 1) & 1, kErrTimeoutTmemFull, a.err) ||
            !mbar_wait_to(&bars->full[s], round & 1, kErrTimeoutFull, a.err))
          break;
        tc_fence_after();
        const uint32_t pf = smem_u32(sF + s * kTileF), pt = smem_u32(sT + s * kTileT);
        const int ng = min(G, a.kgroups - ks * G);
        // K slices of 64 values = 32 bytes; those past the last scale tile
        // hold only padding
#pragma unroll
        for (int kk = 0; kk < BK / 64; ++kk) {
          const int g = kk * G / 4;
          if (g < ng) {
            // mxfp4: a tile of four scales serves two slices
            const uint32_t c = sf0 + g * 4 * (1 + TB);
            mma_fp4<FMT == MXB_FP4_NV>(tbase, desc_kmajor_sw128(pf + kk * 32),
                                       desc_kmajor_sw128(pt + kk * 32),
                                       (FMT == MXB_FP4_MX && (kk & 1)) ? i2 : i0, c, c + 4,
                                       (i > 0 || kk > 0) ? 1u : 0u);
          }
        }
        mma_commit(&bars->empty[s]);
        mma_commit(&bars->sf_free[i & 1]);
      }
      mma_commit(&bars->acc);  // of all that were issued, also where a wait gave up
    }
  } else if (warp >= 2 + kEpiWarps) {
    // Scales: every warp fills the lane quarter of TMEM that it may write (each
    // quarter holds all 32 rows of a scale column).
    const int t = threadIdx.x - 32 * (2 + kEpiWarps);
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const int frb = n0 >> 7, trb = m0 >> 7;
    constexpr int kChunks = kSfTiles * 32;  // 16-byte pieces of a stage
    auto fetch = [&](int i) {  // stage i -> its slot; tile order [group][features, token blocks]
      if (i < nk) {
        const int ks = k_lo + i;
        uint8_t* dst = sS + (i % kSfRing) * kSfTiles * 512;
#pragma unroll
        for (int x0 = 0; x0 < kChunks; x0 += 32 * kSfWarps) {
          const int x = x0 + t, tile = x >> 5, g = tile / (1 + TB), b = tile % (1 + TB);
          const int64_t rb = b == 0 ? frb : trb + b - 1;
          if ((kChunks % (32 * kSfWarps) == 0 || x < kChunks) && ks * G + g < a.kgroups &&
              (b == 0 || rb < a.tok_rblocks))
            cp_async16(dst + x * 16, (b == 0 ? a.fs : a.ts) +
                                         ((size_t)rb * a.kgroups + (size_t)ks * G + g) * 512 + (x & 31) * 16);
        }
      }
      cp_async_commit();
    };
    bool ok = true;
#pragma unroll
    for (int i = 0; i < kSfRing - 1; ++i) fetch(i);
    for (int i = 0; i < nk; ++i) {
      cp_async_wait<kSfRing - 2>();
      asm volatile("bar.sync 1, %0;" ::"n"(32 * kSfWarps) : "memory");
      // all warps are past stage i - 1: its slot takes stage i + kSfRing - 1
      fetch(i + kSfRing - 1);
      // after a wait that gave up the loop runs on (the block barrier above
      // needs every warp), without further waits
      if (i >= 2)
        ok = ok && mbar_wait_warp_to(&bars->sf_free[i & 1], ((i >> 1) - 1) & 1, kErrTimeoutTmemEmpty, a.err);
      tc_fence_after();
      const uint8_t* src = sS + (i % kSfRing) * kSfTiles * 512 + lane * 16;
      const uint32_t dst = tbase + kAcc + (i & 1) * kSfCols + lanes;
#pragma unroll
      for (int x = 0; x < kSfTiles; x += 4) {  // four tiles = 16 columns a store
        uint32_t r[16];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint4 v = *reinterpret_cast<const uint4*>(src + (x + k) * 512);
          r[4 * k] = v.x;
          r[4 * k + 1] = v.y;
          r[4 * k + 2] = v.z;
          r[4 * k + 3] = v.w;
        }
        tmem_st16(dst + x * 4, r);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->sf_ready[i & 1]);
    }
    cp_async_wait<0>();
  }
  __syncwarp();  // warps 0 and 1 ran on one lane

  // ── epilogue ──
  const bool epi = warp >= 2 && warp < 2 + kEpiWarps;
  const int q = warp & 3, half = (warp - 2) >> 2;  // TMEM lane quarter, column half
  constexpr int kPer = NT >= 64 ? 32 : NT / 2;     // columns per tcgen05.ld
  // the factors' product, and a power of two for where it leaves the range that
  // keeps it and its products with the sums normal (a sum of zero times an
  // infinite factor would be NaN, a subnormal one has few bits)
  float factor = 1.0f, post = 1.0f;
  if (FMT == MXB_FP4_NV) {
    const float ga = *a.fg, gb = *a.tg;
    factor = __fmul_rn(ga, gb);
    if (!(factor >= 0x1p-90f && factor <= 0x1p90f)) {
      const bool low = factor < 1.0f;
      factor = low ? __fmul_rn(__fmul_rn(fminf(ga, gb), 0x1p120f), fmaxf(ga, gb))
                   : __fmul_rn(__fmul_rn(fmaxf(ga, gb), 0x1p-120f), fminf(ga, gb));
      post = low ? 0x1p-120f : 0x1p120f;
    }
  }
  auto scaled = [&](float sum) {
    return FMT == MXB_FP4_NV ? __fmul_rn(__fmul_rn(sum, factor), post) : sum;
  };
  OutT* out = static_cast<OutT*>(a.out);
  if (a.splits == 1) {
    if (epi && mbar_wait_warp_to(&bars->acc, 0, kErrTimeoutDone, a.err)) {
      tc_fence_after();
      const int n = n0 + q * 32 + lane;
      const float bv = a.bias && n < a.N ? a.bias[n] : 0.0f;
      // a half's columns: NT / 2 of them, at least 8
#pragma unroll
      for (int cb = 0; cb < (NT >= 64 ? NT / 64 : 1); ++cb) {
        const int c0 = half * (NT / 2) + cb * kPer;
        if (m0 + c0 >= a.M) break;
        uint32_t r[32];
        tmem_ld32(tbase + ((uint32_t)(q * 32) << 16) + c0, r);
        tmem_wait_ld();
        tmem_landed(r);
        if (n < a.N) {
          OutT* o = out + (size_t)(m0 + c0) * a.N + n;
#pragma unroll
          for (int j = 0; j < kPer; ++j)
            if (m0 + c0 + j < a.M)
              store1(o + (size_t)j * a.N, __fadd_rn(scaled(__uint_as_float(r[j])), bv));
        }
      }
    }
  } else {
    // partial tile -> the idle stage buffers, [token][feature] floats
    float* part = reinterpret_cast<float*>(smem);
    if (epi && nk > 0 && mbar_wait_warp_to(&bars->acc, 0, kErrTimeoutDone, a.err)) {
      tc_fence_after();
#pragma unroll
      for (int cb = 0; cb < (NT >= 64 ? NT / 64 : 1); ++cb) {
        const int c0 = half * (NT / 2) + cb * kPer;
        if (m0 + c0 >= a.M) break;
        uint32_t r[32];
        tmem_ld32(tbase + ((uint32_t)(q * 32) << 16) + c0, r);
        tmem_wait_ld();
        tmem_landed(r);
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          part[(c0 + j) * BM + q * 32 + lane] = __uint_as_float(r[j]);
      }
    }
    cluster_sync();
    // each rank adds its share of the tokens, four features a thread
    const int toks = min(NT, a.M - m0);
    const int ranks = min(a.splits, (a.ksteps + per - 1) / per);  // ranks with K values
    const uint32_t base = smem_u32(part);
    for (int u = split * kThreads + threadIdx.x; u < toks * (BM / 4); u += a.splits * kThreads) {
      const int t = u / (BM / 4), f = (u % (BM / 4)) * 4;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int r = 0; r < ranks; ++r) {
        const float4 w = ld_cluster_f4(base + (uint32_t)(t * BM + f) * 4u, (uint32_t)r);
        v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
      }
      const float e[4] = {v.x, v.y, v.z, v.w};
      OutT* o = out + (size_t)(m0 + t) * a.N + n0 + f;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n0 + f + j < a.N)
          store1(o + j, __fadd_rn(scaled(e[j]), a.bias ? a.bias[n0 + f + j] : 0.0f));
    }
    cluster_sync();  // the partial tiles are read: the CTAs may go
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    if (nk > 0) mbar_wait_to(&bars->acc, 0, kErrTimeoutDone, a.err);
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tbase, kCols);
  }
}

template <int FMT, int NT, typename OutT>
int launch(const CUtensorMap& tf, const CUtensorMap& tt, const Args& a, cudaStream_t st) {
  auto kern = fp4_gemm_kernel<FMT, NT, OutT>;
  constexpr size_t smem = smem_bytes<FMT, NT>();
  MXB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(cdiv(a.N, BM) * a.splits), (unsigned)cdiv(a.M, NT));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)a.splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  MXB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, tf, tt, a));
  MXB_LAUNCH_CHECK();
  return MXB_OK;
}

template <int FMT, typename OutT>
int dispatch(const void* fcodes, const void* tcodes, Args& a, cudaStream_t st) {
  const int64_t ft = cdiv(a.N, BM);
  CUtensorMap tf, tt;
  auto maps = [&](int rows_f, int rows_t) {
    return encode_tmap_2d(&tf, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, fcodes, (uint64_t)a.kbytes,
                          (uint64_t)a.N, BK / 2, rows_f, CU_TENSOR_MAP_SWIZZLE_128B) &&
           encode_tmap_2d(&tt, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, tcodes, (uint64_t)a.kbytes,
                          (uint64_t)a.M, BK / 2, rows_t, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  // Tokens per tile: the smallest that holds them all, so a step of few
  // tokens pays an MMA of that width (1 x 4096 x 11008 8.0 us, 13.3 with 128
  // columns; 32 x 8192 x 8192 10.6, 12.8)
  const int nt = a.M <= 16 ? 16 : a.M <= 32 ? 32 : a.M <= 64 ? 64 : 128;
  // K splits while they fill the SMs (two CTAs each for narrow tiles; a wide
  // tile's partial sums cost more than the second CTA saves: 128 x 4096 x 4096
  // 8.1 us with 4 splits, 11.3 with 8), at least two stages each.  More splits
  // shorten the stages' time / splits and lengthen the sum, so that the best is
  // near the root of the stages: tokens x K x features 16 x 4096 x 4096 takes
  // 6.7 us with 8, 5.8 with 4 or 5, 8.7 with one; 8 x 2048 x 1000 4.1 with 4, 4.6
  // with 2, 5.3 with one.
  const int64_t tiles = ft * cdiv(a.M, nt);
  int64_t splits = (nt >= 128 ? kSMs : 2 * kSMs) / tiles;
  if (splits > a.ksteps / 2) splits = a.ksteps / 2;
  if (splits > kMaxSplit) splits = kMaxSplit;
  while (splits * splits > 2 * (int64_t)a.ksteps) --splits;
  a.splits = (int)(splits < 1 ? 1 : splits);
  if (!maps(BM, nt)) return MXB_E_CUDA;
  switch (nt) {
    case 16: return launch<FMT, 16, OutT>(tf, tt, a, st);
    case 32: return launch<FMT, 32, OutT>(tf, tt, a, st);
    case 64: return launch<FMT, 64, OutT>(tf, tt, a, st);
    default: return launch<FMT, 128, OutT>(tf, tt, a, st);
  }
}

}  // namespace fp4g
}  // namespace mxb

extern "C" int mxb_fp4_matmul(const void* a_codes, const void* a_scales, const float* a_global,
                              const void* b_codes, const void* b_scales, const float* b_global,
                              int64_t M, int64_t K, int64_t N, int fmt, const float* bias,
                              void* out, int out_dtype, void* stream) {
  if (fmt != MXB_FP4_MX && fmt != MXB_FP4_NV) return MXB_E_DTYPE;
  if (out_dtype != MXB_F32 && out_dtype != MXB_BF16) return MXB_E_DTYPE;
  if (M < 0 || N < 0 || K <= 0) return MXB_E_SHAPE;
  if (M > 65535 * 128 || N >= (int64_t)1 << 30 || K >= (int64_t)1 << 30) return MXB_E_SHAPE;
  if (M == 0 || N == 0) return MXB_OK;
  const bool nv = fmt == MXB_FP4_NV;
  if (!a_codes || !a_scales || !b_codes || !b_scales || !out || nv != (a_global != nullptr) ||
      nv != (b_global != nullptr))
    return MXB_E_ARG;
  if (((uintptr_t)a_codes | (uintptr_t)a_scales | (uintptr_t)b_codes | (uintptr_t)b_scales) % 16 ||
      (uintptr_t)out % (out_dtype == MXB_BF16 ? 2 : 4))
    return MXB_E_ALIGN;
  fp4g::Args a = {};
  a.fs = static_cast<const uint8_t*>(b_scales);
  a.ts = static_cast<const uint8_t*>(a_scales);
  a.fg = b_global;
  a.tg = a_global;
  a.bias = bias;
  a.out = out;
  a.err = device_error_ptr();
  a.M = (int)M;
  a.N = (int)N;
  a.kbytes = (int)(cdiv(K, 32) * 16);
  a.kgroups = (int)cdiv(cdiv(K, nv ? 16 : 32), 4);
  a.ksteps = (int)cdiv(K, fp4g::BK);
  a.tok_rblocks = (int)cdiv(M, 128);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (nv)
    return out_dtype == MXB_BF16
               ? fp4g::dispatch<MXB_FP4_NV, __nv_bfloat16>(b_codes, a_codes, a, st)
               : fp4g::dispatch<MXB_FP4_NV, float>(b_codes, a_codes, a, st);
  return out_dtype == MXB_BF16 ? fp4g::dispatch<MXB_FP4_MX, __nv_bfloat16>(b_codes, a_codes, a, st)
                               : fp4g::dispatch<MXB_FP4_MX, float>(b_codes, a_codes, a, st);
}
