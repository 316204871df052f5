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
//   warp 0     TMA producer: codes of 128 features and NT tokens (256 K values
//              = 128 bytes a row, 128-byte swizzle) and their scale tiles
//              (bulk copies; the stored order is the tensor core's) a stage;
//   warp 1     TMEM allocation; per stage copies the scale tiles to TMEM
//              (tcgen05.cp) and issues 4 MMAs of K = 64;
//   warps 2-9  epilogue: tcgen05.ld, factor, bias, rounding, store.
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
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kMaxSplit = 8;  // portable cluster size

constexpr int kTileF = BM * BK / 2;  // 16 KB of feature codes

template <int FMT>
constexpr int groups() { return FMT == MXB_FP4_NV ? 4 : 2; }  // scale tiles per stage and 128 rows
template <int NT>
constexpr int tok_blocks() { return (NT + 127) / 128; }
template <int FMT, int NT>
constexpr int stage_bytes() {
  return kTileF + (NT < 8 ? 8 : NT) * BK / 2 + (1 + tok_blocks<NT>()) * groups<FMT>() * 512;
}
template <int NT>
constexpr int stages() { return NT >= 256 ? 4 : NT >= 128 ? 5 : 6; }
template <int NT>
constexpr int acc_cols() { return NT < 32 ? 32 : NT; }
// scale columns: per group 4 for the features, 4 per 128 tokens
template <int FMT, int NT>
constexpr int sf_cols() { return groups<FMT>() * 4 * (1 + tok_blocks<NT>()); }
constexpr int pow2_cols(int c) { return c <= 64 ? 64 : c <= 128 ? 128 : c <= 256 ? 256 : 512; }
template <int FMT, int NT>
constexpr int tmem_cols() { return pow2_cols(acc_cols<NT>() + sf_cols<FMT, NT>()); }

constexpr int kBarBytes = 256;
template <int FMT, int NT>
constexpr size_t smem_bytes() {
  return 1024 + (size_t)stages<NT>() * stage_bytes<FMT, NT>() + kBarBytes;
}

struct Bars {
  uint64_t full[6];
  uint64_t empty[6];
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

template <typename OutT>
__device__ __forceinline__ void store1(OutT* p, float v) {
  if constexpr (sizeof(OutT) == 2) *p = __float2bfloat16_rn(v);
  else *p = v;
}

template <int FMT, int NT, typename OutT>
__global__ void __launch_bounds__(kThreads)
    fp4_gemm_kernel(const __grid_constant__ CUtensorMap tmap_f,
                    const __grid_constant__ CUtensorMap tmap_t, const Args a) {
  constexpr int S = stages<NT>(), G = groups<FMT>(), TB = tok_blocks<NT>();
  constexpr int kTileT = NT * BK / 2;
  constexpr int kStage = stage_bytes<FMT, NT>();
  constexpr int kAcc = acc_cols<NT>(), kCols = tmem_cols<FMT, NT>();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  // [S feature tiles][S token tiles][S scale tiles][barriers]
  uint8_t* sF = smem;
  uint8_t* sT = sF + S * kTileF;
  uint8_t* sS = sT + S * kTileT;
  Bars* bars = reinterpret_cast<Bars*>(smem + S * kStage);
  constexpr int kScaleStage = (1 + TB) * G * 512;

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
      const int frb = n0 >> 7, trb = m0 >> 7;
      for (int i = 0; i < nk; ++i) {
        const int s = i % S, round = i / S, ks = k_lo + i;
        if (round > 0 && !mbar_wait_to(&bars->empty[s], (round - 1) & 1, kErrTimeoutEmpty, a.err))
          break;
        const int ng = min(G, a.kgroups - ks * G);              // scale tiles of this stage
        const int tb = min(TB, a.tok_rblocks - trb);            // existing token scale blocks
        mbar_expect_tx(&bars->full[s], kTileF + kTileT + (uint32_t)(1 + tb) * ng * 512);
        tma_load_2d(sF + s * kTileF, &tmap_f, &bars->full[s], ks * (BK / 2), n0);
        tma_load_2d(sT + s * kTileT, &tmap_t, &bars->full[s], ks * (BK / 2), m0);
        uint8_t* sc = sS + s * kScaleStage;
        bulk_load_g2s(sc, a.fs + ((size_t)frb * a.kgroups + (size_t)ks * G) * 512, ng * 512,
                      &bars->full[s]);
        for (int b = 0; b < tb; ++b)
          bulk_load_g2s(sc + (1 + b) * G * 512,
                        a.ts + ((size_t)(trb + b) * a.kgroups + (size_t)ks * G) * 512, ng * 512,
                        &bars->full[s]);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t sf0 = tbase + kAcc;
      bool ok = true;
      for (int i = 0; i < nk; ++i) {
        const int s = i % S, round = i / S, ks = k_lo + i;
        if (!mbar_wait_to(&bars->full[s], round & 1, kErrTimeoutFull, a.err)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t sc = smem_u32(sS + s * kScaleStage);
        const uint32_t pf = smem_u32(sF + s * kTileF), pt = smem_u32(sT + s * kTileT);
        const int ng = min(G, a.kgroups - ks * G);
#pragma unroll
        for (int g = 0; g < G; ++g) {
          if (g < ng) {
            const uint32_t c = sf0 + g * 4 * (1 + TB);
            tmem_cp_32x128(c, desc_rows16(sc + g * 512));
#pragma unroll
            for (int b = 0; b < TB; ++b)
              tmem_cp_32x128(c + 4 * (1 + b), desc_rows16(sc + ((1 + b) * G + g) * 512));
          }
        }
        // K slices of 64 values = 32 bytes; those past the last scale tile
        // hold only padding
#pragma unroll
        for (int kk = 0; kk < BK / 64; ++kk) {
          const int g = kk * G / 4;
          if (g < ng) {
            const uint32_t c = sf0 + g * 4 * (1 + TB);
            // mxfp4: a tile of four scales serves two slices
            constexpr uint32_t i0 = make_idesc_fp4(FMT == MXB_FP4_MX, BM, NT, 0);
            constexpr uint32_t i2 = make_idesc_fp4(FMT == MXB_FP4_MX, BM, NT, 2);
            mma_fp4<FMT == MXB_FP4_NV>(tbase, desc_kmajor_sw128(pf + kk * 32),
                                       desc_kmajor_sw128(pt + kk * 32),
                                       (FMT == MXB_FP4_MX && (kk & 1)) ? i2 : i0, c, c + 4,
                                       (i > 0 || kk > 0) ? 1u : 0u);
          }
        }
        mma_commit(&bars->empty[s]);
      }
      if (ok) mma_commit(&bars->acc);
    }
  }

  __syncwarp();  // warps 0 and 1 ran on one lane

  // ── epilogue ──
  const bool epi = warp >= 2;
  const int q = warp & 3, half = (warp - 2) >> 2;  // TMEM lane quarter, column half
  constexpr int kPer = NT >= 64 ? 32 : NT / 2;     // columns per tcgen05.ld
  float factor = 1.0f;
  if (FMT == MXB_FP4_NV) factor = __fmul_rn(*a.fg, *a.tg);
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
              store1(o + (size_t)j * a.N, __fadd_rn(__fmul_rn(__uint_as_float(r[j]), factor), bv));
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
          store1(o + j, __fadd_rn(__fmul_rn(e[j], factor), a.bias ? a.bias[n0 + f + j] : 0.0f));
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
  // Tokens per tile: the smallest that holds them all, so a step of few
  // tokens pays an MMA of that width; from 129 tokens on 256 where that still
  // fills the SMs, else 128.
  const int64_t ft = cdiv(a.N, BM);
  int nt = a.M <= 16 ? 16 : a.M <= 32 ? 32 : a.M <= 64 ? 64 : 128;
  if (a.M > 128 && ft * cdiv(a.M, 256) >= kSMs) nt = 256;
  // K splits: while the tiles leave half of the SMs idle, at least two stages each
  const int64_t tiles = ft * cdiv(a.M, nt);
  int splits = 1;
  while (splits < kMaxSplit && tiles * splits * 2 <= kSMs && a.ksteps >= splits * 4) splits *= 2;
  a.splits = splits;
  CUtensorMap tf, tt;
  if (!encode_tmap_2d(&tf, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, fcodes, (uint64_t)a.kbytes,
                      (uint64_t)a.N, BK / 2, BM, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !encode_tmap_2d(&tt, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, tcodes, (uint64_t)a.kbytes,
                      (uint64_t)a.M, BK / 2, nt, CU_TENSOR_MAP_SWIZZLE_128B))
    return MXB_E_CUDA;
  switch (nt) {
    case 16: return launch<FMT, 16, OutT>(tf, tt, a, st);
    case 32: return launch<FMT, 32, OutT>(tf, tt, a, st);
    case 64: return launch<FMT, 64, OutT>(tf, tt, a, st);
    case 128: return launch<FMT, 128, OutT>(tf, tt, a, st);
    default: return launch<FMT, 256, OutT>(tf, tt, a, st);
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
