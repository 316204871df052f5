// Product of two int8 matrices with one scale a token and one a feature:
//
//   C[m, n] = sa[m] sb[n] sum_k a[m, k] b[n, k] (+ bias[n])
//
// The sum is the tensor core's exact int32 (kind::i8), so neither the split of K
// nor the tiles change a result; the epilogue rounds fl(fl(fl(P) sa) sb) to fp32 step by
// step, the order of the framework's other integer products, then adds the bias
// (rounded to fp32 as well) and rounds to the output's type.
#include "mxb_common.cuh"
#include "mxb_internal.h"

#include <cuda.h>

#define MXB_ERROR_WORD_BY_POINTER
#include "tc_ptx.cuh"

using namespace mxb;

namespace mxb {
namespace i8g {

constexpr int BK = 128;  // K values (bytes) a stage: a 128-byte swizzled row
// |a b| <= 2^14: sums of up to this many of them fit an int32
constexpr int64_t kMaxK = 131071;

struct Args {
  const float* sf;  // feature scales, sf_step apart (0: one for all)
  const float* st;  // token scales
  const float* bias;
  void* out;
  int* err;
  int M, N;  // tokens, features
  int ksteps;
  int splits;
  int sf_step, st_step;
};

template <typename OutT>
__device__ __forceinline__ void store1(OutT* p, float v) {
  if constexpr (sizeof(OutT) == 2) *p = __float2bfloat16_rn(v);
  else *p = v;
}
// The value of a sum P under its two scales: 0 + x turns -0 into +0, as an
// accumulator that starts from 0 does.
__device__ __forceinline__ float scaled(int p, float st, float sf, float bias) {
  return __fadd_rn(__fmul_rn(__fmul_rn((float)p, st), sf), bias);
}

// ── few tokens or few tiles ─────────────────────────────────────────────────
// The 128 rows of an MMA are features, its NT columns tokens: one token costs an
// MMA of N = 16, and a warp of the epilogue holds 32 adjacent features of a token,
// which leave as one run.  One CTA owns a 128 x NT tile or, with split K, one of
// `splits` ranges of it; those CTAs form a cluster and add their partial tiles
// over distributed shared memory.  1 token, 4096 -> 11008 (45 MB): 11.4 us a call in a graph
// over the weights of ten layers = 4.0 TB/s from HBM, 8.8 over one that stays in L2; about 5
// of them are the start and the end of a launch.  77 tokens, 2000 -> 1000: 8.4 us.
//   warp 0     TMA producer;  warp 1  TMEM allocation and MMAs;
//   warps 2-9  epilogue
constexpr int BM = 128;
constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kMaxSplit = 8;  // portable cluster size
constexpr int kTileF = BM * BK;
constexpr int kBarBytes = 256;

template <int NT>
constexpr int stages() { return NT >= 128 ? 3 : NT == 64 ? 4 : 5; }
template <int NT>
constexpr int stage_bytes() { return kTileF + NT * BK; }
template <int NT>
constexpr int acc_cols() { return NT < 32 ? 32 : NT; }
template <int NT>
constexpr size_t smem_bytes() { return 1024 + (size_t)stages<NT>() * stage_bytes<NT>() + kBarBytes; }

struct Bars {
  uint64_t full[5], empty[5];
  uint64_t acc;
  uint32_t tmem_base;
};
static_assert(sizeof(Bars) <= kBarBytes, "barrier block overflows its slot");

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
__device__ __forceinline__ int4 ld_cluster_i4(uint32_t saddr, uint32_t rank) {
  uint32_t a;
  int4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a));
  return v;
}

// N columns of the accumulator.  A half of a 16- or 32-token tile is 8 or 16 columns of the
// 32 allocated: 32 at once would read past them.
template <int N>
__device__ __forceinline__ void acc_ld(uint32_t taddr, uint32_t (&r)[N]) {
  if constexpr (N == 8) tmem_ld8(taddr, r);
  else if constexpr (N == 16) tmem_ld16(taddr, r);
  else tmem_ld32(taddr, r);
  tmem_wait_ld();
  tmem_landed(r);
}

template <int NT, typename OutT>
__global__ void __launch_bounds__(kThreads, 2)
    int8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_f,
                     const __grid_constant__ CUtensorMap tmap_t, const Args a) {
  constexpr int S = stages<NT>(), kTileT = NT * BK, kAcc = acc_cols<NT>();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  // [S feature tiles][S token tiles][barriers]
  uint8_t* sF = smem;
  uint8_t* sT = sF + S * kTileF;
  Bars* bars = reinterpret_cast<Bars*>(sT + S * kTileT);

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
    tmem_alloc(&bars->tmem_base, kAcc);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = bars->tmem_base;
  pdl_trigger();
  pdl_wait();  // the setup above overlaps the end of the kernel before

  if (warp == 0) {
    if (lane == 0) {
      int i = 0;
      for (; i < nk; ++i) {
        const int s = i % S, round = i / S, ks = k_lo + i;
        if (round > 0 && !mbar_wait_to(&bars->empty[s], (round - 1) & 1, kErrTimeoutEmpty, a.err))
          break;
        mbar_expect_tx(&bars->full[s], kTileF + kTileT);
        tma_load_2d(sF + s * kTileF, &tmap_f, &bars->full[s], ks * BK, n0);
        tma_load_2d(sT + s * kTileT, &tmap_t, &bars->full[s], ks * BK, m0);
      }
      // the last copies land before the CTA may end, also where a wait gave up
      for (int j = max(i - S, 0); j < i; ++j)
        mbar_wait_to(&bars->full[j % S], (j / S) & 1, kErrTimeoutFull, a.err);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t id = make_idesc(/*S32*/ 2, /*signed*/ 1, 0, 0, BM, NT);
      for (int i = 0; i < nk; ++i) {
        const int s = i % S, round = i / S;
        if (!mbar_wait_to(&bars->full[s], round & 1, kErrTimeoutFull, a.err)) break;
        tc_fence_after();
        const uint32_t pf = smem_u32(sF + s * kTileF), pt = smem_u32(sT + s * kTileT);
#pragma unroll
        for (int kk = 0; kk < BK / 32; ++kk)
          mma_i8(tbase, desc_kmajor_sw128(pf + kk * 32), desc_kmajor_sw128(pt + kk * 32), id,
                 (i > 0 || kk > 0) ? 1u : 0u);
        mma_commit(&bars->empty[s]);
      }
      mma_commit(&bars->acc);  // of all that were issued, also where a wait gave up
    }
  }
  __syncwarp();  // warps 0 and 1 ran on one lane

  // ── epilogue ──
  const bool epi = warp >= 2;
  const int q = warp & 3, half = (warp - 2) >> 2;  // TMEM lane quarter, column half
  constexpr int kPer = NT >= 64 ? 32 : NT / 2;     // columns per tcgen05.ld
  constexpr int kLoads = NT >= 64 ? NT / 64 : 1;   // of them a half
  static_assert(NT / 2 + kLoads * kPer <= kAcc, "columns outside the allocation");
  OutT* out = static_cast<OutT*>(a.out);
  if (a.splits == 1) {
    if (epi && mbar_wait_warp_to(&bars->acc, 0, kErrTimeoutDone, a.err)) {
      tc_fence_after();
      const int n = n0 + q * 32 + lane;
      const float sf = n < a.N ? a.sf[(int64_t)n * a.sf_step] : 0.0f;
      const float bv = a.bias && n < a.N ? a.bias[n] : 0.0f;
#pragma unroll
      for (int cb = 0; cb < kLoads; ++cb) {
        const int c0 = half * (NT / 2) + cb * kPer;
        if (m0 + c0 >= a.M) break;
        uint32_t r[kPer];
        acc_ld(tbase + ((uint32_t)(q * 32) << 16) + c0, r);
        if (n < a.N) {
          OutT* o = out + (size_t)(m0 + c0) * a.N + n;
          const float* st = a.st + (int64_t)(m0 + c0) * a.st_step;
#pragma unroll
          for (int j = 0; j < kPer; ++j)
            if (m0 + c0 + j < a.M)
              store1(o + (size_t)j * a.N, scaled((int)r[j], __ldg(st + j * a.st_step), sf, bv));
        }
      }
    }
  } else {
    // partial tile -> the idle stage buffers, [token][feature]
    int* part = reinterpret_cast<int*>(smem);
    if (epi && nk > 0 && mbar_wait_warp_to(&bars->acc, 0, kErrTimeoutDone, a.err)) {
      tc_fence_after();
#pragma unroll
      for (int cb = 0; cb < kLoads; ++cb) {
        const int c0 = half * (NT / 2) + cb * kPer;
        if (m0 + c0 >= a.M) break;
        uint32_t r[kPer];
        acc_ld(tbase + ((uint32_t)(q * 32) << 16) + c0, r);
#pragma unroll
        for (int j = 0; j < kPer; ++j) part[(c0 + j) * BM + q * 32 + lane] = (int)r[j];
      }
    }
    cluster_sync();
    // each rank adds its share of the tokens, four features a thread
    const int toks = min(NT, a.M - m0);
    const int ranks = min(a.splits, (a.ksteps + per - 1) / per);  // ranks with K values
    const uint32_t base = smem_u32(part);
    for (int u = split * kThreads + threadIdx.x; u < toks * (BM / 4); u += a.splits * kThreads) {
      const int t = u / (BM / 4), f = (u % (BM / 4)) * 4;
      int e[4] = {0, 0, 0, 0};
      for (int r = 0; r < ranks; ++r) {
        const int4 w = ld_cluster_i4(base + (uint32_t)(t * BM + f) * 4u, (uint32_t)r);
        e[0] += w.x; e[1] += w.y; e[2] += w.z; e[3] += w.w;
      }
      const float st = a.st[(int64_t)(m0 + t) * a.st_step];
      OutT* o = out + (size_t)(m0 + t) * a.N + n0 + f;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n0 + f + j < a.N)
          store1(o + j, scaled(e[j], st, a.sf[(int64_t)(n0 + f + j) * a.sf_step],
                               a.bias ? a.bias[n0 + f + j] : 0.0f));
    }
    cluster_sync();  // the partial tiles are read: the CTAs may go
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    if (nk > 0) mbar_wait_to(&bars->acc, 0, kErrTimeoutDone, a.err);
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tbase, kAcc);
  }
}

template <int NT, typename OutT>
int launch(const CUtensorMap& tf, const CUtensorMap& tt, const Args& a, cudaStream_t st) {
  auto kern = int8_gemm_kernel<NT, OutT>;
  constexpr size_t smem = smem_bytes<NT>();
  MXB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(cdiv(a.N, BM) * a.splits), (unsigned)cdiv(a.M, NT));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)a.splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  MXB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, tf, tt, a));
  MXB_LAUNCH_CHECK();
  return MXB_OK;
}

// ── many tokens ─────────────────────────────────────────────────────────────
// A pair of CTAs (cta_group::2) owns a tile of 256 tokens x 256 features: each loads
// its 128 tokens and half of the features, and the pair's MMAs (M = 256) read both
// halves, so that an SM draws 64 bytes a cycle of operands at the full rate where one
// CTA's 128 x 128 tile draws 128.  Pairs walk the list of tiles; the accumulators are
// double (2 x 256 columns of TMEM), so that the epilogue of a tile runs beside the
// products of the next.
//   warp 0      TMA producer (either CTA; both count on the leader's barriers);
//   warp 1      MMAs (the leader's);  warps 2, 3  TMEM allocation, idle;
//   warps 4-11  epilogue: a thread a token and half of the columns; 32 tokens x 128
//               bytes leave as one TMA store from shared memory.
// 4096 tokens, 8192 -> 8192: 174 us in short runs = 3.2 POP/s (292 on 128 x 128 tiles), 194
// to 203 by machine where the power limit holds the clock down; 2048 tokens, 4096 -> 11008: 65
// and 75 to 78 us (344 tiles for 74 pairs).  1024 x 8192 x 8192: 55 to 59 us, tensor pipe
// 61 % (128 tiles, two rounds), each operand read from HBM once.
namespace wide {

constexpr int kEpi = 8;
constexpr int kThreads = 128 + 32 * kEpi;
constexpr int kA = 128 * BK;            // a CTA's tokens of a stage
constexpr int kOut = 32 * 128;          // a warp's piece of the output
constexpr int BN = 256;                 // features of a pair
struct Cfg {
  static constexpr int kB = BN / 2 * BK;  // and features of a stage
  static constexpr int kStage = kA + kB;
  static constexpr int S = 6;
  static constexpr size_t oOut = (size_t)S * kStage, oBars = oOut + kEpi * kOut;
  static constexpr size_t kSmem = 1024 + oBars + 512;
};

struct Bars {
  uint64_t full[Cfg::S], empty[Cfg::S];
  uint64_t acc[2], acc_free[2];
  uint32_t tmem_base;
};
static_assert(sizeof(Bars) <= 512, "barrier block overflows its slot");

struct Tiles {
  int m, n, total;  // tiles along the tokens and the features
};

__device__ __forceinline__ uint32_t rank_of() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// The address of a shared variable in the pair's leader.
__device__ __forceinline__ uint32_t in_leader(const void* p) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(0));
  return a;
}
// A TMA load into this CTA whose bytes count on the leader's barrier (no multicast).
__device__ __forceinline__ void load_pair(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrive on `bar` of both CTAs when all MMAs issued so far are complete.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void arrive_remote(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Tile i: runs of 8 tiles along the tokens, so that the pairs at work share both
// operands in L2.
__device__ __forceinline__ void tile_at(const Tiles& t, int i, int& m, int& n) {
  const int band = 8 * t.n, b = i / band, rows = min(8, t.m - 8 * b), r = i - b * band;
  n = r / rows;
  m = 8 * b + (r - n * rows);
}

template <typename OutT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    int8_wide_kernel(const __grid_constant__ CUtensorMap tmap_f, const __grid_constant__ CUtensorMap tmap_t,
                     const __grid_constant__ CUtensorMap tmap_o, const Args a, const Tiles tiles) {
  using C = Cfg;
  constexpr int S = C::S;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  Bars* bars = reinterpret_cast<Bars*>(smem + C::oBars);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = rank_of();
  const int first = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->acc[b], 1);
      mbar_init(&bars->acc_free[b], 2 * kEpi);
    }
    fence_barrier_init();
    prefetch_tmap(&tmap_f);
    prefetch_tmap(&tmap_t);
    prefetch_tmap(&tmap_o);
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&bars->tmem_base)),
                 "r"(2 * BN)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are set up
  tc_fence_after();
  const uint32_t tbase = bars->tmem_base;
  pdl_trigger();
  pdl_wait();

  if (warp == 0) {
    if (lane == 0) {
      int s = 0, round = 0, issued = 0;
      bool ok = true;
      for (int i = first; i < tiles.total && ok; i += pairs) {
        int m, n;
        tile_at(tiles, i, m, n);
        const int y_t = m * 256 + (int)rank * 128, y_f = n * BN + (int)rank * (BN / 2);
        for (int k = 0; k < a.ksteps; ++k) {
          if (round > 0 && !mbar_wait_to(&bars->empty[s], (round - 1) & 1, kErrTimeoutEmpty, a.err)) {
            ok = false;
            break;
          }
          if (rank == 0) mbar_expect_tx(&bars->full[s], 2 * C::kStage);
          const uint32_t bar = in_leader(&bars->full[s]);
          uint8_t* dst = smem + s * C::kStage;
          load_pair(dst, &tmap_t, bar, k * BK, y_t);
          load_pair(dst + kA, &tmap_f, bar, k * BK, y_f);
          ++issued;
          if (++s == S) {
            s = 0;
            ++round;
          }
        }
      }
      // the pair's last copies land before it may end (the leader counts both CTAs'), also
      // where a wait gave up
      if (rank == 0)
        for (int j = max(issued - S, 0); j < issued; ++j)
          mbar_wait_to(&bars->full[j % S], (j / S) & 1, kErrTimeoutFull, a.err);
    }
  } else if (warp == 1 && rank == 0) {
    if (lane == 0) {
      constexpr uint32_t id = make_idesc(/*S32*/ 2, /*signed*/ 1, 0, 0, 256, BN);
      const uint64_t da = desc_kmajor_sw128(smem_u32(smem)), db = desc_kmajor_sw128(smem_u32(smem + kA));
      int s = 0, round = 0, t = 0;
      bool ok = true;
      for (int i = first; i < tiles.total && ok; i += pairs, ++t) {
        const int b = t & 1;
        if (t >= 2) ok = mbar_wait_to(&bars->acc_free[b], ((t >> 1) - 1) & 1, kErrTimeoutTmemEmpty, a.err);
        if (!ok) break;
        tc_fence_after();
        const uint32_t acc = tbase + b * BN;
        for (int k = 0; k < a.ksteps; ++k) {
          if (!mbar_wait_to(&bars->full[s], round & 1, kErrTimeoutFull, a.err)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t off = (uint32_t)(s * C::kStage) >> 4;
#pragma unroll
          for (int kk = 0; kk < BK / 32; ++kk)
            mma_pair(acc, da + off + kk * 2, db + off + kk * 2, id, (k > 0 || kk > 0) ? 1u : 0u);
          commit_pair(&bars->empty[s]);
          if (++s == S) {
            s = 0;
            ++round;
          }
        }
        commit_pair(&bars->acc[b]);  // of all that were issued, also where a wait gave up
      }
    }
  } else if (warp >= 4) {
    // ── epilogue ──
    const int q = warp & 3, half = (warp - 4) >> 2;
    uint8_t* stage = smem + C::oOut + (warp - 4) * kOut;
    constexpr int kCols = 128 / sizeof(OutT);  // a piece's columns: 64 or 32
    int t = 0;
    for (int i = first; i < tiles.total; i += pairs, ++t) {
      int m, n;
      tile_at(tiles, i, m, n);
      const int b = t & 1, row0 = m * 256 + (int)rank * 128 + q * 32;
      if (!mbar_wait_warp_to(&bars->acc[b], (t >> 1) & 1, kErrTimeoutDone, a.err)) break;
      tc_fence_after();
      const float st = row0 + lane < a.M ? __ldg(a.st + (int64_t)(row0 + lane) * a.st_step) : 0.0f;
      const uint32_t acc = tbase + b * BN + ((uint32_t)(q * 32) << 16) + half * (BN / 2);
      const int c0 = n * BN + half * (BN / 2);
#pragma unroll 1
      for (int p = 0; p < BN / 2; p += kCols) {
        // the piece before has been read
        if (lane == 0) bulk_wait_read();
        __syncwarp();
#pragma unroll
        for (int x = 0; x < kCols; x += 32) {
          uint32_t r[32];
          tmem_ld32(acc + p + x, r);
          tmem_wait_ld();
          tmem_landed(r);
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const int col = c0 + p + x + j;
            float4 sf = make_float4(0.0f, 0.0f, 0.0f, 0.0f), bv = sf;
            if (col < a.N) {  // N is a multiple of 4
              if (a.sf_step) sf = __ldg(reinterpret_cast<const float4*>(a.sf + col));
              else sf.x = sf.y = sf.z = sf.w = __ldg(a.sf);
              if (a.bias) bv = __ldg(reinterpret_cast<const float4*>(a.bias + col));
            }
            const float v0 = scaled((int)r[j], st, sf.x, bv.x), v1 = scaled((int)r[j + 1], st, sf.y, bv.y);
            const float v2 = scaled((int)r[j + 2], st, sf.z, bv.z), v3 = scaled((int)r[j + 3], st, sf.w, bv.w);
            if constexpr (sizeof(OutT) == 4) {
              *reinterpret_cast<float4*>(stage + lane * 128 + (((j / 4) ^ (lane & 7)) << 4)) =
                  make_float4(v0, v1, v2, v3);
            } else {
              const __nv_bfloat162 lo = __floats2bfloat162_rn(v0, v1), hi = __floats2bfloat162_rn(v2, v3);
              // 16-byte chunk (x + j) / 8 of the row, its half j / 4 % 2
              *reinterpret_cast<uint2*>(stage + lane * 128 + ((((x + j) / 8) ^ (lane & 7)) << 4) + (j & 4) * 2) =
                  make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
            }
          }
        }
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0 && row0 < a.M && c0 + p < a.N) {
          tma_store_2d(&tmap_o, stage, c0 + p, row0);
          bulk_commit();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_remote(in_leader(&bars->acc_free[b]));
    }
    if (lane == 0) bulk_wait_read();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // no CTA ends while its pair may still read or signal it
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tbase), "r"(2 * BN));
  }
}

template <typename OutT>
int launch(const CUtensorMap& tf, const CUtensorMap& tt, const CUtensorMap& to, const Args& a, cudaStream_t st) {
  using C = Cfg;
  static_assert(C::kSmem <= 227 * 1024, "shared memory");
  auto kern = int8_wide_kernel<OutT>;
  MXB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem));
  Tiles t;
  t.m = (int)cdiv(a.M, 256);
  t.n = (int)cdiv(a.N, BN);
  t.total = t.m * t.n;
  const int pairs = t.total < kSMs / 2 ? t.total : kSMs / 2;
  MXB_CUDA_TRY(launch_pdl(kern, dim3((unsigned)(2 * pairs)), kThreads, C::kSmem, st, tf, tt, to, a, t));
  MXB_LAUNCH_CHECK();
  return MXB_OK;
}

}  // namespace wide

// Rows of K bytes that start anywhere -> rows of Kp, zero from K on: a warp a row, 16
// bytes a lane from five words that lie in memory as such (64 x 8001 x 8000: 58 us byte by
// byte).
__global__ void __launch_bounds__(256)
    pad_rows_kernel(const uint8_t* __restrict__ a, int64_t ra, const uint8_t* __restrict__ b, int64_t rb, int K,
                    int Kp, uint8_t* __restrict__ out) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, warps = gridDim.x * 8;
  for (int64_t row = blockIdx.x * 8 + (threadIdx.x >> 5); row < ra + rb; row += warps) {
    const bool of_a = row < ra;
    const uint8_t* lo = of_a ? a : b;
    const uint8_t* hi = lo + (of_a ? ra : rb) * K;  // the operand's bytes, and no others, are read
    const uint8_t* src = lo + (of_a ? row : row - ra) * K;
    auto word = [&](const uint8_t* p) -> uint32_t {
      if (p >= lo && p + 4 <= hi) return __ldg(reinterpret_cast<const uint32_t*>(p));
      uint32_t w = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (p + j >= lo && p + j < hi) w |= (uint32_t)__ldg(p + j) << (8 * j);
      return w;
    };
    for (int k = lane * 16; k < Kp; k += 512) {
      const uint8_t* p = src + k;
      const uint32_t off = (uint32_t)((uintptr_t)p & 3);
      p -= off;
      uint32_t w[5];
#pragma unroll
      for (int j = 0; j < 5; ++j) w[j] = word(p + 4 * j);
      const int left = K - k;  // bytes of the row from here on
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = __funnelshift_r(w[j], w[j + 1], 8 * off);
        const int n = left - 4 * j;
        if (n < 4) w[j] &= n <= 0 ? 0u : (1u << (8 * n)) - 1u;
      }
      *reinterpret_cast<uint4*>(out + row * Kp + k) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// How a product is cut: tokens a CTA (0: CTA pairs) and K splits.
struct Cut {
  int nt, splits;
};

// Up to 64 tokens the smallest tile that holds them all, so that few tokens pay an MMA of
// their width, and K splits while they fill the SMs, as many as the root of twice the
// stages at most (more shorten the stages' time / splits and lengthen the sum).  Beyond,
// what costs least by the times that the kernels took (microseconds): a stage of a 128 x
// 128 tile 0.42 alone on an SM and 0.53 for two, of a 128 x 64 tile 0.33 and 0.40, of a
// pair's 256 x 256 tile 0.38; 6 or 8 around them, 4.5 to join splits, which have to win by
// a fifth.  E.g. (auto / the other kernels' best): 160 x 4096 x 11008 18.8 / 22.5, 256 x
// 11008 x 4096 23.4 / 28.8, 700 x 4096 x 11008 32.9 / 39.4, 2000 x 2048 x 2048 14.5 /
// 16.4.
//
// Clusters have to fit all at once: one too many starts when the first ones have gone (1 x
// 4096 x 4736, weights from HBM: 37 clusters of 8 11.2 us, of 6 7.7).  Two CTAs an SM, the
// SMs of a cluster in one GPC: 148 clusters of 2 fit, 91 of 3, 71, 55, 45, 37 and 33 of 4
// to 8 (90 of 3 11.7 us, of 2 12.5; 96 of 3 17.2).  So threes stop at 270 CTAs, more at 256.
Cut cut_of(int64_t M, int64_t N, int64_t ksteps, bool pairs) {
  const int64_t ft = cdiv(N, BM);
  if (M <= 64) {
    const int nt = M <= 16 ? 16 : M <= 32 ? 32 : 64;
    int64_t splits = 2 * kSMs / ft;
    if (splits > ksteps / 2) splits = ksteps / 2;
    if (splits > kMaxSplit) splits = kMaxSplit;
    while (splits * splits > 2 * ksteps) --splits;
    while (splits > 2 && ft * splits > (splits == 3 ? 270 : 256)) --splits;
    return {nt, (int)(splits < 1 ? 1 : splits)};
  }
  Cut best = {0, 1};
  double least = pairs ? 8.0 + 0.38 * ksteps * cdiv(cdiv(M, 256) * cdiv(N, 256), kSMs / 2) : 1e30;
  for (int nt = 64; nt <= 128; nt += 64) {
    if (cdiv(M, nt) > 65535) continue;  // gridDim.y
    double whole = 0.0;
    for (int s = 1; s <= kMaxSplit && (s == 1 || 2 * s <= ksteps); ++s) {
      const int64_t ctas = ft * cdiv(M, nt) * s;
      if (s > 1 && ctas > 256) break;
      const double stage = nt == 64 ? (ctas <= kSMs ? 0.33 : 0.40) : (ctas <= kSMs ? 0.42 : 0.53);
      const double t = 6.0 + stage * cdiv(ksteps, s) * cdiv(ctas, 2 * kSMs) + (s > 1 ? 4.5 : 0.0);
      if (s == 1) whole = t;
      if (t < least && (s == 1 || t < 0.8 * whole)) {
        least = t;
        best = {nt, s};
      }
    }
  }
  return best;
}

template <typename OutT>
int dispatch(const void* fcodes, const void* tcodes, int64_t ldk, Args& a, cudaStream_t st) {
  CUtensorMap tf, tt;
  // pairs write whole TMA lines, and read scales and bias by 16 bytes
  const bool lines = a.N % (16 / (int)sizeof(OutT)) == 0 && (uintptr_t)a.out % 16 == 0 &&
                     ((uintptr_t)a.sf | (uintptr_t)a.bias) % 16 == 0;
  const Cut cut = cut_of(a.M, a.N, a.ksteps, lines);
  if (cut.nt == 0) {
    CUtensorMap to;
    const bool half = sizeof(OutT) == 2;
    if (!encode_tmap_2d(&tf, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, fcodes, (uint64_t)ldk, (uint64_t)a.N, BK, wide::BN / 2,
                        CU_TENSOR_MAP_SWIZZLE_128B) ||
        !encode_tmap_2d(&tt, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, tcodes, (uint64_t)ldk, (uint64_t)a.M, BK, 128,
                        CU_TENSOR_MAP_SWIZZLE_128B) ||
        !encode_tmap_2d(&to, half ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32,
                        sizeof(OutT), a.out, (uint64_t)a.N, (uint64_t)a.M, 128 / sizeof(OutT), 32,
                        CU_TENSOR_MAP_SWIZZLE_128B))
      return MXB_E_CUDA;
    return wide::launch<OutT>(tf, tt, to, a, st);
  }
  const int nt = cut.nt;
  a.splits = cut.splits;
  if (!encode_tmap_2d(&tf, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, fcodes, (uint64_t)ldk, (uint64_t)a.N, BK, BM,
                      CU_TENSOR_MAP_SWIZZLE_128B) ||
      !encode_tmap_2d(&tt, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, tcodes, (uint64_t)ldk, (uint64_t)a.M, BK, nt,
                      CU_TENSOR_MAP_SWIZZLE_128B))
    return MXB_E_CUDA;
  switch (nt) {
    case 16: return launch<16, OutT>(tf, tt, a, st);
    case 32: return launch<32, OutT>(tf, tt, a, st);
    case 64: return launch<64, OutT>(tf, tt, a, st);
    default: return launch<128, OutT>(tf, tt, a, st);
  }
}

int64_t padded(int64_t K) { return (K + 15) / 16 * 16; }

}  // namespace i8g
}  // namespace mxb

extern "C" {

size_t mxb_int8_matmul_workspace_size(int64_t M, int64_t K, int64_t N, int aligned) {
  if (M <= 0 || K <= 0 || N <= 0 || (K % 16 == 0 && aligned)) return 0;
  return (size_t)(M + N) * (size_t)i8g::padded(K);
}

int mxb_int8_matmul(const void* a_codes, const float* a_scales, int a_scale_step, const void* b_codes,
                    const float* b_scales, int b_scale_step, int64_t M, int64_t K, int64_t N,
                    const float* bias, void* out, int out_dtype, void* workspace, size_t workspace_bytes,
                    void* stream) {
  if (out_dtype != MXB_F32 && out_dtype != MXB_BF16) return MXB_E_DTYPE;
  if (M < 0 || N < 0 || K <= 0 || K > i8g::kMaxK) return MXB_E_SHAPE;
  if (M > 65535 * 128 || N >= (int64_t)1 << 30) return MXB_E_SHAPE;
  if ((a_scale_step != 0 && a_scale_step != 1) || (b_scale_step != 0 && b_scale_step != 1)) return MXB_E_ARG;
  if (M == 0 || N == 0) return MXB_OK;
  if (!a_codes || !a_scales || !b_codes || !b_scales || !out) return MXB_E_ARG;
  if (((uintptr_t)a_scales | (uintptr_t)b_scales | (uintptr_t)bias) % 4 ||
      (uintptr_t)out % (out_dtype == MXB_BF16 ? 2 : 4) || (uintptr_t)workspace % 16)
    return MXB_E_ALIGN;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  i8g::Args a = {};
  a.sf = b_scales;
  a.st = a_scales;
  a.sf_step = b_scale_step;
  a.st_step = a_scale_step;
  a.bias = bias;
  a.out = out;
  a.err = device_error_ptr();
  a.M = (int)M;
  a.N = (int)N;
  a.ksteps = (int)cdiv(K, i8g::BK);
  const void *tc = a_codes, *fc = b_codes;
  int64_t ldk = K;
  // TMA wants rows that start at multiples of 16 bytes
  if (K % 16 || ((uintptr_t)a_codes | (uintptr_t)b_codes) % 16) {
    ldk = i8g::padded(K);
    const size_t need = mxb_int8_matmul_workspace_size(M, K, N, 0);
    if (need > 0) {
      if (!workspace || workspace_bytes < need) return MXB_E_WORKSPACE;
      const int64_t blocks = cdiv(M + N, 8);
      MXB_CUDA_TRY(launch_pdl(i8g::pad_rows_kernel, dim3((unsigned)(blocks < 8 * kSMs ? blocks : 8 * kSMs)),
                              256, 0, st, static_cast<const uint8_t*>(a_codes), M,
                              static_cast<const uint8_t*>(b_codes), N, (int)K, (int)ldk,
                              static_cast<uint8_t*>(workspace)));
      MXB_LAUNCH_CHECK();
      tc = workspace;
      fc = static_cast<uint8_t*>(workspace) + M * ldk;
    }
  }
  return out_dtype == MXB_BF16 ? i8g::dispatch<__nv_bfloat16>(fc, tc, ldk, a, st)
                               : i8g::dispatch<float>(fc, tc, ldk, a, st);
}

}  // extern "C"
