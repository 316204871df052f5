// Attention of every query row of a batch over a prefix that they share, on
// tcgen05 (paged_attn.cu describes the cache and the parts that it joins).
//
// With all B * T * G rows of a KV head taken together the prefix is a product
// of two matrices, bound by arithmetic: 4 * rows * keys * dim operations, and
// the work around it, one exponential a score and the unpacking of the codes.
// A CTA owns 128 rows (two groups of 128 from 129 rows on, so that a key is
// unpacked once for 256 rows) and a run of the keys, in tiles of 64:
//   warp 0        TMA producer: raw codes and scales, ring of kStages tiles;
//   warp 1        TMEM allocation, MMA issue: S = Q K^T (fp16 x fp16), two
//                 buffers a row group; O += P V with P read from TMEM;
//   warps 2-5     unpack codes to exact fp16 (K and V tiles have one layout:
//                 K-major for the first product, MN-major for the second),
//                 and lay out the tile's scales;
//   warps 6-..    softmax, a thread a row: S from TMEM, running maximum, sum,
//                 weights back to TMEM over S.
// Scores: Q is fp16 under a power of two per row that puts its largest value
// into [2^14, 2^15), the codes are exact.  Weights: p_j = exp2(s_j - m) times
// 2^6 sv_j / c, c a power of two of at least the largest value scale so far, and m
// following the maximum within 2^8.  While the value scales span less than 2^-14
// of c, a row's largest weight is at least 2^-8, so fp16 keeps 11 bits of those
// down to 2^-6 of it and is off by at most 2^-17 of it below.  From the first tile
// with a wider span on, c is each row's own and follows its largest weight, as
// that may belong to a key whose value scale is far under another's (a wide tile
// costs one more multiplication and comparison a score).  m, sums and outputs
// are fp32; O is rescaled in TMEM only when m or c moves.
// Pairs of codes unpack out of order; Q's columns are stored in the same
// order and O's columns are put back when they are written.
//
// 64 x 8 rows of each of 8 heads over 8192 keys of 128 dims in int8: 34 - 41 us =
// 420 - 500 TFLOP/s (188 us with the 32-row groups of paged_attn.cu).  A 64-key
// tile takes about 3600 cycles; unpacking, softmax and the issue of its products
// about 3000 each, so that eight unpacking warps instead of four, or a warp for
// each product, were no faster.  Q takes 5 us at the start and O 4 at the end.
#include "mxb_common.cuh"
#include "mxb_internal.h"

#include <cuda.h>
#include <cuda_fp16.h>

#define MXB_ERROR_WORD_BY_POINTER
#include "tc_ptx.cuh"

using namespace mxb;

namespace mxb {
namespace pfx {

constexpr int KT = kPrefixKeys;
constexpr int kStages = 3;
constexpr int kSlots = 4;  // scale slots: softmax may lag the unpacking by two tiles
constexpr int kConvWarps = 4;
constexpr float kRoom = 64.0f;  // 2^6
// Value scales below this part of c make a tile wide: of the largest, 2^-11 or 2^-12.
// 64 x 8 rows of 8 heads over 8192 keys take 45 us while all tiles are narrow, 60
// when all are wide, 70 with both (ncu), so a span that a cache has in earnest is
// left narrow.
constexpr float kWide = 0x1p-14f;

template <int BITS, int D, int MT>
struct Cfg {
  static constexpr int RB = D * BITS / 8;
  static constexpr int kRaw = KT * RB;
  static constexpr int kAtom = KT * 128;           // 64 dims of every key
  static constexpr int kPlane = kAtom * (D / 64);  // 16 or 8 KB
  static constexpr int kQAtom = 128 * 128;
  static constexpr int kQ = kQAtom * (D / 64);
  static constexpr int kThreads = 64 + 32 * kConvWarps + 128 * MT;
  static constexpr size_t oK = (size_t)MT * kQ, oV = oK + 2 * kPlane, oRaw = oV + 2 * kPlane;
  static constexpr size_t oRawS = oRaw + (size_t)kStages * 2 * kRaw;
  static constexpr size_t oSc = oRawS + (size_t)kStages * 2 * KT * 4;
  static constexpr size_t oBars = oSc + (size_t)kSlots * (2 * KT + 4) * 4;
  static constexpr size_t kSmem = 1024 + oBars + 512;
  // TMEM: per row group two S buffers of 64 columns, then O
  static constexpr int kCols = MT == 2 ? 512 : 256;
};

struct Bars {
  uint64_t raw_full[kStages], raw_empty[kStages];
  uint64_t kready[2], kfree[2], vready[2], vfree[2];
  uint64_t sready[2][2], pready[2][2], pvdone[2];
  uint64_t scready[kSlots];
  uint64_t qready;
  uint64_t drained;  // every product issued is complete
  uint32_t tmem_base;
  uint32_t gone[kStages];  // bit i: keys 16 i .. of the tile lie behind a number outside the pool
};
static_assert(sizeof(Bars) <= 512, "barrier block overflows its slot");

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t hsub2u(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t hf2(float lo, float hi) {
  const __half2 t = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&t);
}

// Position p of a group of unpacked codes holds dim order(p) of the group: int8
// words give (0, 2), (1, 3); int4 words (0, 4), (1, 5), (2, 6), (3, 7).
template <int BITS>
__host__ __device__ constexpr int order(int p) {
  return BITS == 8 ? ((p & 4) | ((p & 1) << 1) | ((p & 2) >> 1))
                   : ((p & 1) << 2) | (p >> 1);
}

// 16 bytes of codes -> 16 (int8) or 32 (int4) exact fp16 values as 16-byte
// chunks of eight.
template <int BITS>
__device__ __forceinline__ void unpack16(uint4 r, uint4 (&o)[BITS == 8 ? 2 : 4]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
  if constexpr (BITS == 8) {
    uint32_t v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = hsub2u((w[i] & 0x00FF00FFu) ^ 0x64806480u, 0x64806480u);
      v[2 * i + 1] = hsub2u(((w[i] >> 8) & 0x00FF00FFu) ^ 0x64806480u, 0x64806480u);
    }
    o[0] = make_uint4(v[0], v[1], v[2], v[3]);
    o[1] = make_uint4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        v[k] = hsub2u(((w[i] >> (4 * k)) & 0x000F000Fu) ^ 0x64086408u, 0x64086408u);
      o[i] = make_uint4(v[0], v[1], v[2], v[3]);
    }
  }
}

// One raw tile [KT][RB] -> fp16 plane, rows of 128 bytes per 64-dim atom,
// 128-byte swizzle (thread t of the unpackers).  Eight neighbouring lanes take
// chunks of one atom from two (four) rows, so that their 16-byte stores cover
// all banks.
template <int BITS, int D>
__device__ __forceinline__ void unpack_tile(const uint8_t* raw, uint8_t* plane, int t) {
  constexpr int RB = D * BITS / 8, C = RB / 16, N = BITS == 8 ? 2 : 4;  // chunks a row, out per chunk
  constexpr int kAtom = KT * 128, kThr = 32 * kConvWarps;
#pragma unroll
  for (int i0 = 0; i0 < KT * C; i0 += kThr) {
    const int i = i0 + t;
    if (KT * C < kThr && i >= KT * C) break;
    int row, c;
    if (C == 8) {
      c = (i & 3) | (((i >> 3) & 1) << 2);
      row = ((i >> 4) << 1) | ((i >> 2) & 1);
    } else if (C == 4 && BITS == 4) {
      c = (i & 1) | (((i >> 3) & 1) << 1);
      row = ((i >> 4) << 2) | ((i >> 1) & 3);
    } else {
      c = i % C;
      row = i / C;
    }
    const uint4 r = *reinterpret_cast<const uint4*>(raw + row * RB + c * 16);
    uint4 o[N];
    unpack16<BITS>(r, o);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int ch = c * N + k;
      *reinterpret_cast<uint4*>(plane + (ch >> 3) * kAtom + row * 128 + (((ch & 7) ^ (row & 7)) << 4)) = o[k];
    }
  }
}

// A row of the softmax: reference and sum; lc, log2 of the c that its O stands
// under; top_w, log2 of the largest weight stored, or less (kept for wide tiles;
// -8 is what narrow ones reach).
struct Row {
  float mu = 0.0f, m_top = -INFINITY, l = 0.0f, lc = 0.0f, top_w = -8.0f;
  bool ok = true;
};
struct RowTiles {
  Bars* bars;
  const float* sc_slots;
  uint32_t tmem;  // S of this warp's rows; O follows after 128 columns
  int x, lane, keys;  // row group; keys of the run
  float rowf;
  int* err;
};

// One tile of 64 keys; false where a wait gave up, or at the first wide tile (W:
// this one may be wide).
template <int D, bool W>
__device__ __forceinline__ bool softmax_tile(Row& r, const RowTiles& g, int t) {
  const int b = t & 1, slot = t % kSlots;
  r.ok = mbar_wait_warp_to(&g.bars->scready[slot], (t / kSlots) & 1, kErrTimeoutFull, g.err) &&
       mbar_wait_warp_to(&g.bars->sready[g.x][b], (t >> 1) & 1, kErrTimeoutTmemFull, g.err);
  if (!r.ok) return false;
  const float4 of_tile = *reinterpret_cast<const float4*>(g.sc_slots + slot * (2 * KT + 4) + 2 * KT);
  const float lcn = of_tile.x;
  const uint32_t gone = __float_as_uint(of_tile.y);
  if (!W && __float_as_uint(of_tile.z) != 0u) return false;
  tc_fence_after();
  float v[KT];
  {
    uint32_t r0v[32], r1v[32];
    tmem_ld32(g.tmem + b * 64, r0v);
    tmem_ld32(g.tmem + b * 64 + 32, r1v);
    tmem_wait_ld();
    tmem_landed(r0v);
    tmem_landed(r1v);
    const float4* ks = reinterpret_cast<const float4*>(g.sc_slots + slot * (2 * KT + 4));
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      const float4 k0 = ks[j / 4], k1 = ks[8 + j / 4];
      v[j] = __uint_as_float(r0v[j]) * k0.x;
      v[j + 1] = __uint_as_float(r0v[j + 1]) * k0.y;
      v[j + 2] = __uint_as_float(r0v[j + 2]) * k0.z;
      v[j + 3] = __uint_as_float(r0v[j + 3]) * k0.w;
      v[32 + j] = __uint_as_float(r1v[j]) * k1.x;
      v[33 + j] = __uint_as_float(r1v[j + 1]) * k1.y;
      v[34 + j] = __uint_as_float(r1v[j + 2]) * k1.z;
      v[35 + j] = __uint_as_float(r1v[j + 3]) * k1.w;
    }
  }
  const int valid = g.keys - t * KT;
  if (gone) {
#pragma unroll
    for (int j = 0; j < KT; ++j)
      if (gone >> (j >> 4) & 1u) v[j] = -INFINITY;
  }
  if (valid < KT) {
#pragma unroll
    for (int j = 0; j < KT; ++j)
      if (j >= valid) v[j] = -INFINITY;
  }
  float m4[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
  for (int j = 4; j < KT; ++j) m4[j & 3] = fmaxf(m4[j & 3], v[j]);
  const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * g.rowf;
  const float4* vs = reinterpret_cast<const float4*>(g.sc_slots + slot * (2 * KT + 4) + KT);
  bool waited = t == 0;
  float alpha = 1.0f, dm = 0.0f;
  if (t == 0) {
    r.lc = lcn;
    r.top_w = -INFINITY;
  }
  bool rescale = mx > r.m_top || (!W && lcn != r.lc);
  if (__any_sync(0xffffffffu, rescale)) {
    const float m0 = r.m_top == -INFINITY ? -INFINITY : r.mu;
    const float m1 = fmaxf(m0, mx);
    r.mu = m1 == -INFINITY ? 0.0f : m1;
    dm = m0 - r.mu;
    alpha = ex2(dm);
    r.l *= alpha;
    r.m_top = m1 + 8.0f;
    if (!W) {
      alpha *= ex2(r.lc - lcn);
      r.lc = lcn;
    }
    rescale = true;
  }
  uint32_t pk[32];
  float s0 = 0.0f, s1 = 0.0f;
  if (W) {
    // the weights first, then a c for this row that puts its largest so far
    // between 2^-2 and 2^12
    float u4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < KT; j += 4) {
      const float4 w = vs[j / 4];
      const float p0 = ex2(__fmaf_rn(v[j], g.rowf, -r.mu)), p1 = ex2(__fmaf_rn(v[j + 1], g.rowf, -r.mu));
      const float p2 = ex2(__fmaf_rn(v[j + 2], g.rowf, -r.mu)), p3 = ex2(__fmaf_rn(v[j + 3], g.rowf, -r.mu));
      s0 += p0 + p2;
      s1 += p1 + p3;
      v[j] = p0 * w.x;
      v[j + 1] = p1 * w.y;
      v[j + 2] = p2 * w.z;
      v[j + 3] = p3 * w.w;
#pragma unroll
      for (int k = 0; k < 4; ++k) u4[k] = fmaxf(u4[k], v[j + k]);
    }
    const float u = fmaxf(fmaxf(u4[0], u4[1]), fmaxf(u4[2], u4[3]));
    r.top_w = fminf(fmaxf(r.top_w + dm, log2f(u) + (lcn - r.lc)), 200.0f);
    const bool off = r.top_w > 12.0f || (r.top_w < -2.0f && r.top_w > -INFINITY) || lcn - r.lc > 120.0f;
    if (__any_sync(0xffffffffu, off)) {
      if (off) {
        // no further below the tile's c than 2^120: fp32 holds little under that
        const float up = fminf(6.0f - floorf(r.top_w), 120.0f - (lcn - r.lc));
        r.lc -= up;
        r.top_w += up;
        alpha *= ex2(up);
      }
      rescale = true;
    }
    const float up = ex2(lcn - r.lc);
#pragma unroll
    for (int j = 0; j < KT; j += 2) pk[j / 2] = hf2(v[j] * up, v[j + 1] * up);
  }
  if (rescale && t > 0) {
    // O of the tiles before has to be complete; the next product waits
    // for this tile's weights
    r.ok = mbar_wait_warp_to(&g.bars->pvdone[g.x], (t - 1) & 1, kErrTimeoutTmemEmpty, g.err);
    if (!r.ok) return false;
    waited = true;
    tc_fence_after();
#pragma unroll 1
    for (int d = 0; d < D; d += 32) {
      uint32_t o[32];
      tmem_ld32(g.tmem + 128 + d, o);
      tmem_wait_ld();
      tmem_landed(o);
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
      tmem_st32(g.tmem + 128 + d, o);
    }
  }
  if (!W) {
#pragma unroll
    for (int j = 0; j < KT; j += 4) {
      const float4 w = vs[j / 4];
      const float p0 = ex2(__fmaf_rn(v[j], g.rowf, -r.mu)), p1 = ex2(__fmaf_rn(v[j + 1], g.rowf, -r.mu));
      const float p2 = ex2(__fmaf_rn(v[j + 2], g.rowf, -r.mu)), p3 = ex2(__fmaf_rn(v[j + 3], g.rowf, -r.mu));
      s0 += p0 + p2;
      s1 += p1 + p3;
      pk[j / 2] = hf2(p0 * w.x, p1 * w.y);
      pk[j / 2 + 1] = hf2(p2 * w.z, p3 * w.w);
    }
  }
  r.l += s0 + s1;
  // every phase of pvdone is waited for in turn: a parity tells only the
  // last completed phase from the one before it
  if (!waited) {
    r.ok = mbar_wait_warp_to(&g.bars->pvdone[g.x], (t - 1) & 1, kErrTimeoutTmemEmpty, g.err);
    if (!r.ok) return false;
  }
  tmem_st32(g.tmem + b * 64, pk);
  tmem_wait_st();
  tc_fence_before();
  __syncwarp();
  if (g.lane == 0) mbar_arrive(&g.bars->pready[g.x][b]);
  return true;
}
// The wide tiles, apart: in line they cost a call whose tiles are all narrow 2 us of 69.
template <int D>
__device__ __noinline__ Row wide_tiles(Row r, const RowTiles w, int t, int n) {
  while (t < n && softmax_tile<D, true>(r, w, t)) ++t;
  return r;
}

template <int BITS, int D, int MT>
__global__ void __launch_bounds__(Cfg<BITS, D, MT>::kThreads, 1)
    prefix_attn_kernel(const __grid_constant__ CUtensorMap tmap_k,
                       const __grid_constant__ CUtensorMap tmap_v, const PrefixArgs a, int box) {
  using C = Cfg<BITS, D, MT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  Bars* bars = reinterpret_cast<Bars*>(smem + C::oBars);
  float* sc_slots = reinterpret_cast<float*>(smem + C::oSc);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int boxes = KT / box, box_shift = 31 - __clz(box);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bars->raw_full[s], boxes);
      mbar_init(&bars->raw_empty[s], kConvWarps);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->kready[b], kConvWarps);
      mbar_init(&bars->kfree[b], 1);
      mbar_init(&bars->vready[b], kConvWarps);
      mbar_init(&bars->vfree[b], 1);
      for (int x = 0; x < 2; ++x) {
        mbar_init(&bars->sready[x][b], 1);
        mbar_init(&bars->pready[x][b], 4);
      }
      mbar_init(&bars->pvdone[b], 1);
    }
    for (int s = 0; s < kSlots; ++s) mbar_init(&bars->scready[s], kConvWarps);
    mbar_init(&bars->qready, 4 * MT);
    mbar_init(&bars->drained, 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, C::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = bars->tmem_base;
  pdl_trigger();
  pdl_wait();

  const int h = blockIdx.z, r0 = blockIdx.y * 128 * MT;
  const int rows = a.B * a.T * a.G;
  const int tiles = (a.len + KT - 1) / KT, per = (tiles + a.splits - 1) / a.splits;
  const int t_lo = min((int)blockIdx.x * per, tiles), n = min(per, tiles - t_lo);
  auto t_s = [&](int x, int b) { return tbase + (uint32_t)(x * (128 + D) + b * 64); };
  auto t_o = [&](int x) { return tbase + (uint32_t)(x * (128 + D) + 128); };

  if (warp == 0) {
    const int page_mask = (1 << a.page_shift) - 1;
    int i = 0;
    for (; i < n; ++i) {
      const int s = i % kStages, round = i / kStages;
      const int pos = (t_lo + i) * KT + lane * box;
      int p = -1;
      if (lane < boxes && pos < a.len) {
        p = __ldg(a.table + (pos >> a.page_shift));
        if (p < 0 || p >= a.n_pages) {
          if (a.err) atomicCAS(a.err, 0, kErrIndex);
          p = -2;
        }
      }
      const int p16 = __shfl_sync(0xffffffffu, p, lane >> (box_shift - 4));
      const uint32_t gone = __ballot_sync(0xffffffffu, lane < KT / 16 && p16 == -2);
      if (round > 0 && !mbar_wait_warp_to(&bars->raw_empty[s], (round - 1) & 1, kErrTimeoutEmpty, a.err))
        break;
      if (lane == 0) bars->gone[s] = gone;  // before its arrival
      if (lane < boxes) {
        uint64_t* bar = &bars->raw_full[s];
        if (p >= 0) {
          const int row = ((p * a.H + h) << a.page_shift) + (pos & page_mask);
          uint8_t* dst = smem + C::oRaw + (size_t)s * 2 * C::kRaw + lane * box * C::RB;
          float* sc = reinterpret_cast<float*>(smem + C::oRawS) + s * 2 * KT + lane * box;
          mbar_expect_tx(bar, (uint32_t)box * (2 * C::RB + 8));
          const int line = (int)((int64_t)row * C::RB / 128);  // lines of 128 bytes
          tma_load_2d(dst, &tmap_k, bar, 0, line);
          tma_load_2d(dst + C::kRaw, &tmap_v, bar, 0, line);
          bulk_load_g2s(sc, a.k_scales + row, (uint32_t)box * 4, bar);
          bulk_load_g2s(sc + KT, a.v_scales + row, (uint32_t)box * 4, bar);
        } else {
          mbar_arrive(bar);
        }
      }
    }
    // the last copies land before the CTA may end, also where a wait gave up
    for (int j = max(i - kStages, 0); j < i; ++j)
      mbar_wait_warp_to(&bars->raw_full[j % kStages], (j / kStages) & 1, kErrTimeoutFull, a.err);
  } else if (warp == 1) {
    if (lane == 0 && n > 0) {
      constexpr uint32_t id_s = make_idesc(/*F32*/ 1, /*F16*/ 0, 0, 0, 128, KT);
      constexpr uint32_t id_o = make_idesc(1, 0, 0, /*B MN-major*/ 1, 128, D);
      const uint32_t sq = smem_u32(smem), sk = smem_u32(smem + C::oK), sv = smem_u32(smem + C::oV);
      bool ok = mbar_wait_to(&bars->qready, 0, kErrTimeoutFull, a.err);
      auto issue_s = [&](int t) {
        const int b = t & 1;
        ok = ok && mbar_wait_to(&bars->kready[b], (t >> 1) & 1, kErrTimeoutFull, a.err);
        if (!ok) return;
        tc_fence_after();
        for (int x = 0; x < MT; ++x) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            mma_f16(t_s(x, b),
                    desc_kmajor_sw128(sq + x * C::kQ + (kk >> 2) * C::kQAtom + (kk & 3) * 32),
                    desc_kmajor_sw128(sk + b * C::kPlane + (kk >> 2) * C::kAtom + (kk & 3) * 32),
                    id_s, kk > 0 ? 1u : 0u);
          mma_commit(&bars->sready[x][b]);
        }
        mma_commit(&bars->kfree[b]);
      };
      issue_s(0);
      for (int t = 0; t < n && ok; ++t) {
        const int b = t & 1;
        if (t + 1 < n) {
          // S of the next tile goes over P of the last one: that product has to
          // be complete, since MMAs of different shapes need not run in the
          // order they are issued (the softmax of tile t runs meanwhile)
          if (t > 0) ok = mbar_wait_to(&bars->pvdone[MT - 1], (t - 1) & 1, kErrTimeoutTmemEmpty, a.err);
          if (ok) issue_s(t + 1);
        }
        ok = ok && mbar_wait_to(&bars->vready[b], (t >> 1) & 1, kErrTimeoutFull, a.err);
        for (int x = 0; x < MT && ok; ++x) {
          ok = mbar_wait_to(&bars->pready[x][b], (t >> 1) & 1, kErrTimeoutTmemFull, a.err);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < KT / 16; ++kk)
            mma_f16_ts(t_o(x), t_s(x, b) + kk * 8,
                       desc_mnmajor_sw128(sv + b * C::kPlane + kk * 16 * 128, C::kAtom), id_o,
                       (t > 0 || kk > 0) ? 1u : 0u);
          mma_commit(&bars->pvdone[x]);
        }
        if (ok) mma_commit(&bars->vfree[b]);
      }
      mma_commit(&bars->drained);
    }
  } else if (warp < 2 + kConvWarps) {
    const int t = threadIdx.x - 64;
    float c = 0.0f;  // power of two above every value scale so far (0: none)
    uint32_t least = 0x7F800000u;  // bits of the smallest so far
    for (int i = 0; i < n; ++i) {
      const int s = i % kStages, b = i & 1, slot = i % kSlots;
      if (!mbar_wait_warp_to(&bars->raw_full[s], (i / kStages) & 1, kErrTimeoutFull, a.err)) break;
      const uint8_t* raw = smem + C::oRaw + (size_t)s * 2 * C::kRaw;
      const float* rsc = reinterpret_cast<const float*>(smem + C::oRawS) + s * 2 * KT;
      if (i >= 2 && !mbar_wait_warp_to(&bars->kfree[b], ((i >> 1) - 1) & 1, kErrTimeoutEmpty, a.err)) break;
      {
        // scales: every warp finds the tile's largest value scale for itself
        const int valid = a.len - (t_lo + i) * KT;
        const uint32_t gone = bars->gone[s];
        float v0 = lane < valid ? rsc[KT + lane] : 0.0f;
        float v1 = lane + 32 < valid ? rsc[KT + lane + 32] : 0.0f;
        if (gone) {  // nothing was copied for these keys
          if (gone >> (lane >> 4) & 1u) v0 = 0.0f;
          if (gone >> (2 + (lane >> 4)) & 1u) v1 = 0.0f;
        }
        // bits of non-negative floats rise with them (no NaN passes the fmaxf)
        const float mx = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fmaxf(v0, v1), 0.0f))));
        if (mx > c || c == 0.0f) {
          // four times the next power of two, between 2^-100 and 2^100
          const int ex = min(max((int)(__float_as_uint(mx) >> 23) + 3, 27), 227);
          c = __uint_as_float((uint32_t)ex << 23);
        }
        least = min(least, __reduce_min_sync(0xffffffffu, min(lane < valid ? __float_as_uint(v0) : least,
                                                              lane + 32 < valid ? __float_as_uint(v1) : least)));
        float* sl = sc_slots + slot * (2 * KT + 4);
        if (warp < 4) {  // the first two of these warps: 32 keys each
          const int j = (warp - 2) * 32 + lane;
          sl[j] = j < valid ? rsc[j] * a.scale_log2 : 0.0f;
          sl[KT + j] = (warp == 2 ? v0 : v1) * (kRoom / c);
        } else if (warp == 4 && lane == 0) {
          const bool wide = __uint_as_float(least) < c * kWide;
          *reinterpret_cast<float4*>(sl + 2 * KT) =
              make_float4((float)((int)(__float_as_uint(c) >> 23) - 127), __uint_as_float(gone),
                          __uint_as_float(wide), 0.0f);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->scready[slot]);
      }
      unpack_tile<BITS, D>(raw, smem + C::oK + b * C::kPlane, t);
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->kready[b]);
      if (i >= 2 && !mbar_wait_warp_to(&bars->vfree[b], ((i >> 1) - 1) & 1, kErrTimeoutEmpty, a.err)) break;
      unpack_tile<BITS, D>(raw + C::kRaw, smem + C::oV + b * C::kPlane, t);
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bars->vready[b]);
        mbar_arrive(&bars->raw_empty[s]);
      }
    }
  } else {
    const int x = (warp - 2 - kConvWarps) >> 2, q4 = warp & 3;
    const int lr = q4 * 32 + lane, row = r0 + x * 128 + lr;
    const uint32_t lane_sel = (uint32_t)(q4 * 32) << 16;
    const bool live = row < rows;
    int64_t id = 0;  // output row
    if (live) {
      const int b = row / (a.T * a.G), rr = row - b * a.T * a.G, t = rr / a.G;
      id = ((int64_t)b * a.T + t) * ((int64_t)a.H * a.G) + (int64_t)h * a.G + (rr - t * a.G);
    }
    // ── Q row: bf16 -> fp16 under a power of two, columns in unpack order ──
    float rowf;
    {
      const uint4* qp = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.q) + id * D);
      uint4 raw[D / 8];
#pragma unroll
      for (int ch = 0; ch < D / 8; ++ch) raw[ch] = __ldg(qp + ch);
      float top = 0.0f;
#pragma unroll
      for (int ch = 0; ch < D / 8; ++ch) {
        const uint32_t w[4] = {raw[ch].x, raw[ch].y, raw[ch].z, raw[ch].w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w[i] << 16)),
                                 fabsf(__uint_as_float(w[i] & 0xffff0000u))));
      }
      const int ex = (int)(__float_as_uint(top) >> 23);
      const int up = !live || ex == 0 || ex == 255 ? 127 : min(127 + 14 + 127 - ex, 227);
      const float f = live ? __uint_as_float((uint32_t)up << 23) : 0.0f;
      rowf = __uint_as_float((uint32_t)(254 - up) << 23);
      uint8_t* dst = smem + (size_t)x * C::kQ;
#pragma unroll
      for (int ch = 0; ch < D / 8; ++ch) {
        const uint32_t w[4] = {raw[ch].x, raw[ch].y, raw[ch].z, raw[ch].w};
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[2 * i] = live ? __uint_as_float(w[i] << 16) * f : 0.0f;
          v[2 * i + 1] = live ? __uint_as_float(w[i] & 0xffff0000u) * f : 0.0f;
        }
        const uint4 o = make_uint4(hf2(v[order<BITS>(0)], v[order<BITS>(1)]),
                                   hf2(v[order<BITS>(2)], v[order<BITS>(3)]),
                                   hf2(v[order<BITS>(4)], v[order<BITS>(5)]),
                                   hf2(v[order<BITS>(6)], v[order<BITS>(7)]));
        *reinterpret_cast<uint4*>(dst + (ch >> 3) * C::kQAtom + lr * 128 + (((ch & 7) ^ (lr & 7)) << 4)) = o;
      }
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->qready);
    }
    Row r;
    const RowTiles w = {bars, sc_slots, t_s(x, 0) + lane_sel, x, lane, a.len - t_lo * KT, rowf, a.err};
    int t = 0;
    while (t < n && softmax_tile<D, false>(r, w, t)) ++t;
    if (t < n && r.ok) r = wide_tiles<D>(r, w, t, n);  // the scales' range only grows
    // ── this split's part ──
    if (r.ok && n > 0) mbar_wait_warp_to(&bars->pvdone[x], (n - 1) & 1, kErrTimeoutDone, a.err);
    tc_fence_after();
    const int64_t pr = (int64_t)blockIdx.x * a.n_rows + id;
#pragma unroll 1
    for (int d = 0; d < D; d += 32) {
      uint32_t v[32];
      if (n > 0) {
        tmem_ld32(t_o(x) + lane_sel + d, v);
        tmem_wait_ld();
        tmem_landed(v);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0u;
      }
      if (live) {
#pragma unroll
        for (int g8 = 0; g8 < 32; g8 += 8) {
          float o[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) o[order<BITS>(i)] = __uint_as_float(v[g8 + i]);
          // a whole 32-byte sector a lane
          asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(
                           a.o + pr * D + d + g8),
                       "f"(o[0]), "f"(o[1]), "f"(o[2]), "f"(o[3]), "f"(o[4]), "f"(o[5]), "f"(o[6]),
                       "f"(o[7])
                       : "memory");
        }
      }
    }
    if (live) {
      // O = 2^m' sum: m' = m + log2(c / room)
      reinterpret_cast<float4*>(a.ml)[pr] =
          r.m_top == -INFINITY ? make_float4(-INFINITY, r.l, -INFINITY, 0.0f)  // l: 0, or of NaN scores
                             : make_float4(r.mu, r.l, r.mu + (r.lc - 6.0f), 0.0f);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    if (n > 0) mbar_wait_warp_to(&bars->drained, 0, kErrTimeoutDone, a.err);
    tc_fence_after();
    tmem_dealloc(tbase, C::kCols);
  }
}

template <int BITS, int D, int MT>
int launch(const CUtensorMap& tk, const CUtensorMap& tv, const PrefixArgs& a, int box, cudaStream_t st) {
  using C = Cfg<BITS, D, MT>;
  auto kern = prefix_attn_kernel<BITS, D, MT>;
  static_assert(C::kSmem <= 227 * 1024, "shared memory");
  MXB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem));
  const dim3 grid((unsigned)a.splits, (unsigned)cdiv((int64_t)a.B * a.T * a.G, 128 * MT), (unsigned)a.H);
  MXB_CUDA_TRY(launch_pdl(kern, grid, C::kThreads, C::kSmem, st, tk, tv, a, box));
  MXB_LAUNCH_CHECK();
  return MXB_OK;
}

template <int BITS, int D>
int launch_mt(const CUtensorMap& tk, const CUtensorMap& tv, const PrefixArgs& a, int box, cudaStream_t st) {
  return prefix_rows_per_cta((int64_t)a.B * a.T * a.G) == 256 ? launch<BITS, D, 2>(tk, tv, a, box, st)
                                                              : launch<BITS, D, 1>(tk, tv, a, box, st);
}

}  // namespace pfx

int prefix_rows_per_cta(int64_t rows) { return rows > 128 ? 256 : 128; }

int prefix_attention(const PrefixArgs& a, cudaStream_t st) {
  CUtensorMap tk, tv;
  const int page = 1 << a.page_shift, box = page < pfx::KT ? page : pfx::KT;
  const uint64_t rb = (uint64_t)a.dim * a.bits / 8, lines = (uint64_t)a.n_pages * a.H * page * rb / 128;
  const uint32_t box_lines = (uint32_t)(box * rb / 128);
  if (!encode_tmap_2d(&tk, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.k_codes, 128, lines, 128, box_lines,
                      CU_TENSOR_MAP_SWIZZLE_NONE) ||
      !encode_tmap_2d(&tv, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.v_codes, 128, lines, 128, box_lines,
                      CU_TENSOR_MAP_SWIZZLE_NONE))
    return MXB_E_CUDA;
  if (a.bits == 8)
    return a.dim == 128 ? pfx::launch_mt<8, 128>(tk, tv, a, box, st)
                        : pfx::launch_mt<8, 64>(tk, tv, a, box, st);
  return a.dim == 128 ? pfx::launch_mt<4, 128>(tk, tv, a, box, st)
                      : pfx::launch_mt<4, 64>(tk, tv, a, box, st);
}

}  // namespace mxb
