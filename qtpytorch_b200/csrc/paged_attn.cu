// Attention over the paged quantized KV cache, with a prefix that the whole
// batch shares read once for all.
//
//   s_j = scale * sk_j (q . kc_j),  o = sum_j exp(s_j - m) sv_j vc_j / sum_j exp(s_j - m)
//
// with int8 / int4 codes kc, vc and one scale per key and head.  The codes are
// small integers, exact in bf16: they go to the MMAs as they are, sk_j
// multiplies a score and sv_j a probability, so a key costs two fp32
// multiplies a row instead of 2 D.  One pass with a running maximum and sum;
// both, and the outputs, are fp32.  Probabilities are rounded to bf16 for
// their product (2^-9 relative each, as the output itself is).
//
// The problem is bound by the bytes of the codes for few query rows.  A warp
// is on its own: it walks tiles of 32 keys through a private ring of shared
// memory that its own lanes fill by TMA (the pool is a matrix of head rows, a
// box never leaves a page), so there is no block-wide barrier in the loop and
// all of a CTA's rings are in flight at once.  The products run transposed,
// S^T = K Q^T and O^T = V^T P^T: keys (then head dims) take the 16 rows of the
// MMA and query rows its 8 columns, so 8 grouped heads waste nothing.  K rows
// and V columns come from ldmatrix as 16-bit pairs of codes, and the order of
// the contraction index is permuted (the same for Q) to what the byte order of
// the codes gives, so that unpacking is two or three instructions a pair.
//
// Work is split over keys when there are few rows; partial results (m, l, O)
// are joined by a second kernel, as are the prefix's and the sequences' own.
#include "mxb_common.cuh"
#include "mxb_internal.h"

#include <cuda.h>

#define MXB_ERROR_WORD_BY_POINTER
#include "tc_ptx.cuh"

using namespace mxb;

namespace mxb {
namespace pattn {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kTile = 32;    // keys per warp tile
constexpr int kStages = 3;

template <int BITS, int D>
struct Geo {
  static constexpr int RB = D * BITS / 8;       // bytes of a head row: 128, 64 or 32
  static constexpr int kTileBytes = kTile * RB;
  static constexpr int kRing = kStages * (2 * kTileBytes + 2 * kTile * 4);
  static constexpr CUtensorMapSwizzle kSwz = RB == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                                             : RB == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                        : CU_TENSOR_MAP_SWIZZLE_32B;
  // byte offset of 16-byte chunk c of row r in a tile (the TMA swizzle)
  __device__ static uint32_t at(int r, int c) {
    const int x = RB == 128 ? (r & 7) : RB == 64 ? ((r >> 1) & 3) : ((r >> 2) & 1);
    return (uint32_t)(r * RB + ((c ^ x) << 4));
  }
};

struct Args {
  const __nv_bfloat16* q;  // [B][T][Hq][D]
  const float* ks;
  const float* vs;
  const int* table;        // [B][width] (sequences) or [width] (prefix)
  const int* lengths;      // null: the prefix
  int64_t n_pages;
  int width, page_shift, box;
  int B, T, H, G;
  int prefix_len;
  int rows;                // query rows per unit (T * G, or B * T * G for the prefix)
  int row_tiles;           // per unit and KV head
  int splits;
  float scale_log2;
  // outputs: partials [part][row][D] / [part][row][2], or the result itself
  float* po;
  float* pml;
  int part0;
  int64_t n_rows;          // B * T * Hq
  __nv_bfloat16* out;      // direct result (one part), else null
  float* lse;
  int* err;
};

__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ uint32_t movm(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t bsub2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t bf2(float lo, float hi) {
  const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&t);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Bytes 0 and 2 of w, two's complement int8 -> bf16 pair: with u the low seven
// bits and s the sign, (128 + u) - (128 + 128 s), all three exact in bf16.
__device__ __forceinline__ uint32_t i8pair(uint32_t w) {
  return bsub2((w & 0x007F007Fu) | 0x43004300u, (w & 0x00800080u) | 0x43004300u);
}
// Low nibbles of both halves of w, two's complement int4 -> bf16 pair:
// (128 + (code + 8)) - 136.
__device__ __forceinline__ uint32_t i4pair(uint32_t w) {
  return bsub2((w & 0x000F000Fu) ^ 0x43084308u, 0x43084308u);
}

// Index within a 16-value contraction step of the pairs that the code bytes
// give: the k-th value (0..7 of the lane's eight a 32-value chunk, 0..3 of the
// four a 16-value chunk) that pair p (b0 / b1 of step st) holds.
template <int BITS>
__device__ __forceinline__ int qdim(int step, int c, int pair, int e) {
  if (BITS == 8) return step * 16 + 4 * c + pair + 2 * e;  // bytes (0, 2), then (1, 3)
  const int i = (step & 1) * 2 + pair;                     // nibbles (i, i + 4)
  return (step >> 1) * 32 + 8 * c + i + 4 * e;
}

template <int BITS, int D, int NT>
__global__ void __launch_bounds__(kThreads)
    paged_attn_kernel(const __grid_constant__ CUtensorMap tmap_k,
                      const __grid_constant__ CUtensorMap tmap_v, const Args a) {
  using Ge = Geo<BITS, D>;
  constexpr int kSteps = D / 16, kMT = D / 16;
  constexpr int R = 8 * NT;  // query rows per CTA
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  __shared__ uint64_t full[kWarps][kStages];
  __shared__ float sm_m[kWarps][R], sm_l[kWarps][R];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;

  pdl_trigger();
  pdl_wait();
  const int split = blockIdx.x;
  const int h = blockIdx.y / a.row_tiles, r0 = (blockIdx.y % a.row_tiles) * R;
  const int unit = blockIdx.z;
  const bool own = a.lengths != nullptr;
  int len = own ? a.lengths[unit] : a.prefix_len;
  const int64_t cap = (int64_t)a.width << a.page_shift;
  if (len > cap) {
    if (threadIdx.x == 0 && a.err) atomicCAS(a.err, 0, kErrIndex);
    len = (int)cap;
  }
  len = max(len, 0);
  const int tiles = (len + kTile - 1) / kTile;
  const int per = (tiles + a.splits - 1) / a.splits;
  const int t_lo = min(split * per, tiles), t_hi = min(t_lo + per, tiles);
  const int* table = a.table + (own ? (int64_t)unit * a.width : 0);

  // ring of this warp: [stages][K tile][V tile], then the scales
  uint8_t* ring = smem + warp * (kStages * 2 * Ge::kTileBytes);
  float* rs = reinterpret_cast<float*>(smem + kWarps * kStages * 2 * Ge::kTileBytes) +
              warp * (kStages * 2 * kTile);
  const int boxes = kTile / a.box;
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&full[warp][s], boxes);
    fence_barrier_init();
  }
  __syncwarp();

  const int page_mask = (1 << a.page_shift) - 1;
  // page numbers are fetched one tile before the copies that need them
  auto page_of = [&](int tile) -> int {
    const int pos = tile * kTile + lane * a.box;
    if (lane >= boxes || tile >= t_hi || pos >= len) return -1;
    int p = __ldg(table + (pos >> a.page_shift));
    if (p < 0 || p >= a.n_pages) {
      if (a.err) atomicCAS(a.err, 0, kErrIndex);
      p = 0;
    }
    return p;
  };
  auto issue = [&](int tile, int s, int p) {
    if (lane < boxes) {
      if (p >= 0) {
        const int pos = tile * kTile + lane * a.box;
        const int row = ((p * a.H + h) << a.page_shift) + (pos & page_mask);
        const uint32_t bytes = (uint32_t)a.box * (2 * Ge::RB + 8);
        uint8_t* k = ring + s * 2 * Ge::kTileBytes + lane * a.box * Ge::RB;
        float* sc = rs + s * 2 * kTile + lane * a.box;
        uint64_t* bar = &full[warp][s];
        mbar_expect_tx(bar, bytes);
        tma_load_2d(k, &tmap_k, bar, 0, row);
        tma_load_2d(k + Ge::kTileBytes, &tmap_v, bar, 0, row);
        bulk_load_g2s(sc, a.ks + row, (uint32_t)a.box * 4, bar);
        bulk_load_g2s(sc + kTile, a.vs + row, (uint32_t)a.box * 4, bar);
      } else {
        mbar_arrive(&full[warp][s]);
      }
    }
  };

  // fill the ring
  int next_page = -1;
  {
    int pg[kStages];
#pragma unroll
    for (int s = 0; s < kStages; ++s) pg[s] = page_of(t_lo + warp + s * kWarps);
#pragma unroll
    for (int s = 0; s < kStages; ++s)
      if (t_lo + warp + s * kWarps < t_hi) issue(t_lo + warp + s * kWarps, s, pg[s]);
    next_page = page_of(t_lo + warp + kStages * kWarps);
  }

  // query rows as B fragments (columns = rows r0 + 8 n + g), and the number
  // of keys that each of this lane's two columns per n-tile sees
  uint32_t qf[NT][kSteps][2];
  int limit[NT][2];
  int lim_min = len;
  auto row_id = [&](int r, int& t) -> int64_t {  // row of the unit -> row of the output
    int b = unit, rr = r;
    if (!own) {
      b = r / (a.T * a.G);
      rr = r - b * a.T * a.G;
    }
    t = rr / a.G;
    return ((int64_t)b * a.T + t) * ((int64_t)a.H * a.G) + (int64_t)h * a.G + (rr - t * a.G);
  };
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = r0 + 8 * n + g;
    int t;
    const bool live = r < a.rows;
    const __nv_bfloat16* qp = a.q + (live ? row_id(r, t) : 0) * D;
#pragma unroll
    for (int st = 0; st < kSteps; ++st)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const uint16_t lo = live ? __bfloat16_as_ushort(qp[qdim<BITS>(st, c, p, 0)]) : 0;
        const uint16_t hi = live ? __bfloat16_as_ushort(qp[qdim<BITS>(st, c, p, 1)]) : 0;
        qf[n][st][p] = (uint32_t)lo | ((uint32_t)hi << 16);
      }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int rr = r0 + 8 * n + 2 * c + e;
      limit[n][e] = len;
      if (own && rr < a.rows) limit[n][e] = len - (a.T - 1 - rr / a.G);
    }
  }
  if (own) lim_min = len - (a.T - 1);

  float o[kMT][NT][4];
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int j = 0; j < kMT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[j][n][e] = 0.0f;
    m[n][0] = m[n][1] = -INFINITY;
    l[n][0] = l[n][1] = 0.0f;
  }

  bool ok = true;
  int it = 0;
  for (int tile = t_lo + warp; tile < t_hi; tile += kWarps, ++it) {
    const int s = it % kStages;
    ok = mbar_wait_warp_to(&full[warp][s], (it / kStages) & 1, kErrTimeoutFull, a.err);
    if (!ok) break;
    const uint32_t kt = smem_u32(ring + s * 2 * Ge::kTileBytes);
    const uint32_t vt = kt + Ge::kTileBytes;
    const float* sc = rs + s * 2 * kTile;

    // ── S^T = K Q^T: 32 keys x R rows ──
    float sa[2][NT][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sa[mt][n][e] = 0.0f;
#pragma unroll
    for (int j = 0; j < Ge::RB / 16; ++j) {
      uint32_t w[4];
      ldsm4(kt + Ge::at(lane, j), w);
      if constexpr (BITS == 8) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const uint32_t a0 = i8pair(w[2 * mt]), a1 = i8pair(w[2 * mt + 1]);
          const uint32_t a2 = i8pair(w[2 * mt] >> 8), a3 = i8pair(w[2 * mt + 1] >> 8);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816(sa[mt][n], a0, a1, a2, a3, qf[n][j][0], qf[n][j][1]);
        }
      } else {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const uint32_t a0 = i4pair(w[2 * mt] >> (8 * z)), a1 = i4pair(w[2 * mt + 1] >> (8 * z));
            const uint32_t a2 = i4pair(w[2 * mt] >> (8 * z + 4));
            const uint32_t a3 = i4pair(w[2 * mt + 1] >> (8 * z + 4));
#pragma unroll
            for (int n = 0; n < NT; ++n)
              mma16816(sa[mt][n], a0, a1, a2, a3, qf[n][2 * j + z][0], qf[n][2 * j + z][1]);
          }
      }
    }
    // ── scores, running maximum ──
    float kscale[4], vscale[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      kscale[i] = sc[8 * i + g] * a.scale_log2;
      vscale[i] = sc[kTile + 8 * i + g];
    }
    const int key0 = tile * kTile + g;
    const bool ragged = (tile + 1) * kTile > lim_min;  // some key is hidden from some row
    uint32_t pb[2][NT][2];
    bool grew = false;
    float alpha[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float& v = sa[i >> 1][n][(i & 1) * 2 + e];
          v *= kscale[i];
          if (ragged && key0 + 8 * i >= limit[n][e]) v = -INFINITY;
          mx[e] = fmaxf(mx[e], v);
        }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], w));
        const float mn = fmaxf(m[n][e], mx[e]);
        const float mu = mn == -INFINITY ? 0.0f : mn;  // no key yet: every weight is 0
        alpha[n][e] = ex2(m[n][e] - mu);
        grew |= mn != m[n][e];
        m[n][e] = mn;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float& v = sa[i >> 1][n][(i & 1) * 2 + e];
          const float p = ex2(v - mu);
          sum += p;
          // a hidden key's scale may be anything, NaN included
          v = (ragged && key0 + 8 * i >= limit[n][e]) ? 0.0f : p * vscale[i];
        }
        l[n][e] = l[n][e] * alpha[n][e] + sum;
      }
      // keys x rows -> rows x keys: the B fragment of the second product
#pragma unroll
      for (int i = 0; i < 4; ++i)
        pb[i >> 1][n][i & 1] = movm(bf2(sa[i >> 1][n][(i & 1) * 2], sa[i >> 1][n][(i & 1) * 2 + 1]));
    }
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
      for (int j = 0; j < kMT; ++j)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          o[j][n][0] *= alpha[n][0];
          o[j][n][1] *= alpha[n][1];
          o[j][n][2] *= alpha[n][0];
          o[j][n][3] *= alpha[n][1];
        }
    }
    // ── O^T += V^T P^T ──
#pragma unroll
    for (int j = 0; j < Ge::RB / 16; ++j) {
      uint32_t w[4];
      ldsm4t(vt + Ge::at(lane, j), w);
      if constexpr (BITS == 8) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const uint32_t a0 = i8pair(w[2 * mt]), a1 = i8pair(w[2 * mt] >> 8);
          const uint32_t a2 = i8pair(w[2 * mt + 1]), a3 = i8pair(w[2 * mt + 1] >> 8);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816(o[j][n], a0, a1, a2, a3, pb[mt][n][0], pb[mt][n][1]);
        }
      } else {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const uint32_t a0 = i4pair(w[2 * mt] >> (8 * z)), a1 = i4pair(w[2 * mt] >> (8 * z + 4));
            const uint32_t a2 = i4pair(w[2 * mt + 1] >> (8 * z));
            const uint32_t a3 = i4pair(w[2 * mt + 1] >> (8 * z + 4));
#pragma unroll
            for (int n = 0; n < NT; ++n)
              mma16816(o[2 * j + z][n], a0, a1, a2, a3, pb[mt][n][0], pb[mt][n][1]);
          }
      }
    }
    __syncwarp();  // the stage is read
    const int nt = tile + kStages * kWarps;
    if (nt < t_hi) {
      issue(nt, s, next_page);
      next_page = page_of(nt + kWarps);
    }
  }

  // ── join the warps ──
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], w);
      if (g == 0) {
        sm_m[warp][8 * n + 2 * c + e] = m[n][e];
        sm_l[warp][8 * n + 2 * c + e] = l[n][e];
      }
    }
  __syncthreads();  // every ring is idle
  constexpr int P = D + 4;  // row pitch in floats
  float* so = reinterpret_cast<float*>(smem) + warp * R * P;
#pragma unroll
  for (int j = 0; j < kMT; ++j) {
    // dims of this lane's accumulator rows g and g + 8
    const int d = BITS == 8 ? 16 * j + 2 * g : 32 * (j >> 1) + 4 * g + 2 * (j & 1);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        *reinterpret_cast<float2*>(so + (8 * n + 2 * c + e) * P + d) =
            make_float2(o[j][n][e], o[j][n][2 + e]);
  }
  __syncthreads();
  const float* s0 = reinterpret_cast<const float*>(smem);
  for (int u = threadIdx.x; u < R * (D / 4); u += kThreads) {
    const int r = u / (D / 4), d = (u % (D / 4)) * 4;
    if (r0 + r >= a.rows) break;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, sm_m[w][r]);
    const float mu = mx == -INFINITY ? 0.0f : mx;
    float sum = 0.0f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = ex2(sm_m[w][r] - mu);
      const float4 x = *reinterpret_cast<const float4*>(s0 + (w * R + r) * P + d);
      sum += f * sm_l[w][r];
      v.x += f * x.x; v.y += f * x.y; v.z += f * x.z; v.w += f * x.w;
    }
    int t;
    const int64_t id = row_id(r0 + r, t);
    if (a.out) {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      *reinterpret_cast<uint2*>(a.out + id * D + d) =
          make_uint2(bf2(v.x * inv, v.y * inv), bf2(v.z * inv, v.w * inv));
      if (a.lse && d == 0)
        a.lse[id] = sum == 0.0f ? -INFINITY : (mu + __log2f(sum)) * 0.69314718055994531f;
    } else {
      const int64_t pr = (int64_t)(a.part0 + split) * a.n_rows + id;
      *reinterpret_cast<float4*>(a.po + pr * D + d) = v;
      if (d == 0) *reinterpret_cast<float2*>(a.pml + pr * 2) = make_float2(mx, sum);
    }
  }
}

// One warp a row: joins the parts in order.
template <int D>
__global__ void __launch_bounds__(128)
    paged_join_kernel(const float* __restrict__ po, const float* __restrict__ pml, int parts,
                      int64_t n_rows, __nv_bfloat16* __restrict__ out, float* __restrict__ lse) {
  const int64_t row = blockIdx.x * (int64_t)4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  pdl_trigger();
  pdl_wait();
  if (row >= n_rows) return;
  constexpr int V = D / 32;
  float mx = -INFINITY;
  for (int p = lane; p < parts; p += 32) mx = fmaxf(mx, pml[((int64_t)p * n_rows + row) * 2]);
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
  const float mu = mx == -INFINITY ? 0.0f : mx;
  float sum = 0.0f, v[V];
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = 0.0f;
  for (int p = 0; p < parts; ++p) {
    const int64_t pr = (int64_t)p * n_rows + row;
    const float2 ml = *reinterpret_cast<const float2*>(pml + pr * 2);
    const float f = ex2(ml.x - mu);
    sum += f * ml.y;
    if (f == 0.0f && ml.y == ml.y) continue;  // an empty or vanishing part
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] += f * po[pr * D + lane * V + i];
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  __nv_bfloat16* o = out + row * D + lane * V;
#pragma unroll
  for (int i = 0; i < V; i += 2) *reinterpret_cast<uint32_t*>(o + i) = bf2(v[i] * inv, v[i + 1] * inv);
  if (lse && lane == 0)
    lse[row] = sum == 0.0f ? -INFINITY : (mu + __log2f(sum)) * 0.69314718055994531f;
}

template <int BITS, int D, int NT>
int launch(const CUtensorMap& tk, const CUtensorMap& tv, const Args& a, int units, cudaStream_t st) {
  auto kern = paged_attn_kernel<BITS, D, NT>;
  constexpr size_t ring = (size_t)kWarps * Geo<BITS, D>::kRing;
  constexpr size_t join = (size_t)kWarps * 8 * NT * (D + 4) * 4;
  constexpr size_t smem = 1024 + (ring > join ? ring : join);
  MXB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  MXB_CUDA_TRY(launch_pdl(kern, dim3((unsigned)a.splits, (unsigned)(a.row_tiles * a.H), (unsigned)units),
                          kThreads, smem, st, tk, tv, a));
  MXB_LAUNCH_CHECK();
  return MXB_OK;
}

template <int BITS, int D>
int launch_nt(const CUtensorMap& tk, const CUtensorMap& tv, const Args& a, int nt, int units,
              cudaStream_t st) {
  switch (nt) {
    case 1: return launch<BITS, D, 1>(tk, tv, a, units, st);
    case 2: return launch<BITS, D, 2>(tk, tv, a, units, st);
    default: return launch<BITS, D, 4>(tk, tv, a, units, st);
  }
}

int launch_any(const CUtensorMap& tk, const CUtensorMap& tv, const Args& a, int bits, int dim,
               int nt, int units, cudaStream_t st) {
  if (bits == 8)
    return dim == 128 ? launch_nt<8, 128>(tk, tv, a, nt, units, st)
                      : launch_nt<8, 64>(tk, tv, a, nt, units, st);
  return dim == 128 ? launch_nt<4, 128>(tk, tv, a, nt, units, st)
                    : launch_nt<4, 64>(tk, tv, a, nt, units, st);
}

// How a call is cut: column tiles of 8 query rows per CTA, CTAs per unit over
// the keys.
struct Plan {
  int nt_own, tiles_own, splits_own;  // the sequences' own keys (0 splits: none)
  int nt_pre, tiles_pre, splits_pre;  // the shared prefix
  int parts() const { return splits_own + splits_pre; }
};

int nt_of(int64_t rows) { return rows <= 8 ? 1 : rows <= 16 ? 2 : 4; }

// Splits over the keys until two CTAs an SM are busy, each with at least one
// tile a warp.
int splits_of(int64_t units, int64_t keys) {
  const int64_t most = cdiv(keys, kTile * kWarps);
  int64_t s = cdiv(2 * kSMs, units);
  s = s < most ? s : most;
  return (int)(s < 1 ? 1 : s > 128 ? 128 : s);
}

Plan make_plan(int64_t B, int64_t T, int64_t H, int64_t G, int64_t max_keys, int64_t prefix) {
  Plan p = {};
  p.nt_own = nt_of(T * G);
  p.tiles_own = (int)cdiv(T * G, 8 * p.nt_own);
  // with no own keys possible the sequences' launch still writes the empty rows
  if (max_keys > 0 || prefix == 0) p.splits_own = splits_of(B * H * p.tiles_own, max_keys);
  if (prefix > 0) {
    p.nt_pre = nt_of(B * T * G);
    p.tiles_pre = (int)cdiv(B * T * G, 8 * p.nt_pre);
    p.splits_pre = splits_of(H * p.tiles_pre, prefix);
  }
  return p;
}

}  // namespace pattn
}  // namespace mxb

extern "C" {

size_t mxb_paged_attention_workspace_size(int64_t B, int64_t T, int heads, int group, int dim,
                                          int page, int64_t width, int64_t prefix_len) {
  if (B <= 0 || T <= 0 || heads <= 0 || group <= 0 || dim <= 0 || page <= 0) return 0;
  const pattn::Plan p = pattn::make_plan(B, T, heads, group, width * page, prefix_len);
  if (p.parts() <= 1) return 0;
  return (size_t)p.parts() * (size_t)(B * T * heads * group) * (size_t)(dim + 2) * sizeof(float);
}

int mxb_paged_attention(const void* q, int64_t B, int64_t T, int heads, int group, int dim,
                        const void* k_codes, const float* k_scales, const void* v_codes,
                        const float* v_scales, int64_t n_pages, int page, int bits,
                        const int* table, int64_t width, const int* lengths,
                        const int* prefix_table, int64_t prefix_width, int64_t prefix_len,
                        float scale, void* out, float* lse, void* workspace,
                        size_t workspace_bytes, void* stream) {
  const int rc = kv_pool_check(n_pages, heads, page, dim, bits, k_codes, k_scales, v_codes, v_scales);
  if (rc != MXB_OK) return rc;
  if (B < 0 || B > 65535 || T < 0 || T > 65535 || group <= 0 || group > 1024 || width < 0 ||
      prefix_len < 0 || width * page > INT32_MAX - 64 || prefix_len > INT32_MAX - 64 ||
      prefix_len > prefix_width * page || B * T * group > INT32_MAX / 2)
    return MXB_E_SHAPE;
  if (B == 0 || T == 0) return MXB_OK;
  if (!q || !out || !lengths || (width > 0 && !table) || (prefix_len > 0 && !prefix_table))
    return MXB_E_ARG;
  if (((uintptr_t)q | (uintptr_t)out) % 16) return MXB_E_ALIGN;
  const pattn::Plan p = pattn::make_plan(B, T, heads, group, width * page, prefix_len);
  if ((int64_t)p.tiles_own * heads > 65535 || (int64_t)p.tiles_pre * heads > 65535)
    return MXB_E_SHAPE;
  const size_t need =
      mxb_paged_attention_workspace_size(B, T, heads, group, dim, page, width, prefix_len);
  if (need > 0 && (!workspace || workspace_bytes < need)) return MXB_E_WORKSPACE;
  if ((uintptr_t)workspace % 16) return MXB_E_ALIGN;
  cudaStream_t st = static_cast<cudaStream_t>(stream);

  CUtensorMap tk, tv;
  const int box = page < pattn::kTile ? page : pattn::kTile;
  const uint64_t rb = (uint64_t)dim * bits / 8, rows = (uint64_t)n_pages * heads * page;
  const int swz = rb == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                  : rb == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                             : CU_TENSOR_MAP_SWIZZLE_32B;
  if (!encode_tmap_2d(&tk, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, k_codes, rb, rows, (uint32_t)rb, box, swz) ||
      !encode_tmap_2d(&tv, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, v_codes, rb, rows, (uint32_t)rb, box, swz))
    return MXB_E_CUDA;

  pattn::Args a = {};
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.ks = k_scales;
  a.vs = v_scales;
  a.n_pages = n_pages;
  a.page_shift = 31 - __builtin_clz((unsigned)page);
  a.box = box;
  a.B = (int)B;
  a.T = (int)T;
  a.H = heads;
  a.G = group;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.n_rows = B * T * heads * group;
  a.err = device_error_ptr();
  const bool direct = p.parts() == 1;
  a.out = direct ? static_cast<__nv_bfloat16*>(out) : nullptr;
  a.lse = direct ? lse : nullptr;
  a.po = static_cast<float*>(workspace);
  a.pml = a.po ? a.po + (size_t)p.parts() * a.n_rows * dim : nullptr;
  if (p.splits_pre > 0) {
    a.table = prefix_table;
    a.lengths = nullptr;
    a.width = (int)prefix_width;
    a.prefix_len = (int)prefix_len;
    a.rows = (int)(B * T * group);
    a.row_tiles = p.tiles_pre;
    a.splits = p.splits_pre;
    a.part0 = p.splits_own;
    const int r = pattn::launch_any(tk, tv, a, bits, dim, p.nt_pre, 1, st);
    if (r != MXB_OK) return r;
  }
  if (p.splits_own > 0) {
    a.table = table;
    a.lengths = lengths;
    a.width = (int)width;
    a.prefix_len = 0;
    a.rows = (int)(T * group);
    a.row_tiles = p.tiles_own;
    a.splits = p.splits_own;
    a.part0 = 0;
    const int r = pattn::launch_any(tk, tv, a, bits, dim, p.nt_own, (int)B, st);
    if (r != MXB_OK) return r;
  }
  if (!direct) {
    const unsigned grid = (unsigned)cdiv(a.n_rows, 4);
    MXB_CUDA_TRY(launch_pdl(dim == 128 ? pattn::paged_join_kernel<128> : pattn::paged_join_kernel<64>,
                            dim3(grid), 128, 0, st, a.po, a.pml, p.parts(), a.n_rows,
                            static_cast<__nv_bfloat16*>(out), lse));
    MXB_LAUNCH_CHECK();
  }
  return MXB_OK;
}

}  // extern "C"
