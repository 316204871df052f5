// Attention over the paged quantized KV cache, with a prefix that the whole
// batch shares read once for all.
//
//   s_j = scale * sk_j (q . kc_j),  o = sum_j exp(s_j - m) sv_j vc_j / sum_j exp(s_j - m)
//
// with int8 / int4 codes kc, vc and one scale per key and head.  One pass with
// a running maximum and sum; both, and the outputs, are fp32.
//
// The codes are small integers and go to the MMAs as such (bf16 or fp16, both
// exact): sk_j multiplies a score, and sv_j joins the exponent of the weight
// of the second product, exp2(s_j + log2 sv_j - m'), with a running maximum m'
// of its own.  The weights are then at most 1 with a 1 in every row's range,
// so fp16 (11 bits) holds them whatever the scales are, and a key costs a few
// fp32 operations a row instead of 2 D.
//
// For few query rows the bytes of the codes are the bound.  A warp is on its
// own: it walks tiles of 32 keys through a private ring of shared memory that
// its own lanes fill by TMA (the pool is a matrix of head rows, a box never
// leaves a page), so there is no block-wide barrier in the loop and all of a
// CTA's rings are in flight at once.  The products run transposed, S^T = K Q^T
// and O^T = V^T P^T: keys (then head dims) take the 16 rows of the MMA and
// query rows its 8 columns, so 8 grouped heads waste nothing.  K rows and V
// columns come from ldmatrix as 16-bit pairs of codes, and the order of the
// contraction index is permuted (the same for Q) to what the byte order of the
// codes gives.  Unpacking: a mask and an exclusive or put a code under a fixed
// exponent, which leaves code + offset; for K the offset is taken out once, in
// the accumulator's start -offset * sum(q) (in fp32: the D / 16 + 4 additions may
// each be off by 2^-23 of (offset + code) sum|q| sk, offset 1152 or 136), for V by
// one packed subtraction.
//
// Work: the tiles of all sequences, heads and row groups form one list, which
// the CTAs share out in equal runs (lengths are known on the device only), so
// a batch of very different lengths keeps every SM busy to the end; short units
// (make_plan) get a CTA each instead.  A run may hold several units or a part of
// one; a unit's first part goes to a row buffer, a later part to its CTA's
// buffer, and a second kernel joins them with the parts of the shared prefix.
// Rows with a single part are written directly.
//
// 2 x 131072 keys and less, 4 rows of each of 8 heads of 128 dims in int8 (346 MB):
// 69 - 72 us = 4.8 - 5.0 TB/s, 62 without any arithmetic.  24 rows of 64 dims in int4
// take about 1000 instructions a tile for 2 KB of codes and are bound by their latency
// (0.47 issued a cycle with 12 warps an SM): 50 us for 48 x up to 6000 keys.
#include "mxb_common.cuh"
#include "mxb_internal.h"

#include <cuda.h>
#include <cuda_fp16.h>

#define MXB_ERROR_WORD_BY_POINTER
#include "tc_ptx.cuh"

using namespace mxb;

namespace mxb {
namespace pattn {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kTile = 32;    // keys per warp tile

// CTAs per SM, by what their registers and rings leave room for
__host__ __device__ constexpr int ctas(int nt, int rb, int dim) {
  return nt == 1 ? (rb == 32 ? 4 : 3) : (dim == 64 && nt <= 3) ? 3 : 2;
}

template <int BITS, int D, int NT>
struct Geo {
  static constexpr int RB = D * BITS / 8;       // bytes of a head row: 128, 64 or 32
  static constexpr int kTileBytes = kTile * RB;
  // ring depth: 100 to 200 KB in flight an SM
  static constexpr int kCtas = ctas(NT, RB, D);
  static constexpr int kStages = RB == 128 ? (NT >= 2 ? 3 : 2) : RB == 64 ? (kCtas == 2 ? 4 : 3) : 4;
  static constexpr int R = 8 * NT;              // query rows per CTA
  static constexpr int kPitch = D + 4;          // floats of a row in the join buffer
  static constexpr size_t kRing = (size_t)kWarps * kStages * (2 * kTileBytes + 2 * kTile * 4);
  static constexpr size_t kJoin = (size_t)kWarps * R * kPitch * 4;
  // where it fits the join buffer lies beside the ring, so the next unit's
  // loads start before the join
  static constexpr size_t kStatic = 2048 + (NT >= 3 && D == 128 ? 9 * 1024 : 0);
  static constexpr bool kApart = kCtas * (1024 + kRing + kJoin + kStatic) <= 228 * 1024;
  static constexpr size_t kSmem = 1024 + (kApart ? kRing + kJoin : kRing > kJoin ? kRing : kJoin);
  static_assert(kCtas * (kSmem + kStatic) <= 228 * 1024, "CTAs fit an SM");
  // The pool is copied as lines of 128 bytes (one, two or four head rows): the
  // TMA unit takes its time by the line, so 32-byte rows one by one held int4
  // tiles of 64 dims to 285 cycles each.  Byte offset of 16-byte chunk 0 of
  // head row r in a tile under the 128-byte swizzle; chunk c lies at that
  // address ^ (c << 4).
  __device__ static uint32_t at(int r) {
    const uint32_t byte = (uint32_t)(r * RB), line = byte >> 7;
    return (line << 7) | ((((byte >> 4) & 7) ^ (line & 7)) << 4);
  }
};

// Results of a key range: [rows][D] weighted sums relative to 2^m', and
// (m, l, m', 0) per row.
struct Part {
  float* o;
  float4* ml;
};

struct Args {
  const __nv_bfloat16* q;  // [B][T][Hq][D]
  const float* ks;
  const float* vs;
  const int* table;        // [B][width] (sequences) or [width] (prefix)
  const int* lengths;      // null: the prefix
  int64_t n_pages;
  int width, page_shift, box_shift;  // box: keys per copy, a page's or a tile's
  int B, T, H, G;
  int prefix_len;
  int rows;                // query rows per unit (T * G, or B * T * G for the prefix)
  int row_tiles;           // per unit and KV head
  int splits;              // prefix: CTAs over the keys
  float scale_log2;
  Part main, cta;          // sequences: by output row / by CTA; prefix: main by split and row
  int64_t* plan;           // [0] tiles per CTA, [1 + b] first tile of sequence b
  int64_t n_rows;          // B * T * Hq
  bool whole;              // one unit per CTA, no plan
  bool direct;             // rows with one part go straight to out
  __nv_bfloat16* out;
  float* lse;
  int* err;
  // TREE: query t sees newest key i of its sequence where tree[b tree_b + t tree_t + i]
  // is not 0
  const uint8_t* tree;
  int64_t tree_b, tree_t;
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
template <bool HALF>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (HALF)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t hsub2u(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t bf2(float lo, float hi) {
  const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&t);
}
__device__ __forceinline__ uint32_t hf2(float lo, float hi) {
  const __half2 t = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&t);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// Arrive on bar (one of its counted arrivals) when this thread's cp.async are done.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^(x - ref) of a running maximum; nothing seen yet gives 0
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.0f : m; }

// What turns a weighted sum relative to 2^mw into the output: 2^(mw - m) / sum.
// No weight seen (no keys, or value scales of zero): the sum is 0 already, and
// without a reference the power could be infinite.
__device__ __forceinline__ float norm_of(float m, float mw, float sum) {
  return mw == -INFINITY ? 0.0f : ex2(mw - base_of(m)) / sum;
}

// Two codes as 16-bit floats.  K: int8 bytes 0 and 2 of w -> fp16 1152 + code
// ((code + 128) in the mantissa of 1024); int4 low nibbles of both halves ->
// bf16 136 + code ((code + 8) in the mantissa of 128).  V: exact fp16 codes;
// int4 nibble 1 (HI) stays where it is in the mantissa, 16 times its code,
// which saves its shift: the factor leaves with the result.
template <int BITS>
struct Codes;
template <>
struct Codes<8> {
  static constexpr float kOffset = 1152.0f;
  static constexpr bool kHalfQ = true;
  static constexpr float kHiScale = 1.0f;
  __device__ static uint32_t k(uint32_t w) { return (w & 0x00FF00FFu) ^ 0x64806480u; }
  template <bool HI>
  __device__ static uint32_t v(uint32_t w) {
    return hsub2u(k(HI ? w >> 8 : w), 0x64806480u);
  }
};
template <>
struct Codes<4> {
  static constexpr float kOffset = 136.0f;
  static constexpr bool kHalfQ = false;
  static constexpr float kHiScale = 1.0f / 16.0f;
  __device__ static uint32_t k(uint32_t w) { return (w & 0x000F000Fu) ^ 0x43084308u; }
  template <bool HI>
  __device__ static uint32_t v(uint32_t w) {
    return HI ? hsub2u((w & 0x00F000F0u) ^ 0x64806480u, 0x64806480u)
              : hsub2u((w & 0x000F000Fu) ^ 0x64086408u, 0x64086408u);
  }
};

// Sum over the block (kThreads) of one value a thread, and its exclusive prefix.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t& before, int64_t* sm) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t t = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += t;
  }
  if (lane == 31) sm[warp] = inc;
  __syncthreads();
  int64_t total = 0, pre = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) pre += sm[w];
    total += sm[w];
  }
  __syncthreads();
  before = pre + inc - v;
  return total;
}

template <int BITS, int D, int NT, bool TREE>
__global__ void __launch_bounds__(kThreads, Geo<BITS, D, NT>::kCtas)
    paged_attn_kernel(const __grid_constant__ CUtensorMap tmap_k,
                      const __grid_constant__ CUtensorMap tmap_v, const Args a) {
  using Ge = Geo<BITS, D, NT>;
  using Cd = Codes<BITS>;
  constexpr int kSteps = D / 16, kMT = D / 16, kStages = Ge::kStages;
  constexpr int R = Ge::R;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  __shared__ uint64_t full[kWarps][kStages];
  __shared__ float sm_m[kWarps][R], sm_l[kWarps][R], sm_v[kWarps][R];
  __shared__ int64_t sm_scan[kWarps];
  __shared__ int sm_b, sm_off;
  // with many rows the query fragments, the same for all warps, live in
  // shared memory: in registers they would spill
  constexpr bool kQs = NT >= 3 && D == 128;
  __shared__ uint2 sq[kQs ? NT * kSteps * 32 : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;

  // ring of this warp: [stages][K tile][V tile], then the scales
  uint8_t* ring = smem + warp * (kStages * 2 * Ge::kTileBytes);
  float* rs = reinterpret_cast<float*>(smem + kWarps * kStages * 2 * Ge::kTileBytes) +
              warp * (kStages * 2 * kTile);
  float* join = reinterpret_cast<float*>(smem + (Ge::kApart ? Ge::kRing : 0));
  const int box = 1 << a.box_shift, boxes = kTile >> a.box_shift;
  if (lane == 0) {
    // one arrival a box (its copies' bytes), one a lane (its scales)
    for (int s = 0; s < kStages; ++s) mbar_init(&full[warp][s], boxes + 32);
    fence_barrier_init();
  }
  __syncwarp();
  pdl_trigger();
  pdl_wait();

  const bool own = a.lengths != nullptr;
  const int hr = a.H * a.row_tiles;  // units per sequence
  const int64_t cap = (int64_t)a.width << a.page_shift;
  auto len_of = [&](int b) -> int {
    int n = own ? __ldg(a.lengths + b) : a.prefix_len;
    return (int)min((int64_t)max(n, 0), cap);
  };
  auto tiles_of = [&](int n) { return (n + kTile - 1) / kTile; };

  // ── this CTA's run of the tile list ──
  int b = 0, u = 0;             // sequence, unit within it
  int t_lo = 0, t_hi = 0;       // tiles of the current segment
  int64_t left = 0;             // tiles of the run, the segment's included
  int len, n_tiles;
  if (!own) {  // prefix: blockIdx.x = split, blockIdx.y = unit
    u = blockIdx.y;
    len = len_of(0);
    n_tiles = tiles_of(len);
    const int per = (n_tiles + a.splits - 1) / a.splits;
    t_lo = min((int)blockIdx.x * per, n_tiles);
    t_hi = min(t_lo + per, n_tiles);
    left = t_hi - t_lo;
  } else if (a.whole) {
    b = blockIdx.x / hr;
    u = blockIdx.x - b * hr;
    len = len_of(b);
    if (u == 0 && threadIdx.x == 0 && a.err && __ldg(a.lengths + b) > cap)
      atomicCAS(a.err, 0, kErrIndex);
    n_tiles = tiles_of(len);
    t_hi = n_tiles;
    left = n_tiles;
  } else {
    int64_t total = 0, before, n0 = 0, before0 = 0;
    for (int b0 = 0; b0 < a.B; b0 += kThreads) {
      const int i = b0 + threadIdx.x;
      int n = 0;
      if (i < a.B) {
        n = __ldg(a.lengths + i);
        if (n > cap && blockIdx.x == 0 && a.err) atomicCAS(a.err, 0, kErrIndex);
        n = tiles_of((int)min((int64_t)max(n, 0), cap));
      }
      total += block_scan((int64_t)n * hr, before, sm_scan);
      if (b0 == 0) {
        n0 = (int64_t)n * hr;
        before0 = before;
      }
    }
    // equal runs, of a tile a warp or a unit's average length at least: a CTA
    // takes about 5 us a unit, so short units are not put one after another
    auto share = [&](uint32_t n) {
      return (int64_t)(total >> 31 ? (total + n - 1) / n : ((uint32_t)total + n - 1) / n);
    };
    const int64_t per = max(share(gridDim.x), min(share((uint32_t)(a.B * hr)), (int64_t)kWarps));
    const int64_t lo = blockIdx.x * per, hi = min(lo + per, total);
    if (blockIdx.x == 0 && threadIdx.x == 0) a.plan[0] = per;
    int64_t base = 0;
    for (int b0 = 0; b0 < a.B && (blockIdx.x == 0 || base <= lo); b0 += kThreads) {
      const int i = b0 + threadIdx.x;
      int64_t n = n0;
      before = before0;
      if (a.B > kThreads) {  // one scan was not all
        n = i < a.B ? (int64_t)tiles_of(len_of(i)) * hr : 0;
        const int64_t sum = block_scan(n, before, sm_scan);
        before += base;
        base += sum;
      }
      if (i < a.B && blockIdx.x == 0) a.plan[1 + i] = before;
      if (lo < hi && lo >= before && lo < before + n) {
        sm_b = i;
        sm_off = (int)(lo - before);
      }
    }
    __syncthreads();
    if (lo >= hi) return;
    b = sm_b;
    len = len_of(b);
    n_tiles = tiles_of(len);
    u = sm_off / n_tiles;  // a sequence has fewer than 2^31 tiles (checked at the launch)
    t_lo = sm_off - u * n_tiles;
    left = hi - lo;
    t_hi = (int)min((int64_t)n_tiles, t_lo + left);
  }

  const int page_mask = (1 << a.page_shift) - 1;
  const int* table = a.table + (own ? (int64_t)b * a.width : 0);
  // page numbers are fetched one tile before the copies that need them
  auto page_of = [&](int tile) -> int {
    const int pos = tile * kTile + (lane << a.box_shift);
    return lane < boxes && tile < t_hi && pos < len ? __ldg(table + (pos >> a.page_shift)) : 0;
  };
  // Keys behind a number outside the pool are not copied and hidden from every
  // row: once the warp has met one, each tile looks its numbers up again (below).
  bool bad_pages = false;
  auto issue = [&](int tile, int h, int s, int p) {
    const bool used = lane < boxes && tile * kTile + (lane << a.box_shift) < len;
    const bool bad = used && (uint32_t)p >= (uint32_t)a.n_pages;  // n_pages < 2^31
    if (bad && a.err) atomicCAS(a.err, 0, kErrIndex);
    bad_pages = __any_sync(0xffffffffu, bad) || bad_pages;
    if (!used || bad) p = -1;
    uint64_t* bar = &full[warp][s];
    if (lane < boxes) {
      if (p >= 0) {
        const int pos = tile * kTile + (lane << a.box_shift);
        const int row = ((p * a.H + h) << a.page_shift) + (pos & page_mask);
        uint8_t* k = ring + s * 2 * Ge::kTileBytes + (lane << a.box_shift) * Ge::RB;
        mbar_expect_tx(bar, (uint32_t)box * 2 * Ge::RB);
        const int line = row / (128 / Ge::RB);
        tma_load_2d(k, &tmap_k, bar, 0, line);
        tma_load_2d(k + Ge::kTileBytes, &tmap_v, bar, 0, line);
      } else {
        mbar_arrive(bar);
      }
    }
    // a lane's two scales: a bulk copy each would cost the TMA unit as much as
    // a tile of codes (attend_long without them 8 us shorter)
    const int kp = __shfl_sync(0xffffffffu, p, lane >> a.box_shift);
    const int pos = tile * kTile + lane;
    if (kp >= 0) {
      const int row = ((kp * a.H + h) << a.page_shift) + (pos & page_mask);
      float* sc = rs + s * 2 * kTile + lane;
      cp_async4(sc, a.ks + row);
      cp_async4(sc + kTile, a.vs + row);
    }
    cp_async_arrive(bar);
  };
  bool ok = true;  // no wait of this warp gave up
  int next_page = -1;
  int stage = 0;  // ring position of the warp's next tile, and its parity
  uint32_t round = 0;
  const uint32_t lane_at = smem_u32(ring) + Ge::at(lane);
  auto fill = [&]() {
    int pg[kStages];
#pragma unroll
    for (int i = 0; i < kStages; ++i) pg[i] = page_of(t_lo + warp + i * kWarps);
#pragma unroll
    for (int i = 0; i < kStages; ++i)
      if (ok && t_lo + warp + i * kWarps < t_hi)
        issue(t_lo + warp + i * kWarps, u / a.row_tiles,
              stage + i < kStages ? stage + i : stage + i - kStages, pg[i]);
    next_page = page_of(t_lo + warp + kStages * kWarps);
  };
  fill();

  while (true) {
    const int h = u / a.row_tiles, r0 = (u - h * a.row_tiles) * R;
    const bool first = t_lo == 0, last = t_hi == n_tiles;
    auto row_id = [&](int r) -> int64_t {  // row of the unit -> row of the output
      int bb = b, rr = r;
      if (!own) {
        bb = r / (a.T * a.G);
        rr = r - bb * a.T * a.G;
      }
      const int t = rr / a.G;
      return ((int64_t)bb * a.T + t) * ((int64_t)a.H * a.G) + (int64_t)h * a.G + (rr - t * a.G);
    };

    // query rows as B fragments (columns = rows r0 + 8 n + g), the sum that
    // takes the codes' offset out, and how many keys each of this lane's two
    // columns per n-tile sees
    uint32_t qf[NT][kSteps][2];
    float start[NT][2], cfac[NT][2];
    int limit[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = r0 + 8 * n + g;
      const bool live = r < a.rows;
      const uint4* qp = reinterpret_cast<const uint4*>(a.q + (live ? row_id(r) : 0) * D);
      uint32_t raw[kSteps][2];  // bf16 pairs in memory order, 4 values a step
      if (BITS == 8) {
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {  // values 16 st + 4 c ..
          const uint2 w = __ldg(reinterpret_cast<const uint2*>(qp) + st * 4 + c);
          raw[st][0] = w.x;
          raw[st][1] = w.y;
        }
      } else {
#pragma unroll
        for (int j = 0; j < kSteps / 2; ++j) {  // values 32 j + 8 c ..
          const uint4 w = __ldg(qp + j * 4 + c);
          raw[2 * j][0] = w.x;
          raw[2 * j][1] = w.y;
          raw[2 * j + 1][0] = w.z;
          raw[2 * j + 1][1] = w.w;
        }
      }
      float sum = 0.0f, fac = 1.0f;
      if constexpr (BITS == 8) {
        // bf16 -> fp16 under a power of two that puts the row's largest value
        // into [2^14, 2^15): eight bits of every value down to 2^-29 of it
        float top = 0.0f;
#pragma unroll
        for (int st = 0; st < kSteps; ++st)
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            if (!live) raw[st][p] = 0u;
            top = fmaxf(top, fmaxf(fabsf(__uint_as_float(raw[st][p] << 16)),
                                   fabsf(__uint_as_float(raw[st][p] & 0xffff0000u))));
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int ex = (int)(__float_as_uint(top) >> 23);  // biased
        // 2^(14 - (ex - 127)), at most 2^100
        const int up = ex == 0 || ex == 255 ? 127 : min(127 + 14 + 127 - ex, 227);
        const float f = __uint_as_float((uint32_t)up << 23);
        fac = __uint_as_float((uint32_t)(254 - up) << 23);  // its inverse
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
          const float v0 = __uint_as_float(raw[st][0] << 16) * f;
          const float v1 = __uint_as_float(raw[st][0] & 0xffff0000u) * f;
          const float v2 = __uint_as_float(raw[st][1] << 16) * f;
          const float v3 = __uint_as_float(raw[st][1] & 0xffff0000u) * f;
          qf[n][st][0] = hf2(v0, v2);  // bytes 0, 2 of a code word, then 1, 3
          qf[n][st][1] = hf2(v1, v3);
          const float2 s0 = __half22float2(*reinterpret_cast<__half2*>(&qf[n][st][0]));
          const float2 s1 = __half22float2(*reinterpret_cast<__half2*>(&qf[n][st][1]));
          sum += (s0.x + s0.y) + (s1.x + s1.y);
        }
      } else {
#pragma unroll
        for (int j = 0; j < kSteps / 2; ++j) {
          uint32_t x[4] = {raw[2 * j][0], raw[2 * j][1], raw[2 * j + 1][0], raw[2 * j + 1][1]};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (!live) x[i] = 0u;
            sum += __uint_as_float(x[i] << 16) + __uint_as_float(x[i] & 0xffff0000u);
          }
          // values (i, i + 4): nibbles i of the two halves of a code word
          qf[n][2 * j][0] = __byte_perm(x[0], x[2], 0x5410);
          qf[n][2 * j][1] = __byte_perm(x[0], x[2], 0x7632);
          qf[n][2 * j + 1][0] = __byte_perm(x[1], x[3], 0x5410);
          qf[n][2 * j + 1][1] = __byte_perm(x[1], x[3], 0x7632);
        }
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      sum *= -Cd::kOffset;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        start[n][e] = __shfl_sync(0xffffffffu, sum, (2 * c + e) * 4);
        cfac[n][e] = __shfl_sync(0xffffffffu, fac, (2 * c + e) * 4);
        const int rr = r0 + 8 * n + 2 * c + e;
        limit[n][e] = len;
        if (own && rr < a.rows) limit[n][e] = TREE ? len - a.T : len - (a.T - 1 - rr / a.G);
      }
    }
    const int lim_min = own ? len - (TREE ? a.T : a.T - 1) : len;
    if constexpr (kQs) {
      if (warp == 0) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int st = 0; st < kSteps; ++st)
            sq[(n * kSteps + st) * 32 + lane] = make_uint2(qf[n][st][0], qf[n][st][1]);
      }
      __syncthreads();
    }
    auto q_of = [&](int n, int st) -> uint2 {
      if constexpr (kQs) return sq[(n * kSteps + st) * 32 + lane];
      else return make_uint2(qf[n][st][0], qf[n][st][1]);
    };

    float o[kMT][NT][4];
    // references of the sums and of the weights, and the values beyond which
    // they move (-inf: nothing seen)
    float mu[NT][2], l[NT][2], wu[NT][2], m_top[NT][2], w_top[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < kMT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][n][e] = 0.0f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m_top[n][e] = w_top[n][e] = -INFINITY;
        mu[n][e] = wu[n][e] = l[n][e] = 0.0f;
      }
    }

    for (int tile = t_lo + warp; ok && tile < t_hi; tile += kWarps) {
      const int s = stage;
      ok = mbar_wait_warp_to(&full[warp][s], round, kErrTimeoutFull, a.err);
      if (!ok) {
        // the warp's copies in flight, this one among them, before the CTA may
        // end; from here on it only keeps the others' barriers company
#pragma unroll 1
        for (int i = 0; i < kStages && tile + i * kWarps < t_hi; ++i) {
          mbar_wait_warp_to(&full[warp][stage], round, kErrTimeoutFull, a.err);
          if (++stage == kStages) {
            stage = 0;
            round ^= 1u;
          }
        }
        break;
      }
      if (++stage == kStages) {
        stage = 0;
        round ^= 1u;
      }
      const uint32_t kt = lane_at + s * 2 * Ge::kTileBytes;
      const uint32_t vt = kt + Ge::kTileBytes;
      const float* sc = rs + s * 2 * kTile;

      // ── S^T = K Q^T: 32 keys x R rows ──
      float sa[2][NT][4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) sa[mt][n][e] = start[n][e & 1];
#pragma unroll
      for (int j = 0; j < Ge::RB / 16; ++j) {
        uint32_t w[4];
        ldsm4(kt ^ (j << 4), w);
        constexpr int Z = BITS == 8 ? 1 : 2, SH = BITS;  // steps a chunk; shift to the second pair
#pragma unroll
        for (int z = 0; z < Z; ++z) {
          uint32_t f[2][4];
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            f[mt][0] = Cd::k(w[2 * mt] >> (8 * z));
            f[mt][1] = Cd::k(w[2 * mt + 1] >> (8 * z));
            f[mt][2] = Cd::k(w[2 * mt] >> (8 * z + SH));
            f[mt][3] = Cd::k(w[2 * mt + 1] >> (8 * z + SH));
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint2 qv = q_of(n, Z * j + z);
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
              mma16816<Cd::kHalfQ>(sa[mt][n], f[mt][0], f[mt][1], f[mt][2], f[mt][3], qv.x, qv.y);
          }
        }
      }
      // ── scores and the weights' exponents ──
      float kscale[4], lv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        kscale[i] = sc[8 * i + g] * a.scale_log2;
        lv[i] = lg2(sc[kTile + 8 * i + g]);
      }
      // One column tile after the other, to keep few values alive; the two
      // columns of an accumulator pair go through packed operations.
      const int key0 = tile * kTile + g;
      bool ragged = (tile + 1) * kTile > lim_min;  // some key is hidden from some row
      uint32_t hide = 0;  // 16-key halves of the tile behind bad page numbers
      if (bad_pages) {
        ragged = true;
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
          const int key = tile * kTile + 16 * i;
          const int p = key < len ? __ldg(table + (key >> a.page_shift)) : 0;
          hide |= ((uint32_t)p >= (uint32_t)a.n_pages ? 1u : 0u) << i;
        }
      }
      uint32_t pb[2][NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        uint64_t v2[4], w2[4];  // s, s + log2 sv
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint64_t f = pack2(kscale[i], kscale[i]);
          if (BITS == 8) f = fmul2(f, pack2(cfac[n][0], cfac[n][1]));
          v2[i] = fmul2(pack2(sa[i >> 1][n][(i & 1) * 2], sa[i >> 1][n][(i & 1) * 2 + 1]), f);
          w2[i] = fadd2(v2[i], pack2(lv[i], lv[i]));
        }
        if (ragged) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float2 v = unpack2(v2[i]), w = unpack2(w2[i]);
            const int key = (hide >> (i >> 1)) & 1u ? INT32_MAX : key0 + 8 * i;
            if constexpr (TREE) {
              // from limit on the T newest keys, as far as the row's mask names them
              if (key >= limit[n][0]) {
                const int rr = r0 + 8 * n + 2 * c, at = key - limit[n][0];
                const uint8_t* mask = a.tree + b * a.tree_b + at;
                if (key >= len || rr >= a.rows || !__ldg(mask + rr / a.G * a.tree_t)) v.x = w.x = -INFINITY;
                if (key >= len || rr + 1 >= a.rows || !__ldg(mask + (rr + 1) / a.G * a.tree_t))
                  v.y = w.y = -INFINITY;
              }
            } else {
              if (key >= limit[n][0]) v.x = w.x = -INFINITY;  // whatever its scales hold
              if (key >= limit[n][1]) v.y = w.y = -INFINITY;
            }
            v2[i] = pack2(v.x, v.y);
            w2[i] = pack2(w.x, w.y);
          }
        }
        // the references move only when a sum's terms pass 2^64 or a weight 2^8
        // (fp16 holds 2^15), so most tiles need no exchange between lanes
        float mx[2], mw[2];
        bool move = false;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          auto of = [&](uint64_t p) { return e ? unpack2(p).y : unpack2(p).x; };
          mx[e] = fmaxf(fmaxf(of(v2[0]), of(v2[1])), fmaxf(of(v2[2]), of(v2[3])));
          mw[e] = fmaxf(fmaxf(of(w2[0]), of(w2[1])), fmaxf(of(w2[2]), of(w2[3])));
          move |= mx[e] > m_top[n][e] || mw[e] > w_top[n][e];
        }
        if (__any_sync(0xffffffffu, move)) {
          float alpha[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
              mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], x));
              mw[e] = fmaxf(mw[e], __shfl_xor_sync(0xffffffffu, mw[e], x));
            }
            // the larger of the reference (where there is one) and the tile's
            const float m0 = m_top[n][e] == -INFINITY ? -INFINITY : mu[n][e];
            const float w0 = w_top[n][e] == -INFINITY ? -INFINITY : wu[n][e];
            const float m1 = fmaxf(m0, mx[e]), w1 = fmaxf(w0, mw[e]);
            mu[n][e] = base_of(m1);
            wu[n][e] = base_of(w1);
            l[n][e] *= ex2(m0 - mu[n][e]);
            alpha[e] = ex2(w0 - wu[n][e]);
            m_top[n][e] = m1 + 64.0f;
            w_top[n][e] = w1 + 8.0f;
          }
#pragma unroll
          for (int j = 0; j < kMT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][n][e] *= alpha[e & 1];
        }
        // weights: keys x rows -> rows x keys, the B fragment of the second product
        const uint64_t mu2 = pack2(mu[n][0], mu[n][1]), wu2 = pack2(wu[n][0], wu[n][1]);
        uint64_t sum = pack2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 v = unpack2(fsub2(v2[i], mu2)), w = unpack2(fsub2(w2[i], wu2));
          sum = fadd2(sum, pack2(ex2(v.x), ex2(v.y)));
          pb[i >> 1][n][i & 1] = movm(hf2(ex2(w.x), ex2(w.y)));
        }
        l[n][0] += unpack2(sum).x;
        l[n][1] += unpack2(sum).y;
      }
      // ── O^T += V^T P^T ──
#pragma unroll
      for (int j = 0; j < Ge::RB / 16; ++j) {
        uint32_t w[4];
        ldsm4t(vt ^ (j << 4), w);
        constexpr int Z = BITS == 8 ? 1 : 2;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int z = 0; z < Z; ++z) {
            const uint32_t w0 = w[2 * mt] >> (8 * z), w1 = w[2 * mt + 1] >> (8 * z);
            const uint32_t a0 = Cd::template v<false>(w0), a1 = Cd::template v<true>(w0);
            const uint32_t a2 = Cd::template v<false>(w1), a3 = Cd::template v<true>(w1);
#pragma unroll
            for (int n = 0; n < NT; ++n)
              mma16816<true>(o[Z * j + z][n], a0, a1, a2, a3, pb[mt][n][0], pb[mt][n][1]);
          }
      }
      __syncwarp();  // the stage is read
      const int nt = tile + kStages * kWarps;
      if (nt < t_hi) {
        issue(nt, h, s, next_page);
        next_page = page_of(nt + kWarps);
      }
    }

    // ── the next segment, its loads already in flight during the join ──
    const int cb = b, cu = u;
    left -= t_hi - t_lo;
    const bool more = left > 0;
    if (more) {
      t_lo = 0;
      if (++u == hr) {
        u = 0;
        do {  // sequences without keys have no tiles
          ++b;
          len = len_of(b);
        } while (len == 0);
        table = a.table + (int64_t)b * a.width;
        n_tiles = tiles_of(len);
      }
      t_hi = (int)min((int64_t)n_tiles, left);
      if (Ge::kApart) fill();
    }

    // ── join the warps ──
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], x);
        if (g == 0) {
          sm_m[warp][8 * n + 2 * c + e] = m_top[n][e] == -INFINITY ? -INFINITY : mu[n][e];
          sm_l[warp][8 * n + 2 * c + e] = l[n][e];
          sm_v[warp][8 * n + 2 * c + e] = w_top[n][e] == -INFINITY ? -INFINITY : wu[n][e];
        }
      }
    if (!Ge::kApart) __syncthreads();  // every ring is idle
    constexpr int P = Ge::kPitch;
    float* so = join + warp * R * P;
#pragma unroll
    for (int j = 0; j < kMT; ++j) {
      // dims of this lane's accumulator rows g and g + 8
      const int d = BITS == 8 ? 16 * j + 2 * g : 32 * (j >> 1) + 4 * g + 2 * (j & 1);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<float2*>(so + (8 * n + 2 * c + e) * P + d) =
              make_float2(o[j][n][e], o[j][n][2 + e] * Cd::kHiScale);
    }
    __syncthreads();
    const bool direct = a.direct && first && last;
    for (int i = threadIdx.x; i < R * (D / 4); i += kThreads) {
      const int r = i / (D / 4), d = (i % (D / 4)) * 4;
      if (r0 + r >= a.rows) break;
      float mx = -INFINITY, mw = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        mx = fmaxf(mx, sm_m[w][r]);
        mw = fmaxf(mw, sm_v[w][r]);
      }
      const float mu = base_of(mx), wu = base_of(mw);
      float sum = 0.0f;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2(sm_v[w][r] - wu);
        const float4 x = *reinterpret_cast<const float4*>(join + (w * R + r) * P + d);
        sum += ex2(sm_m[w][r] - mu) * sm_l[w][r];
        v.x += f * x.x; v.y += f * x.y; v.z += f * x.z; v.w += f * x.w;
      }
      // row of the output: the unit's h and b are those before the advance
      int bb = cb, rr = r0 + r;
      if (!own) {
        bb = rr / (a.T * a.G);
        rr -= bb * a.T * a.G;
      }
      const int t = rr / a.G, hh = cu / a.row_tiles;
      const int64_t id = ((int64_t)bb * a.T + t) * ((int64_t)a.H * a.G) + (int64_t)hh * a.G + (rr - t * a.G);
      if (direct) {
        const float inv = norm_of(mx, mw, sum);
        *reinterpret_cast<uint2*>(a.out + id * D + d) =
            make_uint2(bf2(v.x * inv, v.y * inv), bf2(v.z * inv, v.w * inv));
        if (a.lse && d == 0)
          a.lse[id] = sum == 0.0f ? -INFINITY : (mu + __log2f(sum)) * 0.69314718055994531f;
      } else {
        const Part& p = own && !first ? a.cta : a.main;
        const int64_t pr = own ? (first ? id : (int64_t)blockIdx.x * R + r)
                               : (int64_t)blockIdx.x * a.n_rows + id;
        *reinterpret_cast<float4*>(p.o + pr * D + d) = v;
        if (d == 0) p.ml[pr] = make_float4(mx, sum, mw, 0.0f);
      }
    }
    if (!more) break;
    // where the join buffer lies over the rings, its ordinary stores come before
    // the copies (async proxy) of the next unit to the same bytes
    if (!Ge::kApart) fence_proxy_async_shared();
    __syncthreads();  // the join buffer is read
    if (!Ge::kApart) fill();
  }
}

// Joins the parts of rows: the sequence's own, by CTA, then the prefix's, by split.
struct JoinArgs {
  Part main, cta, pre;
  const int64_t* plan;  // null: a unit has one part
  const int* lengths;   // null: no keys of its own
  int64_t cap, n_rows;
  int pre_parts, T, H, G, row_tiles, R;
  int tile_shift;  // log2 of the keys of a tile of the plan
  bool direct;  // rows with one part of their own are written already
  __nv_bfloat16* out;
  float* lse;
};

// A row's parts p0, p0 + step, .. summed, lane l with dims l * D / 32 on.
template <int D>
struct RowSum {
  static constexpr int V = D / 32, U = 4;  // U parts in flight
  float mu = -INFINITY, wu = -INFINITY, sum = 0.0f, v[V];

  // parts of a row, of them its own, and where the CTAs' buffers hold those
  __device__ static int count(const JoinArgs& a, uint32_t row, int& own, int64_t& c_at) {
    const uint32_t bt = row / (uint32_t)(a.H * a.G);
    const int hq = (int)(row - bt * (uint32_t)(a.H * a.G)), h = hq / a.G;
    const int b = (int)(bt / (uint32_t)a.T), rr = (int)(bt - (uint32_t)b * a.T) * a.G + (hq - h * a.G);
    own = 0;
    c_at = 0;
    if (a.lengths) {
      const int64_t n = (min((int64_t)max(__ldg(a.lengths + b), 0), a.cap) + (1 << a.tile_shift) - 1) >> a.tile_shift;
      if (n > 0) {
        own = 1;
        if (a.plan) {
          const int64_t per = a.plan[0];
          const int64_t f0 = a.plan[1 + b] + ((int64_t)h * a.row_tiles + rr / a.R) * n;
          const int64_t c0 = f0 / per;
          own = (int)((f0 + n - 1) / per - c0) + 1;
          c_at = c0 * a.R + rr % a.R;
        }
      }
    }
    return own + a.pre_parts;
  }

  __device__ void add(const JoinArgs& a, uint32_t row, int own, int64_t c_at, int parts, int p0, int step) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = 0.0f;
    for (; p0 < parts; p0 += step * U) {
      float4 ml[U];
      float x[U][V];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int p = p0 + i * step;
        ml[i] = make_float4(-INFINITY, 0.0f, -INFINITY, 0.0f);
#pragma unroll
        for (int k = 0; k < V; ++k) x[i][k] = 0.0f;
        if (p < parts) {
          const bool pre = p >= own;
          const Part& q = pre ? a.pre : p == 0 ? a.main : a.cta;
          const int64_t at = pre ? (int64_t)(p - own) * a.n_rows + row
                                 : p == 0 ? (int64_t)row : c_at + (int64_t)p * a.R;
          ml[i] = q.ml[at];
          if constexpr (V == 4) {
            const float4 t = *reinterpret_cast<const float4*>(q.o + at * D + lane * V);
            x[i][0] = t.x; x[i][1] = t.y; x[i][2] = t.z; x[i][3] = t.w;
          } else {
            const float2 t = *reinterpret_cast<const float2*>(q.o + at * D + lane * V);
            x[i][0] = t.x; x[i][1] = t.y;
          }
        }
      }
      float m1 = mu, w1 = wu;
#pragma unroll
      for (int i = 0; i < U; ++i) {
        m1 = fmaxf(m1, ml[i].x);
        w1 = fmaxf(w1, ml[i].z);
      }
      const float mb = base_of(m1), wb = base_of(w1), fm = ex2(mu - mb), fw = ex2(wu - wb);
      sum *= fm;
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] *= fw;
#pragma unroll
      for (int i = 0; i < U; ++i) {
        sum += ex2(ml[i].x - mb) * ml[i].y;
        const float f = ex2(ml[i].z - wb);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] += f * x[i][k];
      }
      mu = m1;
      wu = w1;
    }
  }
};

__device__ __forceinline__ float lse_of(float mx, float sum) {
  return sum == 0.0f ? -INFINITY : (mx + __log2f(sum)) * 0.69314718055994531f;
}

// RPB rows a block.  One: all warps share its parts, then add up in order.
// kWarps: a warp a row, which needs no second step; a row of more than
// kJoinAlone parts (one long sequence in a batch) still gets the whole block.
// Many rows have few parts and cost instructions: 4096 rows of 10 parts take
// 5 us less with a warp each (4608 rows of 7 to 10 parts the same).  Few rows
// cost the chain of their parts: 64 rows of 28 parts 12 us more with a warp each.
constexpr int kJoinAlone = 32;
constexpr int64_t kJoinManyRows = 1024;
template <int D, int RPB>
__global__ void __launch_bounds__(kThreads) paged_join_kernel(const JoinArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int V = D / 32;
  __shared__ float sv[kWarps][D], sm[kWarps], ss[kWarps], sw[kWarps];
  pdl_trigger();
  pdl_wait();
  int own;
  int64_t c_at;
  auto together = [&](uint32_t row, int parts) {
    RowSum<D> r;
    r.add(a, row, own, c_at, parts, warp, kWarps);
    if (lane == 0) {
      sm[warp] = r.mu;
      ss[warp] = r.sum;
      sw[warp] = r.wu;
    }
#pragma unroll
    for (int k = 0; k < V; ++k) sv[warp][lane * V + k] = r.v[k];
    __syncthreads();
    if (threadIdx.x >= D / 2) return;
    float mx = -INFINITY, mw = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      mx = fmaxf(mx, sm[w]);
      mw = fmaxf(mw, sw[w]);
    }
    const float mt = mx, wt = mw;
    mx = base_of(mx);
    mw = base_of(mw);
    float total = 0.0f, o0 = 0.0f, o1 = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      total += ex2(sm[w] - mx) * ss[w];
      const float f = ex2(sw[w] - mw);
      o0 += f * sv[w][2 * threadIdx.x];
      o1 += f * sv[w][2 * threadIdx.x + 1];
    }
    const float inv = norm_of(mt, wt, total);
    reinterpret_cast<uint32_t*>(a.out + (int64_t)row * D)[threadIdx.x] = bf2(o0 * inv, o1 * inv);
    if (a.lse && threadIdx.x == 0) a.lse[row] = lse_of(mx, total);
  };
  if constexpr (RPB == 1) {
    const int parts = RowSum<D>::count(a, blockIdx.x, own, c_at);
    if (!(a.direct && own == 1)) together(blockIdx.x, parts);
  } else {
    const uint32_t row = blockIdx.x * RPB + warp;
    bool split = false;
    if (row < a.n_rows) {
      const int parts = RowSum<D>::count(a, row, own, c_at);
      split = parts > kJoinAlone;
      if (!split && !(a.direct && own == 1)) {
        RowSum<D> r;
        r.add(a, row, own, c_at, parts, 0, 1);
        const float inv = norm_of(r.mu, r.wu, r.sum);
        uint32_t* o = reinterpret_cast<uint32_t*>(a.out + (int64_t)row * D) + lane * (V / 2);
        if constexpr (V == 4)
          *reinterpret_cast<uint2*>(o) = make_uint2(bf2(r.v[0] * inv, r.v[1] * inv),
                                                    bf2(r.v[2] * inv, r.v[3] * inv));
        else
          *o = bf2(r.v[0] * inv, r.v[1] * inv);
        if (a.lse && lane == 0) a.lse[row] = lse_of(base_of(r.mu), r.sum);
      }
    }
    if (__syncthreads_or(split)) {
      for (int w = 0; w < RPB; ++w) {
        const uint32_t other = blockIdx.x * RPB + w;
        if (other >= a.n_rows) break;
        const int parts = RowSum<D>::count(a, other, own, c_at);
        if (parts > kJoinAlone) {
          __syncthreads();  // the row before is read
          together(other, parts);
        }
      }
    }
  }
}

// How a call is cut: column tiles of 8 query rows per CTA, CTAs for the
// sequences' own keys and splits of the prefix.
struct Plan {
  int nt_own, tiles_own, ctas_own;        // ctas_own 0: no own keys possible
  bool whole;                             // a unit per CTA
  int rows_own, tile_own;                 // query rows a CTA and keys a tile, of the own keys
  bool tensor;                            // own keys on tree_attn.cu
  bool join;                              // rows may have several parts
  int nt_pre, tiles_pre, splits_pre;      // splits_pre 0: no prefix; nt_pre 0: prefix_attn.cu
  size_t o_plan, o_main, o_cta, o_pre, bytes;  // workspace offsets
};

int nt_of(int64_t rows) { return rows <= 8 ? 1 : rows <= 16 ? 2 : rows <= 24 ? 3 : 4; }

// Rows of a tree a KV head from which its own keys go to the tcgen05 kernel, which
// costs the same for 40 rows as for 128.  Microseconds of a call, there and in groups of
// up to 32 rows, 8 heads of 128 dims in int8: 8 sequences of up to 8000 keys, 64 rows
// 91 / 98, 128 rows 98 / 159; 16 of up to 700, 64 rows 35 / 35, 256 rows 47 / 115; 4
// heads of 64 dims in int4, 24 of up to 6000: 56 rows 72 / 71, 104 rows 76 / 124.  Where
// every tile of keys finds an SM of its own, from 25 rows on (1 x 700 keys, 32 rows 22 /
// 27).
constexpr int64_t kTreeRows = 64;
// Keys up to which it takes a unit a CTA, where half of the SMs get one (16 x 700 keys
// of 256 rows: 47, as a list 82; 1 x 700, 8 units: 45 and 33).
constexpr int64_t kTreeWhole = 1024;

Plan make_plan(int64_t B, int64_t T, int64_t H, int64_t G, int dim, int bits, int64_t max_keys,
               int64_t prefix, bool tree) {
  Plan p = {};
  const int64_t n_rows = B * T * H * G;
  const int rb = dim * bits / 8;
  p.nt_own = nt_of(T * G);
  p.tensor = tree && max_keys > 0 &&
             (T * G >= kTreeRows || (T * G > 24 && B * H * cdiv(max_keys, kTreeKeys) <= kSMs));
  p.rows_own = p.tensor ? tree_rows_per_cta(T * G) : 8 * p.nt_own;
  p.tile_own = p.tensor ? kTreeKeys : kTile;
  p.tiles_own = (int)cdiv(T * G, p.rows_own);
  const int64_t units = B * H * p.tiles_own;
  // Short units: one CTA each, and the hardware shares them out.  The list's
  // even runs cost a plan, a second unit's start in most CTAs (5 us) and a
  // join, and pay only where a unit is long beside that or too few units fill
  // the SMs.  Microseconds, a CTA a unit against the list, 8 heads of 128 dims
  // in int8, lengths uniform up to the width: 64 x 512 keys 19 / 52, 256 x 1024
  // 69 / 126, 64 x 4096 71 / 87 (all full 113 / 108), 16 x 2048 24 / 24 (27 /
  // 31), 16 x 4096 45 / 37, 4 x 2048 18.5 / 15.8, 1 x 1024 11.6 / 13.0.
  const int64_t slots = kSMs * ctas(p.nt_own, rb, dim);
  const int64_t whole_keys = units >= slots ? 4096 : units >= kSMs * 3 / 4 ? 2048 : 1024;
  p.whole = max_keys <= (!p.tensor ? whole_keys : units >= kSMs / 2 ? kTreeWhole : 0) &&
            (max_keys > 0 || prefix == 0);
  if (p.whole) {
    p.ctas_own = (int)units;
  } else if (p.tensor) {
    const int64_t most = units * cdiv(max_keys, kTreeKeys);
    p.ctas_own = (int)(most < kSMs ? most : kSMs);
  } else if (max_keys > 0) {
    const int64_t most = units * cdiv(max_keys, kTile * kWarps);
    p.ctas_own = (int)(most < slots ? most : slots);
  }
  // Many rows: 128-row tensor-core tiles, one CTA an SM.  Microseconds of a
  // call, tiles against groups of up to 32 rows, 8 heads of 128 dims in int8
  // (64 in int4): 24 rows over 512 keys 16.5 / 20.5 (15 / 18.5), over 8192
  // 28 / 25; 28 rows over 512 16.4 / 25.7 (15.6 / 19.5), over 8192 28 / 33
  // (26 / 24.5), over 32768 58 / 62 (51 / 33); 48 rows over 32768 65 / 138.
  const int64_t pre_rows = B * T * G;
  if (prefix > 0 && (pre_rows >= 48 || (pre_rows > 24 && prefix <= 8192))) {
    const int64_t units = H * cdiv(pre_rows, prefix_rows_per_cta(pre_rows));
    const int64_t most = cdiv(prefix, 2 * kPrefixKeys);
    int64_t s = kSMs / units;
    s = s < most ? s : most;
    p.splits_pre = (int)(s < 1 ? 1 : s);
  } else if (prefix > 0) {
    p.nt_pre = nt_of(B * T * G);
    p.tiles_pre = (int)cdiv(B * T * G, 8 * p.nt_pre);
    const int64_t most = cdiv(prefix, kTile * kWarps);
    int64_t s = cdiv(kSMs * ctas(p.nt_pre, rb, dim), H * p.tiles_pre);
    s = s < most ? s : most;
    p.splits_pre = (int)(s < 1 ? 1 : s);
  }
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t o = at;
    at += (n + 255) & ~(size_t)255;
    return o;
  };
  const size_t row = (size_t)dim * 4 + 16;
  p.join = !p.whole || prefix > 0;
  if (p.join) {
    p.o_plan = take(p.whole ? 0 : (size_t)(B + 1) * 8);
    p.o_main = take(p.ctas_own ? (size_t)n_rows * row : 0);
    p.o_cta = take(p.whole ? 0 : (size_t)p.ctas_own * p.rows_own * row);
    p.o_pre = take((size_t)p.splits_pre * n_rows * row);
  }
  p.bytes = at;
  return p;
}

template <int BITS, int D, int NT, bool TREE>
int launch(const CUtensorMap& tk, const CUtensorMap& tv, const Args& a, dim3 grid, cudaStream_t st) {
  auto kern = paged_attn_kernel<BITS, D, NT, TREE>;
  constexpr size_t smem = Geo<BITS, D, NT>::kSmem;
  MXB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  MXB_CUDA_TRY(launch_pdl(kern, grid, kThreads, smem, st, tk, tv, a));
  MXB_LAUNCH_CHECK();
  return MXB_OK;
}

template <int BITS, int D, bool TREE>
int launch_nt(const CUtensorMap& tk, const CUtensorMap& tv, const Args& a, int nt, dim3 grid,
              cudaStream_t st) {
  switch (nt) {
    case 1: return launch<BITS, D, 1, TREE>(tk, tv, a, grid, st);
    case 2: return launch<BITS, D, 2, TREE>(tk, tv, a, grid, st);
    case 3: return launch<BITS, D, 3, TREE>(tk, tv, a, grid, st);
    default: return launch<BITS, D, 4, TREE>(tk, tv, a, grid, st);
  }
}

template <bool TREE>
int launch_any(const CUtensorMap& tk, const CUtensorMap& tv, const Args& a, int bits, int dim,
               int nt, dim3 grid, cudaStream_t st) {
  if (bits == 8)
    return dim == 128 ? launch_nt<8, 128, TREE>(tk, tv, a, nt, grid, st)
                      : launch_nt<8, 64, TREE>(tk, tv, a, nt, grid, st);
  return dim == 128 ? launch_nt<4, 128, TREE>(tk, tv, a, nt, grid, st)
                    : launch_nt<4, 64, TREE>(tk, tv, a, nt, grid, st);
}

Part part_at(void* ws, size_t off, size_t rows, int dim) {
  char* p = static_cast<char*>(ws) + off;
  return {reinterpret_cast<float*>(p), reinterpret_cast<float4*>(p + rows * dim * 4)};
}

// A call; tree null: the causal order of the newest tokens.
int attention(const void* q, int64_t B, int64_t T, int heads, int group, int dim, const void* k_codes,
              const float* k_scales, const void* v_codes, const float* v_scales, int64_t n_pages, int page,
              int bits, const int* table, int64_t width, const int* lengths, const int* prefix_table,
              int64_t prefix_width, int64_t prefix_len, const uint8_t* tree, int64_t tree_b, int64_t tree_t,
              float scale, void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = kv_pool_check(n_pages, heads, page, dim, bits, k_codes, k_scales, v_codes, v_scales);
  if (rc != MXB_OK) return rc;
  if (B < 0 || B > 65535 || T < 0 || T > 65535 || group <= 0 || group > 1024 || width < 0 ||
      prefix_len < 0 || width > (INT32_MAX - 64) / page || prefix_len > INT32_MAX - 64 ||
      prefix_width < 0 || prefix_width > INT32_MAX || prefix_len > prefix_width * page ||
      B * T * group > INT32_MAX / 2)
    return MXB_E_SHAPE;
  if (B == 0 || T == 0) return MXB_OK;
  if (!q || !out || !lengths || (width > 0 && !table) || (prefix_len > 0 && !prefix_table))
    return MXB_E_ARG;
  // parts are stored 32 bytes at a time
  if (((uintptr_t)q | (uintptr_t)out) % 16 || (uintptr_t)workspace % 32) return MXB_E_ALIGN;
  const Plan p =
      make_plan(B, T, heads, group, dim, bits, width * page, prefix_len, tree != nullptr);
  const int64_t pre_rows = B * T * group;
  if ((int64_t)p.tiles_own * heads > 65535 || (int64_t)p.tiles_pre * heads > 65535 ||
      (p.splits_pre > 0 && p.nt_pre == 0 && cdiv(pre_rows, prefix_rows_per_cta(pre_rows)) > 65535) ||
      B * heads * p.tiles_own > INT32_MAX || B * T * heads * group > INT32_MAX ||
      (int64_t)heads * p.tiles_own * (width * page / p.tile_own + 1) > INT32_MAX ||
      (p.tensor && width * page > INT32_MAX - 4 * kTreeKeys))  // its positions are 32 bits, a tile further
    return MXB_E_SHAPE;
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes)) return MXB_E_WORKSPACE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);

  CUtensorMap tk, tv;
  const int box = page < kTile ? page : kTile;
  const uint64_t rb = (uint64_t)dim * bits / 8, lines = (uint64_t)n_pages * heads * page * rb / 128;
  const uint32_t box_lines = (uint32_t)(box * rb / 128);
  if (!encode_tmap_2d(&tk, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, k_codes, 128, lines, 128, box_lines,
                      CU_TENSOR_MAP_SWIZZLE_128B) ||
      !encode_tmap_2d(&tv, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, v_codes, 128, lines, 128, box_lines,
                      CU_TENSOR_MAP_SWIZZLE_128B))
    return MXB_E_CUDA;

  Args a = {};
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.ks = k_scales;
  a.vs = v_scales;
  a.n_pages = n_pages;
  a.page_shift = 31 - __builtin_clz((unsigned)page);
  a.box_shift = 31 - __builtin_clz((unsigned)box);
  a.B = (int)B;
  a.T = (int)T;
  a.H = heads;
  a.G = group;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.n_rows = B * T * heads * group;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.lse = lse;
  a.err = device_error_ptr();
  a.tree = tree;
  a.tree_b = tree_b;
  a.tree_t = tree_t;
  Part pre = {}, own = {}, cta = {};
  if (p.splits_pre > 0) {
    pre = part_at(workspace, p.o_pre, (size_t)p.splits_pre * a.n_rows, dim);
    a.table = prefix_table;
    a.width = (int)prefix_width;
    a.prefix_len = (int)prefix_len;
    a.rows = (int)(B * T * group);
    a.row_tiles = p.tiles_pre;
    a.splits = p.splits_pre;
    a.main = pre;
    int r;
    if (p.nt_pre == 0) {
      PrefixArgs x = {};
      x.q = q;
      x.B = (int)B;
      x.T = (int)T;
      x.H = heads;
      x.G = group;
      x.dim = dim;
      x.bits = bits;
      x.k_codes = k_codes;
      x.v_codes = v_codes;
      x.k_scales = k_scales;
      x.v_scales = v_scales;
      x.n_pages = n_pages;
      x.page_shift = a.page_shift;
      x.table = prefix_table;
      x.len = (int)prefix_len;
      x.splits = p.splits_pre;
      x.scale_log2 = a.scale_log2;
      x.n_rows = a.n_rows;
      x.o = pre.o;
      x.ml = reinterpret_cast<float*>(pre.ml);
      x.err = a.err;
      r = prefix_attention(x, st);
    } else {
      r = launch_any<false>(tk, tv, a, bits, dim, p.nt_pre,
                            dim3((unsigned)p.splits_pre, (unsigned)(p.tiles_pre * heads)), st);
    }
    if (r != MXB_OK) return r;
  }
  a.lengths = lengths;
  a.table = table;
  a.width = (int)width;
  a.rows = (int)(T * group);
  a.row_tiles = p.tiles_own;
  a.whole = p.whole;
  a.direct = p.splits_pre == 0;
  if (p.ctas_own > 0) {
    if (p.join) own = part_at(workspace, p.o_main, (size_t)a.n_rows, dim);
    if (!p.whole) {
      cta = part_at(workspace, p.o_cta, (size_t)p.ctas_own * p.rows_own, dim);
      a.plan = reinterpret_cast<int64_t*>(static_cast<char*>(workspace) + p.o_plan);
    }
    a.main = own;
    a.cta = cta;
    const dim3 grid((unsigned)p.ctas_own);
    int r;
    if (p.tensor) {
      const TreeArgs x = {q, a.B, a.T, a.H, a.G, dim, bits, k_codes, v_codes, k_scales, v_scales, n_pages,
                          a.page_shift, table, a.width, lengths, tree, tree_b, tree_t, a.rows, a.row_tiles,
                          a.scale_log2, own.o, reinterpret_cast<float*>(own.ml), cta.o,
                          reinterpret_cast<float*>(cta.ml), a.plan, a.direct, out, lse, a.err};
      r = tree_attention(x, p.ctas_own, st);
    } else {
      r = tree ? launch_any<true>(tk, tv, a, bits, dim, p.nt_own, grid, st)
               : launch_any<false>(tk, tv, a, bits, dim, p.nt_own, grid, st);
    }
    if (r != MXB_OK) return r;
  }
  if (p.join) {
    JoinArgs j = {own, cta, pre, a.plan, p.ctas_own > 0 ? lengths : nullptr, width * page,
                  a.n_rows, p.splits_pre, (int)T, heads, group, p.tiles_own, p.rows_own,
                  31 - __builtin_clz((unsigned)p.tile_own), a.direct, a.out, lse};
    const bool many = a.n_rows >= kJoinManyRows;
    auto kern = dim == 128 ? (many ? paged_join_kernel<128, kWarps>
                                   : paged_join_kernel<128, 1>)
                           : (many ? paged_join_kernel<64, kWarps>
                                   : paged_join_kernel<64, 1>);
    MXB_CUDA_TRY(launch_pdl(kern, dim3((unsigned)(many ? cdiv(a.n_rows, kWarps) : a.n_rows)),
                            kThreads, 0, st, j));
    MXB_LAUNCH_CHECK();
  }
  return MXB_OK;
}

}  // namespace pattn
}  // namespace mxb

extern "C" {

size_t mxb_paged_attention_workspace_size(int64_t B, int64_t T, int heads, int group, int dim,
                                          int bits, int page, int64_t width, int64_t prefix_len) {
  if (B <= 0 || T <= 0 || heads <= 0 || group <= 0 || dim <= 0 || page <= 0 || bits <= 0) return 0;
  return pattn::make_plan(B, T, heads, group, dim, bits, width * page, prefix_len, false).bytes;
}

int mxb_paged_attention(const void* q, int64_t B, int64_t T, int heads, int group, int dim,
                        const void* k_codes, const float* k_scales, const void* v_codes,
                        const float* v_scales, int64_t n_pages, int page, int bits,
                        const int* table, int64_t width, const int* lengths,
                        const int* prefix_table, int64_t prefix_width, int64_t prefix_len,
                        float scale, void* out, float* lse, void* workspace,
                        size_t workspace_bytes, void* stream) {
  return pattn::attention(q, B, T, heads, group, dim, k_codes, k_scales, v_codes, v_scales, n_pages, page, bits,
                          table, width, lengths, prefix_table, prefix_width, prefix_len, nullptr, 0, 0, scale,
                          out, lse, workspace, workspace_bytes, stream);
}

size_t mxb_tree_attention_workspace_size(int64_t B, int64_t T, int heads, int group, int dim, int bits,
                                         int page, int64_t width, int64_t prefix_len) {
  if (B <= 0 || T <= 0 || heads <= 0 || group <= 0 || dim <= 0 || page <= 0 || bits <= 0) return 0;
  return pattn::make_plan(B, T, heads, group, dim, bits, width * page, prefix_len, true).bytes;
}

int mxb_tree_attention(const void* q, int64_t B, int64_t T, int heads, int group, int dim, const void* k_codes,
                       const float* k_scales, const void* v_codes, const float* v_scales, int64_t n_pages,
                       int page, int bits, const int* table, int64_t width, const int* lengths,
                       const int* prefix_table, int64_t prefix_width, int64_t prefix_len,
                       const uint8_t* tree_mask, int64_t tree_batch_stride, int64_t tree_token_stride,
                       float scale, void* out, float* lse, void* workspace, size_t workspace_bytes,
                       void* stream) {
  if (B > 0 && T > 0 && !tree_mask) return MXB_E_ARG;
  return pattn::attention(q, B, T, heads, group, dim, k_codes, k_scales, v_codes, v_scales, n_pages, page, bits,
                          table, width, lengths, prefix_table, prefix_width, prefix_len, tree_mask,
                          tree_batch_stride, tree_token_stride, scale, out, lse, workspace, workspace_bytes,
                          stream);
}

}  // extern "C"
