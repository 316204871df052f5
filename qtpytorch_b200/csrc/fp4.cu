// Microscaled 4-bit floating point: quantize, dequantize and the per-tensor
// factor (mxfp4: E8M0 scales of 32 elements; nvfp4: E4M3 scales of 16 and one
// fp32 factor g).  Layout and formulas: include/mxb.h.
//
// All three are one pass over HBM: a thread owns 16 consecutive elements of a
// row (an nvfp4 block, half an mxfp4 block), so the block maximum costs no
// shuffle (nvfp4) or one (mxfp4), the codes leave as one 8-byte store and the
// scales of four blocks as one 32-bit store in the tensor-core tile order.
// HBM bounds all of them at size (11008 x 4096): mxfp4 from fp32 31.5 us = 6.5
// TB/s; nvfp4's factor needs a pass of its own before, 28.6 us = 6.3 TB/s;
// dequantized to fp32 31 us = 6.6 TB/s, to bf16 19 us = 6.0 TB/s.  A step's few
// rows are bound by the launch (8 x 4096: 2 us).
#include "mxb_common.cuh"
#include "mxb_internal.h"

#include <cuda_fp16.h>

using namespace mxb;

namespace {

constexpr int kThreads = 256;
constexpr int kE = 16;  // elements per thread (quantize)

__host__ __device__ inline int64_t fp4_blocks(int64_t K, int fmt) {
  return fmt == MXB_FP4_NV ? cdiv(K, 16) : cdiv(K, 32);
}
__host__ __device__ inline int64_t fp4_row_bytes(int64_t K) { return cdiv(K, 32) * 16; }

// byte offset of the first of the four scales (r, 4 * cg .. 4 * cg + 3)
__device__ __forceinline__ size_t sf_offset(int64_t r, int64_t cg, int64_t groups) {
  return ((size_t)(r >> 7) * groups + cg) * 512 + (size_t)(r & 31) * 16 + (size_t)((r >> 5) & 3) * 4;
}

// Eight floats -> eight E2M1 codes (round to nearest even, saturating), first
// in the low nibble.
__device__ __forceinline__ uint32_t e2m1x8(const float* q) {
  uint32_t w;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(w)
      : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
  return w;
}

__device__ __forceinline__ uint32_t e4m3_of(float v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(v));
  return r & 0xFFu;
}
__device__ __forceinline__ float e4m3_value(uint32_t b) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)b));
  return __half2float(__ushort_as_half((unsigned short)(h & 0xFFFFu)));
}
__device__ __forceinline__ float e8m0_value(uint32_t b) {
  // 2^(b - 127); b = 0 is the subnormal 2^-127, 0xFF is NaN
  return __uint_as_float(b == 0u ? 0x00400000u : b == 255u ? 0x7FC00000u : b << 23);
}

// The tensor's factor from its largest magnitude: amax * fl(1 / 2688), so
// that the largest block's scale is e4m3's 448.
__device__ __forceinline__ float factor_of(float amax) {
  return (amax > 0.0f && amax <= 3.4028235e38f) ? __fmul_rn(amax, 1.0f / 2688.0f) : 1.0f;
}

// Maximum over the block (NaN kept), in every thread.
__device__ __forceinline__ float block_max(float a) {
  __shared__ float s[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a = nan_max(a, __shfl_xor_sync(0xffffffffu, a, o));
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = a;
  __syncthreads();
  a = s[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) a = nan_max(a, s[w]);
  return a;
}

// 32 bytes: a whole sector a lane, so that a warp's lanes, 16 elements apart,
// use all that they touch.
__device__ __forceinline__ void ld32b(const void* p, uint32_t (&r)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
                 "=r"(r[7])
               : "l"(p));
}

// i / d by a product with 2^(31 + s) / d rounded up, exact for i < 2^31 (the
// rounding adds less than 2^s >= d to it).  A division costs some twenty
// instructions beside about 200 for the rest of 16 elements.
struct Div {
  uint32_t d, m, s;  // m = 0: divide
  __device__ __forceinline__ uint32_t operator()(uint32_t i) const { return m ? __umulhi(i, m) >> s : i / d; }
};
Div div_by(uint32_t d, uint64_t top) {
  Div r = {d, 0, 0};
  if (d < 2 || top > (uint64_t)1 << 31) return r;
  uint32_t l = 1;
  while (l < 31 && ((uint64_t)1 << l) < d) ++l;
  if (((uint64_t)1 << l) < d) return r;
  r.m = (uint32_t)((((uint64_t)1 << (31 + l)) + d - 1) / d);
  r.s = l - 1;
  return r;
}

// Up to 16 elements of a row from column c0 on; zero past K.  vec: rows are
// 32-byte aligned.
template <typename InT>
__device__ __forceinline__ void load16(const InT* __restrict__ row, int64_t c0, int64_t K, bool vec,
                                       float (&v)[kE]) {
  if (vec && c0 + kE <= K) {
    if constexpr (sizeof(InT) == 4) {
      uint32_t a[8], b[8];
      ld32b(row + c0, a);
      ld32b(row + c0 + 8, b);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = __uint_as_float(a[i]);
        v[8 + i] = __uint_as_float(b[i]);
      }
    } else {
      uint32_t w[8];
      ld32b(row + c0, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kE; ++i) v[i] = c0 + i < K ? load_as_f32(row, c0 + i) : 0.0f;
  }
}

// Largest |x| of each block's share of the tensor (NaN kept) -> part[block].
// The quantize kernel reduces the at most kAmaxBlocks values, so there is no
// atomic and nothing to clear.
constexpr int kAmaxBlocks = 6 * kSMs;
template <typename InT>
__global__ void __launch_bounds__(kThreads) fp4_amax_kernel(const InT* __restrict__ x, int64_t K,
                                                            int64_t ldx, Div gpr,
                                                            uint32_t items, bool vec,
                                                            float* __restrict__ part) {
  pdl_trigger();
  pdl_wait();
  float a = 0.0f;
  const uint64_t step = (uint64_t)gridDim.x * kThreads;
  for (uint64_t i = blockIdx.x * (uint64_t)kThreads + threadIdx.x; i < items; i += 2 * step) {
    float v[2][kE];
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // two in flight
      const uint64_t j = i + h * step < items ? i + h * step : i;
      const uint32_t r = gpr((uint32_t)j), c = (uint32_t)j - r * gpr.d;
      load16(x + (int64_t)r * ldx, (int64_t)c * kE, K, vec, v[h]);
    }
#pragma unroll
    for (int j = 0; j < kE; ++j) a = nan_max(a, nan_max(fabsf(v[0][j]), fabsf(v[1][j])));
  }
  a = block_max(a);
  if (threadIdx.x == 0) part[blockIdx.x] = a;
}

// Largest |x| of a small tensor, found by every cluster of kSmallCluster blocks
// for itself: a launch less than with fp4_amax_kernel, which costs a call of
// this size more than the extra reads from L2.  A call and its kernels, with and
// without: 8 x 4096 bf16 8.8 and 6.2 us, 16 and 6.2; 64 x 4096 (the limit) 8.8 and
// 8.2, 13.8 and 6.2; 256 x 4096 17.6 and 16.4, 12.8 and 6.9.
constexpr int kSmallCluster = 8;
constexpr int64_t kSmallItems = (int64_t)kSmallCluster * kThreads * 8;
template <typename InT>
__device__ __forceinline__ float cluster_amax(const InT* __restrict__ x, uint32_t rows, int64_t K,
                                              int64_t ldx, bool vec) {
  __shared__ float mine;
  uint32_t rank;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const uint32_t gpr = (uint32_t)((K + kE - 1) / kE), items = rows * gpr;
  float a = 0.0f;
  for (uint32_t i = rank * kThreads + threadIdx.x; i < items; i += kSmallCluster * kThreads) {
    const uint32_t r = i / gpr, c = i - r * gpr;
    float v[kE];
    load16(x + (int64_t)r * ldx, (int64_t)c * kE, K, vec, v);
#pragma unroll
    for (int j = 0; j < kE; ++j) a = amax_step(a, v[j]);
  }
  a = block_max(a);
  if (threadIdx.x == 0) mine = a;
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
  const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(&mine));
#pragma unroll
  for (int p = 0; p < kSmallCluster; ++p) {
    uint32_t ra;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(at), "r"(p));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(ra));
    a = nan_max(a, v);
  }
  // no block leaves while another may still read its value
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
  return a;
}

// gpr: 16-element groups per row, covering whole tiles of four scales;
// items: rows * gpr groups, then one 32-bit word per four scales of each
// padding row.  parts: -1 the factor from the cluster's own pass over x, 0 given.
// part: the blocks' maxima (parts > 0), else null; the blocks then run
// from the end of the tensor, whose rows the maximum pass left in L2.
template <typename InT, int FMT>
__global__ void __launch_bounds__(kThreads)
    fp4_quant_kernel(const InT* __restrict__ x, uint32_t rows, int64_t K, int64_t ldx, Div gpr,
                     uint32_t items, uint32_t pad_words, uint32_t groups, bool vec,
                     const float* __restrict__ part, int parts, float* __restrict__ gscale,
                     uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  pdl_trigger();
  pdl_wait();
  float g = 1.0f;
  if (FMT == MXB_FP4_NV) {
    if (part) {
      float a = 0.0f;
      for (int p = threadIdx.x; p < parts; p += kThreads) a = nan_max(a, part[p]);
      g = factor_of(block_max(a));
      if (blockIdx.x == 0 && threadIdx.x == 0) *gscale = g;
    } else if (parts < 0) {
      g = factor_of(cluster_amax(x, rows, K, ldx, vec));
      if (blockIdx.x == 0 && threadIdx.x == 0) *gscale = g;
    } else {
      g = *gscale;
    }
  }
  const int64_t rb = fp4_row_bytes(K);
  const uint32_t blocks = (uint32_t)(((uint64_t)items + pad_words + kThreads - 1) / kThreads);
  auto item_of = [&](uint32_t blk0) -> uint64_t {
    return (part ? blocks - 1 - blk0 : blk0) * (uint64_t)kThreads + threadIdx.x;
  };
  float next[kE];
  auto fetch = [&](uint32_t blk0) {  // the values of a later item
    if (blk0 >= blocks) return;
    const uint64_t i = item_of(blk0);
    if (i < items) {
      const uint32_t r = gpr((uint32_t)i), c = (uint32_t)i - r * gpr.d;
      load16(x + (int64_t)r * ldx, (int64_t)c * kE, K, vec, next);
    } else {
#pragma unroll
      for (int j = 0; j < kE; ++j) next[j] = 0.0f;
    }
  };
  fetch(blockIdx.x);
  for (uint32_t blk0 = blockIdx.x; blk0 < blocks; blk0 += gridDim.x) {
    const uint64_t i = item_of(blk0);
    const bool mine = i < items;
    if (!mine && i - items < pad_words) {
      const uint32_t w = (uint32_t)(i - items);
      const uint32_t r = rows + w / groups;
      *reinterpret_cast<uint32_t*>(scales + sf_offset(r, w % groups, groups)) = 0u;
    }
    const uint32_t r = mine ? gpr((uint32_t)i) : 0u, c = mine ? (uint32_t)i - r * gpr.d : 0u;
    float v[kE];
#pragma unroll
    for (int j = 0; j < kE; ++j) v[j] = next[j];
    fetch(blk0 + gridDim.x);
    float a = 0.0f;
#pragma unroll
    for (int j = 0; j < kE; ++j) a = amax_step(a, v[j]);
    if (FMT == MXB_FP4_MX) a = nan_max(a, __shfl_xor_sync(0xffffffffu, a, 1));
    const bool finite = a <= 3.4028235e38f;
    uint32_t sb;
    float q[kE];
    if (FMT == MXB_FP4_MX) {
      // floor(log2(a)) is the exponent field; subnormals fall under the clamp
      sb = (uint32_t)max((int)(__float_as_uint(a) >> 23) - 2, 0);
      const float inv = __uint_as_float((254u - sb) << 23);  // exact: a power of two
#pragma unroll
      for (int j = 0; j < kE; ++j) q[j] = __fmul_rn(v[j], inv);
      if (!finite) sb = 255u;
    } else {
      sb = e4m3_of(fminf(__fdiv_rn(a, __fmul_rn(6.0f, g)), 448.0f));
      const float s = __fmul_rn(e4m3_value(sb), g);
      const float rs = __frcp_rn(s);
      // (under a given factor far too small a quotient may pass fp32's range)
      if (s >= 7.9e-31f && s <= 1.2e30f && __fmul_rn(a, rs) <= 3.4028235e38f) {
        // x / s by Markstein's corrected product (r correctly rounded, the
        // residual exact in an FMA): three operations instead of a division.  The
        // residual is taken as q0 s - x: for x = -0 that is +0, and -0 stays -0.
#pragma unroll
        for (int j = 0; j < kE; ++j) {
          const float q0 = __fmul_rn(v[j], rs);
          q[j] = __fmaf_rn(-__fmaf_rn(q0, s, -v[j]), rs, q0);
        }
      } else {
#pragma unroll
        for (int j = 0; j < kE; ++j) q[j] = s > 0.0f ? __fdiv_rn(v[j], s) : __fmul_rn(v[j], 0.0f);
      }
      if (!finite) sb = 0x7Fu;
    }
    uint2 w = make_uint2(e2m1x8(q), e2m1x8(q + 8));
    if (!finite) w = make_uint2(0u, 0u);
    if (mine && (int64_t)c * 8 < rb)
      *reinterpret_cast<uint2*>(codes + (size_t)r * rb + (size_t)c * 8) = w;
    // four scales -> one word.  A group of four blocks starts at a multiple of
    // 8 (mxfp4) or 4 (nvfp4) items, and gpr is a multiple of that, so its lanes
    // sit in one warp and one row.
    constexpr int L = FMT == MXB_FP4_MX ? 2 : 1;
    if ((int64_t)c * kE >= K) sb = 0u;  // blocks past the row
    uint32_t word = sb;
    word |= __shfl_down_sync(0xffffffffu, word, L) << 8;
    word |= __shfl_down_sync(0xffffffffu, word, 2 * L) << 16;
    if (mine && (c & (4 * L - 1)) == 0)
      *reinterpret_cast<uint32_t*>(scales + sf_offset(r, c / (4 * L), groups)) = word;
  }
}

// Two E2M1 codes (one byte) -> two floats.
__device__ __forceinline__ float2 e2m1x2_value(uint32_t byte) {
  uint32_t h;
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\t}"
      : "=r"(h)
      : "r"(byte));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}

__device__ __forceinline__ void st32b(void* p, const uint32_t (&r)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// A thread makes 16 values of one scale (8 bytes of codes) and writes them in
// whole sectors; kU of them in flight.  ALIGN: every row of out starts at a
// multiple of 32 bytes, of 16, or neither (0).  4097 x 1000 bf16: 5 us by 16 bytes;
// 4097 x 1001 8.9, 41 with a thread's values stored one by one.
template <typename OutT, int FMT, int ALIGN>
__global__ void __launch_bounds__(kThreads)
    fp4_dequant_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                       const float* __restrict__ gscale, int64_t K, Div cpr, uint32_t items,
                       uint32_t groups, OutT* __restrict__ out) {
  constexpr int kU = 2;
  constexpr int kPerBlk = FMT == MXB_FP4_NV ? 1 : 2;  // items per scale
  const int lane = threadIdx.x & 31;
  pdl_trigger();
  pdl_wait();
  const float g = FMT == MXB_FP4_NV ? *gscale : 1.0f;
  const int64_t rb = fp4_row_bytes(K);
  const uint64_t i0 = blockIdx.x * (uint64_t)(kThreads * kU) + threadIdx.x;  // may pass 32 bits
  uint2 w[kU];
  uint32_t sb[kU], rr[kU], cc[kU];
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    const uint64_t i = i0 + (uint64_t)u * kThreads;
    w[u] = make_uint2(0u, 0u);
    sb[u] = rr[u] = cc[u] = 0u;
    if (i < items) {
      const uint32_t r = cpr((uint32_t)i), c = (uint32_t)i - r * cpr.d;
      w[u] = __ldg(reinterpret_cast<const uint2*>(codes + (size_t)r * rb + (size_t)c * 8));
      const uint32_t blk = c / kPerBlk;
      sb[u] = __ldg(scales + sf_offset(r, blk >> 2, groups) + (blk & 3));
      rr[u] = r;
      cc[u] = c;
    }
  }
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    const bool live = i0 + (uint64_t)u * kThreads < items;
    if (!live && ALIGN >= 16) continue;
    const float s = FMT == MXB_FP4_NV ? __fmul_rn(e4m3_value(sb[u]), g) : e8m0_value(sb[u]);
    float v[kE];
#pragma unroll
    for (int j = 0; j < kE / 2; ++j) {
      const float2 t = e2m1x2_value(((j < 4 ? w[u].x : w[u].y) >> (8 * (j & 3))) & 0xFFu);
      v[2 * j] = __fmul_rn(t.x, s);
      v[2 * j + 1] = __fmul_rn(t.y, s);
    }
    const int64_t c0 = (int64_t)cc[u] * kE;
    OutT* o = out + (int64_t)rr[u] * K + c0;
    constexpr int W = 16 / (int)sizeof(OutT);  // values of 16 bytes
    constexpr int P = 4 / (int)sizeof(OutT);   // of a word
    uint32_t p[kE / P];
#pragma unroll
    for (int j = 0; j < kE / P; ++j) {
      if constexpr (P == 1) {
        p[j] = __float_as_uint(v[j]);
      } else {
        const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        p[j] = *reinterpret_cast<const uint32_t*>(&t);
      }
    }
    if (ALIGN >= 32 && c0 + kE <= K) {
#pragma unroll
      for (int h = 0; h < kE / P; h += 8) {
        uint32_t w8[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w8[j] = p[h + j];
        st32b(o + h * P, w8);
      }
    } else if constexpr (ALIGN >= 16) {
#pragma unroll
      for (int h = 0; h < kE / W; ++h) {
        if (c0 + (h + 1) * W <= K) {
          *reinterpret_cast<uint4*>(o + h * W) = make_uint4(p[4 * h], p[4 * h + 1], p[4 * h + 2], p[4 * h + 3]);
        } else {
#pragma unroll
          for (int j = 4 * h; j < 4 * h + 4; ++j)
            if (c0 + j * P < K) reinterpret_cast<uint32_t*>(o)[j] = p[j];
        }
      }
    } else {
      // a warp's 512 values through shared memory, so that its lanes write
      // neighbours
      __shared__ float stage[kThreads / 32][32 * (kE + 1)];
      float* t = stage[threadIdx.x >> 5];
#pragma unroll
      for (int j = 0; j < kE; ++j) t[lane * (kE + 1) + j] = v[j];
      __syncwarp();
      const int j = lane % kE;
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        const int src = 2 * e + lane / kE;
        const int64_t at = __shfl_sync(0xffffffffu, live ? (int64_t)rr[u] * K + c0 : -1, src);
        const int64_t c = __shfl_sync(0xffffffffu, (int)cc[u], src) * (int64_t)kE + j;
        if (at >= 0 && c < K) out[at + j] = static_cast<OutT>(t[src * (kE + 1) + j]);
      }
      __syncwarp();
    }
  }
}

template <typename InT>
int quantize_t(const InT* x, int64_t rows, int64_t K, int64_t ldx, int fmt, float* g, int derive,
               uint8_t* codes, uint8_t* scales, float* part, cudaStream_t st) {
  const int64_t groups = cdiv(fp4_blocks(K, fmt), 4);
  const int64_t gpr = groups * (fmt == MXB_FP4_NV ? 4 : 8);
  const int64_t items = rows * gpr, pad = (cdiv(rows, 128) * 128 - rows) * groups;
  if (items + pad >= (int64_t)1 << 32) return MXB_E_SHAPE;
  const bool vec = ((uintptr_t)x % 32) == 0 && (ldx * (int64_t)sizeof(InT)) % 32 == 0;
  int parts = 0;
  const bool small = derive && rows * cdiv(K, kE) <= kSmallItems;
  if (derive && !small) {
    // rows without gaps are one long row: only the start's alignment counts
    // (4097 x 1001 fp32 29 -> 18 us, the quantize kernel's 10 included)
    const bool flat = ldx == K;
    const int64_t ak = flat ? rows * K : K, agpr = cdiv(ak, kE), aitems = flat ? agpr : rows * agpr;
    const int64_t blocks = cdiv(aitems, kThreads);
    const bool avec = flat ? ((uintptr_t)x % 32) == 0 : vec;
    parts = (int)(blocks < kAmaxBlocks ? blocks : kAmaxBlocks);
    MXB_CUDA_TRY(launch_pdl(fp4_amax_kernel<InT>, dim3((unsigned)parts), kThreads, 0, st, x, ak, flat ? ak : ldx,
                            div_by((uint32_t)agpr, aitems), (uint32_t)aitems, avec, part));
    MXB_LAUNCH_CHECK();
  }
  auto kern = fmt == MXB_FP4_NV ? fp4_quant_kernel<InT, MXB_FP4_NV> : fp4_quant_kernel<InT, MXB_FP4_MX>;
  // with a factor to find every block first reduces the maxima, so there are
  // only as many blocks as fit
  int64_t blocks = cdiv(items + pad, kThreads);
  if (derive && !small && blocks > 4 * kSMs) blocks = 4 * kSMs;
  if (small) {
    blocks = cdiv(blocks, kSmallCluster) * kSmallCluster;
    parts = -1;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kSmallCluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = small ? 2 : 1;
  MXB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, x, (uint32_t)rows, K, ldx, div_by((uint32_t)gpr, items), (uint32_t)items,
                                  (uint32_t)pad, (uint32_t)groups, vec,
                                  (const float*)(derive && !small ? part : nullptr), parts, g, codes,
                                  scales));
  MXB_LAUNCH_CHECK();
  return MXB_OK;
}

template <typename OutT>
int dequantize_t(const uint8_t* codes, const uint8_t* scales, const float* g, int64_t rows,
                 int64_t K, int fmt, OutT* out, cudaStream_t st) {
  const int64_t cpr = cdiv(K, kE), items = rows * cpr;
  const int64_t groups = cdiv(fp4_blocks(K, fmt), 4);
  const int64_t grid = cdiv(items, 2 * kThreads);
  if (items >= (int64_t)1 << 32) return MXB_E_SHAPE;
  const uint64_t at = (uintptr_t)out | (uint64_t)K * sizeof(OutT);
  const int align = at % 32 == 0 ? 32 : at % 16 == 0 ? 16 : 0;
  const bool nv = fmt == MXB_FP4_NV;
  auto kern = align == 32 ? (nv ? fp4_dequant_kernel<OutT, MXB_FP4_NV, 32> : fp4_dequant_kernel<OutT, MXB_FP4_MX, 32>)
              : align == 16 ? (nv ? fp4_dequant_kernel<OutT, MXB_FP4_NV, 16>
                                  : fp4_dequant_kernel<OutT, MXB_FP4_MX, 16>)
                            : (nv ? fp4_dequant_kernel<OutT, MXB_FP4_NV, 0>
                                  : fp4_dequant_kernel<OutT, MXB_FP4_MX, 0>);
  MXB_CUDA_TRY(launch_pdl(kern, dim3((unsigned)grid), kThreads, 0, st, codes, scales, g, K,
                          div_by((uint32_t)cpr, items), (uint32_t)items, (uint32_t)groups, out));
  MXB_LAUNCH_CHECK();
  return MXB_OK;
}

bool fmt_ok(int fmt) { return fmt == MXB_FP4_MX || fmt == MXB_FP4_NV; }
bool io_ok(int dt) { return dt == MXB_F32 || dt == MXB_BF16; }

}  // namespace

extern "C" {

size_t mxb_fp4_code_bytes(int64_t rows, int64_t K) {
  return rows <= 0 || K <= 0 ? 0 : (size_t)rows * (size_t)fp4_row_bytes(K);
}

size_t mxb_fp4_scale_bytes(int64_t rows, int64_t K, int fmt) {
  if (rows <= 0 || K <= 0 || !fmt_ok(fmt)) return 0;
  return (size_t)cdiv(rows, 128) * (size_t)cdiv(fp4_blocks(K, fmt), 4) * 512;
}

size_t mxb_fp4_quantize_workspace_size(int64_t rows, int64_t K, int fmt, int derive) {
  return rows > 0 && K > 0 && fmt == MXB_FP4_NV && derive ? kAmaxBlocks * sizeof(float) : 0;
}

int mxb_fp4_quantize(const void* x, int x_dtype, int64_t rows, int64_t K, int64_t ldx, int fmt,
                     float* global_scale, int derive, void* codes, void* scales, void* workspace,
                     size_t workspace_bytes, void* stream) {
  if (!fmt_ok(fmt) || !io_ok(x_dtype)) return MXB_E_DTYPE;
  if (rows < 0 || K < 0 || (rows > 1 && ldx < K)) return MXB_E_SHAPE;
  if (rows == 0 || K == 0) return MXB_OK;
  if (!x || !codes || !scales || (fmt == MXB_FP4_NV) != (global_scale != nullptr)) return MXB_E_ARG;
  if ((uintptr_t)codes % 16 || (uintptr_t)scales % 16 || (uintptr_t)workspace % 4 ||
      (uintptr_t)x % (x_dtype == MXB_BF16 ? 2 : 4))
    return MXB_E_ALIGN;
  const bool d = fmt == MXB_FP4_NV && derive != 0;
  if (d && (!workspace || workspace_bytes < mxb_fp4_quantize_workspace_size(rows, K, fmt, 1)))
    return MXB_E_WORKSPACE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  float* ws = static_cast<float*>(workspace);
  uint8_t* c = static_cast<uint8_t*>(codes);
  uint8_t* s = static_cast<uint8_t*>(scales);
  if (x_dtype == MXB_BF16)
    return quantize_t(static_cast<const __nv_bfloat16*>(x), rows, K, ldx, fmt, global_scale, d, c, s,
                      ws, st);
  return quantize_t(static_cast<const float*>(x), rows, K, ldx, fmt, global_scale, d, c, s, ws, st);
}

int mxb_fp4_dequantize(const void* codes, const void* scales, const float* global_scale,
                       int64_t rows, int64_t K, int fmt, void* out, int out_dtype, void* stream) {
  if (!fmt_ok(fmt) || !io_ok(out_dtype)) return MXB_E_DTYPE;
  if (rows < 0 || K < 0) return MXB_E_SHAPE;
  if (rows == 0 || K == 0) return MXB_OK;
  if (!codes || !scales || !out || (fmt == MXB_FP4_NV) != (global_scale != nullptr))
    return MXB_E_ARG;
  if ((uintptr_t)codes % 16 || (uintptr_t)scales % 16 || (uintptr_t)out % (out_dtype == MXB_BF16 ? 2 : 4))
    return MXB_E_ALIGN;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const uint8_t* c = static_cast<const uint8_t*>(codes);
  const uint8_t* s = static_cast<const uint8_t*>(scales);
  if (out_dtype == MXB_BF16)
    return dequantize_t(c, s, global_scale, rows, K, fmt, static_cast<__nv_bfloat16*>(out), st);
  return dequantize_t(c, s, global_scale, rows, K, fmt, static_cast<float*>(out), st);
}

}  // extern "C"
