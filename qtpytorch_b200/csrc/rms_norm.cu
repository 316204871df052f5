// Root-mean-square norm of rows, with the residual's addition in front and int8
// codes with one scale a row behind:
//
//   h = x + r,  y = h w / sqrt(mean(h^2) + eps),
//   s = max(amax|y|, 1e-12) / 127,  code = rint(y / s)   (ties to even)
//
// The quotient is 127 u / amax|u| of u = h w: the root cancels, so a row's sum
// of squares and its largest u are found in the same pass and the codes need one
// reduction, not two.
//
// The codes are the ones of this formula in 64 bits.  The fp32 quotient is off by at
// most 127 * 5 * 2^-24 (h, u, amax, the factor 127 / amax and the product with it are
// rounded once each); where it comes within 127 * 2^-21 of a border between two codes
// it is found again in 64 bits from x, r and w.  There h, u and 127 u are rounded to 53
// bits, which hold them unless the terms lie far apart (0.5 + 2^-60 of a largest 127
// is a tie).  That meets 1 value in 8000.  The largest u is found in 64 bits too, among
// those within 2^-21 of the fp32 one.  Rows that hold infinities or NaN, or whose
// values leave the range in which all this holds, rows of zeros among them, take a slow
// path in 64 bits (4096 x 8192 bf16 with a residual: every second row zero 155 us, all 247).
//
// One pass over HBM: a row stays in the registers of its block, 8 NC values a
// thread.  What bounds it beside HBM is the issue of its instructions and the chain of a
// row (two reductions, two barriers).  4096 x 8192 bf16 with a residual (235 MB): 43 us =
// 5.4 TB/s in pairs of values with four rows an SM, 51 one value at a time with three, 109
// where each correction in 64 bits stood in line.  Rows copied to shared memory ahead of
// their turn by blocks that stay: 50.  8 x 4096: 3.0 us; 1001 x 1999 fp32, value by value:
// 9 us, 13 with 32 values a thread.
#include "mxb_common.cuh"
#include "mxb_internal.h"

using namespace mxb;

namespace {

constexpr int kWarpRows = 8;     // rows a block where a row is a warp's
constexpr int kMaxRow = 32768;   // 1024 threads of 32 values

// 8 consecutive values as they lie in memory (16-byte aligned).
template <typename T>
struct Raw8;
template <>
struct Raw8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = __ldg(reinterpret_cast<const float4*>(p));
    b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  }
  __device__ __forceinline__ void get(uint64_t (&v)[4]) const {
    v[0] = pack2(a.x, a.y); v[1] = pack2(a.z, a.w);
    v[2] = pack2(b.x, b.y); v[3] = pack2(b.z, b.w);
  }
};
template <>
struct Raw8<__nv_bfloat16> {
  uint4 r;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { r = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void get(uint64_t (&v)[4]) const {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = pack2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
};
__device__ __forceinline__ void store8(float* p, const uint64_t (&v)[4]) {
  reinterpret_cast<ulonglong2*>(p)[0] = make_ulonglong2(v[0], v[1]);
  reinterpret_cast<ulonglong2*>(p)[1] = make_ulonglong2(v[2], v[3]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const uint64_t (&v)[4]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2(v[i]);
    const __nv_bfloat162 t = __floats2bfloat162_rn(f.x, f.y);
    w[i] = *reinterpret_cast<const uint32_t*>(&t);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <typename InT, typename WT>
struct Row {
  const InT* x;
  const InT* r;  // null: none
  const WT* w;
  int d;
  __device__ __forceinline__ double h64(int i) const {
    double h = (double)load_as_f32(x, i);
    if (r) h += (double)load_as_f32(r, i);
    return h;
  }
  __device__ __forceinline__ float h32(int i) const {
    float h = load_as_f32(x, i);
    if (r) h = __fadd_rn(h, load_as_f32(r, i));
    return h;
  }
  __device__ __forceinline__ double u64(int i) const { return h64(i) * (double)load_as_f32(w, i); }
};

struct Shared {
  float ssq[32], top[32];
  double dsq[32], dtop[32];
  unsigned long long most;  // bits of the largest |u| in 64 bits
};

// The slow path: everything in 64 bits, the row read again.  t of n threads;
// the reductions are the warp's, then (n > 32) the block's.
template <typename InT, typename WT>
__device__ __noinline__ void row_in_64_bits(const Row<InT, WT>& row, double eps, int t, int n, Shared* sm,
                                            int8_t* code, float* scale, InT* h_out) {
  double ssq = 0.0, top = 0.0;
  bool bad = false;  // an infinity or NaN
  for (int i = t; i < row.d; i += n) {
    const double h = row.h64(i), u = fabs(row.u64(i));
    if (h_out) store1(h_out + i, row.h32(i));
    bad |= !(u <= 1.7976931348623157e308) || !(fabs(h) <= 1.7976931348623157e308);
    ssq += h * h;
    top = fmax(top, u);
  }
  if (bad) ssq = __longlong_as_double(0x7ff8000000000000ll);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    ssq += __shfl_xor_sync(0xffffffffu, ssq, o);
    top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  if (n > 32) {
    if ((t & 31) == 0) {
      sm->dsq[t >> 5] = ssq;
      sm->dtop[t >> 5] = top;
    }
    __syncthreads();
    ssq = top = 0.0;
    for (int i = 0; i < n >> 5; ++i) {
      ssq += sm->dsq[i];
      top = fmax(top, sm->dtop[i]);
    }
  }
  const double root = sqrt(ssq / row.d + eps);
  // no root (eps 0 and a row of zeros) leaves 0 / 0
  const bool ok = root > 0.0 && root <= 1.7976931348623157e308;
  const double den = fmax(top, 1e-12 * root);
  for (int i = t; i < row.d; i += n)
    code[i] = ok ? (int8_t)__double2int_rn(__ddiv_rn(127.0 * row.u64(i), den)) : (int8_t)0;
  if (t == 0) *scale = ok ? (float)(den / root / 127.0) : __int_as_float(0x7fc00000);
}

__device__ __forceinline__ float nan_max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// A row's sum of squares and largest |u|: the warp's, then the block's.
template <bool WARP>
__device__ __forceinline__ void reduce(float& ssq, float& top, Shared& sm, int t, int n) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    ssq += __shfl_xor_sync(0xffffffffu, ssq, o);
    top = nan_max(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  if constexpr (!WARP) {
    if ((t & 31) == 0) {
      sm.ssq[t >> 5] = ssq;
      sm.top[t >> 5] = top;
    }
    __syncthreads();
    const int lane = t & 31, warps = n >> 5;
    ssq = lane < warps ? sm.ssq[lane] : 0.0f;
    top = lane < warps ? sm.top[lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      ssq += __shfl_xor_sync(0xffffffffu, ssq, o);
      top = nan_max(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
  }
}

// Squares and products in the range in which fp32 holds them to 2^-24, the largest y
// above what the scale's lower bound asks for.
__device__ __forceinline__ bool in_range(float ssq, float top, float inv_d, double eps) {
  const float root = sqrtf(fmaf(ssq, inv_d, (float)eps));
  return ssq >= 1e-30f && ssq <= 1e37f && top >= 1e-30f && top <= 1e37f && top >= 1.01e-12f * root;
}

// Value j of a thread's chunk c.
template <bool VEC>
__device__ __forceinline__ int index_of(int c, int j, int t, int n) {
  return VEC ? (c * n + t) * 8 + j : (c * 8 + j) * n + t;
}
// Elements that need 64 bits: a bit each, so that there is one place that reads them again.
template <bool VEC>
__device__ __forceinline__ int index_of_bit(uint32_t bits, int t, int n) {
  const int b = __ffs(bits) - 1;
  return index_of<VEC>(b >> 3, b & 7, t, n);
}

// 8 values of h taken into the sum of squares; u and its largest.
__device__ __forceinline__ void take8(const uint64_t (&xv)[4], const uint64_t (&wv)[4], uint64_t (&u)[4],
                                      uint64_t& ssq, float& top) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    ssq = ffma2(xv[j], xv[j], ssq);
    u[j] = fmul2(xv[j], wv[j]);
    const float2 v = unpack2(u[j]);
    top = nan_max3(top, fabsf(v.x), fabsf(v.y));
  }
}

// The largest |u| in 64 bits of this thread's, whose largest in fp32 is `mine`: of those
// that fp32 cannot tell from the row's largest.
template <int NC, bool VEC, typename RowT>
__device__ __forceinline__ double largest(const uint64_t (&u)[NC][4], float mine, float top, const RowT& row, int t,
                                          int n) {
  const float near_top = top * (1.0f - 0x1p-21f);
  double most = 0.0;
  if (mine >= near_top) {
    uint32_t bits = 0;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 v = unpack2(u[c][j]);
        bits |= fabsf(v.x) >= near_top ? 1u << (8 * c + 2 * j) : 0u;
        bits |= fabsf(v.y) >= near_top ? 2u << (8 * c + 2 * j) : 0u;
      }
    for (; bits; bits &= bits - 1) most = fmax(most, fabs(row.u64(index_of_bit<VEC>(bits, t, n))));
  }
  return most;
}

// Codes and scale.
template <int NC, bool VEC, typename RowT>
__device__ __forceinline__ void put_codes(const uint64_t (&u)[NC][4], double most, float ssq, double eps,
                                          const RowT& row, int t, int n, int8_t* code, float* scale) {
  constexpr float kNear = 0.5f - 127.0f * 0x1p-21f, kRound = 12582912.0f;  // 1.5 * 2^23
  const int d = row.d;
  const float factor = __fdiv_rn(127.0f, (float)most);
  const uint64_t f2 = pack2(factor, factor), r2 = pack2(kRound, kRound), minus = pack2(-1.0f, -1.0f);
  float far = 0.0f;  // largest distance from the code taken
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    uint32_t q[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint64_t v = fmul2(u[c][j], f2), k = fadd2(v, r2);
      const float2 off = unpack2(fadd2(v, ffma2(k, minus, r2))), kk = unpack2(k);
      q[2 * j] = __float_as_uint(kk.x);  // the code in the low byte
      q[2 * j + 1] = __float_as_uint(kk.y);
      far = fmaxf(fmaxf(far, fabsf(off.x)), fabsf(off.y));
    }
    if constexpr (VEC) {
      uint32_t p[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
        p[i] = __byte_perm(__byte_perm(q[4 * i], q[4 * i + 1], 0x0040), __byte_perm(q[4 * i + 2], q[4 * i + 3], 0x0040),
                           0x5410);
      if (index_of<VEC>(c, 0, t, n) < d)
        *reinterpret_cast<uint2*>(code + index_of<VEC>(c, 0, t, n)) = make_uint2(p[0], p[1]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (index_of<VEC>(c, j, t, n) < d) code[index_of<VEC>(c, j, t, n)] = (int8_t)q[j];
    }
  }
  if (far > kNear) {  // over what this thread has just stored
    uint32_t bits = 0;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 v = unpack2(fmul2(u[c][j], f2));
        bits |= fabsf(v.x - rintf(v.x)) > kNear ? 1u << (8 * c + 2 * j) : 0u;
        bits |= fabsf(v.y - rintf(v.y)) > kNear ? 2u << (8 * c + 2 * j) : 0u;
      }
    for (; bits; bits &= bits - 1) {
      const int i = index_of_bit<VEC>(bits, t, n);
      code[i] = (int8_t)__double2int_rn(__ddiv_rn(127.0 * row.u64(i), most));
    }
  }
  if (t == 0) *scale = (float)(most / sqrt((double)ssq / d + eps) / 127.0);
}

// WARP: a warp a row, kWarpRows of them a block; otherwise a block of up to MAX
// threads a row, MIN of them on an SM.
template <typename InT, typename WT, int NC, int MAX, int MIN, bool VEC, bool WARP>
__global__ void __launch_bounds__(WARP ? 32 * kWarpRows : MAX, MIN)
    rms_norm_kernel(const InT* __restrict__ x, const InT* __restrict__ r, int64_t rows, int d, int64_t ldx,
                    int64_t ldr, const WT* __restrict__ w, double eps, float inv_d, int8_t* __restrict__ codes,
                    float* __restrict__ scales, InT* __restrict__ h_out) {
  __shared__ Shared sm;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x, n = WARP ? 32 : blockDim.x;
  const int64_t at = WARP ? (int64_t)blockIdx.x * kWarpRows + (threadIdx.x >> 5) : (int64_t)blockIdx.x;
  pdl_trigger();
  if (!WARP && t == 0) sm.most = 0;
  pdl_wait();
  if (WARP && at >= rows) return;
  const Row<InT, WT> row = {x + at * ldx, r ? r + at * ldr : nullptr, w, d};
  int8_t* code = codes + at * d;
  InT* ho = h_out ? h_out + at * d : nullptr;
  if (d > kMaxRow) {  // longer than the registers
    row_in_64_bits(row, eps, t, n, &sm, code, scales + at, ho);
    return;
  }
  auto index = [&](int c, int j) { return index_of<VEC>(c, j, t, n); };
  uint64_t u[NC][4];
  uint64_t sq2 = 0;
  float top = 0.0f;
  if constexpr (VEC) {
    // x and r of the whole row on their way at once; as many registers as u takes after
    Raw8<InT> xr[NC], rr[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (index(c, 0) < d) {
        xr[c].load(row.x + index(c, 0));
        if (r) rr[c].load(row.r + index(c, 0));
      }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (index(c, 0) < d) {
        Raw8<WT> wr;
        wr.load(w + index(c, 0));
        uint64_t h[4], v[4];
        xr[c].get(h);
        if (r) {
          rr[c].get(v);
#pragma unroll
          for (int j = 0; j < 4; ++j) h[j] = fadd2(h[j], v[j]);
        }
        if (ho) store8(ho + index(c, 0), h);
        wr.get(v);
        take8(h, v, u[c], sq2, top);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) u[c][j] = 0;
      }
    }
  } else {
    uint64_t h[NC][4];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i0 = index(c, 2 * j), i1 = index(c, 2 * j + 1);
        h[c][j] = pack2(i0 < d ? row.h32(i0) : 0.0f, i1 < d ? row.h32(i1) : 0.0f);
        u[c][j] = pack2(i0 < d ? load_as_f32(w, i0) : 0.0f, i1 < d ? load_as_f32(w, i1) : 0.0f);
      }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i0 = index(c, 2 * j), i1 = index(c, 2 * j + 1);
        const float2 v = unpack2(h[c][j]);
        if (ho && i0 < d) store1(ho + i0, v.x);
        if (ho && i1 < d) store1(ho + i1, v.y);
      }
      take8(h[c], u[c], u[c], sq2, top);
    }
  }
  const float mine = top;
  const float2 sq = unpack2(sq2);
  float ssq = sq.x + sq.y;
  reduce<WARP>(ssq, top, sm, t, n);
  if (!in_range(ssq, top, inv_d, eps)) {  // the same for the whole row
    row_in_64_bits<InT, WT>(row, eps, t, n, &sm, code, scales + at, nullptr);
    return;
  }
  double most = largest<NC, VEC>(u, mine, top, row, t, n);
  if constexpr (WARP) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = fmax(most, __shfl_xor_sync(0xffffffffu, most, o));
  } else {
    // bits of non-negative numbers rise with them
    if (most > 0.0) atomicMax(&sm.most, (unsigned long long)__double_as_longlong(most));
    __syncthreads();
    most = __longlong_as_double((long long)sm.most);
  }
  put_codes<NC, VEC>(u, most, ssq, eps, row, t, n, code, scales + at);
}

struct NormArgs {
  const void *x, *r, *w;
  int64_t rows, d, ldx, ldr;
  double eps;
  int8_t* codes;
  float* scales;
  void* h;
};

template <typename InT, typename WT, int NC, int MAX, int MIN, bool VEC, bool WARP>
int launch(const NormArgs& a, int threads, cudaStream_t st) {
  const int64_t blocks = WARP ? cdiv(a.rows, kWarpRows) : a.rows;
  MXB_CUDA_TRY(launch_pdl(rms_norm_kernel<InT, WT, NC, MAX, MIN, VEC, WARP>, dim3((unsigned)blocks),
                          WARP ? 32 * kWarpRows : threads, 0, st, static_cast<const InT*>(a.x),
                          static_cast<const InT*>(a.r), a.rows, (int)a.d, a.ldx, a.ldr,
                          static_cast<const WT*>(a.w), a.eps, (float)(1.0 / (double)a.d), a.codes, a.scales,
                          static_cast<InT*>(a.h)));
  MXB_LAUNCH_CHECK();
  return MXB_OK;
}

template <typename InT, typename WT, bool VEC>
int by_size(const NormArgs& a, cudaStream_t st) {
  // threads of a row with 8 nc values each
  auto threads = [&](int nc) { return (int)cdiv(cdiv(a.d, 8 * nc), 32) * 32; };
  if (a.d > kMaxRow) return launch<InT, WT, 1, 1024, 1, VEC, false>(a, 1024, st);
  if (a.d <= 1024 && a.rows > kSMs) {
    return a.d <= 256   ? launch<InT, WT, 1, 32, 4, VEC, true>(a, 32, st)
           : a.d <= 512 ? launch<InT, WT, 2, 32, 4, VEC, true>(a, 32, st)
                        : launch<InT, WT, 4, 32, 3, VEC, true>(a, 32, st);
  }
  // few rows, or values loaded one by one: as many threads as a row has use for
  if ((a.rows <= 2 * kSMs || !VEC) && threads(1) <= 1024)
    return launch<InT, WT, 1, 1024, 1, VEC, false>(a, threads(1), st);
  if constexpr (VEC) {
    // 64 registers a thread hold a row of bf16 on its way and its u, of fp32 they do not
    // (80 bytes of spills; 4096 x 4096 with a residual 50 us, 44 with three rows an SM)
    constexpr int kRows = sizeof(InT) == 2 ? 4 : 3;
    if (threads(4) <= 256) return launch<InT, WT, 4, 256, kRows, VEC, false>(a, threads(4), st);
  }
  if (threads(4) <= 512)
    return launch<InT, WT, 4, 512, VEC && sizeof(InT) == 2 ? 2 : 1, VEC, false>(a, threads(4), st);
  return launch<InT, WT, 4, 1024, 1, VEC, false>(a, threads(4), st);
}

template <typename InT>
int by_type(const NormArgs& a, int w_dtype, cudaStream_t st) {
  constexpr int64_t per = 16 / sizeof(InT);
  const bool vec = a.d % 8 == 0 && a.ldx % per == 0 && (!a.r || a.ldr % per == 0) &&
                   ((uintptr_t)a.x | (uintptr_t)a.r | (uintptr_t)a.w | (uintptr_t)a.h | (uintptr_t)a.codes) % 16 == 0;
  if (w_dtype == MXB_BF16)
    return vec ? by_size<InT, __nv_bfloat16, true>(a, st) : by_size<InT, __nv_bfloat16, false>(a, st);
  return vec ? by_size<InT, float, true>(a, st) : by_size<InT, float, false>(a, st);
}

}  // namespace

extern "C" int mxb_rms_norm_quantize(const void* x, const void* residual, int x_dtype, int64_t rows, int64_t d,
                                     int64_t x_stride, int64_t residual_stride, const void* weight, int w_dtype,
                                     double eps, void* codes, float* scales, void* sum, void* stream) {
  if ((x_dtype != MXB_F32 && x_dtype != MXB_BF16) || (w_dtype != MXB_F32 && w_dtype != MXB_BF16))
    return MXB_E_DTYPE;
  if (rows < 0 || rows > INT32_MAX || d <= 0 || d > (int64_t)1 << 30) return MXB_E_SHAPE;
  if (!(eps >= 0.0 && eps <= 1e30)) return MXB_E_ARG;
  if (rows == 0) return MXB_OK;
  if (!x || !weight || !codes || !scales) return MXB_E_ARG;
  const uintptr_t xa = x_dtype == MXB_BF16 ? 2 : 4, wa = w_dtype == MXB_BF16 ? 2 : 4;
  if (((uintptr_t)x | (uintptr_t)residual | (uintptr_t)sum) % xa || (uintptr_t)weight % wa ||
      (uintptr_t)scales % 4)
    return MXB_E_ALIGN;
  if (x_stride < 0 || residual_stride < 0) return MXB_E_SHAPE;
  // the inputs are read again after codes and sum are written
  auto meets = [&](const void* p, int64_t n, uintptr_t size) {
    const uintptr_t lo = (uintptr_t)p, hi = lo + (uintptr_t)n * size;
    auto over = [&](const void* out, uintptr_t bytes) {
      return p && out && lo < (uintptr_t)out + bytes && (uintptr_t)out < hi;
    };
    return over(sum, (uintptr_t)(rows * d) * xa) || over(codes, (uintptr_t)(rows * d)) ||
           over(scales, (uintptr_t)rows * 4);
  };
  if (meets(x, (rows - 1) * x_stride + d, xa) || meets(residual, (rows - 1) * residual_stride + d, xa) ||
      meets(weight, d, wa))
    return MXB_E_ARG;
  const NormArgs a = {x, residual, weight, rows, d, x_stride, residual_stride, eps, static_cast<int8_t*>(codes),
                      scales, sum};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return x_dtype == MXB_BF16 ? by_type<__nv_bfloat16>(a, w_dtype, st) : by_type<float>(a, w_dtype, st);
}
