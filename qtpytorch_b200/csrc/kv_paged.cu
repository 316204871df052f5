// Paged quantized KV cache: quantize tokens into their slots as they are
// written, and read ragged histories back through a page table.
//
// Pool: codes [pages][heads][page][D * bits / 8], scales [pages][heads][page]
// fp32, for K and for V; slot = page number * page + offset.  The codes and
// scales of a head row are those of mxb_quantize with block = D.
//
// Both kernels are one pass over HBM.  Write: D / 8 lanes own a head row (one
// 16-byte load of bf16 each), so the row maximum is 3 or 4 shuffles and a
// row's codes leave as one run.  Read: a thread produces 16 bytes of output.
// 4 x 4096 tokens of 8 heads of 128 dims between bf16 and int4 (85 MB): write 23 us
// = 3.7 TB/s, read 19.6 us = 4.3 TB/s, at 0.8 instructions issued a cycle as near
// the ALU's limit as HBM's; a step's 32 tokens are bound by the launch.  In the read,
// rows found by a product instead of a division, and codes as the low bits of 2^23,
// were slower (21.7 us).
#include "mxb_common.cuh"
#include "mxb_internal.h"

using namespace mxb;

namespace {

constexpr int kThreads = 256;
constexpr int kErrIndexCode = 8;  // tc_ptx.cuh kErrIndex

// Eight consecutive values.
__device__ __forceinline__ void load8v(const float* p, bool vec, float (&v)[8]) {
  if (vec) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p));
    const float4 b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = p[i];
  }
}
__device__ __forceinline__ void load8v(const __nv_bfloat16* p, bool vec, float (&v)[8]) {
  if (vec) {
    const uint4 r = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __bfloat162float(p[i]);
  }
}

// One head row's eight values of this lane -> codes and scale in the slot.
template <int BITS, int D>
__device__ __forceinline__ void put_row(const float (&x)[8], float a, int64_t r, int part,
                                        uint8_t* __restrict__ codes, float* __restrict__ scales) {
  constexpr float m = BITS == 8 ? 127.0f : 7.0f;
  // the integer quantizer's order of roundings (quantize.cu block_factor)
  const float si = __fmul_rn(__frcp_rn(nan_max(a, 1e-12f)), m);
  uint32_t c[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    c[j] = __float_as_uint(__fadd_rn(__fmul_rn(x[j], si), 12582912.0f)) & (BITS == 8 ? 255u : 15u);
  if (!(si > 0.0f && si <= 3.4028235e38f)) {  // an infinity or NaN in the row
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = 0u;
  }
  uint8_t* dst = codes + r * (D * BITS / 8) + part * BITS;
  if (BITS == 8) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24,
                                                c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24);
  } else {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) w |= c[j] << (4 * j);
    *reinterpret_cast<uint32_t*>(dst) = w;
  }
  if (part == 0) scales[r] = __frcp_rn(si);
}

// A lane takes its eight values of a key and of the value beside it: two loads
// in flight, and the slot's address once for both.
template <typename InT, int BITS, int D>
__global__ void __launch_bounds__(kThreads)
    kv_write_kernel(const InT* __restrict__ k, const InT* __restrict__ v, int64_t T, int H,
                    int64_t k_ts, int64_t k_hs, int64_t v_ts, int64_t v_hs, bool vec,
                    const int64_t* __restrict__ slots, int64_t n_slots, int page_shift,
                    uint8_t* __restrict__ kc, float* __restrict__ ks, uint8_t* __restrict__ vc,
                    float* __restrict__ vs, int* __restrict__ err) {
  constexpr int L = D / 8;
  pdl_trigger();
  pdl_wait();
  // 32-bit index: T * H < 2^31 (checked at the launch)
  const uint32_t row = blockIdx.x * (uint32_t)(kThreads / L) + threadIdx.x / L;
  const int part = threadIdx.x % L;
  const bool live = row < (uint32_t)(T * H);
  const uint32_t t32 = live ? row / (uint32_t)H : 0u;
  const int64_t t = t32;
  const int h = live ? (int)(row - t32 * (uint32_t)H) : 0;
  float x[8], y[8];
  int64_t slot = -1;
  if (live) {
    slot = slots[t];
    load8v(k + t * k_ts + h * k_hs + part * 8, vec, x);
    load8v(v + t * v_ts + h * v_hs + part * 8, vec, y);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = y[j] = 0.0f;
  }
  float a = 0.0f, b = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    a = amax_step(a, x[j]);
    b = amax_step(b, y[j]);
  }
#pragma unroll
  for (int o = L >> 1; o > 0; o >>= 1) {
    a = nan_max(a, __shfl_xor_sync(0xffffffffu, a, o));
    b = nan_max(b, __shfl_xor_sync(0xffffffffu, b, o));
  }
  if (slot < 0) return;  // padding token
  if (slot >= n_slots) {
    if (part == 0 && err) atomicCAS(err, 0, kErrIndexCode);
    return;
  }
  const int64_t pg = slot >> page_shift;
  const int64_t r = ((pg * H + h) << page_shift) + (slot & ((1 << page_shift) - 1));
  put_row<BITS, D>(x, a, r, part, kc, ks);
  put_row<BITS, D>(y, b, r, part, vc, vs);
}

// blockIdx.y: sequence, blockIdx.z: 0 the keys, 1 the values.  A thread makes
// 16 bytes of output; kU of them in flight.
template <typename OutT, int BITS, int D>
__global__ void __launch_bounds__(kThreads)
    kv_read_kernel(const uint8_t* __restrict__ kc, const float* __restrict__ ks,
                   const uint8_t* __restrict__ vc, const float* __restrict__ vs,
                   const int* __restrict__ table, int width, const int* __restrict__ lengths,
                   int64_t n_pages, int H, int page_shift, uint32_t max_len, OutT* __restrict__ ko,
                   OutT* __restrict__ vo, int* __restrict__ err) {
  constexpr int E = 16 / sizeof(OutT), C = D / E, kU = 4;
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.y;
  const bool val = blockIdx.z != 0;
  const uint8_t* codes = val ? vc : kc;
  const float* scales = val ? vs : ks;
  OutT* out = (val ? vo : ko) + (int64_t)b * max_len * H * D;
  const uint32_t len = (uint32_t)max(lengths[b], 0), rows = max_len * (uint32_t)H;
  constexpr uint32_t kRows = kThreads / C;  // head rows per block and step
  const uint32_t row0 = blockIdx.x * (kRows * kU) + threadIdx.x / C;
  const int part = threadIdx.x % C;
  uint64_t w[kU];
  float s[kU];
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    const uint32_t row = row0 + u * kRows;
    w[u] = 0;
    s[u] = 0.0f;
    if (row < rows) {
      const uint32_t pos = row / (uint32_t)H;
      const int h = (int)(row - pos * (uint32_t)H);
      if (pos < len) {
        const uint32_t at = pos >> page_shift;
        const int pg = at < (uint32_t)width ? table[(int64_t)b * width + at] : -1;
        if (pg >= 0 && pg < n_pages) {
          const int64_t r =
              (((int64_t)pg * H + h) << page_shift) + (pos & ((1u << page_shift) - 1u));
          const uint8_t* p = codes + r * (D * BITS / 8) + part * (E * BITS / 8);
          if (E * BITS == 64) w[u] = __ldg(reinterpret_cast<const unsigned long long*>(p));
          else if (E * BITS == 32) w[u] = __ldg(reinterpret_cast<const uint32_t*>(p));
          else w[u] = __ldg(reinterpret_cast<const uint16_t*>(p));
          s[u] = __ldg(scales + r);
        } else if (err) {
          atomicCAS(err, 0, kErrIndexCode);
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    const uint32_t row = row0 + u * kRows;
    if (row >= rows) continue;
    float v[E];
#pragma unroll
    for (int j = 0; j < E; ++j)
      v[j] = __fmul_rn((float)sext((uint32_t)(w[u] >> (j * BITS)), BITS), s[u]);
    OutT* o = out + (int64_t)row * D + part * E;
    if (sizeof(OutT) == 4) {
      __stcs(reinterpret_cast<float4*>(o), make_float4(v[0], v[1], v[2], v[3]));
    } else {
      uint32_t p[E / 2];
#pragma unroll
      for (int j = 0; j < E / 2; ++j) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        p[j] = *reinterpret_cast<const uint32_t*>(&t);
      }
      __stcs(reinterpret_cast<uint4*>(o), make_uint4(p[0], p[1], p[2 % (E / 2)], p[3 % (E / 2)]));
    }
  }
}

__global__ void __launch_bounds__(kThreads)
    narrow_i64_kernel(const int64_t* __restrict__ src, int64_t n, int* __restrict__ dst) {
  pdl_trigger();
  pdl_wait();
  const int64_t i = blockIdx.x * (int64_t)kThreads + threadIdx.x;
  if (i < n) dst[i] = (int)max(min(src[i], (int64_t)INT32_MAX), (int64_t)INT32_MIN);
}

int shift_of(int page) { return 31 - __builtin_clz((unsigned)page); }

struct WriteArgs {
  int64_t T;
  int H;
  int64_t k_ts, k_hs, v_ts, v_hs;
  const int64_t* slots;
  int64_t n_slots;
  int page;
  uint8_t *kc, *vc;
  float *ks, *vs;
};

template <typename InT, int BITS, int D>
int write_t(const void* k, const void* v, const WriteArgs& a, cudaStream_t st) {
  const int64_t blocks = cdiv(a.T * a.H * (D / 8), kThreads);
  if (a.T * a.H >= (int64_t)1 << 31) return MXB_E_SHAPE;
  const int64_t per = 16 / sizeof(InT);
  const bool vec = ((uintptr_t)k | (uintptr_t)v) % 16 == 0 && a.k_ts % per == 0 &&
                   a.k_hs % per == 0 && a.v_ts % per == 0 && a.v_hs % per == 0;
  MXB_CUDA_TRY(launch_pdl(kv_write_kernel<InT, BITS, D>, dim3((unsigned)blocks), kThreads, 0, st,
                          static_cast<const InT*>(k), static_cast<const InT*>(v), a.T, a.H, a.k_ts,
                          a.k_hs, a.v_ts, a.v_hs, vec, a.slots, a.n_slots, shift_of(a.page), a.kc,
                          a.ks, a.vc, a.vs, device_error_ptr()));
  MXB_LAUNCH_CHECK();
  return MXB_OK;
}

struct ReadArgs {
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int* table;
  int width;
  const int* lengths;
  int64_t B, n_pages;
  int H, page;
  int64_t max_len;
};

template <typename OutT, int BITS, int D>
int read_t(const ReadArgs& a, void* ko, void* vo, cudaStream_t st) {
  const int64_t rows = a.max_len * a.H, blocks = cdiv(rows * (D / (16 / (int64_t)sizeof(OutT))), kThreads * 4);
  if (rows >= (int64_t)1 << 31) return MXB_E_SHAPE;
  MXB_CUDA_TRY(launch_pdl(kv_read_kernel<OutT, BITS, D>, dim3((unsigned)blocks, (unsigned)a.B, 2),
                          kThreads, 0, st, a.kc, a.ks, a.vc, a.vs, a.table, a.width, a.lengths,
                          a.n_pages, a.H, shift_of(a.page), (uint32_t)a.max_len,
                          static_cast<OutT*>(ko), static_cast<OutT*>(vo), device_error_ptr()));
  MXB_LAUNCH_CHECK();
  return MXB_OK;
}

template <typename T, template <typename, int, int> class F, typename... A>
int by_format(int bits, int dim, A&&... a) {
  if (bits == 8) return dim == 128 ? F<T, 8, 128>::run(a...) : F<T, 8, 64>::run(a...);
  return dim == 128 ? F<T, 4, 128>::run(a...) : F<T, 4, 64>::run(a...);
}
template <typename T, int BITS, int D>
struct Write {
  template <typename... A>
  static int run(A&&... a) { return write_t<T, BITS, D>(a...); }
};
template <typename T, int BITS, int D>
struct Read {
  template <typename... A>
  static int run(A&&... a) { return read_t<T, BITS, D>(a...); }
};

}  // namespace

namespace mxb {
// The pool's geometry, shared by the three entry points.
int kv_pool_check(int64_t n_pages, int heads, int page, int dim, int bits, const void* kc,
                  const void* ks, const void* vc, const void* vs) {
  if (bits != 4 && bits != 8) return MXB_E_DTYPE;
  if (dim != 64 && dim != 128) return MXB_E_SHAPE;
  if (page < 16 || (page & (page - 1)) != 0 || page > 1024) return MXB_E_SHAPE;
  if (n_pages <= 0 || heads <= 0 || heads > 65535) return MXB_E_SHAPE;
  // head rows are tensor-map coordinates
  if (n_pages > (int64_t)INT32_MAX / page / heads) return MXB_E_SHAPE;
  if (!kc || !ks || !vc || !vs) return MXB_E_ARG;
  if (((uintptr_t)kc | (uintptr_t)ks | (uintptr_t)vc | (uintptr_t)vs) % 16) return MXB_E_ALIGN;
  return MXB_OK;
}
}  // namespace mxb

extern "C" {

int mxb_narrow_i64(const int64_t* src, int64_t n, int* dst, void* stream) {
  if (n < 0 || n > ((int64_t)INT32_MAX - 1) * kThreads) return MXB_E_SHAPE;
  if (n == 0) return MXB_OK;
  if (!src || !dst) return MXB_E_ARG;
  MXB_CUDA_TRY(launch_pdl(narrow_i64_kernel, dim3((unsigned)cdiv(n, kThreads)), kThreads, 0,
                          static_cast<cudaStream_t>(stream), src, n, dst));
  MXB_LAUNCH_CHECK();
  return MXB_OK;
}

int mxb_kv_write(const void* k, const void* v, int x_dtype, int64_t T, int heads, int dim,
                 int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                 int64_t v_head_stride, const int64_t* slots, int64_t n_pages, int page, int bits,
                 void* k_codes, float* k_scales, void* v_codes, float* v_scales, void* stream) {
  if (x_dtype != MXB_F32 && x_dtype != MXB_BF16) return MXB_E_DTYPE;
  const int rc = kv_pool_check(n_pages, heads, page, dim, bits, k_codes, k_scales, v_codes, v_scales);
  if (rc != MXB_OK) return rc;
  if (T < 0) return MXB_E_SHAPE;
  if (T == 0) return MXB_OK;
  if (!k || !v || !slots) return MXB_E_ARG;
  if (((uintptr_t)k | (uintptr_t)v) % (x_dtype == MXB_BF16 ? 2 : 4)) return MXB_E_ALIGN;
  WriteArgs a = {T, heads, k_token_stride, k_head_stride, v_token_stride, v_head_stride, slots,
                 n_pages * page, page, static_cast<uint8_t*>(k_codes),
                 static_cast<uint8_t*>(v_codes), k_scales, v_scales};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return x_dtype == MXB_BF16 ? by_format<__nv_bfloat16, Write>(bits, dim, k, v, a, st)
                             : by_format<float, Write>(bits, dim, k, v, a, st);
}

int mxb_kv_read(const void* k_codes, const float* k_scales, const void* v_codes,
                const float* v_scales, int64_t n_pages, int heads, int page, int dim, int bits,
                const int* table, int64_t width, const int* lengths, int64_t B, int64_t max_len,
                void* k_out, void* v_out, int out_dtype, void* stream) {
  if (out_dtype != MXB_F32 && out_dtype != MXB_BF16) return MXB_E_DTYPE;
  const int rc = kv_pool_check(n_pages, heads, page, dim, bits, k_codes, k_scales, v_codes, v_scales);
  if (rc != MXB_OK) return rc;
  if (B < 0 || B > 65535 || max_len < 0 || max_len > INT32_MAX || width < 0 || width > INT32_MAX)
    return MXB_E_SHAPE;
  if (B == 0 || max_len == 0) return MXB_OK;
  if ((width > 0 && !table) || !lengths || !k_out || !v_out) return MXB_E_ARG;
  if (((uintptr_t)k_out | (uintptr_t)v_out) % 16) return MXB_E_ALIGN;
  ReadArgs a = {static_cast<const uint8_t*>(k_codes), static_cast<const uint8_t*>(v_codes),
                k_scales, v_scales, table, (int)width, lengths, B, n_pages, heads, page, max_len};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return out_dtype == MXB_BF16 ? by_format<__nv_bfloat16, Read>(bits, dim, a, k_out, v_out, st)
                               : by_format<float, Read>(bits, dim, a, k_out, v_out, st);
}

}  // extern "C"
