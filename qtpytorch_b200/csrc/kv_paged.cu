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

#include <type_traits>

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

// ── append: keys and queries rotated on the way ─────────────────────────────
// Pair i of a head row, (i, i + rot / 2) or with ILV (2 i, 2 i + 1), turns by
// position * inv_freq[i].  A block takes TB tokens: it finds their cosines and
// sines once, in 64 bits as float pairs hi + lo, and turns every head of q and k
// with the fp32 halves.
//
// A key's codes and scale are those of the quantizer fed the rotation in 64 bits
// rounded to fp32, bit for bit.  The fp32 rotation is off by at most
// 4 * 2^-24 of the row's largest value, so only the values within 2^-20 of the
// largest and those whose quotient comes within m 2^-20 of a border between two
// codes are turned again in 64 bits.
//
// 16384 tokens of 32 + 8 heads of 128 dims, bf16 into int4 (353 MB): 88 us = 4.0 TB/s; 95
// with 8 values of a query row a lane, one at a time, 52 of them without queries (of those
// 1 for the angles, 4 for what 64 bits decide): the chain of a row of keys (its load, three
// reductions, two reciprocals) at 32 warps an SM.  Keys loaded a row ahead (76 registers,
// three blocks) 98, more query rows in flight slower, 48 registers no faster.  32 tokens:
// 4.1 us.
struct Rotary {
  const int64_t* pos;  // [axes][axis_stride]
  int64_t axis_stride;
  const float* inv_freq;
  int pairs;      // rot / 2
  int end[3];     // first pair of axes 1 to 3
};

struct AppendRows {
  const void *q, *k, *v;
  int64_t T;
  int Hq, H;  // Hq 0: no queries
  int q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;  // strides below 2^31, their products are not
  bool vec;
};

// Four values as they lie in memory, for loads in flight.
template <typename T>
struct Raw4;
template <>
struct Raw4<float> {
  float4 r;
  __device__ __forceinline__ void load(const float* p, bool vec) {
    if (vec) r = __ldg(reinterpret_cast<const float4*>(p));
    else r = make_float4(p[0], p[1], p[2], p[3]);
  }
  __device__ __forceinline__ void get(float (&v)[4]) const {
    v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w;
  }
};
template <>
struct Raw4<__nv_bfloat16> {
  uint2 r;
  __device__ __forceinline__ void load(const __nv_bfloat16* p, bool vec) {
    if (vec) {
      r = __ldg(reinterpret_cast<const uint2*>(p));
    } else {
      const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
      r = make_uint2(q[0] | (uint32_t)q[1] << 16, q[2] | (uint32_t)q[3] << 16);
    }
  }
  __device__ __forceinline__ void get(float (&v)[4]) const {
    v[0] = __uint_as_float(r.x << 16);
    v[1] = __uint_as_float(r.x & 0xffff0000u);
    v[2] = __uint_as_float(r.y << 16);
    v[3] = __uint_as_float(r.y & 0xffff0000u);
  }
};
__device__ __forceinline__ void store4(float* p, const float (&v)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float (&v)[4]) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
  *reinterpret_cast<uint2*>(p) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// Eight bf16 values as they lie in memory (16-byte aligned), in pairs.
struct Raw8 {
  uint4 r;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { r = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void get(uint64_t (&v)[4]) const {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = pack2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
};
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

// cos and sin of an angle in 64 bits, however large: in turns, as a product and its
// rounding error, so that the whole turns leave exactly.
__device__ __forceinline__ void turn64(double angle, double& c, double& s) {
  constexpr double kHi = 0.15915494309189535, kLo = -9.839338337591243e-18;  // 1 / (2 pi)
  const double t = __dmul_rn(angle, kHi), lo = fma(angle, kLo, fma(angle, kHi, -t));
  sincospi(2.0 * ((t - rint(t)) + lo), &s, &c);
}

constexpr int kAppendTokens = 4;  // at most, a block
// Token of row u of a block, `per` rows a token: a division costs a fifth of a row's work.
__device__ __forceinline__ int token_of(int u, int per) {
  static_assert(kAppendTokens == 4, "three borders");
  return (u >= per) + (u >= 2 * per) + (u >= 3 * per);
}
__device__ __forceinline__ int64_t offset_of(int t, int ts, int h, int hs) {
  return (int64_t)t * ts + (int64_t)h * hs;
}

// Q16: a lane takes 16 values of a query row in pairs (bf16, aligned, whole runs of 8
// pairs), otherwise 8.
template <typename InT, int BITS, int D, bool ILV, bool Q16>
__global__ void __launch_bounds__(kThreads)
    kv_append_kernel(const AppendRows a, const Rotary ro, int TB, const int64_t* __restrict__ slots,
                     int64_t n_slots, int page_shift, InT* __restrict__ q_out, uint8_t* __restrict__ kc,
                     float* __restrict__ ks, uint8_t* __restrict__ vc, float* __restrict__ vs,
                     int* __restrict__ err) {
  constexpr int L = D / 8, kRows = kThreads / L;
  constexpr float m = BITS == 8 ? 127.0f : 7.0f;
  __shared__ float4 hi[kAppendTokens][D / 4];  // cosines and sines of two pairs
  __shared__ float4 lo[kAppendTokens][D / 4];  // (cos, sin) of two pairs
  pdl_trigger();
  pdl_wait();
  const int64_t t0 = (int64_t)blockIdx.x * TB;
  const int tokens = (int)min((int64_t)TB, a.T - t0);
  const int part = threadIdx.x % L, q_rows = tokens * a.Hq, kv_rows = tokens * a.H;
  // this lane's two runs of four values, and whether they turn
  const bool turns = part < ro.pairs / 4;
  const int oa = ILV || !turns ? part * 8 : part * 4, ob = ILV || !turns ? oa + 4 : ro.pairs + part * 4;
  const InT* q = static_cast<const InT*>(a.q) + t0 * a.q_ts;
  const InT* k = static_cast<const InT*>(a.k) + t0 * a.k_ts;
  const InT* v = static_cast<const InT*>(a.v) + t0 * a.v_ts + part * 8;
  // rows of queries, kU of them in flight; the first while the angles are found
  constexpr int QE = Q16 ? 8 : 4, QL = D / (2 * QE), kQRows = kThreads / QL, kU = 16 / QE;
  const int q_part = threadIdx.x % QL;
  const bool q_turns = q_part < ro.pairs / QE;
  const int qa = q_part * (ILV || !q_turns ? 2 * QE : QE), qb = ILV || !q_turns ? qa + QE : ro.pairs + qa;
  using Raw = std::conditional_t<Q16, Raw8, Raw4<InT>>;
  Raw ra[kU], rb[kU];
  auto load_q = [&](int u0) {
#pragma unroll
    for (int i = 0; i < kU; ++i) {
      const int u = u0 + i * kQRows;
      if (u < q_rows) {
        const int t = token_of(u, a.Hq);
        const InT* p = q + offset_of(t, a.q_ts, u - t * a.Hq, a.q_hs);
        if constexpr (Q16) {
          ra[i].load(p + qa);
          rb[i].load(p + qb);
        } else {
          ra[i].load(p + qa, a.vec);
          rb[i].load(p + qb, a.vec);
        }
      }
    }
  };
  int u0 = threadIdx.x / QL;
  load_q(u0);
  q_out += t0 * a.Hq * D;
  for (int i = threadIdx.x; i < tokens * ro.pairs; i += kThreads) {
    const int t = i / ro.pairs, p = i - t * ro.pairs;
    const int axis = (p >= ro.end[0]) + (p >= ro.end[1]) + (p >= ro.end[2]);
    double c, s;
    turn64(__dmul_rn((double)ro.pos[axis * ro.axis_stride + t0 + t], (double)__ldg(ro.inv_freq + p)), c, s);
    const float ch = (float)c, sh = (float)s;
    float* at = reinterpret_cast<float*>(&hi[t][p >> 1]) + (p & 1);
    at[0] = ch;
    at[2] = sh;
    reinterpret_cast<float2*>(lo[t])[p] = make_float2((float)(c - (double)ch), (float)(s - (double)sh));
  }
  __syncthreads();
  // pair j of this lane: values (j, j + 4), or (2 j, 2 j + 1)
  auto first = [](int j) { return ILV ? 2 * j : j; };
  auto second = [](int j) { return ILV ? 2 * j + 1 : j + 4; };
  auto turn = [&](int t, const float (&x)[8], float (&y)[8], float (&cs)[8]) {
    if (turns) {
      const float4 c0 = hi[t][part * 2], c1 = hi[t][part * 2 + 1];
      cs[0] = c0.x; cs[1] = c0.z; cs[2] = c0.y; cs[3] = c0.w;
      cs[4] = c1.x; cs[5] = c1.z; cs[6] = c1.y; cs[7] = c1.w;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float v0 = x[first(j)], v1 = x[second(j)], c = cs[2 * j], s = cs[2 * j + 1];
        y[first(j)] = fmaf(v0, c, -__fmul_rn(v1, s));
        y[second(j)] = fmaf(v0, s, __fmul_rn(v1, c));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = x[j];
    }
  };
  [[maybe_unused]] auto get8 = [](const Raw4<InT>& r0, const Raw4<InT>& r1, float (&x)[8]) {
    r0.get(*reinterpret_cast<float (*)[4]>(x));
    r1.get(*reinterpret_cast<float (*)[4]>(x + 4));
  };
  while (u0 < q_rows) {
#pragma unroll
    for (int i = 0; i < kU; ++i) {
      const int u = u0 + i * kQRows;
      if (u < q_rows) {
        const int t = token_of(u, a.Hq);
        InT* o = q_out + u * D;  // u counts a token's heads in their order
        if constexpr (Q16) {
          uint64_t x0[4], x1[4];
          ra[i].get(x0);
          rb[i].get(x1);
          if (q_turns) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float4 f = hi[t][q_part * 4 + j];
              if constexpr (ILV) {  // two pairs lie in x0[2 j], x0[2 j + 1], then in x1
                uint64_t* x = j < 2 ? x0 + 2 * j : x1 + 2 * j - 4;
                const float2 v0 = unpack2(x[0]), v1 = unpack2(x[1]);
                x[0] = pack2(fmaf(v0.x, f.x, -__fmul_rn(v0.y, f.z)), fmaf(v0.x, f.z, __fmul_rn(v0.y, f.x)));
                x[1] = pack2(fmaf(v1.x, f.y, -__fmul_rn(v1.y, f.w)), fmaf(v1.x, f.w, __fmul_rn(v1.y, f.y)));
              } else {
                const uint64_t c = pack2(f.x, f.y), s = pack2(f.z, f.w), ns = pack2(-f.z, -f.w), v0 = x0[j];
                x0[j] = ffma2(v0, c, fmul2(x1[j], ns));
                x1[j] = ffma2(v0, s, fmul2(x1[j], c));
              }
            }
          }
          store8(o + qa, x0);
          store8(o + qb, x1);
        } else {
          float x[8], y[8], cs[8];
          get8(ra[i], rb[i], x);
          turn(t, x, y, cs);
          store4(o + qa, *reinterpret_cast<float (*)[4]>(y));
          store4(o + qb, *reinterpret_cast<float (*)[4]>(y + 4));
        }
      }
    }
    u0 += kU * kQRows;
    load_q(u0);
  }
  // keys, with the values beside them; a warp goes through its loop as one
  for (int u1 = threadIdx.x / 32 * (32 / L); u1 < kv_rows; u1 += kRows) {
    const int u = u1 + (threadIdx.x % 32) / L;
    const bool live = u < kv_rows;
    const int t = live ? token_of(u, a.H) : 0, h = live ? u - t * a.H : 0;
    float x[8], y[8], w[8], cs[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = w[j] = 0.0f;
    int64_t slot = -1;
    if (live) {
      const InT* p = k + offset_of(t, a.k_ts, h, a.k_hs);
      Raw4<InT> r0, r1;
      r0.load(p + oa, a.vec);
      r1.load(p + ob, a.vec);
      slot = slots[t0 + t];
      load8v(v + offset_of(t, a.v_ts, h, a.v_hs), a.vec, w);
      get8(r0, r1, x);
    }
    turn(t, x, y, cs);
    // value j turned in 64 bits, rounded to fp32
    auto again = [&](int j) -> float {
      const int i = ILV ? j >> 1 : j & 3;
      const float2 l = reinterpret_cast<const float2*>(lo[t])[part * 4 + i];
      const double c = (double)cs[2 * i] + (double)l.x, s = (double)cs[2 * i + 1] + (double)l.y;
      const double v0 = (double)x[first(i)], v1 = (double)x[second(i)];
      return (float)(j == first(i) ? v0 * c - v1 * s : v0 * s + v1 * c);
    };
    float top = 0.0f, top_v = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      top = amax_step(top, y[j]);
      top_v = amax_step(top_v, w[j]);
    }
    const float mine = top;
#pragma unroll
    for (int o = L >> 1; o > 0; o >>= 1) {
      top = nan_max(top, __shfl_xor_sync(0xffffffffu, top, o));
      top_v = nan_max(top_v, __shfl_xor_sync(0xffffffffu, top_v, o));
    }
    if (ro.pairs > 0) {
      const float near_top = top * (1.0f - 0x1p-20f);
      float best = 0.0f;
      if (!(mine < near_top)) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!(fabsf(y[j]) < near_top)) best = amax_step(best, turns ? again(j) : y[j]);
      }
#pragma unroll
      for (int o = L >> 1; o > 0; o >>= 1) best = nan_max(best, __shfl_xor_sync(0xffffffffu, best, o));
      top = best;
    }
    if (!live || slot < 0) continue;
    if (slot >= n_slots) {
      if (part == 0 && err) atomicCAS(err, 0, kErrIndexCode);
      continue;
    }
    const int64_t r = (((slot >> page_shift) * a.H + h) << page_shift) + (slot & ((1 << page_shift) - 1));
    put_row<BITS, D>(w, top_v, r, part, vc, vs);
    const float si = __fmul_rn(__frcp_rn(nan_max(top, 1e-12f)), m);
    const bool ok = si > 0.0f && si <= 3.4028235e38f;  // no infinity or NaN in the row
    float far = 0.0f;  // largest distance from a whole number
    constexpr float kNear = 0.5f - m * 0x1p-20f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      w[j] = __fmul_rn(y[j], si);
      far = fmaxf(far, fabsf(w[j] - rintf(w[j])));
    }
    if (turns && far > kNear) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (fabsf(w[j] - rintf(w[j])) > kNear) w[j] = __fmul_rn(again(j), si);
    }
    uint32_t c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      c[j] = ok ? __float_as_uint(__fadd_rn(w[j], 12582912.0f)) & (BITS == 8 ? 255u : 15u) : 0u;
    uint8_t* dst = kc + r * (D * BITS / 8);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint8_t* d = dst + (i ? ob : oa) * BITS / 8;
      const uint32_t b = c[4 * i] | c[4 * i + 1] << BITS | c[4 * i + 2] << (2 * BITS) | c[4 * i + 3] << (3 * BITS);
      if (BITS == 8) *reinterpret_cast<uint32_t*>(d) = b;
      else *reinterpret_cast<uint16_t*>(d) = (uint16_t)b;
    }
    if (part == 0) ks[r] = __frcp_rn(si);
  }
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

struct AppendArgs {
  AppendRows rows;
  Rotary ro;
  bool interleaved;
  const int64_t* slots;
  int64_t n_slots;
  int page;
  void* q_out;
  uint8_t *kc, *vc;
  float *ks, *vs;
};

template <typename InT, int BITS, int D>
int append_t(const AppendArgs& a, cudaStream_t st) {
  AppendRows r = a.rows;
  const int64_t per = 16 / sizeof(InT);
  r.vec = ((uintptr_t)r.q | (uintptr_t)r.k | (uintptr_t)r.v) % 16 == 0 && (r.Hq == 0 || (r.q_ts % per == 0 && r.q_hs % per == 0)) &&
          r.k_ts % per == 0 && r.k_hs % per == 0 && r.v_ts % per == 0 && r.v_hs % per == 0;
  // a block's tokens share nothing but its threads: one each until the SMs are full
  const int64_t tb = cdiv(r.T, 4 * kSMs);
  const int TB = (int)(tb < kAppendTokens ? tb : kAppendTokens);
  const dim3 grid((unsigned)cdiv(r.T, TB));
  auto go = [&](auto kern) -> int {
    MXB_CUDA_TRY(launch_pdl(kern, grid, kThreads, 0, st, r, a.ro, TB, a.slots, a.n_slots, shift_of(a.page),
                            static_cast<InT*>(a.q_out), a.kc, a.ks, a.vc, a.vs, device_error_ptr()));
    MXB_LAUNCH_CHECK();
    return MXB_OK;
  };
  if constexpr (sizeof(InT) == 2) {
    if (r.vec && a.ro.pairs % 8 == 0)
      return a.interleaved ? go(kv_append_kernel<InT, BITS, D, true, true>)
                           : go(kv_append_kernel<InT, BITS, D, false, true>);
  }
  return a.interleaved ? go(kv_append_kernel<InT, BITS, D, true, false>)
                       : go(kv_append_kernel<InT, BITS, D, false, false>);
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
struct Append {
  template <typename... A>
  static int run(A&&... a) { return append_t<T, BITS, D>(a...); }
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

int mxb_kv_append(const void* q, const void* k, const void* v, int x_dtype, int64_t T, int q_heads, int heads,
                  int dim, int64_t q_token_stride, int64_t q_head_stride, int64_t k_token_stride,
                  int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                  const int64_t* positions, int axes, int64_t axis_stride, const float* inv_freq, int rot,
                  const int* sections, int interleaved, const int64_t* slots, int64_t n_pages, int page,
                  int bits, void* k_codes, float* k_scales, void* v_codes, float* v_scales, void* q_out,
                  void* stream) {
  if (x_dtype != MXB_F32 && x_dtype != MXB_BF16) return MXB_E_DTYPE;
  const int rc = kv_pool_check(n_pages, heads, page, dim, bits, k_codes, k_scales, v_codes, v_scales);
  if (rc != MXB_OK) return rc;
  if (T < 0 || q_heads < 0 || q_heads > 65535 || rot < 0 || rot > dim || rot % 8 || axes < 1 || axes > 4)
    return MXB_E_SHAPE;
  if (T > ((int64_t)1 << 31)) return MXB_E_SHAPE;
  for (int64_t stride : {q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride})
    if (stride < 0 || stride > INT32_MAX) return MXB_E_SHAPE;
  if (axes > 1 && !sections) return MXB_E_ARG;
  Rotary ro = {positions, axis_stride, inv_freq, rot / 2, {INT32_MAX, INT32_MAX, INT32_MAX}};
  int64_t at = 0;
  for (int i = 0; i < axes && axes > 1; ++i) {
    if (sections[i] < 0) return MXB_E_SHAPE;
    if (i > 0) ro.end[i - 1] = (int)at;
    at += sections[i];
  }
  if (axes > 1 && at != rot / 2) return MXB_E_SHAPE;
  if (T == 0) return MXB_OK;
  if (!k || !v || !slots || (q_heads > 0 && (!q || !q_out)) || (rot > 0 && (!positions || !inv_freq)))
    return MXB_E_ARG;
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) % (x_dtype == MXB_BF16 ? 2 : 4) ||
      (q_heads > 0 && (uintptr_t)q_out % 16) || ((uintptr_t)positions | (uintptr_t)slots) % 8 ||
      (uintptr_t)inv_freq % 4)
    return MXB_E_ALIGN;
  AppendArgs a = {{q_heads > 0 ? q : nullptr, k, v, T, q_heads, heads, (int)q_token_stride, (int)q_head_stride,
                   (int)k_token_stride, (int)k_head_stride, (int)v_token_stride, (int)v_head_stride, false},
                  ro, interleaved != 0, slots, n_pages * page, page, q_out, static_cast<uint8_t*>(k_codes),
                  static_cast<uint8_t*>(v_codes), k_scales, v_scales};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return x_dtype == MXB_BF16 ? by_format<__nv_bfloat16, Append>(bits, dim, a, st)
                             : by_format<float, Append>(bits, dim, a, st);
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
