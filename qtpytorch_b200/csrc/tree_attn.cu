// Attention of many query rows of a sequence, a tree of drafted tokens, over its
// own paged history, on tcgen05 (paged_attn.cu describes the cache, the list of
// tiles that CTAs share out and the parts that it joins).
//
// The T * G rows of a KV head meet the same keys, so that S = Q K^T and O = P V are
// products of matrices: 4 T G keys dim operations, and an exponential a score.  A
// CTA owns 128 rows or 256 and walks tiles of 128 keys:
//   warp 0        MMA issue and TMEM allocation;
//   warp 1        TMA producer: raw codes and scales, a ring of steps of 64 or 128 keys
//                 of K or V;
//   warps 2-17    softmax: S from TMEM, running maximum, sum, weights (fp16) back to
//                 TMEM over S;
//   warps 18-21   unpack codes to exact fp16 in shared memory (one layout for K and
//                 V: K-major for the first product, MN-major for the second), and
//                 lay out a tile's scales.
// Two streams of softmax warps take turns on the tensor cores, one multiplying
// while the other exponentiates: with 256 rows the two halves of the rows, with 128
// the even and the odd tiles of the same rows, joined at the end of a unit.
//
// A softmax warp has 16 rows, in the fragment layout of 16 x 8 pieces: a lane holds 2
// rows and a quarter of the keys.  Four such warps a scheduler hide one another's
// latencies (with 32 rows a warp, a thread a row or not, a warp issued an instruction
// every 8 cycles and a tile took 9000), and the keys' scales cost a quarter of the
// shared memory reads that a thread a row makes.
//
// Scores: Q is fp16 under a power of two per row that puts its largest value into
// [2^14, 2^15), the codes are exact.  Weights: p_j = exp2(s_j - m) times 2^6 sv_j /
// c, c a power of two of at least the largest value scale so far, m following the
// maximum within 2^8.  While the value scales span less than 2^-14 of c, a row's
// largest weight is at least 2^-8, so fp16 keeps 11 bits of those down to 2^-6 of it
// and is off by at most 2^-17 of it below.  From the first tile with a wider span
// on, c is each row's own and follows its largest weight.  m, sums and outputs are
// fp32; O is rescaled in TMEM only when m or c moves.
//
// 16 sequences of up to 8192 keys, 64 x 4 rows of each of 8 heads of 128 dims in int8
// (86 GFLOP): 220 us = 390 TFLOP/s, 599 in groups of 32 rows.  A tile takes 7500 cycles
// where its products take 2100: a stream's scores, exponentials and products follow one
// another, and two streams of 16-row warps at one instruction in 5 cycles each do not
// cover that.  The instruction cache is the narrow place: code that was longer (straight
// instead of looped, pieces of 64 keys, more roles' special cases in line or out of it)
// was slower each time (245 -> 304, 220 -> 258, 220 -> 236 us), also with fewer waits.
// Waits that poll took 7 %; a segment costs about 12 us more than its tiles (Q, the first
// references, the part).  148 units of one sequence each: 2.1 us a tile of 128 rows x 64
// dims, 3.1 of 128 x 128, 4.1 of 256 x 128.
#include "mxb_common.cuh"
#include "mxb_internal.h"

#include <cuda.h>
#include <cuda_fp16.h>

#define MXB_ERROR_WORD_BY_POINTER
#include "tc_ptx.cuh"

using namespace mxb;

namespace mxb {
namespace tree {

constexpr int KT = kTreeKeys;  // 128
constexpr int kSoftWarps = 16, kFirstSoft = 2, kFirstUnpack = kFirstSoft + kSoftWarps;
constexpr int kThreads = 32 * (kFirstUnpack + 4);
constexpr int kSlots = 4;      // scale slots: a tile's is written after S of the tile two before
constexpr int kSlotF = 2 * KT + 8;  // key scales, value scales, header
constexpr float kRoom = 64.0f;      // 2^6
constexpr float kWide = 0x1p-14f;

template <int BITS, int D, int MT>
struct Cfg {
  static constexpr int RB = D * BITS / 8;
  static constexpr int kAtom = KT * 128;           // 64 dims of every key
  static constexpr int kPlane = kAtom * (D / 64);  // 32 or 16 KB
  static constexpr int kQAtom = 128 * 128;
  static constexpr int kQ = kQAtom * (D / 64);
  // exchange of two streams, 32 columns at a time: 16 values a thread, and (m, l, m') of its 2 rows
  static constexpr int kX = 32 * (kSoftWarps / 2) * 16 * 4, kXml = 32 * (kSoftWarps / 2) * 32;
  static constexpr size_t oK = (size_t)MT * kQ, oV = oK + 2 * kPlane, oSc = oV + 2 * kPlane;
  static constexpr size_t oX = oSc + (size_t)kSlots * kSlotF * 4;
  static constexpr size_t oBars = oX + (MT == 1 ? kX + kXml : 0);
  // ring of raw codes, kKeys keys of K (with both scales of those) or of V a step: 8 KB,
  // or a whole tile where that is less (in steps of 64 keys the barriers of int4 tiles of
  // 64 dims took longer than their codes)
  static constexpr int kKeys = RB == 128 ? 64 : 128, kSteps = KT / kKeys;  // steps of K, and of V, a tile
  static constexpr int kStep = kKeys * RB, kSlot = kStep + 8 * kKeys;
  static constexpr size_t oRaw = oBars + 768;
  static constexpr int kRing = D == 128 ? 3 : 6;
  static constexpr size_t kSmem = 1024 + oRaw + (size_t)kRing * kSlot;
  static constexpr int kPieces = kStep / 16 / 128;  // 16-byte pieces of a step a thread
};
constexpr int kMaxRing = 6;

struct Bars {
  uint64_t kready[2], kfree[2], vready[2], vfree[2];
  uint64_t sready[2], pready[2], pvdone[2];
  uint64_t scready[kSlots];
  uint64_t raw_full[kMaxRing], raw_empty[kMaxRing];
  uint64_t qready, xfull, xfree;
  uint64_t drained;  // every product issued is complete
  int64_t scan[24];
  uint32_t tmem_base;
  int b, off;
  uint32_t gone[kMaxRing];  // bit i: keys 16 i .. of the step lie behind a number outside the pool
};
static_assert(sizeof(Bars) <= 768 && kThreads / 32 <= 24, "barrier block overflows its slot");

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
__device__ __forceinline__ uint32_t bf2(float lo, float hi) {
  const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
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

// Piece j of thread t: row and 16-byte column of a step's codes.  Eight
// neighbouring lanes take pieces of one atom from two (four) rows, so that their
// 16-byte stores of unpacked values cover all banks.
template <int BITS, int D>
__device__ __forceinline__ void piece(int j, int t, int& row, int& c) {
  constexpr int C = D * BITS / 128;
  const int i = j * 128 + t;
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
}

// S of 16 rows x 32 keys: registers 4 i + 2 h + e hold row 8 h + lane / 4, key 8 i + 2
// (lane % 4) + e.
__device__ __forceinline__ void tmem_ld_16x32(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
// P of 16 rows x 32 keys, two a column: registers 2 i + h hold row 8 h + lane / 4, keys
// 8 i + 2 (lane % 4) and the next.
__device__ __forceinline__ void tmem_st_16x32h(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st_16x32(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// After tmem_wait_ld: no use of the registers before it.
__device__ __forceinline__ void landed16(uint32_t (&r)[16]) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_get(uint32_t taddr, uint32_t (&r)[16]) {
  __syncwarp();
  tmem_ld_16x32(taddr, r);
  tmem_wait_ld();
  landed16(r);
}

template <int BITS, int D>
__device__ __forceinline__ void put_piece(uint4 r, uint8_t* plane, int row, int c) {
  constexpr int N = BITS == 8 ? 2 : 4, kAtom = KT * 128;
  uint4 o[N];
  unpack16<BITS>(r, o);
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int ch = c * N + k;
    *reinterpret_cast<uint4*>(plane + (ch >> 3) * kAtom + row * 128 + (((ch & 7) ^ (row & 7)) << 4)) = o[k];
  }
}

// A place in the list of tiles: tile t of [t_lo, t_hi) of unit u of sequence b,
// `left` tiles from the segment's start to the end of the CTA's run.
struct Place {
  int b, u, t, t_lo, t_hi, n_tiles, len;
  int64_t left;

  __device__ __forceinline__ static int len_of(const TreeArgs& a, int b) {
    const int64_t cap = (int64_t)a.width << a.page_shift;
    return (int)min((int64_t)max(__ldg(a.lengths + b), 0), cap);
  }
  __device__ __forceinline__ void start(const TreeArgs& a, int first) {
    len = len_of(a, b);
    n_tiles = (len + KT - 1) / KT;
    t = t_lo = first;
    t_hi = (int)min((int64_t)n_tiles, t_lo + left);
  }
  // The segment after this one; false: there is none.
  __device__ __forceinline__ bool next_segment(const TreeArgs& a) {
    left -= t_hi - t_lo;
    if (left <= 0) return false;
    if (++u == a.H * a.row_tiles) {
      u = 0;
      do {  // sequences without keys have no tiles
        ++b;
      } while (len_of(a, b) == 0);
    }
    start(a, 0);
    return true;
  }
  __device__ __forceinline__ bool next_tile(const TreeArgs& a) {
    return ++t < t_hi || next_segment(a);
  }
};

// Sum over the warp, or the block, of one value a thread, and its exclusive prefix.
__device__ __forceinline__ int64_t warp_scan(int64_t v, int64_t& before) {
  int64_t inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t t = __shfl_up_sync(0xffffffffu, inc, o);
    if ((threadIdx.x & 31) >= o) inc += t;
  }
  before = inc - v;
  return __shfl_sync(0xffffffffu, inc, 31);
}
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
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) pre += sm[w];
    total += sm[w];
  }
  __syncthreads();
  before = pre + inc - v;
  return total;
}

// A lane's two rows of the softmax, 8 k + lane / 4 of the warp's 16: reference and sum
// (of the lane's own keys); lc, log2 of the c that O stands under; top_w, log2 of the
// largest weight of wide tiles, or less.
struct Rows {
  float mu[2], m_top[2], l[2], lc[2], top_w[2];
};
struct Tile {
  const float* slot;
  uint32_t s, o;        // TMEM: S (P over it) and O of this warp's rows
  bool first;           // no O yet
};

// Which of a lane's scores of a tile that reaches the tree are hidden by the masks of its
// rows: bit 4 i + 2 k + e of a word of 32 keys for key 8 i + 2 (lane % 4) + e of row 8 k +
// lane / 4.  key0: the tile's first key, from the tree's first one on.
__device__ __forceinline__ uint4 tree_bits(int key0, int T, const uint8_t* mask, int64_t mask_t, const int (&tok)[2]) {
  const uint8_t* row[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) row[k] = mask + min(tok[k], T - 1) * mask_t;
  uint4 all = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    uint32_t bits = 0;
    const int k0 = key0 + 32 * c + 2 * (threadIdx.x & 3);
    if (key0 + 32 * c + 32 > 0) {
      // all bytes at once, those of other places are not looked at
      uint32_t seen[4][2][2];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) seen[i][k][e] = __ldg(row[k] + max(min(k0 + 8 * i + e, T - 1), 0));
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int at = k0 + 8 * i + e;
            const bool off = at >= 0 && (at >= T || tok[k] >= T || seen[i][k][e] == 0u);
            bits |= (off ? 1u : 0u) << (4 * i + 2 * k + e);
          }
    }
    all = make_uint4(all.y, all.z, all.w, bits);  // four turns: each word in its place
  }
  __syncwarp();
  return all;
}

// Multiplies the D columns of O, and with them the P of `pieces` pieces of this tile,
// of the lane's rows by 2^x, in place.
template <int D>
__device__ __noinline__ void rescale(uint32_t o_at, uint32_t s_at, bool has_o, int pieces, float x0, float x1) {
  const float by[2] = {ex2(x0), ex2(x1)};
  tmem_wait_st();
  if (has_o) {
#pragma unroll 1
    for (int d = 0; d < D; d += 32) {
      uint32_t o[16];
      tmem_get(o_at + d, o);
#pragma unroll
      for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * by[(i >> 1) & 1]);
      tmem_st_16x32(o_at + d, o);
    }
  }
  // 32 columns of P are two pieces; where the second is none of them it is put back as it was
#pragma unroll 1
  for (int c = 0; c < pieces; c += 2) {
    uint32_t p[16];
    tmem_get(s_at + 16 * c, p);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p[i]));
      const uint32_t y = hf2(f.x * by[(i >> 1) & 1], f.y * by[(i >> 1) & 1]);
      if (i < 8 || c + 1 < pieces) p[i] = y;
    }
    tmem_st_16x32(s_at + 16 * c, p);
  }
  tmem_wait_st();
}

// The softmax of one tile in one pass over S; P is in TMEM afterwards.  References and
// c move where a piece's scores or weights ask for it, and take O and the P before
// that piece along; they are whole powers of two, so that a P that moves with them is
// not rounded again (but where it becomes subnormal).  The loop over pieces of 32 keys
// is not unrolled: three roles share the instruction cache, and four pieces in a row,
// the next one's S on its way, took 304 us where the loop takes 245.
template <int D>
__device__ __forceinline__ void softmax_tile(Rows& r, const Tile& g, const float (&rowf)[2], uint4 hidden) {
  const float* head = g.slot + 2 * KT;
  const float lcn = head[0];
  const bool wide = __float_as_uint(head[1]) != 0u;
  const uint4 gone = *reinterpret_cast<const uint4*>(head + 4);
  const int lane = threadIdx.x & 31;
  if (__builtin_expect((gone.x | gone.y | gone.z | gone.w) != 0u, 0)) {  // for both rows of a lane
    auto of = [&](uint32_t w) -> uint32_t {
      uint32_t bits = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) bits |= (w >> (8 * i + 2 * (lane & 3)) & 3u) * 5u << (4 * i);
      return bits;
    };
    hidden = make_uint4(hidden.x | of(gone.x), hidden.y | of(gone.y), hidden.z | of(gone.z), hidden.w | of(gone.w));
  }
  if (g.first) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      r.mu[k] = r.l[k] = 0.0f;
      r.m_top[k] = r.top_w[k] = -INFINITY;
      r.lc[k] = lcn;
    }
  }
  bool turn = !wide && lcn != r.lc[0];  // the narrow tiles' c is one for all rows
  uint64_t sum[2] = {0, 0};
  const float* ks = g.slot + 2 * (lane & 3);
#pragma unroll 1
  for (int c = 0; c < 4; ++c, ks += 32) {
    const uint32_t h = hidden.x;
    hidden = make_uint4(hidden.y, hidden.z, hidden.w, h);
    uint32_t s[16];
    uint64_t v[2][4];
    tmem_get(g.s + 32 * c, s);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t k2 = *reinterpret_cast<const uint64_t*>(ks + 8 * i);
#pragma unroll
      for (int k = 0; k < 2; ++k)
        v[k][i] = fmul2(pack2(__uint_as_float(s[4 * i + 2 * k]), __uint_as_float(s[4 * i + 2 * k + 1])), k2);
    }
    if (__builtin_expect(h != 0u, 0)) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float2 x = unpack2(v[k][i]);
          if (h >> (4 * i + 2 * k) & 1u) x.x = -INFINITY;
          if (h >> (4 * i + 2 * k + 1) & 1u) x.y = -INFINITY;
          v[k][i] = pack2(x.x, x.y);
        }
    }
    float mx[2], up[2] = {1.0f, 1.0f};
    bool move = turn || wide;
    turn = false;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float2 x0 = unpack2(v[k][0]), x1 = unpack2(v[k][1]), x2 = unpack2(v[k][2]), x3 = unpack2(v[k][3]);
      mx[k] = fmaxf(fmaxf(fmaxf(x0.x, x0.y), fmaxf(x1.x, x1.y)), fmaxf(fmaxf(x2.x, x2.y), fmaxf(x3.x, x3.y))) * rowf[k];
      move |= mx[k] > r.m_top[k];
    }
    if (__builtin_expect(__any_sync(0xffffffffu, move), 0)) {
      float by[2];  // log2 of what O and P are multiplied with
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        mx[k] = fmaxf(mx[k], __shfl_xor_sync(0xffffffffu, mx[k], 1));
        mx[k] = fmaxf(mx[k], __shfl_xor_sync(0xffffffffu, mx[k], 2));
        by[k] = 0.0f;
        if (mx[k] > r.m_top[k]) {
          const float m0 = r.m_top[k] == -INFINITY ? -INFINITY : r.mu[k];
          const float m1 = ceilf(fmaxf(m0, mx[k]));
          by[k] = m0 - m1;
          const float alpha = ex2(by[k]);
          const float2 t = unpack2(sum[k]);
          sum[k] = pack2(t.x * alpha, t.y * alpha);
          r.l[k] *= alpha;
          r.mu[k] = m1;
          r.m_top[k] = m1 + 8.0f;
        }
        if (wide) {
          // a c for the row that puts its largest weight so far between 2^-2 and 2^12
          float u = 0.0f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 x = unpack2(ffma2(v[k][i], pack2(rowf[k], rowf[k]), pack2(-r.mu[k], -r.mu[k])));
            u = fmaxf(u, h >> (4 * i + 2 * k) & 1u ? 0.0f : ex2(x.x) * ks[KT + 8 * i]);
            u = fmaxf(u, h >> (4 * i + 2 * k + 1) & 1u ? 0.0f : ex2(x.y) * ks[KT + 8 * i + 1]);
          }
          u = fmaxf(u, __shfl_xor_sync(0xffffffffu, u, 1));
          u = fmaxf(u, __shfl_xor_sync(0xffffffffu, u, 2));
          r.top_w[k] = fminf(fmaxf(r.top_w[k] + by[k], log2f(u) + (lcn - r.lc[k])), 200.0f);
          if (r.top_w[k] > 12.0f || (r.top_w[k] < -2.0f && r.top_w[k] > -INFINITY) || lcn - r.lc[k] > 120.0f) {
            // no further below the tile's c than 2^120: fp32 holds little under that
            const float x = fminf(6.0f - floorf(r.top_w[k]), 120.0f - (lcn - r.lc[k]));
            r.lc[k] -= x;
            r.top_w[k] += x;
            by[k] += x;
          }
          up[k] = ex2(lcn - r.lc[k]);
        } else {
          by[k] += r.lc[k] - lcn;
          r.lc[k] = lcn;
        }
      }
      if (__any_sync(0xffffffffu, by[0] != 0.0f || by[1] != 0.0f) && !(g.first && c == 0))
        rescale<D>(g.o, g.s, !g.first, c, by[0], by[1]);
    }
    uint32_t pk[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t w = *reinterpret_cast<const uint64_t*>(ks + KT + 8 * i);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float2 x = unpack2(ffma2(v[k][i], pack2(rowf[k], rowf[k]), pack2(-r.mu[k], -r.mu[k])));
        const uint64_t p = pack2(ex2(x.x), ex2(x.y));
        sum[k] = fadd2(sum[k], p);
        uint64_t q = fmul2(p, w);
        q = fmul2(q, pack2(up[k], up[k]));
        const float2 y = unpack2(q);
        pk[2 * i + k] = hf2(y.x, y.y);
      }
    }
    if (__builtin_expect(h != 0u, 0)) {  // whatever their scales hold
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (h >> (4 * i + 2 * k) & 1u) pk[2 * i + k] &= 0xffff0000u;
          if (h >> (4 * i + 2 * k + 1) & 1u) pk[2 * i + k] &= 0x0000ffffu;
        }
    }
    __syncwarp();
    tmem_st_16x32h(g.s + 16 * c, pk);
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float2 x = unpack2(sum[k]);
    r.l[k] += x.x + x.y;
  }
  tmem_wait_st();
  tc_fence_before();
}

// A row's 32 columns, 8 i + 2 c and the next in m[i] of lane c of four -> columns 8 c ..
// of lane c, in the order of the dims.
template <int BITS>
__device__ __forceinline__ void eight_columns(float2 (&m)[4], float (&o)[8]) {
  const int c = threadIdx.x & 3;
#pragma unroll
  for (int s = 1; s < 4; s <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (!(i & s)) {
        const bool hi = c & s;
        float2 t = hi ? m[i] : m[i | s];
        t.x = __shfl_xor_sync(0xffffffffu, t.x, s);
        t.y = __shfl_xor_sync(0xffffffffu, t.y, s);
        if (hi) m[i] = t;
        else m[i | s] = t;
      }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    o[order<BITS>(2 * j)] = m[j].x;
    o[order<BITS>(2 * j + 1)] = m[j].y;
  }
}

template <int BITS, int D, int MT>
__global__ void __launch_bounds__(kThreads, 1)
    tree_attn_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                     const TreeArgs a, int box) {
  using C = Cfg<BITS, D, MT>;
  constexpr int R = 128 * MT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  Bars* bars = reinterpret_cast<Bars*>(smem + C::oBars);
  float* slots = reinterpret_cast<float*>(smem + C::oSc);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->kready[b], 4);
      mbar_init(&bars->kfree[b], 1);
      mbar_init(&bars->vready[b], 4);
      mbar_init(&bars->vfree[b], 1);
      mbar_init(&bars->sready[b], 1);
      mbar_init(&bars->pready[b], kSoftWarps / 2);
      mbar_init(&bars->pvdone[b], 1);
    }
    for (int s = 0; s < kSlots; ++s) mbar_init(&bars->scready[s], 4);
    for (int s = 0; s < C::kRing; ++s) {
      mbar_init(&bars->raw_full[s], C::kKeys / box);
      mbar_init(&bars->raw_empty[s], 4);
    }
    mbar_init(&bars->qready, kSoftWarps / 2 * MT);
    mbar_init(&bars->xfull, kSoftWarps / 2);
    mbar_init(&bars->xfree, kSoftWarps / 2);
    mbar_init(&bars->drained, 1);
    fence_barrier_init();
  }
  if (warp == 0) {
    tmem_alloc(&bars->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = bars->tmem_base;
  pdl_trigger();
  pdl_wait();

  // ── this CTA's run of the list: equal shares of all tiles ──
  const int hr = a.H * a.row_tiles;
  const int64_t cap = (int64_t)a.width << a.page_shift;
  Place at;
  bool any;
  if (a.plan == nullptr) {  // a unit a CTA
    at.b = blockIdx.x / hr;
    at.u = blockIdx.x - at.b * hr;
    if (at.u == 0 && threadIdx.x == 0 && a.err && __ldg(a.lengths + at.b) > cap) atomicCAS(a.err, 0, kErrIndex);
    at.left = (Place::len_of(a, at.b) + KT - 1) / KT;
    any = at.left > 0;
    if (any) {
      at.start(a, 0);
    } else if (a.direct) {  // a sequence without keys: zeros
      const int h = at.u / a.row_tiles, r0 = (at.u - h * a.row_tiles) * R;
      for (int i = threadIdx.x; i < R * (D / 8); i += kThreads) {
        const int row = r0 + i / (D / 8), tok = row / a.G;
        if (row >= a.rows) break;
        const int64_t id = ((int64_t)at.b * a.T + tok) * ((int64_t)a.H * a.G) + (int64_t)h * a.G + (row - tok * a.G);
        reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + id * D)[i % (D / 8)] = make_uint4(0u, 0u, 0u, 0u);
        if (a.lse && i % (D / 8) == 0) a.lse[id] = -INFINITY;
      }
    }
  } else {
    // every warp for itself where the batch is small, otherwise the block together
    const bool alone = a.B <= 512;
    const int width = alone ? 32 : kThreads, me = alone ? lane : threadIdx.x;
    auto tiles_of = [&](int i) -> int64_t {
      return i < a.B ? (int64_t)((Place::len_of(a, i) + KT - 1) / KT) * hr : 0;
    };
    auto scan = [&](int64_t v, int64_t& before) {
      return alone ? warp_scan(v, before) : block_scan(v, before, bars->scan);
    };
    int64_t total = 0, before, base = 0;
    for (int b0 = 0; b0 < a.B; b0 += width) {
      const int i = b0 + me;
      if (i < a.B && blockIdx.x == 0 && a.err && __ldg(a.lengths + i) > cap) atomicCAS(a.err, 0, kErrIndex);
      total += scan(tiles_of(i), before);
    }
    const int64_t per = max((total + gridDim.x - 1) / gridDim.x, (int64_t)1);
    const int64_t lo = blockIdx.x * per, hi = min(lo + per, total);
    if (blockIdx.x == 0 && threadIdx.x == 0) a.plan[0] = per;
    int at_b = 0, at_off = 0;
    for (int b0 = 0; b0 < a.B && (blockIdx.x == 0 || base <= lo); b0 += width) {
      const int i = b0 + me;
      const int64_t n = tiles_of(i), sum = scan(n, before);
      before += base;
      base += sum;
      if (i < a.B && blockIdx.x == 0 && (!alone || warp == 0)) a.plan[1 + i] = before;
      const bool here = lo < hi && lo >= before && lo < before + n;
      if (alone) {
        const uint32_t who = __ballot_sync(0xffffffffu, here);
        if (who) {
          at_b = __shfl_sync(0xffffffffu, i, __ffs(who) - 1);
          at_off = __shfl_sync(0xffffffffu, (int)(lo - before), __ffs(who) - 1);
        }
      } else if (here) {
        bars->b = i;
        bars->off = (int)(lo - before);
      }
    }
    if (!alone) {
      __syncthreads();
      at_b = bars->b;
      at_off = bars->off;
    }
    any = lo < hi;
    if (any) {
      at.b = at_b;
      at.left = hi - lo;
      const int n = (Place::len_of(a, at.b) + KT - 1) / KT;
      at.u = at_off / n;
      at.start(a, at_off - at.u * n);
    }
  }
  auto t_s = [&](int g) { return tbase + (uint32_t)(g * KT); };
  auto t_o = [&](int g) { return tbase + (uint32_t)(2 * KT + g * D); };

  if (warp < kFirstSoft) {
    if (warp == 0) {
      if (lane == 0 && any) {
        constexpr uint32_t id_s = make_idesc(/*F32*/ 1, /*F16*/ 0, 0, 0, 128, KT);
        constexpr uint32_t id_o = make_idesc(1, 0, 0, /*B MN-major*/ 1, 128, D);
        // descriptors count in units of 16 bytes, and stay within their 14 bits
        const uint64_t dq = desc_kmajor_sw128(smem_u32(smem)), dk = desc_kmajor_sw128(smem_u32(smem + C::oK));
        const uint64_t dv = desc_mnmajor_sw128(smem_u32(smem + C::oV), C::kAtom);
        bool ok = true;
        int j0 = 0;                // tiles of the segments before
        int step[2] = {0, 0};      // products P V issued a stream
        uint32_t seg = 0;
        // A stream's turn: P V of its tile io, then S of its tile is over that P.  256 rows:
        // both streams take every tile; 128: the even and the odd ones.
        do {
          const int n = at.t_hi - at.t_lo;
          ok = ok && mbar_sleep_to(&bars->qready, seg & 1, kErrTimeoutFull, a.err);
#pragma unroll 1
          for (int k = 0; k < (MT == 2 ? 2 * n : n) + 2 && ok; ++k) {
            const int g = k & 1, io = MT == 2 ? (k >> 1) - 1 : k - 2, is = io + (MT == 2 ? 1 : 2);
            if (io >= 0) {
              const int j = j0 + io, b = j & 1;
              if (MT == 1 || g == 0) ok = mbar_sleep_to(&bars->vready[b], (j >> 1) & 1, kErrTimeoutFull, a.err);
              ok = ok && mbar_sleep_to(&bars->pready[g], step[g] & 1, kErrTimeoutTmemFull, a.err);
              if (!ok) break;
              tc_fence_after();
              const uint64_t v = dv + (uint32_t)(b * (C::kPlane >> 4));
#pragma unroll 2
              for (int kk = 0; kk < KT / 16; ++kk)
                mma_f16_ts(t_o(g), t_s(g) + kk * 8, v + kk * (16 * 128 >> 4), id_o,
                           (is >= (MT == 2 ? 2 : 4) || kk > 0) ? 1u : 0u);
              mma_commit(&bars->pvdone[g]);
              if (MT == 1 || g == 1) mma_commit(&bars->vfree[b]);
            }
            if (is < n) {
              const int j = j0 + is, b = j & 1;
              // S goes over the stream's P: that product has to be complete
              if (io >= 0) ok = mbar_sleep_to(&bars->pvdone[g], step[g] & 1, kErrTimeoutTmemEmpty, a.err);
              if (MT == 1 || g == 0)
                ok = ok && mbar_sleep_to(&bars->kready[b], (j >> 1) & 1, kErrTimeoutFull, a.err);
              if (!ok) break;
              tc_fence_after();
              const uint64_t q = dq + (MT == 2 ? (uint32_t)(g * (C::kQ >> 4)) : 0u);
              const uint64_t kd = dk + (uint32_t)(b * (C::kPlane >> 4));
#pragma unroll 2
              for (int kk = 0; kk < D / 16; ++kk)
                mma_f16(t_s(g), q + (kk >> 2) * (C::kQAtom >> 4) + (kk & 3) * 2,
                        kd + (kk >> 2) * (C::kAtom >> 4) + (kk & 3) * 2, id_s, kk > 0 ? 1u : 0u);
              mma_commit(&bars->sready[g]);
              if (MT == 1 || g == 1) mma_commit(&bars->kfree[b]);
            }
            if (io >= 0) ++step[g];
          }
          j0 += n;
          ++seg;
        } while (ok && at.next_segment(a));
        mma_commit(&bars->drained);
      }
    } else if (warp == 1) {
      // ── raw codes and scales: a tile's keys in kSteps steps, then its values ──
      const int page_mask = (1 << a.page_shift) - 1, per = box >> 4;  // groups of 16 keys a copy
      // lane i < 8: first head row of keys 16 i .. of a tile; -1 where there are none, -2
      // behind a number outside the pool
      auto rows_of = [&](const Place& p) -> int {
        const int pos = p.t * KT + lane * 16;
        int row = -1;
        if (lane < 8 && pos < p.len) {
          const int pg = __ldg(a.table + (int64_t)p.b * a.width + (pos >> a.page_shift));
          if ((uint32_t)pg < (uint32_t)a.n_pages) {  // n_pages < 2^31
            row = ((pg * a.H + p.u / a.row_tiles) << a.page_shift) + (pos & page_mask);
          } else {
            if (a.err) atomicCAS(a.err, 0, kErrIndex);
            row = -2;
          }
        }
        return row;
      };
      int step = 0;
      if (any) {
        int rows = rows_of(at);
        bool more = true, ok = true;
        while (more && ok) {
          Place next = at;
          more = next.next_tile(a);
          const int next_rows = more ? rows_of(next) : -1;
          for (int q = 0; q < 2 * C::kSteps; ++q, ++step) {
            constexpr int kGroups = C::kKeys / 16;
            const int s = step % C::kRing;
            const bool keys = q < C::kSteps;
            ok = step < C::kRing ||
                 mbar_sleep_warp_to(&bars->raw_empty[s], (step / C::kRing - 1) & 1, kErrTimeoutEmpty, a.err);
            if (!ok) break;
            const int row = __shfl_sync(0xffffffffu, rows, q % C::kSteps * kGroups + lane % kGroups);
            const uint32_t gone = __ballot_sync(0xffffffffu, lane < kGroups && row == -2);
            if (lane == 0) bars->gone[s] = gone;  // before its arrival
            if (lane < kGroups && lane % per == 0) {
              uint64_t* bar = &bars->raw_full[s];
              if (row >= 0) {
                uint8_t* dst = smem + C::oRaw + (size_t)s * C::kSlot;
                mbar_expect_tx(bar, (uint32_t)box * (C::RB + (keys ? 8 : 0)));
                tma_load_2d(dst + lane * 16 * C::RB, keys ? &tmap_k : &tmap_v, bar, 0,
                            (int)((int64_t)row * C::RB / 128));  // lines of 128 bytes
                if (keys) {
                  float* sc = reinterpret_cast<float*>(dst + C::kStep) + lane * 16;
                  bulk_load_g2s(sc, a.k_scales + row, (uint32_t)box * 4, bar);
                  bulk_load_g2s(sc + C::kKeys, a.v_scales + row, (uint32_t)box * 4, bar);
                }
              } else {
                mbar_arrive(bar);
              }
            }
          }
          at = next;
          rows = next_rows;
        }
        // the last copies land before the CTA may end, also where a wait gave up
        for (int j = max(step - C::kRing, 0); j < step; ++j)
          mbar_sleep_warp_to(&bars->raw_full[j % C::kRing], (j / C::kRing) & 1, kErrTimeoutFull, a.err);
      }
    }
  } else if (warp >= kFirstUnpack) {
    if (any) {
      // ── unpack ──
      const int t = threadIdx.x - 32 * kFirstUnpack, w = warp - kFirstUnpack;
      int step = 0;
      bool more = true, ok = true;
      float c = 0.0f;                // power of two above every value scale so far (0: none)
      uint32_t least = 0x7F800000u;  // bits of the smallest so far
      bool fresh = true;             // a segment's first tile
      for (int j = 0; more && ok; ++j) {
        const int b = j & 1, valid = at.len - at.t * KT;  // keys of the tile, from 128 on all
        if (fresh) {
          c = 0.0f;
          least = 0x7F800000u;
        }
        float ks = 0.0f, vs = 0.0f, top = 0.0f;  // of this warp's 32 keys; every warp looks at all value scales
        uint32_t small = least;
        uint4 gone = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 1
        for (int q = 0; q < 2 * C::kSteps; ++q, ++step) {
          const int s = step % C::kRing, part = q % C::kSteps;
          const bool keys = q < C::kSteps, last = part == C::kSteps - 1;
          ok = mbar_sleep_warp_to(&bars->raw_full[s], (step / C::kRing) & 1, kErrTimeoutFull, a.err);
          if (ok && j >= 2 && part == 0)
            ok = mbar_sleep_warp_to(keys ? &bars->kfree[b] : &bars->vfree[b], ((j >> 1) - 1) & 1, kErrTimeoutEmpty, a.err);
          if (!ok) break;
          const uint8_t* src = smem + C::oRaw + (size_t)s * C::kSlot;
          if (keys) {
            const float* sc = reinterpret_cast<const float*>(src + C::kStep);
            const uint32_t bad = bars->gone[s];
#pragma unroll
            for (int x = 0; x < C::kKeys / 32; ++x) {
              const int key = x * 32 + lane, word = part * (C::kKeys / 32) + x;
              const bool some = word * 32 + lane < valid && !(bad >> (key >> 4) & 1u);
              const float v = some ? sc[C::kKeys + key] : 0.0f;  // nothing was copied for the others
              top = fmaxf(top, v);
              if (some) small = min(small, __float_as_uint(v));
              const uint32_t off = __ballot_sync(0xffffffffu, !some);
              if (word == 0) gone.x = off;
              else if (word == 1) gone.y = off;
              else if (word == 2) gone.z = off;
              else gone.w = off;
              if (w == word) {
                ks = some ? sc[key] : 0.0f;
                vs = v;
              }
            }
          }
          uint8_t* plane = smem + (keys ? C::oK : C::oV) + b * C::kPlane;
          uint4 raw[C::kPieces];
#pragma unroll
          for (int i = 0; i < C::kPieces; ++i) {
            int row, cc;
            piece<BITS, D>(i, t, row, cc);
            raw[i] = *reinterpret_cast<const uint4*>(src + row * C::RB + cc * 16);
          }
#pragma unroll
          for (int i = 0; i < C::kPieces; ++i) {
            int row, cc;
            piece<BITS, D>(i, t, row, cc);
            put_piece<BITS, D>(raw[i], plane, part * C::kKeys + row, cc);
          }
          if (last) fence_proxy_async_shared();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&bars->raw_empty[s]);
            if (last) mbar_arrive(keys ? &bars->kready[b] : &bars->vready[b]);
          }
          if (keys && last) {
            // bits of non-negative floats rise with them (no NaN passes the fmaxf)
            const float mx = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(top, 0.0f))));
            if (mx > c || c == 0.0f) {
              // four times the next power of two, between 2^-100 and 2^100
              const int ex = min(max((int)(__float_as_uint(mx) >> 23) + 3, 27), 227);
              c = __uint_as_float((uint32_t)ex << 23);
            }
            least = __reduce_min_sync(0xffffffffu, small);
            float* sl = slots + (j & 3) * kSlotF;
            sl[t] = ks * a.scale_log2;
            sl[KT + t] = vs * (kRoom / c);
            if (t == 0) {
              const bool wide = __uint_as_float(least) < c * kWide;
              sl[2 * KT] = (float)((int)(__float_as_uint(c) >> 23) - 127);
              sl[2 * KT + 1] = __uint_as_float(wide ? 1u : 0u);
              *reinterpret_cast<uint4*>(sl + 2 * KT + 4) = gone;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->scready[j & 3]);
          }
        }
        const int u0 = at.u, b0 = at.b;
        more = at.next_tile(a);
        fresh = at.u != u0 || at.b != b0;
      }
    }
  } else {
    if (any) {
      // ── softmax ──
      constexpr int kGroup = kSoftWarps / 2;
      const int g = (warp - kFirstSoft) / kGroup, w16 = (warp - kFirstSoft) % kGroup;  // stream, warp of it
      const int lane0 = (warp & 3) * 32 + (w16 >> 2) * 16;  // its first TMEM lane, and row
      const uint32_t lane_sel = (uint32_t)lane0 << 16;
      const int xt = w16 * 32 + lane;
      float* xbuf = reinterpret_cast<float*>(smem + C::oX) + xt;
      float4* xml = reinterpret_cast<float4*>(smem + C::oX + C::kX) + xt;
      bool ok = true;
      int j0 = 0, step = 0, xs = 0;
      do {
        const int n = at.t_hi - at.t_lo;
        const int h = at.u / a.row_tiles, r0 = (at.u - h * a.row_tiles) * R + (MT == 2 ? g * 128 : 0) + lane0;
        auto row_id = [&](int row) -> int64_t {  // row of the unit -> row of the output
          const int t = row / a.G;
          return ((int64_t)at.b * a.T + t) * ((int64_t)a.H * a.G) + (int64_t)h * a.G + (row - t * a.G);
        };
        // ── Q rows, two lanes each: bf16 -> fp16 under a power of two, columns in unpack order ──
        float rowf[2];
        {
          constexpr int N = D / 16;  // 16-byte pieces a lane, every other of its row
          const int row = r0 + (lane >> 1);
          const bool live = row < a.rows;
          const uint4* qp = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.q) +
                                                           (live ? row_id(row) : 0) * D) + (lane & 1);
          uint4 raw[N];
#pragma unroll
          for (int i = 0; i < N; ++i) raw[i] = __ldg(qp + 2 * i);
          float top = 0.0f;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const uint32_t x[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
              top = fmaxf(top, fmaxf(fabsf(__uint_as_float(x[j] << 16)), fabsf(__uint_as_float(x[j] & 0xffff0000u))));
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          const int ex = (int)(__float_as_uint(top) >> 23);
          const int up = !live || ex == 0 || ex == 255 ? 127 : min(127 + 14 + 127 - ex, 227);
          const float f = live ? __uint_as_float((uint32_t)up << 23) : 0.0f;
          const float inv = __uint_as_float((uint32_t)(254 - up) << 23);
#pragma unroll
          for (int k = 0; k < 2; ++k) rowf[k] = __shfl_sync(0xffffffffu, inv, (8 * k + (lane >> 2)) * 2);
          if (MT == 2 || g == 0) {
            const int lr = lane0 + (lane >> 1);
            uint8_t* dst = smem + (MT == 2 ? (size_t)g * C::kQ : 0) + lr * 128;
#pragma unroll
            for (int i = 0; i < N; ++i) {
              const uint32_t x[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
              float v[8];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                v[2 * j] = live ? __uint_as_float(x[j] << 16) * f : 0.0f;
                v[2 * j + 1] = live ? __uint_as_float(x[j] & 0xffff0000u) * f : 0.0f;
              }
              const uint4 o = make_uint4(hf2(v[order<BITS>(0)], v[order<BITS>(1)]),
                                         hf2(v[order<BITS>(2)], v[order<BITS>(3)]),
                                         hf2(v[order<BITS>(4)], v[order<BITS>(5)]),
                                         hf2(v[order<BITS>(6)], v[order<BITS>(7)]));
              const int ch = 2 * i + (lane & 1);
              *reinterpret_cast<uint4*>(dst + (ch >> 3) * C::kQAtom + (((ch & 7) ^ (lr & 7)) << 4)) = o;
            }
            fence_proxy_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->qready);
          }
        }
        int tok[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) tok[k] = (r0 + 8 * k + (lane >> 2)) / a.G;
        Rows r = {};
        Tile tile;
        tile.s = t_s(g) + lane_sel;
        tile.o = t_o(g) + lane_sel;
        const int hist = at.len - a.T;  // keys before the tree
        const uint8_t* mask = a.tree + (int64_t)at.b * a.tree_b;
        const int i0 = MT == 2 ? 0 : g, di = MT == 2 ? 1 : 2;
        for (int i = i0; i < n && ok; i += di, ++step) {
          const int j = j0 + i, key0 = (at.t_lo + i) * KT - hist;
          uint4 hidden = make_uint4(0u, 0u, 0u, 0u);
          // while the codes are on their way
          if (__builtin_expect(key0 + KT > 0, 0)) hidden = tree_bits(key0, a.T, mask, a.tree_t, tok);
          ok = mbar_sleep_warp_to(&bars->scready[j & 3], (j >> 2) & 1, kErrTimeoutFull, a.err) &&
               mbar_sleep_warp_to(&bars->sready[g], step & 1, kErrTimeoutTmemFull, a.err);
          if (!ok) break;
          tc_fence_after();
          tile.slot = slots + (j & 3) * kSlotF;
          tile.first = i < di;
          softmax_tile<D>(r, tile, rowf, hidden);
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->pready[g]);
        }
        const bool some = i0 < n;  // this stream had tiles
        if (some && ok) ok = mbar_sleep_warp_to(&bars->pvdone[g], (step - 1) & 1, kErrTimeoutDone, a.err);
        if (!ok) break;
        tc_fence_after();
        // ── the segment's part: O = 2^m' sum, m' = m + log2(c / room) ──
        float4 ml[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float l = r.l[k];
          l += __shfl_xor_sync(0xffffffffu, l, 1);
          l += __shfl_xor_sync(0xffffffffu, l, 2);
          const bool none = !some || r.m_top[k] == -INFINITY;  // l: 0, or of NaN scores
          ml[k] = none ? make_float4(-INFINITY, l, -INFINITY, 0.0f)
                       : make_float4(r.mu[k], l, r.mu[k] + (r.lc[k] - 6.0f), 0.0f);
        }
        const bool both = MT == 1 && n > 1;
        if (MT == 1 && g == 1 && !both) {  // a single tile: nothing to hand over
          j0 += n;
          continue;
        }
        float f0[2] = {1.0f, 1.0f}, f1[2] = {0.0f, 0.0f}, inv[2] = {0.0f, 0.0f};
        const bool first = at.t_lo == 0, direct = a.direct && first && at.t_hi == at.n_tiles;
        int64_t id[2], part[2];
#pragma unroll 1
        for (int d = 0; d < D; d += 32) {
          uint32_t v[16];
          tmem_get(t_o(g) + lane_sel + d, v);
          if (both) {
            // the odd tiles' stream hands its rows to the even tiles', 32 columns at a time
            if (g == 1) {
              if (xs > 0) ok = mbar_sleep_warp_to(&bars->xfree, (xs - 1) & 1, kErrTimeoutEmpty, a.err);
              if (!ok) break;
              if (d == 0) {
                xml[0] = ml[0];
                xml[32 * kGroup] = ml[1];
              }
#pragma unroll
              for (int i = 0; i < 16; ++i) xbuf[i * 32 * kGroup] = __uint_as_float(v[i]);
              __syncwarp();
              if (lane == 0) mbar_arrive(&bars->xfull);
              ++xs;
              continue;
            }
            ok = mbar_sleep_warp_to(&bars->xfull, xs & 1, kErrTimeoutFull, a.err);
            if (!ok) break;
            if (d == 0) {
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const float4 x = ml[k], y = xml[k * 32 * kGroup];
                const float mx = fmaxf(x.x, y.x), mw = fmaxf(x.z, y.z);
                const float mb = mx == -INFINITY ? 0.0f : mx, wb = mw == -INFINITY ? 0.0f : mw;
                f0[k] = ex2(x.z - wb);
                f1[k] = ex2(y.z - wb);
                // the sum of NaN scores alone stands beside no maximum
                ml[k] = make_float4(mx, mx == -INFINITY ? x.y + y.y : ex2(x.x - mb) * x.y + ex2(y.x - mb) * y.y, mw,
                                    0.0f);
              }
            }
#pragma unroll
            for (int i = 0; i < 16; ++i)
              v[i] = __float_as_uint(f0[(i >> 1) & 1] * __uint_as_float(v[i]) +
                                     f1[(i >> 1) & 1] * xbuf[i * 32 * kGroup]);
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->xfree);
            ++xs;
          }
          if (d == 0) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int row = r0 + 8 * k + (lane >> 2);
              id[k] = row < a.rows ? row_id(row) : -1;
              part[k] = first ? id[k] : (int64_t)blockIdx.x * R + row - (at.u - h * a.row_tiles) * R;
              const float mb = ml[k].x == -INFINITY ? 0.0f : ml[k].x, l = ml[k].y;
              inv[k] = l != l ? l : ml[k].z == -INFINITY ? 0.0f : ex2(ml[k].z - mb) / l;  // NaN scores: NaN
              if (id[k] >= 0 && (lane & 3) == 0) {
                if (!direct) reinterpret_cast<float4*>(first ? a.main_ml : a.cta_ml)[part[k]] = ml[k];
                else if (a.lse) a.lse[id[k]] = l == 0.0f ? -INFINITY : (mb + __log2f(l)) * 0.69314718055994531f;
              }
            }
          }
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            // a lane's 32 bytes, four lanes a whole line of the row (columns pair by pair
            // took 3500 cycles more for 32 columns of a part)
            float2 m4[4];
            float o[8];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              m4[i] = make_float2(__uint_as_float(v[4 * i + 2 * k]), __uint_as_float(v[4 * i + 2 * k + 1]));
            eight_columns<BITS>(m4, o);
            const int col = d + 8 * (lane & 3);
            if (id[k] >= 0) {
              if (direct) {
                *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + id[k] * D + col) =
                    make_uint4(bf2(o[0] * inv[k], o[1] * inv[k]), bf2(o[2] * inv[k], o[3] * inv[k]),
                               bf2(o[4] * inv[k], o[5] * inv[k]), bf2(o[6] * inv[k], o[7] * inv[k]));
              } else {
                asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(
                                 (first ? a.main_o : a.cta_o) + part[k] * D + col),
                             "f"(o[0]), "f"(o[1]), "f"(o[2]), "f"(o[3]), "f"(o[4]), "f"(o[5]), "f"(o[6]), "f"(o[7])
                             : "memory");
              }
            }
            __syncwarp();
          }
        }
        __syncwarp();
        tc_fence_before();
        j0 += n;
      } while (ok && at.next_segment(a));
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    if (any) mbar_sleep_warp_to(&bars->drained, 0, kErrTimeoutDone, a.err);
    tc_fence_after();
    tmem_dealloc(tbase, 512);
  }
}

template <int BITS, int D, int MT>
int launch(const CUtensorMap& tk, const CUtensorMap& tv, const TreeArgs& a, int box, int ctas, cudaStream_t st) {
  using C = Cfg<BITS, D, MT>;
  auto kern = tree_attn_kernel<BITS, D, MT>;
  static_assert(C::kSmem <= 227 * 1024, "shared memory");
  MXB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem));
  MXB_CUDA_TRY(launch_pdl(kern, dim3((unsigned)ctas), kThreads, C::kSmem, st, tk, tv, a, box));
  MXB_LAUNCH_CHECK();
  return MXB_OK;
}

template <int BITS, int D>
int launch_mt(const CUtensorMap& tk, const CUtensorMap& tv, const TreeArgs& a, int box, int ctas, cudaStream_t st) {
  return tree_rows_per_cta(a.rows) == 256 ? launch<BITS, D, 2>(tk, tv, a, box, ctas, st)
                                          : launch<BITS, D, 1>(tk, tv, a, box, ctas, st);
}

}  // namespace tree

int tree_rows_per_cta(int64_t rows) { return rows > 128 ? 256 : 128; }

int tree_attention(const TreeArgs& a, int ctas, cudaStream_t st) {
  CUtensorMap tk, tv;
  const uint64_t rb = (uint64_t)a.dim * a.bits / 8;
  const int page = 1 << a.page_shift, keys = rb == 128 ? 64 : 128, box = page < keys ? page : keys;
  const uint64_t lines = (uint64_t)a.n_pages * a.H * page * rb / 128;
  const uint32_t box_lines = (uint32_t)(box * rb / 128);
  if (!encode_tmap_2d(&tk, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.k_codes, 128, lines, 128, box_lines,
                      CU_TENSOR_MAP_SWIZZLE_NONE) ||
      !encode_tmap_2d(&tv, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.v_codes, 128, lines, 128, box_lines,
                      CU_TENSOR_MAP_SWIZZLE_NONE))
    return MXB_E_CUDA;
  if (a.bits == 8)
    return a.dim == 128 ? tree::launch_mt<8, 128>(tk, tv, a, box, ctas, st)
                        : tree::launch_mt<8, 64>(tk, tv, a, box, ctas, st);
  return a.dim == 128 ? tree::launch_mt<4, 128>(tk, tv, a, box, ctas, st)
                      : tree::launch_mt<4, 64>(tk, tv, a, box, ctas, st);
}

}  // namespace mxb
