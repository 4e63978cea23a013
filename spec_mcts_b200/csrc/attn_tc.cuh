// The kernel on tcgen05 of prompt attention: with windows (attn_window_tc.cu), and with changed scores, documents and prefixes (attn_scores.cu).
//
// Two tiles of 128 queries take turns on the tensor cores: S = Q K^T of a tile of 128 keys into tensor memory, P = 2^(S - m) as fp16 over S's
// place, O += P V with P as the A operand from tensor memory.  While the MMAs of one tile of queries run, the other's softmax does.
//   warps 0 - 3, 4 - 7   softmax of the first and second tile of queries: a thread has a row; they write the output
//   warp 8               issues the MMAs (one thread), in the order O += P V of a step, S of the next, tile by tile
//   warp 9               requests tensor copies (one thread): Q, then keys and values in turn through a ring of five tiles
//   warps 10, 11         look through the values that some query of a tile sees in part: see below
// Tensor memory: S (and P) of the two tiles at columns 0 and 128, O at 256 and 384.
//
// m is 7 below a row's largest score, and stays until one passes it by 15, so that O is seldom rescaled; who rescales finds no MMA of its O on the
// way, since S of a step is finished after O += P V of the step before.
// A weight is rounded to fp16: off by 2^-11 of itself at most from 2^-21 of a row's largest on, and by 2^-32 of that below it.  (The sum has them in fp32: with m at the largest
// score itself, 8192 keys at 2^-26 of it were lost to O, but not to the sum.)  Two parts a weight, as for one query over pages, would be another eight of a step's sixteen MMAs
// and 2.5e-4 to 2.9e-4 of the result's norm off 64 bits would be 2.0e-4, which is the rounding of the result.
//
// A masked key has a weight of 0, and 0 times a value that is not finite is no number: in tiles with masked places such values are taken out of
// shared memory before the MMA, and added at the end to the rows that see them (as in attn_window_kernel).  In tiles that all see they stay; a weight
// that fp16 has as 0 makes no number of them there as well, and a row that ends with one takes the sum of what it sees that is not finite.
//
// Every wait is bounded: on expiry the error word is set, what is left is skipped, the CTA's own copies and MMAs are waited for (bounded too),
// and tensor memory is freed.
//
// What bounds it: 16384 positions, window 4096, 64 heads on 8 take 1.66 to 1.70 ms, by the card, 1.13 PFLOP/s and more (68 % of a cuBLAS product's burst rate; at the power limit 1.00 of its 1.40).  The MMAs alone,
// with softmax left out, take 1.469: one of 128 x 128 x 16 takes 87 cycles where 64 would be peak, and the hand-overs of a step the rest: a softmax of 128 keys takes 1750
// cycles (maximum 280, each half of the weights 670) while the other tile's MMAs take 1480.  Steps on the way, ms: P handed on whole 1.89, in halves 1.80; two stages
// of keys and of values, five slots for both 1.72; fewer comparisons and commits in the issuing thread 1.69.  A pair of CTAs that shares keys and values (cta_group::2) 1.80.
#pragma once
#include <math_constants.h>

#include <algorithm>

#include "attn_tiles.cuh"
#include "attn_window.cuh"
#include "q40_tc_common.cuh"
#include "tanh_cap.cuh"

namespace q40 {
namespace window {
namespace tc {

using ttc::elect_one;
using ttc::mbar_arrive;
using ttc::mbar_expect_tx;
using ttc::mbar_init;
using ttc::mbar_wait;

constexpr int THREADS = 384;
constexpr uint32_t TILE = BK * ATTN_D * 2;               // 32 KB: two blocks of 64 dims, rows of 128 bytes
constexpr uint32_t HALF = TILE / 2;
// log2 of a row's largest weight: where the maximum is set, and most.  fp16 holds 2^15
constexpr float WEIGHT_SET = 7.f, WEIGHT_TOP = 15.f;

struct Maps { CUtensorMap q, k, v; };


__device__ __forceinline__ void ld32(uint32_t taddr, float* x) {
  uint32_t* const r = reinterpret_cast<uint32_t*>(x);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,"
      "%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,"
      "%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
      "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// ... of a whole warp, which goes on together or not at all
__device__ __forceinline__ bool all_wait(uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)); }
// A wait while others go through up to n tiles: a wait's limit (measured: 0.59 s) for each 2^16 of them, which take 0.11 s
__device__ __forceinline__ bool long_wait(uint32_t bar, uint32_t parity, int n) {
  for (int i = 0; i <= n >> 16; ++i)
    if (mbar_wait(bar, parity)) return true;
  return false;
}
// D[tmem] (+)= A[smem] * B[smem]
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accum) : "memory");
}
// The B operand [keys][dims] as it lies: dims contiguous, 64 a row of 128 swizzled bytes, blocks of 64 dims a half tile apart, groups
// of eight keys 1024 bytes
__device__ __forceinline__ uint64_t values_desc(uint32_t saddr) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFF);
  d |= (uint64_t)(HALF >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
constexpr uint32_t IDESC = (1u << 4) | ((uint32_t)(BK >> 3) << 17) | ((uint32_t)(BQ >> 4) << 24);       // fp16 in, fp32 out
constexpr uint32_t VALUES_MAJOR = 1u << 16;                                                             // B lies dims first

__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// The lowest n bits, of any n
__device__ __forceinline__ uint32_t below(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; }

// What a form of the kernel knows of its rows.  Here: position p sees what is up to it, less than `window` back or below `sinks`, and scores are as they are
struct Plain {
  using Call = Args;
  static constexpr bool CAP = false, BIAS = false, SPANS = false;
  struct Places { Tiles tiles; Sees sees[2]; };
  template <class B>
  static __device__ __forceinline__ Places places(const Args& a, int row0, int split, Span&, B begin) {
    const Tiles tiles(a, row0, 2 * BQ, split);
    const Places at = {tiles, {tiles.sees(0, BQ, a), tiles.sees(BQ, BQ, a)}};
    begin();
    return at;
  }
  static __device__ __forceinline__ bool keeps(const Args&) { return false; }
};

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// A row's maximum, log2, and sum so far, and its step: the scores of 128 keys from key0 on, at s_at, become weights over their place, in two halves, each of
// which arrive() tells of; O, at o_at, is scaled where the maximum moves
template <class F>
struct Row {
  using Call = typename F::Call;
  float m = -3e38f, l = 0.f;
  Span span = {};                    // where F::SPANS
  float slope = 0.f;                 // where F::BIAS: what a position costs, log2
  int n = 0;                         // tiles of keys so far
  template <class Arrive>
  __device__ __forceinline__ void step(const Call& a, uint32_t s_at, uint32_t o_at, int p, int key0, bool masked, int lane, Arrive arrive) {
    float s[BK];
#pragma unroll
    for (int c = 0; c < 4; ++c) ld32(s_at + 32 * c, s + 32 * c);
    wait_ld();
    Cap k;
    if constexpr (F::CAP) k = cap(a, s);
    float rise = 0.f, begin = 0.f;                 // scores with a bias are log2, less `begin + c rise` in places 16 c .. 16 c + 15
    if constexpr (F::BIAS) bias(a, s, p, key0, k, rise, begin);
    if (masked) {
      const int last = (F::SPANS ? span.last : p) - key0, first = (F::SPANS ? span.start : 0) + a.sinks - key0;
      const int from = (F::SPANS ? max(p - a.window, span.start - 1) : p - a.window) - key0;      // seen: places <= last that are > from or < first
#pragma unroll
      for (int c = 0; c < BK; c += 32) {
        uint32_t seen = below(first - c);
        if (F::SPANS) seen &= ~below(span.start - key0 - c);
        seen = below(last + 1 - c) & (~below(from + 1 - c) | seen);
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (!(seen & (1u << e))) s[c + e] = -CUDART_INF_F;
      }
    }
    // With a cap the largest magnitude is known, which mostly tells that no score of a row passes its maximum
    if (!F::CAP || __any_sync(0xffffffffu, highest(a, k, p, key0) > m + WEIGHT_TOP)) {
      float most;
      if constexpr (F::BIAS) {
        most = -CUDART_INF_F;
#pragma unroll
        for (int c = 0; c < BK; c += 16) {
          float mx[2] = {max3(s[c], s[c + 1], s[c + 2]), max3(s[c + 8], s[c + 9], s[c + 10])};
#pragma unroll
          for (int e = 3; e < 7; e += 2) mx[0] = max3(mx[0], s[c + e], s[c + e + 1]), mx[1] = max3(mx[1], s[c + 8 + e], s[c + 9 + e]);
          most = fmaxf(most, fmaf((float)(c / 16), rise, begin) + max3(fmaxf(mx[0], mx[1]), s[c + 7], s[c + 15]));
        }
      } else {
        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int c = 4; c < BK - 4; c += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], s[c + e], s[c + 4 + e]);
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], s[BK - 4 + e]);
        most = max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]);
        most *= F::CAP ? k.of(most * most) : a.scale_log2;
      }
      const bool passes = most > m + WEIGHT_TOP;
      if (__any_sync(0xffffffffu, passes)) {
        const float now = passes ? most - WEIGHT_SET : m, corr = fmaxf(ex2(m - now), 1.17549435e-38f);      // (never 0: infinities stay)
        m = now;
        l *= corr;
        if (n > 0) {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            float o[32];
            ld32(o_at + 32 * c, o);
            wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= corr;
            st32(o_at + 32 * c, reinterpret_cast<const uint32_t*>(o));
          }
          wait_st();
        }
      }
    }
    const uint64_t scale2 = pack2(a.scale_log2, a.scale_log2), m2 = pack2(-m, -m);
    uint64_t sum[2] = {0, 0};                      // of this step: weight by weight onto l, the low bits of each would be lost to a long sum
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      uint32_t pk[32];
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        float x, y;
        const uint64_t s2 = pack2(s[64 * c + 2 * e], s[64 * c + 2 * e + 1]);
        if constexpr (F::BIAS) {
          const float less = fmaf((float)(4 * c + e / 8), rise, begin) - m;
          unpack2(add2(s2, pack2(less, less)), x, y);
        } else {
          unpack2(fma2(s2, F::CAP ? k.of(mul2(s2, s2)) : scale2, m2), x, y);
        }
        x = ex2(x);
        y = ex2(y);
        sum[e & 1] = add2(sum[e & 1], pack2(x, y));
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(pk[e]) : "f"(y), "f"(x));
      }
      st32(s_at + 32 * c, pk);
      wait_st();
      fence_before();
      __syncwarp();
      if (lane == 0) arrive(c);
    }
    float x, y;
    unpack2(add2(sum[0], sum[1]), x, y);
    l += x + y;
    ++n;
  }
  // A raw score s becomes s of(s^2) in log2: a polynomial while all of a warp's are in its range, else that much of what they have become by 2^x.  (The coefficient of the
  // highest power is above 0 there too, so that a masked -inf stays one)
  struct Cap {
    float x[5], top;                               // top: log2 of a magnitude that no score has passed
    __device__ __forceinline__ float of(float u) const { return fmaf(fmaf(fmaf(fmaf(x[4], u, x[3]), u, x[2]), u, x[1]), u, x[0]); }
    __device__ __forceinline__ uint64_t of(uint64_t u) const {
      uint64_t y = pack2(x[4], x[4]);
#pragma unroll
      for (int i = 3; i >= 0; --i) y = fma2(y, u, pack2(x[i], x[i]));
      return y;
    }
  };
  static __device__ __forceinline__ Cap cap(const Call& a, float (&s)[BK]) {
    float big[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < BK; c += 8)
#pragma unroll
      for (int e = 0; e < 4; ++e) big[e] = max3(big[e], fabsf(s[c + e]), fabsf(s[c + 4 + e]));
    Cap k;
    const float most = max3(fmaxf(big[0], big[1]), big[2], big[3]);
    if (__any_sync(0xffffffffu, most > a.cap_limit)) {
#pragma unroll
      for (int e = 0; e < BK; ++e) s[e] = tanh_by_exp(s[e] * a.cap_exp) * a.cap_out;
      k = {{a.scale_log2, 0.f, 0.f, 0.f, 1e-44f}, a.cap_out * a.scale_log2};
    } else {
#pragma unroll
      for (int i = 0; i < 5; ++i) k.x[i] = a.cap_k[i];
      k.top = most * k.of(most * most);
    }
    return k;
  }
  // What no score of a tile passes, with its bias
  __device__ __forceinline__ float highest(const Call&, const Cap& k, int p, int key0) const {
    if (!F::BIAS) return k.top;
    const float nearest = (float)max(p - key0 - (BK - 1), 0), farthest = (float)max(p - key0, key0 + BK - 1 - p);
    return k.top - slope * (slope >= 0.f ? nearest : farthest);
  }
  // Scores become log2 of what they are with their bias, less what 16 of them share: an instruction for two of them, where whole biases would be two
  __device__ __forceinline__ void bias(const Call& a, float (&s)[BK], int p, int key0, const Cap& k, float& rise, float& begin) const {
    const float at = (float)(key0 - p);
    const bool ahead = __any_sync(0xffffffffu, key0 + BK - 1 > p && span.last > p);          // keys ahead of some row
    uint64_t each[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) each[i] = ahead ? 0 : pack2(slope * (float)(2 * i), slope * (float)(2 * i + 1));
    const uint64_t scale2 = pack2(a.scale_log2, a.scale_log2);
#pragma unroll
    for (int e = 0; e < BK; e += 2) {
      const uint64_t s2 = pack2(s[e], s[e + 1]);
      unpack2(fma2(s2, F::CAP ? k.of(mul2(s2, s2)) : scale2, each[e / 2 % 8]), s[e], s[e + 1]);
    }
    if (ahead) {
#pragma unroll
      for (int e = 0; e < BK; ++e) s[e] = fmaf(-slope, fabsf(at + (float)e), s[e]);
      rise = begin = 0.f;
    } else {
      rise = 16.f * slope;
      begin = slope * at;
    }
  }
  // ... and its output, or a split's partial result.  taken_out: values that are not finite were taken out of tiles that `sees` say are seen in part
  // stage: 8 KB of shared memory of this warp's
  template <class T, class S>
  __device__ __forceinline__ void write(const Call& a, uint32_t o_at, int p, int h, int hk, const T& tiles, const S (&sees)[2], bool taken_out, unsigned char* stage,
                                        int lane) const {
    const float inv = l != 0.f ? 1.f / l : 0.f;
    const bool no_document = F::SPANS && span.last < p, there = p <= tiles.p_last && !(no_document && F::keeps(a));
    // Where CTAs come in waves: all of a row at once, and rows by way of shared memory, sixteen lanes a row (4001 tokens in nine documents 76.3 -> 72.4 us; in one wave 77
    // tokens take 6.9 this way, and 6.3 as below).  The rows' place is that of the queries, whose copy has landed
    if (F::SPANS && gridDim.x > 148 && a.splits == 1 && a.wide_out && !taken_out) {
      float o[ATTN_D];
#pragma unroll
      for (int c = 0; c < 4; ++c) ld32(o_at + 32 * c, o + 32 * c);
      wait_ld();
      if (n == 0)
#pragma unroll
        for (int e = 0; e < ATTN_D; ++e) o[e] = 0.f;
      uint64_t all[4] = {0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < ATTN_D / 2; ++e) all[e % 4] = add2(all[e % 4], pack2(o[2 * e], o[2 * e + 1]));
      float x, y;
      unpack2(add2(add2(all[0], all[1]), add2(all[2], all[3])), x, y);
      if (!__any_sync(0xffffffffu, x + y != x + y)) {        // else what is no number is looked into below
        uint4* const row = reinterpret_cast<uint4*>(stage) + 16 * lane;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          uint32_t w[4];
#pragma unroll
          for (int d = 0; d < 4; ++d) w[d] = h2_as_u32(__floats2half2_rn(o[8 * e + 2 * d] * inv, o[8 * e + 2 * d + 1] * inv));
          row[e ^ (lane & 7)] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        const uint32_t rows = __ballot_sync(0xffffffffu, there);
        __syncwarp();
        __half* const out = a.o + (int64_t)(p - lane - a.offset) * a.ldo + h * ATTN_D + 8 * (lane & 15);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int r = 2 * i + (lane >> 4);
          if ((rows >> r) & 1) *reinterpret_cast<uint4*>(out + r * a.ldo) = reinterpret_cast<const uint4*>(stage)[16 * r + ((lane & 15) ^ (r & 7))];
        }
        return;
      }
    }
    __half* const out = a.o + (int64_t)(p - a.offset) * a.ldo + h * ATTN_D;
    const int64_t part_at = ((int64_t)blockIdx.y * a.S + (p - a.offset)) * a.H + h;
    if (a.splits > 1 && p <= tiles.p_last) a.pml[part_at] = make_float2(m, no_document ? -1.f : l);
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
      float o[32];
      ld32(o_at + 32 * c, o);
      wait_ld();
      if (n == 0)                                  // none of the split's keys: nothing has been written there
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = 0.f;
      uint64_t all[16];                            // (a sum is no number where one of them is none, and where they are infinite both ways, which does no harm)
#pragma unroll
      for (int e = 0; e < 16; ++e) all[e] = pack2(o[2 * e], o[2 * e + 1]);
#pragma unroll
      for (int e = 8; e > 0; e >>= 1)
#pragma unroll
        for (int d = 0; d < e; ++d) all[d] = add2(all[d], all[d + e]);
      float x, y;
      unpack2(all[0], x, y);
      const bool lost = x + y != x + y && l == l;  // no number, and not by a score: see above
      if ((taken_out || lost) && there) {          // rare, and slow
        uint32_t found = 0;
        for (int j = 0; j < tiles.n; ++j) {
          const int tile = tiles.tile(j), key0 = tile * BK;
          if (!lost && !sees[0].part(tile) && !sees[1].part(tile)) continue;
          for (int k = key0; k < min(key0 + BK, (F::SPANS ? span.last : p) + 1); ++k) {
            const int start = F::SPANS ? span.start : 0;
            if (k < start || (p - k >= a.window && k - start >= a.sinks)) continue;
            const __half* const v = a.v + (int64_t)k * a.ldv + hk * ATTN_D + 32 * c;
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (not_finite(v[e])) {
                o[e] = (lost && !(found & (1u << e)) ? 0.f : o[e]) + __half2float(v[e]);
                found |= 1u << e;
              }
          }
        }
      }
      if (there && a.splits > 1) {
        float4* const part = reinterpret_cast<float4*>(a.po + part_at * ATTN_D + 32 * c);
#pragma unroll
        for (int e = 0; e < 8; ++e) part[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
      } else if (there) {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) w[e] = h2_as_u32(__floats2half2_rn(o[2 * e] * inv, o[2 * e + 1] * inv));
        if (a.wide_out) {
#pragma unroll
          for (int e = 0; e < 4; ++e) reinterpret_cast<uint4*>(out + 32 * c)[e] = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) reinterpret_cast<uint32_t*>(out + 32 * c)[e] = w[e];
        }
      }
    }
  }
};

// Values that are not finite, among `n` pieces of 16 bytes, become zeros, by 64 threads at 0 .. 63 of two warps; whether this warp found any.  (64 bytes of eight
// values a thread and step: magnitudes by maxima of pairs, above all of which is what is not finite)
__device__ __forceinline__ bool take_out(uint4* v, int n, int at) {
  __half2 most[2] = {u32_as_h2(0), u32_as_h2(0)};
#pragma unroll 8
  for (int c = at; c < n; c += 64) {
    const uint4 x = v[c];
    most[0] = __hmax2_nan(__hmax2_nan(most[0], __habs2(u32_as_h2(x.x))), __habs2(u32_as_h2(x.y)));
    most[1] = __hmax2_nan(__hmax2_nan(most[1], __habs2(u32_as_h2(x.z))), __habs2(u32_as_h2(x.w)));
  }
  const __half2 top = __hmax2_nan(most[0], most[1]);
  if (!__any_sync(0xffffffffu, not_finite(__low2half(top)) || not_finite(__high2half(top)))) return false;
  __half* const x = reinterpret_cast<__half*>(v);
  for (int c = at; c < n; c += 64)
    for (int e = 0; e < 8; ++e)
      if (not_finite(x[8 * c + e])) x[8 * c + e] = __ushort_as_half(0);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");           // the MMA reads them
  return true;
}

constexpr int SLOTS = 5;                        // of the ring that keys and values go through in turn
constexpr int LOOKED = 4;                       // barriers of values that are looked through: at most three of them are in the ring
constexpr uint32_t AT_Q = 0, AT_RING = 2 * TILE, AT_BARS = AT_RING + SLOTS * TILE;
enum Bar { Q_FULL, FULL = Q_FULL + 2, EMPTY = FULL + SLOTS, LOOK = EMPTY + SLOTS, READY = LOOK + LOOKED, S_FULL = READY + LOOKED,
           P_HALF = S_FULL + 2, P_FULL = P_HALF + 2, O_DONE = P_FULL + 2, ALL_DONE = O_DONE + 2, BARS };
static_assert(BARS <= 32, "a lane makes a barrier");
constexpr uint32_t SMEM = AT_BARS + 8 * BARS + 48 + 1024;       // (1024: the alignment)

template <class F>
__global__ void __launch_bounds__(THREADS, 1)
attn_tc_kernel(const typename F::Call a, const __grid_constant__ Maps maps, int* err) {
  extern __shared__ unsigned char smem_raw[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t raw0 = ttc::smem_u32(smem_raw), base = (raw0 + 1023u) & ~1023u;
  unsigned char* const gbase = smem_raw + (base - raw0);
  const auto bar = [&](int which) { return base + AT_BARS + 8 * which; };
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(gbase + AT_BARS + 8 * BARS);
  volatile int* const s_failed = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* const s_taken_out = s_failed + 1;
  volatile uint32_t* const s_requested = tmem_slot + 3;          // of each slot: the barrier of its last copy, and 1 + the phase
  const int blocks = (a.S + 2 * BQ - 1) / (2 * BQ);
  const int blk = blocks - 1 - (int)(blockIdx.x / a.H), h = (int)(blockIdx.x % a.H), hk = h / (a.H / a.Hkv);
  const int row0 = blk * 2 * BQ;
  const auto copy = [&](const CUtensorMap* map, uint32_t dst, int head, int row, uint32_t full) {
    mbar_expect_tx(full, TILE);
    ttc::tma_2d(dst, map, head * ATTN_D, row, full);
    ttc::tma_2d(dst + HALF, map, head * ATTN_D + 64, row, full);
  };
  const auto begin = [&]() {
    // (the same for all lanes, which the compiler does not know; places of tiles that come later would be spilled)
    if ((F::SPANS ? __shfl_sync(0xffffffffu, warp, 0) : warp) == 9) {
      if (lane < BARS) mbar_init(bar(lane), lane >= P_HALF && lane < P_FULL + 2 ? 4 : lane >= READY && lane < READY + LOOKED ? 2 : 1);
      if (lane < SLOTS) s_requested[lane] = 0;
      if (lane == 0) *s_failed = *s_taken_out = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      // the first queries are on their way while the others find out which keys they see
      asm volatile("griddepcontrol.wait;" ::: "memory");
      if (elect_one()) {
        copy(&maps.q, base + AT_Q, h, row0, bar(Q_FULL));
      }
      __syncwarp();
    }
  };
  Span span = {};
  const auto where = F::places(a, row0, blockIdx.y, span, begin);
  const auto& tiles = where.tiles;
  const auto& sees = where.sees;
  if (warp == 9) {
    if (elect_one()) {
      if (tiles.n > 0) {
        s_requested[0] = 2 * FULL + 1;
        copy(&maps.k, base + AT_RING, hk, tiles.tile(0) * BK, bar(FULL));
      }
      if (sees[1].last >= 0) copy(&maps.q, base + AT_Q + TILE, h, row0 + BQ, bar(Q_FULL + 1));
    }
    __syncwarp();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ttc::smem_u32(tmem_slot)), "n"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  bool failed = false;
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int i = warp >> 2, p = tiles.p_first + i * BQ + (warp & 3) * 32 + lane;
    const uint32_t quad = (uint32_t)(32 * (warp & 3)) << 16, s_at = tmem + quad + 128 * i, o_at = s_at + 256;
    const auto mine = i ? sees[1] : sees[0];
    Row<F> row;
    row.span = span;
    if constexpr (F::BIAS) row.slope = a.slopes[h] * 1.44269504f;
    for (int j = 0; j < tiles.n; ++j) {
      const int tile = tiles.tile(j);
      if (!mine.some(tile)) continue;
      if (!all_wait(bar(S_FULL + i), row.n & 1)) { failed = true; break; }
      fence_after();
      row.step(a, s_at, o_at, p, tile * BK, !mine.all(tile), lane, [&](int half) { mbar_arrive(bar((half ? P_FULL : P_HALF) + i)); });
    }
    if (!failed && mine.last >= 0) {
      if (!all_wait(bar(O_DONE + i), 0)) failed = true;
      // (write() puts rows where the queries are: who took no step waits for their copy, which nothing else here has waited for)
      if (F::SPANS && row.n == 0 && !all_wait(bar(Q_FULL + i), 0)) failed = true;
      fence_after();
      if (!failed) row.write(a, o_at, p, h, hk, tiles, sees, *s_taken_out, gbase + AT_Q + i * TILE + (warp & 3) * (TILE / 4), lane);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 8) {
      if (elect_one()) {
        bool pending[2] = {false, false}, q_there[2] = {false, false};      // O += P V of the tile before is still to come
        int steps[2] = {0, 0}, slot = 0, looked = 0, v_slot = 0;
        bool v_masked = false, v_there = false;        // the values are in v_slot, the looked-th to be looked through; they have been waited for
        uint32_t phases = 0;                           // of FULL, a bit a slot
        const auto full = [&](int at) { return mbar_wait(bar(FULL + at), (phases >> at) & 1); };
        const auto values_there = [&]() {
          if (v_there) return true;
          v_there = true;
          if (!v_masked) return full(v_slot);
          return mbar_wait(bar(LOOK + looked % LOOKED), (looked / LOOKED) & 1) && mbar_wait(bar(READY + looked % LOOKED), (looked / LOOKED) & 1);
        };
        const auto product = [&](int i) {
          pending[i] = false;
          if (!values_there() || !mbar_wait(bar(P_HALF + i), (steps[i] - 1) & 1)) return false;
          fence_after();
          const uint64_t b = values_desc(base + AT_RING + v_slot * TILE);
#pragma unroll
          for (int ks = 0; ks < BK / 32; ++ks)
            ttc::mma_ts(tmem + 256 + 128 * i, tmem + 128 * i + 8 * ks, b + (uint64_t)((ks * 2048) >> 4), IDESC | VALUES_MAJOR, steps[i] > 1 || ks > 0 ? 1u : 0u);
          if (!mbar_wait(bar(P_FULL + i), (steps[i] - 1) & 1)) return false;
          fence_after();
#pragma unroll
          for (int ks = BK / 32; ks < BK / 16; ++ks)
            ttc::mma_ts(tmem + 256 + 128 * i, tmem + 128 * i + 8 * ks, b + (uint64_t)((ks * 2048) >> 4), IDESC | VALUES_MAJOR, 1u);
          return true;
        };
        for (int j = 0; j < tiles.n && !failed; ++j) {
          const int tile = tiles.tile(j), next = slot + 1 == SLOTS ? 0 : slot + 1;       // keys in `slot`, values in the next
          if (!full(slot)) { failed = true; break; }
          bool scored[2] = {false, false};
          const auto scores = [&](int i) {
            scored[i] = true;
            if (!sees[i].some(tile)) return true;
            if (!q_there[i]) {
              if (!mbar_wait(bar(Q_FULL + i), 0)) return false;
              q_there[i] = true;
            }
            fence_after();
            const uint64_t qd = ttc::kmajor_desc(base + AT_Q + i * TILE), kd = ttc::kmajor_desc(base + AT_RING + slot * TILE);
#pragma unroll
            for (int ks = 0; ks < ATTN_D / 16; ++ks) {
              const uint64_t off = (uint64_t)(((ks >> 2) * HALF + (ks & 3) * 32) >> 4);
              mma_ss(tmem + 128 * i, qd + off, kd + off, IDESC, ks > 0 ? 1u : 0u);
            }
            ttc::commit(bar(S_FULL + i));
            pending[i] = true;
            ++steps[i];
            return true;
          };
          // the second tile's scores do not wait for the first one's weights where it has none to wait for itself
          const bool due = pending[1];                           // a product of the second tile with the values of the tile before
          if (F::SPANS && !due && pending[0] && !scores(1)) { failed = true; break; }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (failed) break;
            if ((i && F::SPANS ? due : pending[i]) && !product(i)) { failed = true; break; }
            if (i == 1 && j > 0) ttc::commit(bar(EMPTY + v_slot));
            if (!(F::SPANS && scored[i]) && !scores(i)) failed = true;
          }
          if (failed) break;
          ttc::commit(bar(EMPTY + slot));
          if (v_masked) ++looked;
          else if (j > 0) phases ^= 1u << v_slot;
          phases ^= 1u << slot;
          v_slot = next;
          v_masked = sees[0].part(tile) || sees[1].part(tile);
          v_there = false;
          slot = next + 1 == SLOTS ? 0 : next + 1;
        }
        for (int i = 0; i < 2; ++i) {
          if (!failed && pending[i] && !product(i)) failed = true;
          ttc::commit(bar(O_DONE + i));
        }
        ttc::commit(bar(ALL_DONE));
      }
      __syncwarp();
    } else if (warp == 9) {
      if (elect_one()) {
        int slot = 1, looked = 0;
        uint32_t full = 1;                             // phases of FULL, a bit a slot
        for (int x = 1; x < 2 * tiles.n; ++x) {        // keys of tile x / 2, or its values; the first are requested
          const int tile = tiles.tile(x >> 1);
          if (x >= SLOTS && !mbar_wait(bar(EMPTY + slot), (x / SLOTS - 1) & 1)) { failed = true; break; }
          const bool look = (x & 1) && (sees[0].part(tile) || sees[1].part(tile));
          const int which = look ? LOOK + looked % LOOKED : FULL + slot;
          s_requested[slot] = 2 * which + 1 + (look ? (looked / LOOKED) & 1 : (full >> slot) & 1);
          copy(x & 1 ? &maps.v : &maps.k, base + AT_RING + slot * TILE, hk, tile * BK, bar(which));
          if (look) ++looked;
          else full ^= 1u << slot;
          if (++slot == SLOTS) slot = 0;
        }
        // queries that see none of a split's keys are waited for by nobody else
        for (int i = 0; i < 2; ++i)
          if (sees[i].last >= 0 && !mbar_wait(bar(Q_FULL + i), 0)) failed = true;
      }
      __syncwarp();
    } else {
      const int at = (warp - 10) * 32 + lane;
      int looked = 0;
      for (int j = 0; j < tiles.n; ++j) {
        const int tile = tiles.tile(j);
        if (!sees[0].part(tile) && !sees[1].part(tile)) continue;
        const int which = looked % LOOKED;
        if (!__all_sync(0xffffffffu, long_wait(bar(LOOK + which), (looked / LOOKED) & 1, tiles.n))) { failed = true; break; }
        ++looked;
        uint4* const v = reinterpret_cast<uint4*>(gbase + AT_RING + (2 * j + 1) % SLOTS * TILE);
        if (take_out(v, (int)TILE / 16, at)) *s_taken_out = 1;
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(READY + which));
      }
    }
  }
  if (!long_wait(bar(ALL_DONE), 0, tiles.n) || failed) *s_failed = 1;
  fence_before();
  __syncthreads();
  if (tid == 0 && *s_failed) {
    q40_set_error(err);
    for (int i = 0; i < 2; ++i)
      if (sees[i].last >= 0) mbar_wait(bar(Q_FULL + i), 0);
    for (int i = 0; i < SLOTS; ++i)
      if (const uint32_t r = s_requested[i]) mbar_wait(bar((int)(r - 1) >> 1), (r - 1) & 1);
  }
  __syncthreads();
  if (warp == 8) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512));
  }
}

// Partial results of a row, in the splits' order: a warp has one, a lane four dims
template <class F>
__global__ void __launch_bounds__(128)
attn_tc_merge_kernel(const typename F::Call a, int64_t rows) {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  float M = -3e38f;
  for (int s = 0; s < a.splits; ++s) M = fmaxf(M, a.pml[s * rows + row].x);
  float x[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f;
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) {
    const float2 ml = a.pml[s * rows + row];
    const float4 o = reinterpret_cast<const float4*>(a.po + (s * rows + row) * ATTN_D)[lane];
    const float f = fmaxf(ex2(ml.x - M), 1.17549435e-38f), y[4] = {o.x, o.y, o.z, o.w};
    l = fmaf(ml.y, f, l);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = fmaf(y[e], f, x[e]);
  }
  if (F::SPANS && l < 0.f && F::keeps(a)) return;               // a row of no document
  const float inv = l != 0.f ? 1.f / l : 0.f;
  __half* const out = a.o + row / a.H * a.ldo + row % a.H * ATTN_D + 4 * lane;
  reinterpret_cast<__half2*>(out)[0] = __floats2half2_rn(x[0] * inv, x[1] * inv);
  reinterpret_cast<__half2*>(out)[1] = __floats2half2_rn(x[2] * inv, x[3] * inv);
}

// Copies of `box` rows of 64 dims out of rows of heads
inline bool make_map(CUtensorMap* m, const __half* x, int heads, int64_t rows, int64_t ld, int box) {
  EncodeTiledFn encode = ttc_encode_fn();
  if (!encode) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)heads * ATTN_D, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t boxes[2] = {64, (cuuint32_t)box}, one[2] = {1, 1};
  return ttc_encode(encode, m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2u, (void*)x, dims, strides, boxes, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class F>
static int launch_form(const typename F::Call& a, int* err, cudaStream_t st) {
  Maps maps;
  const int64_t keys = (int64_t)a.offset + a.S;
  if (!make_map(&maps.q, a.q, a.H, a.S, a.ldq, BQ) || !make_map(&maps.k, a.k, a.Hkv, keys, a.ldk, BK) || !make_map(&maps.v, a.v, a.Hkv, keys, a.ldv, BK))
    return Q40_E_UNSUPPORTED;
  static std::atomic<uint64_t> ready;
  cudaError_t e = q40_allow_smem(ready, (const void*)attn_tc_kernel<F>, (int)SMEM);
  if (e != cudaSuccess) { (void)cudaGetLastError(); return Q40_E_UNSUPPORTED; }
  const int64_t blocks = (int64_t)a.H * ((a.S + 2 * BQ - 1) / (2 * BQ));
  if (blocks > 0x7fffffffLL) return Q40_E_SHAPE;
  e = q40_launch_pdl(attn_tc_kernel<F>, dim3((unsigned)blocks, a.splits), dim3(THREADS), SMEM, st, a, maps, err);
  const int64_t rows = (int64_t)a.S * a.H;
  if (e == cudaSuccess && a.splits > 1) e = q40_launch_pdl(attn_tc_merge_kernel<F>, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, st, a, rows);
  return e == cudaSuccess ? Q40_OK : (int)e;
}

}  // namespace tc
}  // namespace window
}  // namespace q40
