// q40_attn_causal_window's kernel for prompts with enough work: on tcgen05, 256 queries of one head a CTA.
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
#include <math_constants.h>

#include <algorithm>

#include "attn_window.cuh"
#include "q40_tc_common.cuh"

namespace q40 {
namespace window {
namespace tc {

using ttc::elect_one;
using ttc::mbar_arrive;
using ttc::mbar_expect_tx;
using ttc::mbar_init;
using ttc::mbar_wait;

constexpr int BQ = 128, BK = 128, THREADS = 384;            // queries of a CTA's tile, keys of a tile
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

// Which tiles of keys (by number: keys BK t ..) a tile of queries sees some keys of, and all of them.  (Comparisons of numbers that are made once: the
// thread that issues MMAs asks for every tile, and a few hundred cycles of it were a tenth of the time)
struct Sees {
  int last, from, sinks, all_last, all_from, all_sinks;
  // queries at positions first .. end, none if end < first
  __host__ __device__ __forceinline__ Sees(int first, int end, int window, int n_sinks) {
    last = end >= first ? end / BK : -1;
    from = first - window + 1 > 0 ? (first - window + 1) / BK : 0;
    sinks = (n_sinks + BK - 1) / BK;
    all_last = (first + 1) / BK - 1;
    all_from = end - window + 1 > 0 ? (end - window + BK) / BK : 0;
    all_sinks = n_sinks / BK;
  }
  __host__ __device__ __forceinline__ bool some(int t) const { return t <= last && (t >= from || t < sinks); }
  __host__ __device__ __forceinline__ bool all(int t) const { return t <= all_last && (t >= all_from || t < all_sinks); }
  __host__ __device__ __forceinline__ bool part(int t) const { return some(t) && !all(t); }
};

// The tiles of keys that a CTA goes through, tile(0) to tile(n - 1): those that one of its queries sees, or a split's share of them
struct Tiles {
  int p_first, p_last;               // positions of the CTA's first and last query
  int t_first, t_from, j0, n;
  // `rows` queries from row0 on
  __host__ __device__ __forceinline__ Tiles(const Args& a, int row0, int rows, int split) {
    p_first = a.offset + row0;
    p_last = (p_first + rows < a.offset + a.S ? p_first + rows : a.offset + a.S) - 1;
    const int from = p_first - a.window + 1 > 0 ? p_first - a.window + 1 : 0, first = a.sinks < from ? a.sinks : from;
    t_first = (first + BK - 1) / BK;
    t_from = from / BK > t_first ? from / BK : t_first;
    const int all = t_first + p_last / BK + 1 - t_from;
    j0 = (int)((int64_t)all * split / a.splits);
    n = (int)((int64_t)all * (split + 1) / a.splits) - j0;
  }
  __device__ __forceinline__ int tile(int j) const { return j + j0 < t_first ? j + j0 : j + j0 - t_first + t_from; }
  // `count` queries from the first-th on
  __host__ __device__ __forceinline__ Sees sees(int first, int count, const Args& a) const {
    const int end = p_first + first + count - 1;
    return Sees(p_first + first, end < p_last ? end : p_last, a.window, a.sinks);
  }
};

// A row's maximum, log2, and sum so far, and its step: the scores of 128 keys from key0 on, at s_at, become weights over their place, in two halves, each of
// which arrive() tells of; O, at o_at, is scaled where the maximum moves
struct Row {
  float m = -3e38f, l = 0.f;
  int n = 0;                         // tiles of keys so far
  template <class Arrive>
  __device__ __forceinline__ void step(const Args& a, uint32_t s_at, uint32_t o_at, int p, int key0, bool masked, int lane, Arrive arrive) {
    float s[BK];
#pragma unroll
    for (int c = 0; c < 4; ++c) ld32(s_at + 32 * c, s + 32 * c);
    wait_ld();
    if (masked) {
      const int last = p - key0, from = p - a.window - key0, first = a.sinks - key0;      // seen: places <= last that are > from or < first
#pragma unroll
      for (int c = 0; c < BK; c += 32) {
        const uint32_t seen = below(last + 1 - c) & (~below(from + 1 - c) | below(first - c));
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (!(seen & (1u << e))) s[c + e] = -CUDART_INF_F;
      }
    }
    float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
    for (int c = 4; c < BK - 4; c += 8)
#pragma unroll
      for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], s[c + e], s[c + 4 + e]);
#pragma unroll
    for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], s[BK - 4 + e]);
    const float most = max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]) * a.scale_log2;
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
    const uint64_t scale2 = pack2(a.scale_log2, a.scale_log2), m2 = pack2(-m, -m);
    uint64_t sum[2] = {0, 0};                      // of this step: weight by weight onto l, the low bits of each would be lost to a long sum
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      uint32_t pk[32];
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        float x, y;
        unpack2(fma2(pack2(s[64 * c + 2 * e], s[64 * c + 2 * e + 1]), scale2, m2), x, y);
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
  // ... and its output, or a split's partial result.  taken_out: values that are not finite were taken out of tiles that `sees` say are seen in part
  __device__ __forceinline__ void write(const Args& a, uint32_t o_at, int p, int h, int hk, const Tiles& tiles, const Sees (&sees)[2], bool taken_out) const {
    const float inv = l != 0.f ? 1.f / l : 0.f;
    const bool there = p <= tiles.p_last;
    // (rows by way of shared memory, 256 bytes of one at a time: no faster)
    __half* const out = a.o + (int64_t)(p - a.offset) * a.ldo + h * ATTN_D;
    const int64_t part_at = ((int64_t)blockIdx.y * a.S + (p - a.offset)) * a.H + h;
    if (a.splits > 1 && there) a.pml[part_at] = make_float2(m, l);
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
          for (int k = key0; k < min(key0 + BK, p + 1); ++k) {
            if (p - k >= a.window && k >= a.sinks) continue;
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

__global__ void __launch_bounds__(THREADS, 1)
attn_window_tc_kernel(const Args a, const __grid_constant__ Maps maps, int* err) {
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
  const Tiles tiles(a, row0, 2 * BQ, blockIdx.y);
  const Sees sees[2] = {tiles.sees(0, BQ, a), tiles.sees(BQ, BQ, a)};       // (in front of the waits)

  const auto copy = [&](const CUtensorMap* map, uint32_t dst, int head, int row, uint32_t full) {
    mbar_expect_tx(full, TILE);
    ttc::tma_2d(dst, map, head * ATTN_D, row, full);
    ttc::tma_2d(dst + HALF, map, head * ATTN_D + 64, row, full);
  };
  if (warp == 9) {
    if (lane < BARS) mbar_init(bar(lane), lane >= P_HALF && lane < P_FULL + 2 ? 4 : lane >= READY && lane < READY + LOOKED ? 2 : 1);
    if (lane < SLOTS) s_requested[lane] = 0;
    if (lane == 0) *s_failed = *s_taken_out = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    // the first queries and keys are on their way while the others meet
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (elect_one() && tiles.n > 0) {
      copy(&maps.q, base + AT_Q, h, row0, bar(Q_FULL));
      s_requested[0] = 2 * FULL + 1;
      copy(&maps.k, base + AT_RING, hk, tiles.tile(0) * BK, bar(FULL));
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
    const Sees mine = i ? sees[1] : sees[0];
    Row row;
    for (int j = 0; j < tiles.n; ++j) {
      const int tile = tiles.tile(j);
      if (!mine.some(tile)) continue;
      if (!all_wait(bar(S_FULL + i), row.n & 1)) { failed = true; break; }
      fence_after();
      row.step(a, s_at, o_at, p, tile * BK, !mine.all(tile), lane, [&](int half) { mbar_arrive(bar((half ? P_FULL : P_HALF) + i)); });
    }
    if (!failed && mine.last >= 0) {
      if (!all_wait(bar(O_DONE + i), 0)) failed = true;
      fence_after();
      if (!failed) row.write(a, o_at, p, h, hk, tiles, sees, *s_taken_out);
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
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (failed) break;
            if (pending[i] && !product(i)) { failed = true; break; }
            if (i == 1 && j > 0) ttc::commit(bar(EMPTY + v_slot));
            if (!sees[i].some(tile)) continue;
            if (!q_there[i]) {
              if (!mbar_wait(bar(Q_FULL + i), 0)) { failed = true; break; }
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
          if (tiles.n > 0 && sees[i].last >= 0 && !mbar_wait(bar(Q_FULL + i), 0)) failed = true;
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
      if (tiles.n > 0 && sees[i].last >= 0) mbar_wait(bar(Q_FULL + i), 0);
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
__global__ void __launch_bounds__(128)
attn_window_merge_kernel(const Args a, int64_t rows) {
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
  const float inv = l != 0.f ? 1.f / l : 0.f;
  __half* const out = a.o + row / a.H * a.ldo + row % a.H * ATTN_D + 4 * lane;
  reinterpret_cast<__half2*>(out)[0] = __floats2half2_rn(x[0] * inv, x[1] * inv);
  reinterpret_cast<__half2*>(out)[1] = __floats2half2_rn(x[2] * inv, x[3] * inv);
}

}  // namespace tc

int splits_tc(const Args& a) {
  using namespace tc;
  const int64_t blocks = (int64_t)a.H * ((a.S + 2 * BQ - 1) / (2 * BQ));
  Args one = a;
  one.splits = 1;
  const int tiles = Tiles(one, (a.S - 1) / (2 * BQ) * 2 * BQ, 2 * BQ, 0).n;          // of the last block, which has most
  // Least of what a CTA takes for its tiles and what sharing them costs: another launch, and the partial results' way out and back
  // (us; measured: 256 queries x 32 heads, 11 tiles 27.5 alone, 20 in four splits; 512 queries, four tiles 12.7 alone, 19 in two)
  const double tile = a.S > BQ ? 2.1 : 1.4, part = 0.35e-6 * a.S * a.H * (ATTN_D + 2) * sizeof(float);
  int best = 1;
  double least = tile * tiles;
  for (int s = 2; s <= 16 && s * blocks <= 148 && 2 * s <= tiles; ++s) {
    const double t = tile * ((tiles + s - 1) / s) + 3.5 + part * s;
    if (t < least) { least = t; best = s; }
  }
  return best;
}

// Copies of `box` rows of 64 dims out of rows of heads
static bool make_map(CUtensorMap* m, const __half* x, int heads, int64_t rows, int64_t ld, int box) {
  EncodeTiledFn encode = ttc_encode_fn();
  if (!encode) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)heads * ATTN_D, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t boxes[2] = {64, (cuuint32_t)box}, one[2] = {1, 1};
  return ttc_encode(encode, m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2u, (void*)x, dims, strides, boxes, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int launch_tc(const Args& a, int* err, cudaStream_t st) {
  using namespace tc;
  Maps maps;
  const int64_t keys = (int64_t)a.offset + a.S;
  if (!make_map(&maps.q, a.q, a.H, a.S, a.ldq, BQ) || !make_map(&maps.k, a.k, a.Hkv, keys, a.ldk, BK) || !make_map(&maps.v, a.v, a.Hkv, keys, a.ldv, BK))
    return Q40_E_UNSUPPORTED;
  static std::atomic<uint64_t> ready;
  cudaError_t e = q40_allow_smem(ready, (const void*)attn_window_tc_kernel, (int)SMEM);
  if (e != cudaSuccess) { (void)cudaGetLastError(); return Q40_E_UNSUPPORTED; }
  const int64_t blocks = (int64_t)a.H * ((a.S + 2 * BQ - 1) / (2 * BQ));
  if (blocks > 0x7fffffffLL) return Q40_E_SHAPE;
  e = q40_launch_pdl(attn_window_tc_kernel, dim3((unsigned)blocks, a.splits), dim3(THREADS), SMEM, st, a, maps, err);
  const int64_t rows = (int64_t)a.S * a.H;
  if (e == cudaSuccess && a.splits > 1) e = q40_launch_pdl(tc::attn_window_merge_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, st, a, rows);
  return e == cudaSuccess ? Q40_OK : (int)e;
}

}  // namespace window
}  // namespace q40
