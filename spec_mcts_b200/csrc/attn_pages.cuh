// Attention of one query token per sequence over a paged cache of fp16 or of 8-bit codes with a scale for each page and kv head,
// with all keys visible, or the last `window` and the first `sinks`.
//
// The visible keys of a sequence are numbered through (first ones, then the window), so that a window costs nothing but the look-up of
// a key's place, and masked keys are never read.  A unit is a sequence and up to eight query heads of one kv head, whose keys and values are
// read once for all of them; its keys go to CTAs in chunks, whose size goes by the number of keys and of units alone (chunk_of), so that
// results do not depend on how long the tables are.  A unit of one chunk writes its output; the partial results of several meet in page_merge_kernel.
//
// A warp takes 16 keys at a time, of 8-bit ones 32, through a ring of its own (cp.async):
//   scores   A = 16 keys, B = the queries: columns 2i and 2i + 1 are head i's (of two heads, 4i .. 4i + 3; of one, all; of eight, one each)
//   output   A = 16 values transposed, B = the weights, each as two fp16 parts (weight_parts): a head's two columns, or, of eight
//            heads, two products
// Lane (g, t) has the scores of keys g and g + 8.  A key's scale multiplies its score; a value's, vs, its weight, as 2^(s + log2 vs - m),
// where m is the largest s + log2 vs: the weights of the values, and not those of the scores, have to fit in fp16.
//
// What bounds it: many keys, HBM (64 sequences of up to 2048 e4m3 keys of 32 heads 124 us, 6.5 TB/s; 100 windows of 4096 fp16 keys of 8 heads 243 us, 6.9 TB/s), at the
// power limit instructions (18 a key of one head, 39 of eight); few units of eight heads, neither (8 x 65536 int8 keys under 64 heads 158 us where HBM takes 129: at 8 x 16384 issue slots are 54 %
// busy, and a warp, whose ring has one stage, does not copy while it computes); few keys, a warp's chain of 1 us per 32 of them (512 int8 keys of 32 heads 5.9 us, 2000 9.7).
#pragma once
#include <algorithm>
#include <type_traits>

#include "attn_tile.cuh"
#include "pages_common.cuh"
#include "tanh_cap.cuh"

namespace q40 {
namespace pages {

constexpr int MERGE_THREADS = 128;
// Warps of a CTA: eight with one stage of their ring while the units are no more than the SMs, else four with two.  Us, eight / four: 1 x 500 int8 keys of 8 heads
// 5.7 / 6.7, 8 x 500 6.0 / 6.7, 8 x 2000 11.1 / 13.0, 64 units of up to 65536 157 / 152 (four would be better for these, but lengths are not known here, and a table's width is not to decide); fp16 1 x 2000 of 32 heads 9.3 / 10.5.  Eight with two stages (one CTA an SM) 1 x
// 30000 30 where one has 26
constexpr int FEW = 148;                   // units
// Keys of a chunk: one wave of CTAs (two an SM), if that leaves chunks of up to 2048 keys, else about 1200 CTAs, whose chunks even out lengths.  Us: 1 x 30000 keys of
// 8 heads in 30 chunks of 1024 19.9, in 59 of 512 26; 100 x 4100 x 8 heads in chunks for 600 / 1200 / 2400 / 4800 / 9600 CTAs 240 / 240 / 252 / 260 / 268, 64 x 2048 x 32 heads
// 122 / 122 / 122 / 133 / 144.  A second chunk costs a launch, 2 to 3 us: 256 keys of 1 x 500 8.0, 512 6.7
constexpr int CHUNK_MIN = 512, CHUNK_MAX = 8192;
constexpr int CHUNK_WAVE = 2048;
constexpr int64_t MOST_CHUNKS = 65535;     // of a unit, as the grid has it: behind 8192 x 65535 keys chunks are of 16384
constexpr int64_t WAVE = 296, CTAS = 1200; // CTAs that a call is cut into, about: one wave of them, where that leaves chunks of up to CHUNK_WAVE

struct Args {
  const __half* q;         // sequence b, head h at q + b * q_stride + h * 128
  int64_t q_stride;
  const void *k, *v;       // [Hkv, P, 128]
  const float *ks, *vs;    // [Hkv, pages]
  __half* o;               // [B, H, 128]
  PageTable tbl;
  const int32_t* seq_lens;
  int last_page, pages;
  int64_t P;
  int B, L, H, Hkv, window, sinks;
  int groups, heads;       // of a kv head's query heads; heads of a group (the last may have fewer)
  int64_t units;
  int nchunks;             // most of a unit
  float* po;               // [units][nchunks][heads][128], not normalised
  float2* pml;             // ... maximum (log2) and sum
  float scale_log2;
};

// ... and what becomes of scores: capped by a tanh (unless cap_out is 0), less what the distance to the query costs (unless slopes is NULL)
struct ScoreArgs : Args {
  const float* slopes;     // [H]
  float cap_limit, cap_exp, cap_out, cap_k[5];
};
template <bool SCORES>
using Call = std::conditional_t<SCORES, ScoreArgs, Args>;

template <int T>
constexpr int row_bytes = ATTN_D * cache_bytes<T>;
template <int T>
constexpr int keys_of = T == CACHE_F16 ? 16 : 32;         // of a stage: 8 KB
template <int T>
constexpr int stage_bytes = 2 * keys_of<T> * row_bytes<T> + (T == CACHE_F16 ? 0 : 2 * keys_of<T> * 4);
template <int T, int G, int S>
constexpr int warp_bytes = S * stage_bytes<T> > G * ATTN_D * 4 ? S * stage_bytes<T> : G * ATTN_D * 4;

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 r;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(addr));
  return r;
}
__device__ __forceinline__ float lds32(uint32_t addr) {
  float r;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool pred) {
  const int sz = pred ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(sz));
}

// Keys of a chunk for a unit of n keys, by its own length and the number of units alone
__host__ __device__ __forceinline__ int chunk_of(int64_t n, int64_t units) {
  int chunk = CHUNK_MIN;
  const int64_t wave = WAVE / units, all = CTAS > units ? CTAS / units : 1;
  while (chunk < CHUNK_WAVE && chunk * wave < n) chunk *= 2;
  if (wave > 1 && chunk * wave >= n) return chunk;
  chunk = CHUNK_MIN;
  while ((chunk < CHUNK_MAX && chunk * all < n) || chunk * MOST_CHUNKS < n) chunk *= 2;
  return chunk;
}

// Visible keys of a sequence: number n; key i of them is position i below `first`, then i + skip
struct Visible {
  int n, first, skip;
  __device__ __forceinline__ Visible(const Args& a, int b) {
    const int len = a.seq_lens ? min(max(a.seq_lens[b], 0), a.L) : a.L;
    const int lo = a.window > 0 ? max(len - a.window, 0) : 0;
    first = min(a.sinks, lo);
    skip = lo - first;
    n = len - skip;
  }
};

// weight_parts for two products into one sum: neither part is 0 or negative, so that an infinite value comes out as it is (2^-24 more
// than the weight is 2^-38 of the largest one)
__device__ __forceinline__ uint32_t weight_parts_of_one_sum(float p) {
  const __half least = __ushort_as_half(1), h = __hmax_nan(__float2half_rz(p), least);
  return h2_as_u32(__halves2half2(h, __hmax_nan(__float2half_rn(p - __half2float(h)), least)));
}

// Four codes as two pairs of halves
template <int T>
__device__ __forceinline__ uint2 halves_of(uint32_t w) {
  return T == CACHE_I8 ? make_uint2(i8_to_h2(prmt(w, 0x64646464u, 0x4140)), i8_to_h2(prmt(w, 0x64646464u, 0x4342))) : e4m3_to_h4(w);
}
template <int T>
__device__ __forceinline__ uint32_t biased(uint32_t w) { return T == CACHE_I8 ? w ^ 0x80808080u : w; }
// base + i * size in one instruction
__device__ __forceinline__ const unsigned char* row_at(const unsigned char* base, int i, int size) {
  const unsigned char* r;
  asm("mad.wide.s32 %0, %1, %2, %3;" : "=l"(r) : "r"(i), "r"(size), "l"(base));
  return r;
}

// c tanh(s / c) of scores times log2(e): a polynomial while all of a warp's are in its range, else 1 - 2 / (1 + e^2x)
template <int N>
__device__ __forceinline__ void cap(const ScoreArgs& a, float (&s)[N]) {
  float big = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) big = fmaxf(big, fabsf(s[i]));
  if (__any_sync(0xffffffffu, big > a.cap_limit)) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = tanh_by_exp(s[i] * a.cap_exp) * a.cap_out;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] *= tanh_poly(s[i] * s[i], a.cap_k);
  }
}

template <bool SCORES, int T, int G, int S, int NW>
__global__ void __launch_bounds__(NW * 32)
attn_pages_kernel(const Call<SCORES> a) {
  constexpr int D = ATTN_D, RB = row_bytes<T>, KEYS = keys_of<T>, MT = KEYS / 16;
  constexpr int GL = G == 4 ? 0 : G == 2 ? 1 : 2;        // up to four heads: lane t works for head t >> GL
  constexpr int HL = G == 8 ? 2 : 1;                     // heads of a lane
  constexpr int LPR = RB / 16, RPI = 32 / LPR;           // lanes that copy a row, rows a copy instruction
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3, mi = lane >> 3;
  const int unit = blockIdx.x, chunk = blockIdx.y;
  const int group = unit % a.groups, hk = unit / a.groups % a.Hkv, b = unit / a.groups / a.Hkv;
  const int rep = a.H / a.Hkv, h0 = hk * rep + group * a.heads, heads = min(a.heads, rep - group * a.heads);
  const Visible vis(a, b);
  const int size = chunk_of(vis.n, a.units);
  const int64_t begin64 = (int64_t)chunk * size;
  if (begin64 >= vis.n && chunk > 0) return;
  const int begin = (int)begin64, end = (int)min((int64_t)vis.n, begin64 + size);

  extern __shared__ __align__(128) unsigned char rings[];
  constexpr int WB = warp_bytes<T, G, S>;
  const uint32_t ring = smem_u32(rings + warp * WB);
  const unsigned char* const kb = reinterpret_cast<const unsigned char*>(a.k) + (int64_t)hk * a.P * RB + (lane % LPR) * 16;
  const unsigned char* const vb = reinterpret_cast<const unsigned char*>(a.v) + (int64_t)hk * a.P * RB + (lane % LPR) * 16;
  const float *const ks = a.ks + (int64_t)hk * a.pages, *const vs = a.vs + (int64_t)hk * a.pages;

  // place of the keys from i0 on, one a lane (16 keys: again in lanes 16 to 31), looked up one request ahead
  struct Place { int page, slot; };
  const auto place_of = [&](int i0) {
    Place p = {0, 0};
    const int i = i0 + (lane & (KEYS - 1));
    if (i < end) {
      const int pos = i < vis.first ? i : i + vis.skip, pg = a.tbl.page_of(pos);
      // a bad page id must not turn into a wild read: clamp into the pool
      p.page = min(max(a.tbl.id(b, pg), 0), a.last_page);
      p.slot = (int)min((int64_t)p.page * a.tbl.page_size + (pos - pg * a.tbl.page_size), a.P - 1);
    }
    return p;
  };
  const auto request = [&](int i0, int stage, const Place& p) {
    const uint32_t kt = ring + stage * stage_bytes<T>, vt = kt + KEYS * RB;
#pragma unroll
    for (int j = 0; j < KEYS / RPI; ++j) {
      const int r = j * RPI + lane / LPR;
      const bool ok = i0 + r < end;
      const int slot = __shfl_sync(0xffffffffu, p.slot, r);
      const uint32_t at = r * RB + (((lane % LPR) ^ (r & 7)) << 4);
      cp_async16(kt + at, row_at(kb, slot, RB), ok);
      cp_async16(vt + at, row_at(vb, slot, RB), ok);
    }
    if (T != CACHE_F16) {
      static_assert(T == CACHE_F16 || KEYS == 32, "a lane copies the scales of one key");
      const bool ok = i0 + lane < end;
      cp_async4(vt + KEYS * RB + lane * 4, ks + p.page, ok);
      cp_async4(vt + KEYS * RB + KEYS * 4 + lane * 4, vs + p.page, ok);
    }
  };
  constexpr int STEP = NW * KEYS;
  const int mine = begin + warp * KEYS;
  Place next = place_of(mine);
#pragma unroll
  for (int i = 0; i < S; ++i) {
    if (mine + i * STEP < end) request(mine + i * STEP, i, next);
    cp_async_commit();
    next = place_of(mine + (i + 1) * STEP);
  }

  // B fragments of the queries.  fp16: k of step ks are dims 16 ks + 2t, + 1, + 8, + 9 (ldmatrix); codes: 32 t + 4 ks .. + 3, so that a
  // lane reads whole words of its keys
  uint32_t qb[8][2];
  {
    const int head = min(G == 8 ? g : (g >> 1) >> GL, heads - 1);
    const __half* const q = a.q + b * a.q_stride + (int64_t)(h0 + head) * D;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (T == CACHE_F16) {
        qb[i][0] = *reinterpret_cast<const uint32_t*>(q + 16 * i + 2 * t);
        qb[i][1] = *reinterpret_cast<const uint32_t*>(q + 16 * i + 8 + 2 * t);
      } else {
        const uint2 w = *reinterpret_cast<const uint2*>(q + 32 * t + 4 * i);
        qb[i][0] = w.x;
        qb[i][1] = w.y;
      }
    }
  }
  float slope[HL];                               // of the lane's heads, log2
  int newest = 0;                                // the query's position: that of the last key
  float skip = 0.f;
  if constexpr (SCORES) {
#pragma unroll
    for (int j = 0; j < HL; ++j) slope[j] = a.slopes ? a.slopes[h0 + min(HL == 2 ? 2 * t + j : t >> GL, heads - 1)] * 1.44269504f : 0.f;
    newest = vis.n - 1 + vis.skip;
    skip = (float)vis.skip;
  }
  float m[HL], l[HL], acc[8][4];
#pragma unroll
  for (int j = 0; j < HL; ++j) { m[j] = NO_KEY; l[j] = 0.f; }
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;

  int stage = 0;
#pragma unroll 1
  for (int i0 = mine; i0 < end; i0 += STEP) {
    cp_async_wait<S - 1>();
    __syncwarp();
    const uint32_t kt = ring + stage * stage_bytes<T>, vt = kt + KEYS * RB;
    float x[MT][4], sc[2 * MT][HL], lv[2 * MT];    // scores, log2 of the values' scales of keys 8r + g
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float c0[4] = {0.f, 0.f, 0.f, 0.f}, c1[4] = {0.f, 0.f, 0.f, 0.f};
      if constexpr (T == CACHE_F16) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          uint32_t y[4], z[4];
          const int r = (lane & 7) + (mi & 1) * 8;
          ldsm_x4(kt + tile_off(r, 2 * i + (mi >> 1)), y[0], y[1], y[2], y[3]);
          ldsm_x4(kt + tile_off(r, 2 * i + 2 + (mi >> 1)), z[0], z[1], z[2], z[3]);
          mma_f16(c0, y[0], y[1], y[2], y[3], qb[i][0], qb[i][1]);
          mma_f16(c1, z[0], z[1], z[2], z[3], qb[i + 1][0], qb[i + 1][1]);
        }
      } else {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint32_t at = kt + (16 * mt + g) * RB + (((2 * t + c) ^ g) << 4);
          const uint4 y4 = lds128(at), z4 = lds128(at + 8 * RB);
          const uint32_t y[4] = {y4.x, y4.y, y4.z, y4.w}, z[4] = {z4.x, z4.y, z4.z, z4.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint2 u = halves_of<T>(biased<T>(y[w])), v = halves_of<T>(biased<T>(z[w]));
            mma_f16(w & 1 ? c1 : c0, u.x, v.x, u.y, v.y, qb[4 * c + w][0], qb[4 * c + w][1]);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) x[mt][j] = c0[j] + c1[j];
    }
    bool above = false;
    if constexpr (SCORES) {
      float s[2 * MT * HL];
#pragma unroll
      for (int r = 0; r < 2 * MT; ++r) {
        const float scale = T == CACHE_F16 ? a.scale_log2 : a.scale_log2 * lds32(vt + KEYS * RB + (8 * r + g) * 4);
#pragma unroll
        for (int j = 0; j < HL; ++j) s[HL * r + j] = x[r >> 1][2 * (r & 1) + j] * scale;
      }
      if (a.cap_out != 0.f) cap(a, s);
      if (a.slopes) {
        const float far = (float)(newest - vis.skip - i0 - g);       // of key g; another is 8 r nearer, a first key `skip` further away
#pragma unroll
        for (int r = 0; r < 2 * MT; ++r) {
          const float d = far - (float)(8 * r) + (i0 + 8 * r + g < vis.first ? skip : 0.f);
#pragma unroll
          for (int j = 0; j < HL; ++j) s[HL * r + j] = fmaf(-slope[j], d, s[HL * r + j]);
        }
      }
#pragma unroll
      for (int r = 0; r < 2 * MT; ++r)
#pragma unroll
        for (int j = 0; j < HL; ++j) x[r >> 1][2 * (r & 1) + j] = s[HL * r + j];
    }
#pragma unroll
    for (int r = 0; r < 2 * MT; ++r) {
      float scale = SCORES ? 1.f : a.scale_log2;
      lv[r] = 0.f;
      if (T != CACHE_F16) {
        if (!SCORES) scale *= lds32(vt + KEYS * RB + (8 * r + g) * 4);
        const float y = lg2(lds32(vt + KEYS * RB + KEYS * 4 + (8 * r + g) * 4));
        lv[r] = y < -60.f ? -60.f : y;           // a scale of 0: next to nothing.  NaN stays
      }
      const bool there = i0 + 8 * r + g < end;
#pragma unroll
      for (int j = 0; j < HL; ++j) {
        sc[r][j] = there ? x[r >> 1][2 * (r & 1) + j] * scale : -CUDART_INF_F;
        above |= sc[r][j] + lv[r] > m[j] + (WEIGHT_BITS + 1.f);
      }
    }
    // a maximum stays while no weight passes 2^(WEIGHT_BITS + 1), which fp16 holds
    if (__any_sync(0xffffffffu, above)) {
#pragma unroll
      for (int j = 0; j < HL; ++j) {
        float mnew = m[j];
#pragma unroll
        for (int r = 0; r < 2 * MT; ++r) mnew = fmaxf(mnew, sc[r][j] + lv[r] - WEIGHT_BITS);
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) mnew = fmaxf(mnew, __shfl_xor_sync(0xffffffffu, mnew, o));
        const float corr = ex2_some(m[j] - mnew);
        l[j] *= corr;
        m[j] = mnew;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          acc[i][j] *= corr;
          acc[i][2 + j] *= corr;
          if (HL == 1) { acc[i][1] *= corr; acc[i][3] *= corr; }
        }
      }
    }
    uint32_t bh[2 * MT], bl[2 * MT];             // B fragments of the weights' first and second parts
#pragma unroll
    for (int r = 0; r < 2 * MT; ++r) {
      uint32_t pk[HL];                           // both parts of a weight
#pragma unroll
      for (int j = 0; j < HL; ++j) {
        const float w = ex2(sc[r][j] + lv[r] - m[j]);
        l[j] += T == CACHE_F16 ? w : ex2(sc[r][j] - m[j]);
        pk[j] = HL == 1 ? weight_parts(w) : weight_parts_of_one_sum(w);
      }
      if (HL == 1) {
        bh[r] = movmatrix(pk[0]);
      } else {
        bh[r] = movmatrix(prmt(pk[0], pk[HL - 1], 0x5410));
        bl[r] = movmatrix(prmt(pk[0], pk[HL - 1], 0x7632));
      }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      if constexpr (T == CACHE_F16) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint32_t y[4];
          ldsm_x4_t(vt + tile_off((lane & 7) + (mi >> 1) * 8, 2 * i + (mi & 1)), y[0], y[1], y[2], y[3]);
          mma_f16(acc[i], y[0], y[1], y[2], y[3], bh[0], bh[1]);
          if (HL == 2) mma_f16(acc[i], y[0], y[1], y[2], y[3], bl[0], bl[1]);
        }
      } else {
        // keys 2t, 2t + 1 (y, z) and 2t + 8, 2t + 9 (u, v), dims 16 g ..: product i has dims 2i (rows g) and 2i + 1 (rows g + 8) of these
        const auto values = [&](int key) { return lds128(vt + (16 * mt + key) * RB + ((g ^ (key & 7)) << 4)); };
        const uint4 y4 = values(2 * t), z4 = values(2 * t + 1), u4 = values(2 * t + 8), v4 = values(2 * t + 9);
        const uint32_t y[4] = {y4.x, y4.y, y4.z, y4.w}, z[4] = {z4.x, z4.y, z4.z, z4.w}, u[4] = {u4.x, u4.y, u4.z, u4.w}, v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t by = biased<T>(y[w]), bz = biased<T>(z[w]), bu = biased<T>(u[w]), bv = biased<T>(v[w]);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint2 yz = halves_of<T>(prmt(by, bz, half ? 0x7362 : 0x5140)), uv = halves_of<T>(prmt(bu, bv, half ? 0x7362 : 0x5140));
            mma_f16(acc[2 * w + half], yz.x, yz.y, uv.x, uv.y, bh[2 * mt], bh[2 * mt + 1]);
            if (HL == 2) mma_f16(acc[2 * w + half], yz.x, yz.y, uv.x, uv.y, bl[2 * mt], bl[2 * mt + 1]);
          }
        }
      }
    }
    __syncwarp();
    if (i0 + S * STEP < end) request(i0 + S * STEP, stage, next);
    cp_async_commit();
    next = place_of(i0 + (S + 1) * STEP);
    if (++stage == S) stage = 0;
  }
#pragma unroll
  for (int j = 0; j < HL; ++j)
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], o);

  // behind the wait: see page_merge_kernel; and not before most of the work, since the next launch's CTAs take room from what is left of this one
  asm volatile("griddepcontrol.launch_dependents;");
  // the ring, which is empty, takes the warp's outputs
  __shared__ float sm_m[G][NW], sm_l[G][NW];
  float* const out = reinterpret_cast<float*>(rings + warp * WB);
  __syncwarp();
  if (lane < 4) {
    if (HL == 2) {
      sm_m[2 * t][warp] = m[0]; sm_l[2 * t][warp] = l[0];
      sm_m[(2 * t + 1) % G][warp] = m[HL - 1]; sm_l[(2 * t + 1) % G][warp] = l[HL - 1];
    } else if ((lane & ((1 << GL) - 1)) == 0) {
      sm_m[t >> GL][warp] = m[0]; sm_l[t >> GL][warp] = l[0];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d0 = T == CACHE_F16 ? 16 * i + g : 16 * g + 2 * i, d1 = T == CACHE_F16 ? d0 + 8 : d0 + 1;
    if (HL == 2) {
      out[2 * t * D + d0] = acc[i][0]; out[(2 * t + 1) * D + d0] = acc[i][1];
      out[2 * t * D + d1] = acc[i][2]; out[(2 * t + 1) * D + d1] = acc[i][3];
    } else if (GL == 0 || (i & ((1 << GL) - 1)) == (t & ((1 << GL) - 1))) {
      out[(t >> GL) * D + d0] = both_parts(acc[i][0], acc[i][1]);
      out[(t >> GL) * D + d1] = both_parts(acc[i][2], acc[i][3]);
    }
  }
  __syncthreads();
  const bool alone = vis.n <= size;
  const auto write = [&](int j, int d, float M, float Lsum, float x) {
    if (alone) {
      a.o[((int64_t)b * a.H + h0 + j) * D + d] = __float2half_rn(Lsum != 0.f ? x / Lsum : 0.f);
    } else {
      const int64_t at = ((int64_t)unit * a.nchunks + chunk) * a.heads + j;
      a.po[at * D + d] = x;
      if (d == 0) a.pml[at] = make_float2(M, Lsum);
    }
  };
  for (int i = tid; i < heads * D; i += NW * 32) {
    const int j = i / D;
    float M = NO_KEY, Lsum = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, sm_m[j][w]);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = ex2_some(sm_m[j][w] - M);
      Lsum = fmaf(sm_l[j][w], f, Lsum);
      x = fmaf(reinterpret_cast<const float*>(rings + w * WB)[i], f, x);
    }
    write(j, i % D, M, Lsum, x);
  }
}

// The partial results of units of several chunks, in the chunks' order; a CTA has a unit and one of its heads, a thread a dim.  The launch in
// front starts this one when what it waited for is there, so that lengths can be read before its results are
static __global__ void __launch_bounds__(MERGE_THREADS)
page_merge_kernel(const Args a) {
  constexpr int BATCH = 8;                       // chunks whose results are requested together
  const int unit = blockIdx.x / a.heads, j = blockIdx.x % a.heads, tid = threadIdx.x;
  const int group = unit % a.groups, hk = unit / a.groups % a.Hkv, b = unit / a.groups / a.Hkv;
  const int rep = a.H / a.Hkv;
  const Visible vis(a, b);
  const int size = chunk_of(vis.n, a.units), n = (vis.n - 1) / size + 1;
  const int64_t first = (int64_t)unit * a.nchunks * a.heads + j;
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (vis.n <= size || j >= rep - group * a.heads) return;
  float M = NO_KEY, x = 0.f, Lsum = 0.f;
  for (int c0 = 0; c0 < n; c0 += BATCH) {
    float2 ml[BATCH];
    float y[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int64_t at = first + (int64_t)(c0 + i) * a.heads;
      ml[i] = c0 + i < n ? a.pml[at] : make_float2(NO_KEY, 0.f);
      y[i] = c0 + i < n ? a.po[at * ATTN_D + tid] : 0.f;
    }
    float now = M;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) now = fmaxf(now, ml[i].x);
    const float corr = ex2_some(M - now);
    x *= corr;
    Lsum *= corr;
    M = now;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const float f = ex2_some(ml[i].x - M);
      Lsum = fmaf(ml[i].y, f, Lsum);
      x = fmaf(y[i], f, x);
    }
  }
  a.o[((int64_t)b * a.H + hk * rep + group * a.heads + j) * ATTN_D + tid] = __float2half_rn(Lsum != 0.f ? x / Lsum : 0.f);
}

struct Plan { int64_t units; int groups, heads, nchunks; };

static Plan plan_of(int B, int H, int Hkv, int L, int window, int sinks) {
  Plan p;
  const int rep = H / Hkv;
  p.groups = (rep + 7) / 8;
  p.heads = (rep + p.groups - 1) / p.groups;
  p.units = (int64_t)B * Hkv * p.groups;
  const int64_t most = window > 0 ? std::min<int64_t>(L, (int64_t)window + sinks) : L;      // visible keys
  // The most chunks that a unit of up to that many keys has.  While chunks are of one size, longer units have more of them; the size changes
  // behind multiples of one (chunk_of): there, or at the end
  int64_t n = 1;
  const auto at = [&](int64_t keys) {
    keys = std::min(keys, most);
    if (keys > 0) n = std::max(n, (keys + chunk_of(keys, p.units) - 1) / chunk_of(keys, p.units));
  };
  at(most);
  at(CHUNK_MAX * MOST_CHUNKS);
  for (int64_t chunk = CHUNK_MIN; chunk <= CHUNK_MAX; chunk *= 2) {
    at(chunk * (WAVE / p.units));
    at(chunk * std::max<int64_t>(1, CTAS / p.units));
  }
  p.nchunks = (int)std::min<int64_t>(n, 1 << 30);
  return p;
}

template <bool SCORES, int T, int G, int S, int NW>
static cudaError_t launch(const Call<SCORES>& a, int64_t units, cudaStream_t st) {
  static std::atomic<uint64_t> ready;
  constexpr int BYTES = NW * warp_bytes<T, G, S>;
  const cudaError_t e = q40_allow_smem(ready, (const void*)attn_pages_kernel<SCORES, T, G, S, NW>, BYTES);
  if (e != cudaSuccess) return e;
  return q40_launch_pdl(attn_pages_kernel<SCORES, T, G, S, NW>, dim3((unsigned)units, (unsigned)a.nchunks), dim3(NW * 32), BYTES, st, a);
}
template <bool SCORES, int T, int G>
static cudaError_t launch_warps(const Call<SCORES>& a, int64_t units, cudaStream_t st) {
  if (units <= FEW) return launch<SCORES, T, G, 1, 8>(a, units, st);
  return launch<SCORES, T, G, 2, 4>(a, units, st);
}
template <bool SCORES, int T>
static cudaError_t launch_heads(const Call<SCORES>& a, int64_t units, cudaStream_t st) {
  return a.heads > 4 ? launch_warps<SCORES, T, 8>(a, units, st) : a.heads > 2 ? launch_warps<SCORES, T, 4>(a, units, st)
         : a.heads > 1 ? launch_warps<SCORES, T, 2>(a, units, st) : launch_warps<SCORES, T, 1>(a, units, st);
}

// The checks of a call and what its kernels get; Q40_OK with a.B == 0: nothing is to be done
static int args_of(Args& a, const void* page_tbl, int idx_bytes, int64_t tbl_stride, const int32_t* seq_lens, const void* q, int64_t q_stride, const void* kpool,
                   const void* vpool, const float* k_scale, const float* v_scale, int cache_type, void* o, int64_t P, int B, int Lmax, int H, int Hkv, int D,
                   int page_size, int window, int sinks, void* workspace, size_t workspace_bytes) {
  if (!q || !o) return Q40_E_NULL;
  if (D != ATTN_D || (idx_bytes != 2 && idx_bytes != 4) || cache_type < CACHE_F16 || cache_type > CACHE_E4M3) return Q40_E_UNSUPPORTED;
  if (B < 0 || H <= 0 || Hkv <= 0 || H % Hkv != 0 || (int64_t)B * H > 0x7fffffffLL) return Q40_E_SHAPE;
  if (Lmax < 0 || Lmax > (1 << 29) || P < 0 || P > 0x7fffffffLL || page_size <= 0 || window < 0 || sinks < 0 || q_stride < (int64_t)H * D) return Q40_E_SHAPE;
  if (Lmax > 0 && (!page_tbl || !kpool || !vpool || P == 0 || (cache_type != CACHE_F16 && (!k_scale || !v_scale)))) return Q40_E_NULL;
  if (tbl_stride < ((int64_t)Lmax + page_size - 1) / page_size) return Q40_E_SHAPE;
  if (cache_type != CACHE_F16 && P % page_size != 0) return Q40_E_SHAPE;
  a.B = B;
  if (B == 0) return Q40_OK;
  if (!q40_aligned(q, 16) || q_stride % 8 != 0 || !q40_aligned(kpool, 16) || !q40_aligned(vpool, 16) || !q40_aligned(o, 2) ||
      !q40_aligned(k_scale, 4) || !q40_aligned(v_scale, 4) || !q40_aligned(page_tbl, idx_bytes) || !q40_aligned(seq_lens, 4))
    return Q40_E_ALIGN;
  const Plan p = plan_of(B, H, Hkv, Lmax, window, sinks);
  const int64_t parts = p.units * p.nchunks * p.heads;
  if (parts > 0x7fffffffLL || p.nchunks > MOST_CHUNKS) return Q40_E_SHAPE;
  if (p.nchunks > 1) {
    if (!workspace || workspace_bytes < (size_t)parts * (ATTN_D + 2) * sizeof(float)) return Q40_E_WORKSPACE;
    if (!q40_aligned(workspace, 16)) return Q40_E_ALIGN;
  }
  a.q = (const __half*)q; a.q_stride = q_stride; a.k = kpool; a.v = vpool; a.ks = k_scale; a.vs = v_scale; a.o = (__half*)o;
  a.tbl = {page_tbl, tbl_stride, idx_bytes == 4, page_size, page_shift_of(page_size)};
  a.seq_lens = seq_lens; a.P = P; a.last_page = P > 0 ? (int)((P - 1) / page_size) : 0; a.pages = (int)(P / page_size);
  a.L = Lmax; a.H = H; a.Hkv = Hkv; a.window = window; a.sinks = sinks;
  a.groups = p.groups; a.heads = p.heads; a.units = p.units; a.nchunks = p.nchunks;
  a.po = (float*)workspace; a.pml = (float2*)(a.po + parts * ATTN_D);
  a.scale_log2 = attn_scale_log2(D);
  return Q40_OK;
}

template <bool SCORES>
static int enqueue(const Call<SCORES>& a, int cache_type, cudaStream_t st) {
  cudaError_t e = cache_type == CACHE_F16 ? launch_heads<SCORES, CACHE_F16>(a, a.units, st)
                  : cache_type == CACHE_I8 ? launch_heads<SCORES, CACHE_I8>(a, a.units, st) : launch_heads<SCORES, CACHE_E4M3>(a, a.units, st);
  if (e == cudaSuccess && a.nchunks > 1) e = q40_launch_pdl(page_merge_kernel, dim3((unsigned)(a.units * a.heads)), dim3(MERGE_THREADS), 0, st, static_cast<const Args&>(a));
  return e == cudaSuccess ? Q40_OK : (int)e;
}

}  // namespace pages
}  // namespace q40

