// Append of new tokens' keys and values to a paged cache, with the rotary embedding of keys and queries on the way: what
// q40_rope_kv_append does for the Q4_0 cache, for the pages that q40_attn_paged and q40_attn_pages read.  A token's place comes
// from the positions on the device, so that a captured step can be replayed.
//
// A rotated value is x c - y s of fp16 values and tables: products are exact in fp32, their sum rounds once, and once more to fp16 where it
// is kept in fp16 (q40_rope rounds each product too, which is the reference's order for its own cache).
//
// 8 bits: a page's scale is the largest magnitude in it over the largest code.  New rows may raise it; the page's earlier
// rows are then coded anew (code * old / new, rounded again).  A page whose first slot is written starts without one.  A value that is
// not finite makes its page's scale NaN, which whoever reads the page sees, until the page is begun anew.
//
// What bounds it: one token, a chain of four loads (position, page, scale or tables, store; 2.1 us with a launch); prompts, HBM: 4001 tokens of 96 heads in fp16
// 33.0 us, 6.0 TB/s, 8191 of 64 + 2 x 8 heads into int8 pages of 64 56.7 us, 5.7 TB/s (with one head a lane group 83, pages behind the queries 65; its four heads a lane group at eight CTAs an SM spill 44 bytes a thread).
#include "pages_common.cuh"

namespace q40 {
namespace append {

struct Args {
  PageTable tbl;
  int width;               // entries of a sequence's row of the table
  int pages;               // of the pool
  const int32_t* pos;      // [B] of a sequence's first new token
  const int32_t* offsets;  // [B + 1] rows of each sequence's new tokens, or nullptr: row b is sequence b's one token
  const __half *q, *k, *v;
  __half* q_out;           // [T, H * 128]
  int64_t q_stride, k_stride, v_stride;
  const __half *cos_tbl, *sin_tbl;
  int n_pos;
  void *kpool, *vpool;     // [Hkv, P, 128]
  float *k_scale, *v_scale;
  int64_t P;
  int B, T, H, Hkv;
  unsigned page_blocks;    // of the 8-bit launch: blocks in front that have a page; the others rotate queries
};

constexpr int THREADS = 128;
constexpr int EACH = 4;                   // heads of a lane group in large calls
constexpr int64_t MANY = 32768;           // ... of more rows than these: fewer would not fill the SMs with a quarter of the lane groups
constexpr int MOST_ROWS = 1 << 26;        // of a page in 8 bits: its earlier rows are counted through in pieces of 8 bytes, 16 a row, in 32 bits
constexpr int UNITS = THREADS / 8;        // rows of 128 values of a block's pass, eight lanes each

// The last i of [0, n) whose first(i) is not above x (0 where there is none)
template <class F>
__device__ __forceinline__ int last_not_above(int n, int64_t x, F first) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first(mid) <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Sequence and position of row t; false: it belongs to none, or lies in front of the first position
__device__ __forceinline__ bool token_of(const Args& a, int t, int& seq, int64_t& at) {
  if (!a.offsets) {
    seq = t;
    at = a.pos[t];
    return at >= 0;
  }
  seq = last_not_above(a.B, t, [&](int i) { return a.offsets[i]; });
  const int first = a.offsets[seq];
  at = (int64_t)a.pos[seq] + t - first;
  return t >= first && t < a.offsets[seq + 1] && at >= 0;
}

// Page id of a position, or -1 where the table or the pool has none
__device__ __forceinline__ int page_id(const Args& a, int seq, int64_t page) {
  if (page >= a.width) return -1;
  const int id = a.tbl.id(seq, (int)page);
  return (unsigned)id < (unsigned)a.pages ? id : -1;
}

struct Row { float lo[8], hi[8]; };       // of lane i: dims 8i .. 8i + 7 and 64 + 8i ..

__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 x = __half22float2(u32_as_h2(w[j]));
    f[2 * j] = x.x;
    f[2 * j + 1] = x.y;
  }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = h2_as_u32(__floats2half2_rn(f[2 * j], f[2 * j + 1]));
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ Row load_row(const __half* x, int i) {
  Row r;
  unpack8(*reinterpret_cast<const uint4*>(x + 8 * i), r.lo);
  unpack8(*reinterpret_cast<const uint4*>(x + 64 + 8 * i), r.hi);
  return r;
}
struct Turn { float c[8], s[8]; };        // of a position, lane i's
__device__ __forceinline__ Turn turn_of(const Args& a, int64_t at, int i) {
  const int64_t p = at < a.n_pos ? at : a.n_pos - 1;
  Turn t;
  unpack8(*reinterpret_cast<const uint4*>(a.cos_tbl + p * 64 + 8 * i), t.c);
  unpack8(*reinterpret_cast<const uint4*>(a.sin_tbl + p * 64 + 8 * i), t.s);
  return t;
}
__device__ __forceinline__ void rotate(Row& r, const Turn& t) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = r.lo[j], y = r.hi[j];
    r.lo[j] = fmaf(x, t.c[j], -(y * t.s[j]));
    r.hi[j] = fmaf(y, t.c[j], x * t.s[j]);
  }
}

// Heads [h, end) of token t's queries.  Several, so that a token's place and tables are looked up once for them: 8191 tokens of 64 heads
// 83 us with one, 60 with four, 61 with eight
template <int E>
__device__ __forceinline__ void rotate_queries(const Args& a, int t, int h, int end, int i) {
  const __half* const x = a.q + t * a.q_stride + 8 * i;
  __half* const out = a.q_out + (int64_t)t * a.H * ATTN_D + 8 * i;
  constexpr int U = E < 4 ? E : 4;
  int seq;
  int64_t at;
  const bool there = token_of(a, t, seq, at);                     // else zeros
  const Turn turn = turn_of(a, there ? at : 0, i);
#pragma unroll 1
  for (int h0 = h; h0 < end; h0 += U) {
    uint4 lo[U], hi[U];
#pragma unroll
    for (int e = 0; e < U; ++e) {
      const int at_h = min(h0 + e, end - 1) * ATTN_D;
      lo[e] = *reinterpret_cast<const uint4*>(x + at_h);
      hi[e] = *reinterpret_cast<const uint4*>(x + at_h + 64);
    }
#pragma unroll
    for (int e = 0; e < U; ++e) {
      if (h0 + e >= end) break;
      Row r;
      unpack8(lo[e], r.lo);
      unpack8(hi[e], r.hi);
      rotate(r, turn);
      *reinterpret_cast<uint4*>(out + (h0 + e) * ATTN_D) = there ? pack8(r.lo) : make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(out + (h0 + e) * ATTN_D + 64) = there ? pack8(r.hi) : make_uint4(0, 0, 0, 0);
    }
  }
}

// Heads [h, end) of token t's keys, then values, into fp16 pools
template <int E>
__device__ __forceinline__ void append_heads(const Args& a, int t, int h, int end, int i) {
  int seq;
  int64_t at;
  if (!token_of(a, t, seq, at)) return;
  const int64_t page = at / a.tbl.page_size;
  const int id = page_id(a, seq, page);
  if (id < 0) return;
  const int64_t slot = (int64_t)id * a.tbl.page_size + (at - page * a.tbl.page_size);
  if (slot >= a.P) return;                                        // a pool may end inside its last page
  Turn turn = {};
  if (a.cos_tbl && h < a.Hkv) turn = turn_of(a, at, i);
  constexpr int U = E < 4 ? E : 4;
#pragma unroll 1
  for (int h0 = h; h0 < end; h0 += U) {
    uint4 lo[U], hi[U];
#pragma unroll
    for (int e = 0; e < U; ++e) {
      const int he = min(h0 + e, end - 1);
      const __half* const x = (he < a.Hkv ? a.k + t * a.k_stride + he * ATTN_D : a.v + t * a.v_stride + (he - a.Hkv) * ATTN_D) + 8 * i;
      lo[e] = *reinterpret_cast<const uint4*>(x);
      hi[e] = *reinterpret_cast<const uint4*>(x + 64);
    }
#pragma unroll
    for (int e = 0; e < U; ++e) {
      const int he = h0 + e;
      if (he >= end) break;
      const bool is_k = he < a.Hkv;
      if (is_k && a.cos_tbl) {
        Row r;
        unpack8(lo[e], r.lo);
        unpack8(hi[e], r.hi);
        rotate(r, turn);
        lo[e] = pack8(r.lo);
        hi[e] = pack8(r.hi);
      }
      __half* const out = reinterpret_cast<__half*>(is_k ? a.kpool : a.vpool) + ((int64_t)(is_k ? he : he - a.Hkv) * a.P + slot) * ATTN_D + 8 * i;
      *reinterpret_cast<uint4*>(out) = lo[e];
      *reinterpret_cast<uint4*>(out + 64) = hi[e];
    }
  }
}

// fp16 pools.  Eight lanes take E heads of a token: of its queries, or of its keys and values
template <int E>
__global__ void __launch_bounds__(THREADS)
page_append_kernel(const Args a, int64_t units) {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");              // nothing of the previous launch is read before it is done
  const int64_t unit = (int64_t)blockIdx.x * UNITS + (threadIdx.x >> 3);
  const int i = threadIdx.x & 7;
  if (unit >= units) return;
  const int nq = (a.H + E - 1) / E, n = nq + (2 * a.Hkv + E - 1) / E, t = (int)(unit / n), part = (int)(unit - (int64_t)t * n);
  if (part < nq) rotate_queries<E>(a, t, part * E, min((part + 1) * E, a.H), i);
  else append_heads<E>(a, t, (part - nq) * E, min((part - nq + 1) * E, 2 * a.Hkv), i);
}

// Eight values as codes of scale 1 / inv
template <int T>
__device__ __forceinline__ uint2 code8(const float (&f)[8], float inv) {
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const float x = f[j] * inv, y = f[j + 1] * inv;
    uint32_t two;
    if (T == CACHE_I8) {
      const int cx = __float2int_rn(fminf(fmaxf(x, -127.f), 127.f)), cy = __float2int_rn(fminf(fmaxf(y, -127.f), 127.f));
      two = (cx & 0xff) | ((cy & 0xff) << 8);
    } else {
      two = __nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, __NV_E4M3);
    }
    w[j >> 2] |= two << (8 * (j & 2));
  }
  return make_uint2(w[0], w[1]);
}
template <int T>
__device__ __forceinline__ uint2 recode8(uint2 c, float ratio) {
  float f[8];
  const uint32_t w[2] = {c.x, c.y};
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if (T == CACHE_I8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[4 * j + i] = (float)(int8_t)(w[j] >> (8 * i));
    } else {
      const uint2 h = e4m3_to_h4(w[j]);
      const float2 x = __half22float2(u32_as_h2(h.x)), y = __half22float2(u32_as_h2(h.y));
      f[4 * j] = x.x; f[4 * j + 1] = x.y; f[4 * j + 2] = y.x; f[4 * j + 3] = y.y;
    }
  }
  return code8<T>(f, ratio);
}

// 8-bit pools.  The first blocks, which take longest, have a page of a sequence and a kv head each: the first two warps its keys, the others its
// values.  A sequence whose new rows are [o, e) touches at most (e - o) / page_size + 2 pages, so that its blocks can begin at
// o / page_size + 2 * sequence, and nobody counts pages.
template <int T, int E>
__global__ void __launch_bounds__(THREADS, E > 1 ? 8 : 7)
page_append_8bit_kernel(const Args a) {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int i = threadIdx.x & 7;
  if (blockIdx.x >= a.page_blocks) {
    const int64_t unit = (int64_t)(blockIdx.x - a.page_blocks) * UNITS + (threadIdx.x >> 3);
    const int nq = (a.H + E - 1) / E, part = (int)(unit % nq);
    if (unit < (int64_t)a.T * nq) rotate_queries<E>(a, (int)(unit / nq), part * E, min((part + 1) * E, a.H), i);
    return;
  }
  const unsigned block = blockIdx.x;
  const int h = (int)(block % a.Hkv), ps = a.tbl.page_size;
  const int64_t unit = block / a.Hkv;
  int seq, first, end;                     // the sequence's new rows
  int64_t at, page;                        // position of the first of them, page of this block
  if (!a.offsets) {
    seq = first = (int)unit;
    end = first + 1;
    at = a.pos[seq];
    page = at / ps;
  } else {
    seq = last_not_above(a.B, unit, [&](int s) { return (int64_t)max(a.offsets[s], 0) / ps + 2 * (int64_t)s; });
    first = max(a.offsets[seq], 0);
    end = min(a.offsets[seq + 1], a.T);
    at = a.pos[seq];
    page = (at < 0 ? 0 : at / ps) + (unit - (first / ps + 2 * (int64_t)seq));
  }
  // this page's new rows: slots [from, to) of it.  Positions before the first are not written
  const int64_t from_at = max(max(at, page * ps), (int64_t)0), to_at = min(at + end - first, (page + 1) * ps);
  if (from_at >= to_at) return;
  const int id = page_id(a, seq, page);
  if (id < 0) return;
  const int from = (int)(from_at - page * ps), n = (int)(to_at - from_at), row0 = first + (int)(from_at - at);
  const bool is_k = threadIdx.x < 64;
  const int group = (threadIdx.x >> 3) & 7;                       // of the eight that share the rows
  const __half* const x = is_k ? a.k + (int64_t)row0 * a.k_stride + h * ATTN_D : a.v + (int64_t)row0 * a.v_stride + h * ATTN_D;
  const int64_t ld = is_k ? a.k_stride : a.v_stride;
  float* const scale_at = (is_k ? a.k_scale : a.v_scale) + (int64_t)h * a.pages + id;
  const float old = from == 0 ? 0.f : *scale_at;

  const auto value = [&](int j) {
    Row r = load_row(x + j * ld, i);
    if (is_k && a.cos_tbl) rotate(r, turn_of(a, from_at + j, i));
    return r;
  };
  unsigned most = 0;                       // bits of the largest magnitude; what is not finite is above all that is
  Row kept = {};
  for (int j = group; j < n; j += 8) {
    const Row r = value(j);
    if (j == group) kept = r;
#pragma unroll
    for (int d = 0; d < 8; ++d) most = max(most, max(__float_as_uint(fabsf(r.lo[d])), __float_as_uint(fabsf(r.hi[d]))));
  }
  most = __reduce_max_sync(0xffffffffu, most);
  __shared__ unsigned sm_most[4];
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) sm_most[warp] = most;
  __syncthreads();                         // (the old scale has been read)
  most = max(sm_most[warp & 2], sm_most[(warp & 2) + 1]);
  const bool finite = most < 0x7f800000u && old <= 3.402823466e38f;
  const float now = finite ? fmaxf(old, __uint_as_float(most) * cache_top_inv<T>) : CUDART_NAN_F;
  const float inv = now > 0.f ? __frcp_rn(now) : 0.f;
  if ((threadIdx.x & 63) == 0) *scale_at = now;

  uint8_t* const rows = reinterpret_cast<uint8_t*>(is_k ? a.kpool : a.vpool) + ((int64_t)h * a.P + (int64_t)id * ps) * ATTN_D;
  if (now > old && from > 0) {             // the page's earlier rows
    const float ratio = old * inv;
#pragma unroll 4
    for (int e = threadIdx.x & 63; e < from * 16; e += 64) {
      uint2* const c = reinterpret_cast<uint2*>(rows) + e;
      *c = recode8<T>(*c, ratio);
    }
  }
  for (int j = group; j < n; j += 8) {
    const Row r = j == group ? kept : value(j);
    uint2* const out = reinterpret_cast<uint2*>(rows + (int64_t)(from + j) * ATTN_D) + i;
    out[0] = code8<T>(r.lo, inv);
    out[8] = code8<T>(r.hi, inv);
  }
}

}  // namespace append
}  // namespace q40

extern "C" int q40_page_append(const void* page_tbl, int idx_bytes, int64_t tbl_stride, int tbl_width, const int32_t* pos,
                               const int32_t* offsets, const void* q, int64_t q_stride, void* q_out, const void* k, int64_t k_stride,
                               const void* v, int64_t v_stride, const void* cos_tbl, const void* sin_tbl, int n_pos, void* kpool,
                               void* vpool, float* k_scale, float* v_scale, int cache_type, int64_t P, int B, int T, int H, int Hkv, int D,
                               int page_size, void* stream) {
  using namespace q40;
  using namespace q40::append;
  if (!page_tbl || !pos || !k || !v || !kpool || !vpool || !cos_tbl != !sin_tbl || !q != !q_out) return Q40_E_NULL;
  if (cache_type != CACHE_F16 && (!k_scale || !v_scale)) return Q40_E_NULL;
  if (q && !cos_tbl) return Q40_E_NULL;                           // queries come to be rotated
  if (D != ATTN_D || (idx_bytes != 2 && idx_bytes != 4) || cache_type < CACHE_F16 || cache_type > CACHE_E4M3) return Q40_E_UNSUPPORTED;
  if (!q) H = 0;
  if (B < 0 || T < 0 || (q && H <= 0) || Hkv <= 0 || page_size <= 0 || P <= 0 || tbl_width <= 0 || tbl_stride < tbl_width) return Q40_E_SHAPE;
  if (!offsets && T != B) return Q40_E_SHAPE;
  if (cos_tbl && n_pos <= 0) return Q40_E_SHAPE;
  if (cache_type != CACHE_F16 && (P % page_size != 0 || page_size > MOST_ROWS)) return Q40_E_SHAPE;
  const int64_t pages = (P + page_size - 1) / page_size;
  if (pages > 0x7fffffffLL) return Q40_E_SHAPE;
  if (k_stride < (int64_t)Hkv * D || v_stride < (int64_t)Hkv * D || (q && q_stride < (int64_t)H * D)) return Q40_E_SHAPE;
  if (k_stride % 8 != 0 || v_stride % 8 != 0 || (q && q_stride % 8 != 0)) return Q40_E_ALIGN;
  if (!q40_aligned(page_tbl, idx_bytes) || !q40_aligned(pos, 4) || !q40_aligned(offsets, 4) || !q40_aligned(k_scale, 4) || !q40_aligned(v_scale, 4))
    return Q40_E_ALIGN;
  if (!q40_aligned(q, 16) || !q40_aligned(q_out, 16) || !q40_aligned(k, 16) || !q40_aligned(v, 16) || !q40_aligned(cos_tbl, 16) ||
      !q40_aligned(sin_tbl, 16) || !q40_aligned(kpool, 16) || !q40_aligned(vpool, 16))
    return Q40_E_ALIGN;
  if (B == 0 || T == 0) return Q40_OK;
  Args a{};
  a.tbl = {page_tbl, tbl_stride, idx_bytes == 4, page_size, page_shift_of(page_size)};
  a.width = tbl_width; a.pages = (int)pages; a.pos = pos; a.offsets = offsets;
  a.q = (const __half*)q; a.k = (const __half*)k; a.v = (const __half*)v; a.q_out = (__half*)q_out;
  a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride;
  a.cos_tbl = (const __half*)cos_tbl; a.sin_tbl = (const __half*)sin_tbl; a.n_pos = n_pos;
  a.kpool = kpool; a.vpool = vpool; a.k_scale = k_scale; a.v_scale = v_scale; a.P = P;
  a.B = B; a.T = T; a.H = H; a.Hkv = Hkv;
  const cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  // one head a lane group while that leaves few of them: a decode step is over when its longest chain of loads is
  const bool many = (int64_t)T * (H + 2 * Hkv) > MANY;
  const int each = many ? EACH : 1, nq = (H + each - 1) / each;
  if (cache_type == CACHE_F16) {
    const int64_t units = (int64_t)T * (nq + (2 * Hkv + each - 1) / each), blocks = (units + UNITS - 1) / UNITS;
    if (blocks > 0x7fffffffLL) return Q40_E_SHAPE;
    e = q40_launch_pdl(many ? page_append_kernel<EACH> : page_append_kernel<1>, dim3((unsigned)blocks), dim3(THREADS), 0, st, a, units);
  } else {
    const int64_t qb = ((int64_t)T * nq + UNITS - 1) / UNITS, units = offsets ? T / page_size + 2 * (int64_t)B : B;
    if (qb + units * Hkv > 0x7fffffffLL) return Q40_E_SHAPE;
    a.page_blocks = (unsigned)(units * Hkv);
    const dim3 grid((unsigned)(qb + units * Hkv));
    const auto kernel = cache_type == CACHE_I8 ? (many ? page_append_8bit_kernel<CACHE_I8, EACH> : page_append_8bit_kernel<CACHE_I8, 1>)
                                               : (many ? page_append_8bit_kernel<CACHE_E4M3, EACH> : page_append_8bit_kernel<CACHE_E4M3, 1>);
    e = q40_launch_pdl(kernel, grid, dim3(THREADS), 0, st, a);
  }
  return e == cudaSuccess ? Q40_OK : (int)e;
}
