// Attention of a prompt, or of a later chunk of one, with a sliding window and first keys that stay visible: query i, at position
// p = offset + i, attends the keys j <= p with p - j < window or j < sinks.
//
// Small calls: a CTA has 64 queries of one head, the blocks with most keys first, and goes through the tiles of 64 keys that one of its
// queries sees; the tile step is attn_causal_kernel's, with the window in the mask.
//
// A masked key has a weight of 0, and 0 times a value that is not finite is no number.  In a tile that some query sees in part, values
// that are not finite are therefore taken out in shared memory, and added at the end to the queries that see their key: an infinity or NaN comes
// out of a sum whatever its weight is.  In the other tiles they stay; a weight that fp16 has as 0, or a maximum that moves far, makes no number of an infinity
// there as well, and a row that ends with one takes the sum of the values that it sees and that are not finite.
#include "attn_tile.cuh"
#include "attn_window.cuh"

namespace q40 {
namespace window {

constexpr int NWARPS = 4, RB = NWARPS * 16, NT = NWARPS * 32;
constexpr int BITS = 14;                     // log2 of a row's largest weight

__global__ void __launch_bounds__(NT)
attn_window_kernel(const Args a) {
  constexpr int D = ATTN_D;
  extern __shared__ __align__(128) unsigned char smem[];
  const uint32_t sbase = smem_u32(smem);     // [Q rows][stage][K tile | V tile]
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int rblk = (int)((gridDim.x - 1 - blockIdx.x) / a.H), h = (int)(blockIdx.x % a.H), hk = h / (a.H / a.Hkv);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int row0 = rblk * RB, rows = min(RB, a.S - row0);
  // positions of the block's queries, and the keys that one of them sees: below `first`, and from `from` to k_end
  const int p_first = a.offset + row0, p_last = p_first + rows - 1, k_end = p_last + 1;
  const int from = max(0, p_first - a.window + 1), first = min(a.sinks, from);
  const int t_first = (first + TILE_KEYS - 1) / TILE_KEYS, t_from = max(from / TILE_KEYS, t_first);
  const int ntiles = t_first + (k_end + TILE_KEYS - 1) / TILE_KEYS - t_from;
  const auto tile_of = [&](int i) { return i < t_first ? i : i - t_first + t_from; };
  const uint32_t stages = sbase + RB * TILE_ROW_BYTES;

  auto load = [&](int tile, int stage) {
    const int64_t key0 = (int64_t)tile * TILE_KEYS;
    const uint32_t kdst = stages + stage * 2 * TILE_BYTES;
    load_tile<NT>(kdst, kdst + TILE_BYTES, a.k + key0 * a.ldk + hk * D, a.v + key0 * a.ldv + hk * D, a.ldk, a.ldv, k_end - tile * TILE_KEYS, tid);
  };
  for (int idx = tid; idx < RB * 16; idx += NT) {
    const int r = idx >> 4, ch = idx & 15;
    const bool ok = r < rows;
    cp_async16(sbase + tile_off(r, ch), a.q + (int64_t)(ok ? row0 + r : row0) * a.ldq + h * D + ch * 8, ok);
  }
  cp_async_commit();
  load(tile_of(0), 0);
  cp_async_commit();
  cp_async_wait<1>();
  __syncthreads();
  WarpRows w;
  w.init();
  w.load_q(sbase, warp * 16, lane);

  const int p0 = p_first + warp * 16 + g, p1 = p0 + 8;                   // positions of this lane's two rows
  const int warp_first = p_first + warp * 16, warp_last = warp_first + 15;
  bool taken_out = false;
  for (int i = 0; i < ntiles; ++i) {
    const int stage = i & 1, key0 = tile_of(i) * TILE_KEYS;
    if (i + 1 < ntiles) load(tile_of(i + 1), stage ^ 1);
    cp_async_commit();
    cp_async_wait<1>();
    __syncthreads();
    const uint32_t kt = stages + stage * 2 * TILE_BYTES, vt = kt + TILE_BYTES;
    // a tile that all queries of the block see
    const auto all_see = [&](int lo, int hi) { return key0 + TILE_KEYS <= lo + 1 && (key0 > hi - a.window || key0 + TILE_KEYS <= a.sinks); };
    if (!all_see(p_first, p_last)) {
      uint4* const row = reinterpret_cast<uint4*>(smem + RB * TILE_ROW_BYTES + stage * 2 * TILE_BYTES + TILE_BYTES);
      __half2 most = u32_as_h2(0);             // magnitudes: what is not finite is above all that is, or stays
#pragma unroll
      for (int j = 0; j < TILE_BYTES / 16 / NT; ++j) {
        const uint4 x = row[tid + j * NT];
        const uint32_t e[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int c = 0; c < 4; ++c) most = __hmax2_nan(most, __habs2(u32_as_h2(e[c])));
      }
      const bool found = not_finite(__low2half(most)) || not_finite(__high2half(most));
      if (__syncthreads_or(found)) {
        taken_out = true;
        __half* const x = reinterpret_cast<__half*>(row);
        for (int j = tid; j < TILE_BYTES / 2; j += NT)
          if (not_finite(x[j])) x[j] = __ushort_as_half(0);
        __syncthreads();
      }
    }
    if (all_see(min(warp_first, p_last), min(warp_last, p_last))) w.step<false, TILE_KEYS, false, BITS>(kt, vt, a.scale_log2, 0, 0, lane);
    else if (key0 <= warp_last && (key0 + TILE_KEYS > warp_first - a.window + 1 || key0 < a.sinks))
      w.step<true, TILE_KEYS, true, BITS>(kt, vt, a.scale_log2, min(p0, p_last) + 1 - key0, min(p1, p_last) + 1 - key0, lane, p0 - a.window + 1 - key0,
                                    p1 - a.window + 1 - key0, a.sinks - key0);
    __syncthreads();
  }
  cp_async_wait<0>();
  w.finish();
  bool lost[2] = {false, false};             // no number, and not by a score
#pragma unroll
  for (int r = 0; r < 2; ++r) {
#pragma unroll
    for (int dt = 0; dt < 16; ++dt) lost[r] |= w.o[dt][2 * r] != w.o[dt][2 * r] || w.o[dt][2 * r + 1] != w.o[dt][2 * r + 1];
    lost[r] &= w.l[r] == w.l[r];
  }
  if (taken_out || lost[0] || lost[1]) {     // rare, and slow
    uint32_t found[2] = {0, 0};
    for (int i = 0; i < ntiles; ++i) {
      const int key0 = tile_of(i) * TILE_KEYS;
      const bool all = key0 + TILE_KEYS <= p_first + 1 && (key0 > p_last - a.window || key0 + TILE_KEYS <= a.sinks);
      if (all && !lost[0] && !lost[1]) continue;
      for (int j = key0; j < min(key0 + TILE_KEYS, k_end); ++j) {
        const __half* const x = a.v + (int64_t)j * a.ldv + hk * D + 2 * t;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int p = r ? p1 : p0;
          if (p > p_last || j > p || (p - j >= a.window && j >= a.sinks) || (all && !lost[r])) continue;
#pragma unroll
          for (int dt = 0; dt < 16; ++dt)
#pragma unroll
            for (int c = 0; c < 2; ++c)
              if (not_finite(x[dt * 8 + c])) {
                const uint32_t bit = 1u << (2 * dt + c);
                w.o[dt][2 * r + c] = (lost[r] && !(found[r] & bit) ? 0.f : w.o[dt][2 * r + c]) + __half2float(x[dt * 8 + c]);
                found[r] |= bit;
              }
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int p = r ? p1 : p0;
    if (p > p_last) continue;
    const float inv = w.l[r] != 0.f ? 1.f / w.l[r] : 0.f;
    __half* dst = a.o + (int64_t)(p - a.offset) * a.ldo + h * D;
#pragma unroll
    for (int dt = 0; dt < 16; ++dt)
      *reinterpret_cast<__half2*>(dst + dt * 8 + 2 * t) = __floats2half2_rn(w.o[dt][2 * r] * inv, w.o[dt][2 * r + 1] * inv);
  }
}

}  // namespace window
}  // namespace q40

namespace q40 {
namespace window {

static Args args_of(int S, int H, int Hkv, int offset, int window, int sinks) {
  Args a{};
  a.S = S; a.H = H; a.Hkv = Hkv;
  // positions end at offset + S: what is further back, or further on, than that sees or adds nothing more
  a.offset = offset; a.window = min(window, offset + S); a.sinks = min(sinks, offset + S);
  a.scale_log2 = attn_scale_log2(ATTN_D);
  a.splits = 1;
  return a;
}
// Whether the kernel on tcgen05 takes the call.  Us here / there, 32 heads: 64 queries of themselves 4.5 / 5.3, 100 6.5 / 5.5, 256 11.2 / 8.7; a query behind 300 keys of which it sees
// 68 8.0 / 8.7, 64 such queries 11.0 / 8.7; a query behind 4000 with a window of 1024 30.9 / 10.7
static bool wide(const Args& a) { return a.S > 64 || (int64_t)min(a.offset, a.window - 1) + a.S + a.sinks > 128; }
static bool fits(int S, int H, int Hkv, int D, int offset, int window, int sinks) {
  return S >= 0 && H > 0 && Hkv > 0 && H % Hkv == 0 && offset >= 0 && window > 0 && sinks >= 0 && (int64_t)S + offset <= (1 << 30) && D == ATTN_D;
}
static size_t part_bytes(const Args& a) { return (size_t)a.splits * a.S * a.H * (ATTN_D + 2) * sizeof(float); }

}  // namespace window
}  // namespace q40

extern "C" size_t q40_attn_causal_window_workspace_bytes(int S, int H, int Hkv, int D, int offset, int window, int sinks) {
  using namespace q40::window;
  if (!fits(S, H, Hkv, D, offset, window, sinks) || S == 0) return 0;
  Args a = args_of(S, H, Hkv, offset, window, sinks);
  if (!wide(a)) return 0;
  a.splits = splits_tc(a);
  return a.splits == 1 ? 0 : part_bytes(a);
}

extern "C" int q40_attn_causal_window(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, void* o,
                                      int64_t ldo, int S, int H, int Hkv, int D, int offset, int window, int sinks, void* workspace,
                                      size_t workspace_bytes, int* err, void* stream) {
  using namespace q40;
  using namespace q40::window;
  if (!q || !k || !v || !o) return Q40_E_NULL;
  if (D != ATTN_D) return Q40_E_UNSUPPORTED;
  if (!fits(S, H, Hkv, D, offset, window, sinks)) return Q40_E_SHAPE;
  if (ldq < (int64_t)H * D || ldo < (int64_t)H * D || ldk < (int64_t)Hkv * D || ldv < (int64_t)Hkv * D) return Q40_E_SHAPE;
  if (ldq % 8 != 0 || ldk % 8 != 0 || ldv % 8 != 0 || ldo % 2 != 0) return Q40_E_ALIGN;
  if (!q40_aligned(q, 16) || !q40_aligned(k, 16) || !q40_aligned(v, 16) || !q40_aligned(o, 4)) return Q40_E_ALIGN;
  if (S == 0) return Q40_OK;
  Args a = args_of(S, H, Hkv, offset, window, sinks);
  a.q = (const __half*)q; a.k = (const __half*)k; a.v = (const __half*)v; a.o = (__half*)o;
  a.ldq = ldq; a.ldk = ldk; a.ldv = ldv; a.ldo = ldo;
  a.wide_out = ldo % 8 == 0 && q40_aligned(o, 16);
  if (err && wide(a)) {
    if (!q40_aligned(err, 4)) return Q40_E_ALIGN;
    const int splits = splits_tc(a);
    if (splits > 1 && workspace) {
      a.splits = splits;
      if (workspace_bytes < part_bytes(a)) return Q40_E_WORKSPACE;
      if (!q40_aligned(workspace, 16)) return Q40_E_ALIGN;
      a.po = (float*)workspace;
      a.pml = (float2*)(a.po + (size_t)splits * S * H * ATTN_D);
    }
    const int rc = launch_tc(a, err, (cudaStream_t)stream);
    if (rc != Q40_E_UNSUPPORTED) return rc;
    a.splits = 1;
  }
  const size_t smem = RB * TILE_ROW_BYTES + 4 * TILE_BYTES;
  static std::atomic<uint64_t> ready;
  cudaError_t e = q40_allow_smem(ready, (const void*)attn_window_kernel, (int)smem);
  if (e != cudaSuccess) { (void)cudaGetLastError(); return Q40_E_UNSUPPORTED; }
  const int64_t blocks = (int64_t)H * ((S + RB - 1) / RB);
  if (blocks > 0x7fffffffLL) return Q40_E_SHAPE;
  e = q40_launch_pdl(attn_window_kernel, dim3((unsigned)blocks), dim3(NT), smem, (cudaStream_t)stream, a);
  return e == cudaSuccess ? Q40_OK : (int)e;
}
