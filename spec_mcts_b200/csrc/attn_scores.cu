// Prompt attention with changed scores and further masks: scores capped by a tanh, less what the distance of a key costs, documents that see
// themselves alone (the prompts of several requests in one call), and a prefix that sees itself in both directions.
//
// Query i at position p, in a document of positions [s, e) whose first f are its prefix, sees the keys s <= j < e with (j <= p or j - s < f) and (p - j < window or
// j - s < sinks).  Its score of key j is c tanh(x / c) - slope |p - j|, x = q . k / sqrt(128).
//
// The kernel is that of attn_tc.cuh.  What is added, a step of 128 keys a row:
//   cap      tanh(x) = x P(x^2), P of degree 4, while no |x / c| of the warp's rows is above 0.625, in the product that makes the exponent: five packed instructions
//            more for two scores, and 64 of three inputs for the largest magnitude; else 1 - 2 / (1 + e^2x), two more of the sixteen-a-cycle functions a score, of
//            which 2^x takes as long as the MMAs do.  (P of degree 7 in between, up to 1.25: 3920 -> 3444 us where all scores lie there, 16384 positions as below, but 320 ->
//            364 where they lie on both sides, 4001 positions: not taken)
//   bias     two packed instructions for two scores.  Sixteen keys share what their distances have in common; each bias is rounded twice, by 2^-24 of what is
//            left to the nearest of them.  Near keys come first: their scores are the largest, and O, once scaled for each step of a steep slope, is not any more (2079 -> 1762 us)
//   masks    what a row sees is an interval and the first keys of its document: words of bits, in tiles that some row does not see whole
// Documents are looked up by each row; what a tile's first and last row see tells which tiles of keys it goes through.
//
// Us by the card: 16384 positions, window 4096, 64 heads on 8: 1650 with plain scores, 1780 to 1900 with slopes, 1900 with a cap of which no score is above 0.625, 2280 to 2360 with both;
// 3970 and 3910 where scores reach the cap: three of the sixteen-a-cycle functions a score, 2420 for the visible ones alone.  4001 positions of 32 heads in nine
// documents with slopes 66 to 71, where the bytes take 20 and the MMAs 25: 512 CTAs of some ten steps each, 3 us of start and 4 of end around 2 a step, with nothing
// beside them on their SM.  One tile of queries a CTA and two CTAs an SM: 68 (75 with slopes), 2120 for the cap, 2290 for both: not taken, since others lose 5 %.
#include "attn_tc.cuh"

namespace q40 {
namespace window {

struct ScoreArgs : Args {
  const int32_t* documents;          // [n_documents + 1] rows at which they begin and end, or nullptr: all rows are one
  int n_documents;
  const int32_t* prefixes;           // of each document, or nullptr: `prefix` of each
  int prefix;
  int keep;                          // rows of no document are left as they are; else zeros
  const float* slopes;               // [H]
  float cap_limit, cap_exp, cap_out, cap_k[5];
};

namespace tc {

template <bool WITH_CAP, bool WITH_BIAS>
struct Scores {
  using Call = ScoreArgs;
  static constexpr bool CAP = WITH_CAP, BIAS = WITH_BIAS, SPANS = true;
  using Places = SpanPlaces;
  static __device__ __forceinline__ bool keeps(const ScoreArgs& a) { return a.keep; }

  // Every thread of the CTA calls it; a thread that has a row gets its span
  template <class B>
  static __device__ __forceinline__ Places places(const ScoreArgs& a, int row0, int split, Span& mine, B begin) {
    const int n = min(2 * BQ, a.S - row0);
    Span at[4];
    if (a.documents) {
      // Where documents begin is read once by all threads, up to FEW of them; looked up in global memory, a handful took a microsecond
      constexpr int FEW = 256;
      __shared__ Span edges[4];
      __shared__ int begins[FEW];
      asm volatile("griddepcontrol.wait;" ::: "memory");
      const int r = threadIdx.x;
      begin();                                           // (the queries are on their way meanwhile)
      const bool few = a.n_documents < FEW;
      if (few) {
        if (r <= a.n_documents) begins[r] = a.documents[r];
        __syncthreads();
      }
      if (r < 2 * BQ) {
        const int row = row0 + min(r, n - 1);
        mine = few ? span_in(a, row, [&](int k) { return begins[k]; }) : span_in(a, row, [&](int k) { return a.documents[k]; });
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (r == edge_row(e, n)) edges[e] = mine;
      }
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 4; ++e) at[e] = edges[e];
      return SpanPlaces(a, row0, split, at, BIAS);
    } else {
      mine = span_of(a, row0 + min((int)threadIdx.x, n - 1));
#pragma unroll
      for (int e = 0; e < 4; ++e) at[e] = span_of(a, row0 + edge_row(e, n));
      const Places there(a, row0, split, at, BIAS);
      begin();
      return there;
    }
  }
};

}  // namespace tc

static bool fits_scores(int S, int H, int Hkv, int D, int offset, int window, int sinks) {
  return S >= 0 && H > 0 && Hkv > 0 && H % Hkv == 0 && offset >= 0 && window > 0 && sinks >= 0 && (int64_t)S + offset <= (1 << 30) && D == ATTN_D;
}
static int splits_of(int S, int H, int Hkv, int offset, int window, int sinks) {
  Args a{};
  a.S = S; a.H = H; a.Hkv = Hkv; a.offset = offset;
  a.window = std::min(window, offset + S); a.sinks = std::min(sinks, offset + S);
  return splits_tc(a);
}
static size_t part_bytes(int splits, int S, int H) { return (size_t)splits * S * H * (ATTN_D + 2) * sizeof(float); }

}  // namespace window
}  // namespace q40

extern "C" size_t q40_attn_causal_scores_workspace_bytes(int S, int H, int Hkv, int D, int offset, int window, int sinks) {
  using namespace q40::window;
  if (!fits_scores(S, H, Hkv, D, offset, window, sinks) || S == 0) return 0;
  const int splits = splits_of(S, H, Hkv, offset, window, sinks);
  return splits == 1 ? 0 : part_bytes(splits, S, H);
}

extern "C" int q40_attn_causal_scores(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, void* o, int64_t ldo, int S, int H, int Hkv,
                                      int D, int offset, int window, int sinks, float softcap, const float* slopes, const int32_t* documents, int n_documents,
                                      const int32_t* prefixes, int prefix, int keep_rest, void* workspace, size_t workspace_bytes, int* err, void* stream) {
  using namespace q40;
  using namespace q40::window;
  if (!q || !k || !v || !o || !err || (prefixes && !documents)) return Q40_E_NULL;
  if (D != ATTN_D) return Q40_E_UNSUPPORTED;
  if (!fits_scores(S, H, Hkv, D, offset, window, sinks)) return Q40_E_SHAPE;
  if (ldq < (int64_t)H * D || ldo < (int64_t)H * D || ldk < (int64_t)Hkv * D || ldv < (int64_t)Hkv * D) return Q40_E_SHAPE;
  if (softcap != 0.f && !(softcap >= Q40_SOFTCAP_LEAST && softcap <= Q40_SOFTCAP_MOST)) return Q40_E_SHAPE;
  if (prefix < 0 || (documents && (offset != 0 || n_documents < 0 || n_documents >= (1 << 30)))) return Q40_E_SHAPE;
  if (ldq % 8 != 0 || ldk % 8 != 0 || ldv % 8 != 0 || ldo % 2 != 0) return Q40_E_ALIGN;
  if (!q40_aligned(q, 16) || !q40_aligned(k, 16) || !q40_aligned(v, 16) || !q40_aligned(o, 4) || !q40_aligned(err, 4) || !q40_aligned(slopes, 4) ||
      !q40_aligned(documents, 4) || !q40_aligned(prefixes, 4))
    return Q40_E_ALIGN;
  if (S == 0) return Q40_OK;
  ScoreArgs a{};
  a.q = (const __half*)q; a.k = (const __half*)k; a.v = (const __half*)v; a.o = (__half*)o;
  a.ldq = ldq; a.ldk = ldk; a.ldv = ldv; a.ldo = ldo;
  a.S = S; a.H = H; a.Hkv = Hkv;
  const int whole = offset + S;
  a.offset = offset; a.window = std::min(window, whole); a.sinks = std::min(sinks, whole);
  a.wide_out = ldo % 8 == 0 && q40_aligned(o, 16);
  a.scale_log2 = attn_scale_log2(D);
  a.documents = documents; a.n_documents = n_documents; a.prefixes = prefixes; a.prefix = std::min(prefix, whole); a.keep = keep_rest != 0;
  a.slopes = slopes;
  if (softcap != 0.f) {
    const double unit = 1. / (sqrt((double)D) * softcap);          // of a raw score, in caps
    a.cap_limit = (float)(TANH_TO / unit); a.cap_exp = (float)(2. * unit * 1.4426950408889634); a.cap_out = (float)(1. / unit);
    tanh_poly_of(unit, a.cap_k);
    for (float& k : a.cap_k) k = (float)((double)k * a.scale_log2);
  }
  a.splits = 1;
  const int splits = splits_of(S, H, Hkv, offset, window, sinks);
  if (splits > 1 && workspace) {
    a.splits = splits;
    if (workspace_bytes < part_bytes(splits, S, H)) return Q40_E_WORKSPACE;
    if (!q40_aligned(workspace, 16)) return Q40_E_ALIGN;
    a.po = (float*)workspace;
    a.pml = (float2*)(a.po + (size_t)splits * S * H * ATTN_D);
  }
  const cudaStream_t st = (cudaStream_t)stream;
  if (softcap != 0.f) return slopes ? tc::launch_form<tc::Scores<true, true>>(a, err, st) : tc::launch_form<tc::Scores<true, false>>(a, err, st);
  return slopes ? tc::launch_form<tc::Scores<false, true>>(a, err, st) : tc::launch_form<tc::Scores<false, false>>(a, err, st);
}
