// q40_attn_pages_scores: q40_attn_pages with scores that are capped by a tanh, or less by what the distance to the query costs.  Cap and bias are
// a few instructions for each score of a lane, beside some 18 a key and head group (attn_pages.cuh).
#include "attn_pages.cuh"

extern "C" int q40_attn_pages_scores(const void* page_tbl, int idx_bytes, int64_t tbl_stride, const int32_t* seq_lens, const void* q,
                              int64_t q_stride, const void* kpool, const void* vpool, const float* k_scale, const float* v_scale,
                              int cache_type, void* o, int64_t P, int B, int Lmax, int H, int Hkv, int D, int page_size, int window, int sinks, float softcap, const float* slopes,
                              void* workspace, size_t workspace_bytes, void* stream) {
  using namespace q40;
  using namespace q40::pages;
  if (softcap != 0.f && !(softcap >= Q40_SOFTCAP_LEAST && softcap <= Q40_SOFTCAP_MOST)) return Q40_E_SHAPE;
  ScoreArgs a{};
  const int rc = args_of(a, page_tbl, idx_bytes, tbl_stride, seq_lens, q, q_stride, kpool, vpool, k_scale, v_scale, cache_type, o, P, B, Lmax, H, Hkv, D, page_size, window,
                         sinks, workspace, workspace_bytes);
  if (rc != Q40_OK || a.B == 0) return rc;
  if (!q40_aligned(slopes, 4)) return Q40_E_ALIGN;
  a.slopes = slopes;
  if (softcap != 0.f) {
    const double unit = 1. / (softcap * 1.4426950408889634);          // of a score in log2, in caps
    a.cap_limit = (float)(TANH_TO / unit); a.cap_exp = (float)(2. * unit * 1.4426950408889634); a.cap_out = (float)(1. / unit);
    tanh_poly_of(unit, a.cap_k);
  }
  return enqueue<true>(a, cache_type, (cudaStream_t)stream);
}
