// q40_attn_pages: attention of one query token per sequence over a paged cache (attn_pages.cuh).
#include "attn_pages.cuh"

extern "C" size_t q40_attn_pages_workspace_bytes(int B, int H, int Hkv, int L, int window, int sinks) {
  using namespace q40::pages;
  if (B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv != 0 || L <= 0) return 0;
  const Plan p = plan_of(B, H, Hkv, L, window, sinks);
  return p.nchunks == 1 ? 0 : (size_t)p.units * p.nchunks * p.heads * (q40::ATTN_D + 2) * sizeof(float);
}

extern "C" int q40_attn_pages(const void* page_tbl, int idx_bytes, int64_t tbl_stride, const int32_t* seq_lens, const void* q,
                              int64_t q_stride, const void* kpool, const void* vpool, const float* k_scale, const float* v_scale,
                              int cache_type, void* o, int64_t P, int B, int Lmax, int H, int Hkv, int D, int page_size, int window, int sinks,
                              void* workspace, size_t workspace_bytes, void* stream) {
  using namespace q40::pages;
  Args a{};
  const int rc = args_of(a, page_tbl, idx_bytes, tbl_stride, seq_lens, q, q_stride, kpool, vpool, k_scale, v_scale, cache_type, o, P, B, Lmax, H, Hkv, D, page_size, window,
                         sinks, workspace, workspace_bytes);
  return rc != Q40_OK || a.B == 0 ? rc : enqueue<false>(a, cache_type, (cudaStream_t)stream);
}
