// What the append to a paged cache (page_append.cu) and the attention over it (attn_pages.cu) share: what a pool holds, and where.
//
// A pool is [Hkv, P, 128], P token slots of each kv head, of fp16, or of 8-bit codes (signed integers or e4m3) with one fp32
// scale for each page and kv head, [Hkv, P / page_size]: an element is code * scale.
#pragma once
#include <cuda_fp8.h>

#include "attn_common.cuh"

namespace q40 {

enum CacheType { CACHE_F16 = 0, CACHE_I8 = 1, CACHE_E4M3 = 2 };

template <int T>
constexpr int cache_bytes = T == CACHE_F16 ? 2 : 1;
template <int T>
constexpr float cache_top_inv = T == CACHE_I8 ? 1.f / 127.f : 1.f / 448.f;        // one over the code that a page's largest value gets

// Where the tokens of a sequence are: page ids of `width` entries a sequence
struct PageTable {
  const void* ids;         // int16 (unsigned) or int32
  int64_t stride;          // entries from sequence to sequence
  int wide;                // int32
  int page_size, page_shift;      // its log2, or -1
  __device__ __forceinline__ int page_of(int t) const { return page_shift >= 0 ? t >> page_shift : t / page_size; }
  __device__ __forceinline__ int id(int64_t seq, int page) const {
    const int64_t at = seq * stride + page;
    return wide ? reinterpret_cast<const int32_t*>(ids)[at] : (int)reinterpret_cast<const uint16_t*>(ids)[at];
  }
};

static inline int page_shift_of(int page_size) {
  if (page_size <= 0 || (page_size & (page_size - 1)) != 0) return -1;
  int s = 0;
  while ((1 << s) < page_size) ++s;
  return s;
}

// Four e4m3 codes as two pairs of halves: exact
__device__ __forceinline__ uint2 e4m3_to_h4(uint32_t four) {
  uint2 r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}" : "=r"(r.x), "=r"(r.y) : "r"(four));
  return r;
}
// Two signed bytes, which come + 128 with a byte 0x64 above each (the half 1024 + 128 + code), as two halves: exact
__device__ __forceinline__ uint32_t i8_to_h2(uint32_t biased) {
  return h2_as_u32(__hsub2(u32_as_h2(biased), u32_as_h2(0x64806480u)));
}

// 2^x of what is scaled down, never 0: an infinite value stays one
__device__ __forceinline__ float ex2_some(float x) { return fmaxf(ex2(x), 1.17549435e-38f); }

}  // namespace q40
