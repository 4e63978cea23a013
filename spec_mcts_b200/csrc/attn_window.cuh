// What the two kernels of q40_attn_causal_window share.
#pragma once
#include "attn_common.cuh"

namespace q40 {
namespace window {

struct Args {
  const __half *q, *k, *v;    // position-major rows; heads side by side
  __half* o;
  int64_t ldq, ldk, ldv, ldo;
  int S, H, Hkv;
  int offset, window, sinks;
  int wide_out;               // output rows at 16-byte addresses
  float scale_log2;
  int splits;                 // CTAs that share the keys of a block of queries (attn_window_tc.cu): their results, not normalised
  float* po;                  // [splits][S][H][128]
  float2* pml;                // [splits][S][H] maximum (log2) and sum
};

__device__ __forceinline__ bool not_finite(__half x) { return (__half_as_ushort(x) & 0x7c00) == 0x7c00; }

// defined in attn_window_tc.cu: how many splits a call is worth, and the call, with a.splits of them.  `err`: device word, set to 1 if a bounded wait expired.  Q40_E_UNSUPPORTED: nothing was enqueued
int splits_tc(const Args& a);
int launch_tc(const Args& a, int* err, cudaStream_t st);

}  // namespace window
}  // namespace q40
