// Scores capped by a tanh, for the attention kernels: x -> tanh(u x) / u, where u is 1 over the cap in the score's units.
#pragma once
#include "attn_common.cuh"

namespace q40 {

// tanh(y) / y = sum over i of TANH[i] y^2i for |y| <= TANH_TO, off by 1.1e-7 of itself (a fit of least largest relative error, by weighted least squares)
constexpr double TANH[5] = {0.999999893, -0.333319542, 0.13304526, -0.0518218664, 0.0150509449};
constexpr double TANH_TO = 0.625;
// ... as the coefficients of x^2 for tanh(u x) / (u x)
static inline void tanh_poly_of(double u, float (&k)[5]) {
  double power = 1.;
  for (int i = 0; i < 5; ++i, power *= u * u) k[i] = (float)(TANH[i] * power);
}
__device__ __forceinline__ float tanh_poly(float x2, const float (&k)[5]) {
  return fmaf(fmaf(fmaf(fmaf(k[4], x2, k[3]), x2, k[2]), x2, k[1]), x2, k[0]);
}
// tanh(y) for any y, given 2 y log2(e): infinities become +-1, NaN stays; off by some 2^-23
__device__ __forceinline__ float tanh_by_exp(float y) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + ex2(y)));
  return fmaf(-2.f, r, 1.f);
}

}  // namespace q40
