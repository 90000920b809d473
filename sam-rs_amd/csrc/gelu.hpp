// The exact GELU of the reference's MLP, shared by the kernels that apply it to a result.
#pragma once
#include "common.hpp"

namespace samhip {

// 0.5 x (1 + erf(x / sqrt 2)), with 1 + erf(x / sqrt 2) taken as erfc(|x| / sqrt 2) for x < 0 and
// 2 - erfc(|x| / sqrt 2) otherwise, so that negative x loses nothing to cancellation. erfc is the
// Chebyshev fit of Press et al., Numerical Recipes in C (2nd ed., section 6.2, erfcc): fractional
// error below 1.2e-7 for every argument (1.04e-7 measured in float64 against the exact erfc; the f32
// evaluation here stays within 7e-8 of the exact gelu in absolute terms). About 18 instructions
// against some 45 for the device erff, which made this kernel arithmetic-bound.
__device__ __forceinline__ float gelu_erf(float x) {
#pragma clang fp contract(off)
  const float z = fabsf(x) * 0.70710678118654752f;
  const float t = __builtin_amdgcn_rcpf(1.f + 0.5f * z);
  float p = 0.17087277f;
  p = fmaf(t, p, -0.82215223f);
  p = fmaf(t, p, 1.48851587f);
  p = fmaf(t, p, -1.13520398f);
  p = fmaf(t, p, 0.27886807f);
  p = fmaf(t, p, -0.18628806f);
  p = fmaf(t, p, 0.09678418f);
  p = fmaf(t, p, 0.37409196f);
  p = fmaf(t, p, 1.00002368f);
  p = fmaf(t, p, -1.26551223f);
  const float e = t * __builtin_amdgcn_exp2f(fmaf(-z, z, p) * 1.4426950408889634f);
  return 0.5f * x * (x >= 0.f ? 2.f - e : e);
}

// The same for results of 16 bits, with seven instructions less: erfc(z) exp(z^2) as a polynomial of degree 6 in
// t = 1 / (1 + 0.44 z) without constant term, fitted here for the least relative error over 0 <= z <= 14 (6.6e-6; 1.1e-5 with
// f32's roundings, down to x = -12), a fortieth of half a step of f16: of N(0, 1) arguments one f16 result in 240 is the neighbour of the
// exact one's rounding for it. A 4-bit product of 4096 x 5120 and k = 1280 takes 39.1 us with gelu_erf and 36.4 with this in f16, 16384
// rows of it 119 and 109. Halves of the coefficients.
__device__ __forceinline__ float gelu_erf16(float x) {
  const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(x), 0.31112698372208092f, 1.f));
  float p = -0.0721961836f;
  p = fmaf(t, p, 0.172969651f);
  p = fmaf(t, p, 0.0228032338f);
  p = fmaf(t, p, 0.130619835f);
  p = fmaf(t, p, 0.121544765f);
  p = fmaf(t, p, 0.124259499f);
  const float e = p * t * __builtin_amdgcn_exp2f(x * x * -0.72134752044448170f);
  return x * (x >= 0.f ? 1.f - e : e);
}
template <typename T> __device__ __forceinline__ float gelu_for(float x) {
  if constexpr (sizeof(T) == 2)
    return gelu_erf16(x);
  else
    return gelu_erf(x);
}

}  // namespace samhip
