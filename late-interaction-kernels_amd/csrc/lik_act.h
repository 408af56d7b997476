// Activations of the feed-forward blocks.
#pragma once
#include "lik_enc.h"

namespace lik {
namespace enc {

enum { ACT_GELU = 0, ACT_GELU_TANH = 1, ACT_SILU = 2 };

// act(x) and its derivative, for 16-bit outputs
template <int ACT, bool SLOPE>
__device__ __forceinline__ float act_of(float x, float& slope) {
  if constexpr (ACT == ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-x));
    if (SLOPE) slope = s * (1.0f + x * (1.0f - s));
    return x * s;
  } else if constexpr (ACT == ACT_GELU_TANH) {
    // (1 + tanh u) / 2 = sigmoid(2 u), u = sqrt(2 / pi) (x + 0.044715 x^3); 0 or 1 past |x| = 64, whose powers stay finite
    const float z = __builtin_amdgcn_fmed3f(x, -64.0f, 64.0f), z2 = z * z;
    const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-1.5957691216f * z * fmaf(0.044715f, z2, 1.0f)));
    if (SLOPE) slope = s * (1.0f + z * (1.0f - s) * 1.5957691216f * fmaf(0.134145f, z2, 1.0f));
    return x * s;
  } else {
    // cdf(-|x|) = erfc(|x| / sqrt 2) / 2 = poly(s) exp(-x^2 / 2), s = 1 / (1 + p |x| / sqrt 2): Abramowitz and
    // Stegun 7.1.26, absolute error of erf 1.5e-7, so 1e-7 |x| of the activation: far under the 16-bit outputs' rounding but where
    // the activation all but vanishes (relative to it 5e-5 at -3, 5e-4 at -4, 4e-3 at -6); the exponential is the slope's too (the
    // library's erff costs three times as many instructions).
    const float z = fabsf(x), s = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678118f, z, 1.0f));
    const float e = __expf(-0.5f * x * x);
    float q = fmaf(1.061405429f, s, -1.453152027f);
    q = fmaf(q, s, 1.421413741f);
    q = fmaf(q, s, -0.284496736f);
    q = fmaf(q, s, 0.254829592f);
    const float tail = 0.5f * q * s * e;
    const float cdf = x < 0.f ? tail : 1.0f - tail;
    if (SLOPE) slope = fmaf(x, 0.39894228040f * e, cdf);
    return x * cdf;
  }
}
// For fp32 outputs: exponentials and reciprocals to a rounding or two, in half the instructions of the library's (20000 rows 768 ->
// 2304 with gelu 91 us; with expf and divisions 114; with the formula of the 16-bit outputs, which is off by three times as much, 78).
// exp(x) for x up to 0; under 2^-126 it is zero. The product x log2 e is carried on to twice its bits.
__device__ __forceinline__ float exp_f32(float x) {
  x = fmaxf(x, -150.0f);
  const float t = 1.44269504f * x, lo = fmaf(1.92596299e-8f, x, fmaf(1.44269504f, x, -t));  // (log2 e is 1.44269504f + 1.926e-8)
  return __builtin_amdgcn_exp2f(t) * fmaf(0.693147181f, lo, 1.0f);
}
// 1 / x for normal x with a normal result: one step of Newton's
__device__ __forceinline__ float rcp_f32(float x) {
  const float r = __builtin_amdgcn_rcpf(x);
  return fmaf(fmaf(-x, r, 1.0f), r, r);
}
// x / (1 + exp(-w))
__device__ __forceinline__ float sigmoid_times(float x, float w) {
  const float e = exp_f32(-fabsf(w));
  return x * ((w < 0.f ? e : 1.0f) * rcp_f32(1.0f + e));
}
// act(x), as exact as fp32 arithmetic makes it.
template <int ACT>
__device__ __forceinline__ float act_f32_of(float x) {
  if constexpr (ACT == ACT_SILU) {
    return sigmoid_times(x, x);
  } else if constexpr (ACT == ACT_GELU_TANH) {  // (as above)
    const float z = __builtin_amdgcn_fmed3f(x, -64.0f, 64.0f);
    return sigmoid_times(x, 1.5957691216f * z * fmaf(0.044715f, z * z, 1.0f));
  } else {
    // cdf(-|x|) = s q(t) exp(-x^2 / 2), s = 1 / (1 + 0.27 |x|), t = 1 - s = 0.27 |x| s: q of degree 8, fitted to the least relative
    // error of the product for |x| <= 15 (2^-25; the density underflows there), q(0) = 1/2. Where x is negative x cdf is off by
    // some 2^-24 (x^2 + 6) of itself, x^2 of which are the roundings of the exponent and about what those of x itself do.
    const float z = fminf(fabsf(x), 64.0f), s = rcp_f32(fmaf(0.27f, z, 1.0f)), t = 0.27f * z * s;
    float q = fmaf(0.0287802052f, t, -0.104559392f);
    q = fmaf(q, t, 0.0943524241f);
    q = fmaf(q, t, 0.0856105015f);
    q = fmaf(q, t, -0.0914911479f);
    q = fmaf(q, t, -0.401701063f);
    q = fmaf(q, t, 0.974294305f);
    q = fmaf(q, t, -0.977565587f);
    q = fmaf(q, t, 0.5f);
    const float tail = q * s * __builtin_amdgcn_exp2f(-0.72134752f * x * x);
    return x * (x < 0.f ? tail : 1.0f - tail);
  }
}
// Eight at a time, so that one value's chain of instructions fills the other's waits.
template <bool SLOPE>
__device__ __forceinline__ void act8(int act, const float* x, float* y, float* slope) {
  float none;
  auto all = [&](auto A) {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = act_of<decltype(A)::value, SLOPE>(x[e], SLOPE ? slope[e] : none);
  };
  if (act == ACT_SILU) all(std::integral_constant<int, ACT_SILU>{});
  else if (act == ACT_GELU_TANH) all(std::integral_constant<int, ACT_GELU_TANH>{});
  else all(std::integral_constant<int, ACT_GELU>{});
}
// For fp32 outputs.
__device__ __forceinline__ void act8_f32(int act, const float* x, float* y) {
  auto all = [&](auto A) {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = act_f32_of<decltype(A)::value>(x[e]);
  };
  if (act == ACT_SILU) all(std::integral_constant<int, ACT_SILU>{});
  else if (act == ACT_GELU_TANH) all(std::integral_constant<int, ACT_GELU_TANH>{});
  else all(std::integral_constant<int, ACT_GELU>{});
}

}  // namespace enc
}  // namespace lik
