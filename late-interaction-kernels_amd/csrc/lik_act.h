// Activations of the feed-forward blocks.
#pragma once
#include "lik_enc.h"

namespace lik {
namespace enc {

enum { ACT_GELU = 0, ACT_GELU_TANH = 1, ACT_SILU = 2 };

// act(x) and its derivative
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
    // Stegun 7.1.26, absolute error of erf 1.5e-7, far under the 16-bit outputs' rounding; the exponential is
    // the slope's too (the library's erff costs three times as many instructions).
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

}  // namespace enc
}  // namespace lik
