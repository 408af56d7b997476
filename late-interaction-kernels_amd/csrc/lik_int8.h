// Rows as 8-bit integers with a scale each: the definition that the quantising kernels share.
//   s = max(fp32(max|x| / 127), 2^-126),  q = x / s to the nearest integer, ties to even
// q is that of the exact quotient: x * (1 / s) is off by at most 127 * 2^-22 = 3e-5, so only quotients that
// close to a half-integer can be on its wrong side. For those the remainder x - q s decides: it is a whole
// multiple of the smaller of both spacings and at most s, hence exact in one fma (x one binade under s = 2^k is
// the exception, and there the product with 1 / s = 2^-k is exact).
#pragma once
#include "lik_enc.h"

namespace lik {
namespace enc {

// |x| of a chunk's elements as integer bits, which order as the magnitudes do (NaN above everything), joined with m.
template <int EK>
__device__ __forceinline__ uint32_t absmax_bits(const u32x4& w, uint32_t m) {
  if constexpr (EK == EK_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, w[i] & 0x7fffffffu);
    return m;
  } else {  // two 16-bit maxima side by side
    typedef unsigned short us2 __attribute__((ext_vector_type(2)));
    us2 a = __builtin_bit_cast(us2, m);
#pragma unroll
    for (int i = 0; i < 4; ++i) a = __builtin_elementwise_max(a, __builtin_bit_cast(us2, w[i] & 0x7fff7fffu));
    return __builtin_bit_cast(uint32_t, a);
  }
}
template <int EK>
__device__ __forceinline__ uint32_t absmax_join(uint32_t a, uint32_t b) {
  if constexpr (EK == EK_F32) return max(a, b);
  typedef unsigned short us2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(us2, a), __builtin_bit_cast(us2, b)));
}
// The row's scale (NaN where it holds an infinity or a NaN) and what its elements are multiplied by first.
template <int EK>
__device__ __forceinline__ void row_scale(uint32_t m, float& s, float& inv) {
  float amax;
  if constexpr (EK == EK_F32) amax = __uint_as_float(m);
  else amax = el_to_f32<EK>(max(m & 0xffffu, m >> 16));
  const bool fine = amax < INFINITY;
  s = fmaxf(amax / 127.0f, 1.1754943508e-38f);
  inv = fine ? 1.0f / s : 0.f;
  if (!fine) s = __uint_as_float(0x7fc00000u);
}
// The integers of a chunk's elements, 4 to a word; inv = 0: zeros.
template <int EK>
__device__ __forceinline__ void chunk_to_int8(const u32x4& w, float s, float inv, uint32_t* out) {
  constexpr int V = El<EK>::V;
  constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: added, the sum's lowest bits are the nearest integer
  float v[V], y[V], most = 0.f;
  chunk_widen<EK>(w, v);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float q = v[e] * inv;
    y[e] = q + kRound;
    most = fmaxf(most, fabsf(q - (y[e] - kRound)));
  }
  if (most > 0.4999f) {
    const float half = 0.5f * s;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float r = y[e] - kRound, rem = fmaf(-r, s, v[e]);
      if (fabsf(rem) > half || (fabsf(rem) == half && (__float_as_uint(y[e]) & 1u))) y[e] += copysignf(1.0f, rem);
    }
  }
#pragma unroll
  for (int g = 0; g < V / 4; ++g) {
    const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(y[4 * g + 1]), __float_as_uint(y[4 * g]), 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(y[4 * g + 3]), __float_as_uint(y[4 * g + 2]), 0x04000c0cu);
    out[g] = inv == 0.f ? 0u : lo | hi;
  }
}

}  // namespace enc
}  // namespace lik
