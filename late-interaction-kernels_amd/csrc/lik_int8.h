// Rows as 8-bit integers with a scale each: the definition that the quantising kernels share.
//   s = max(fp32(max|x| / 127), 2^-126),  q = x / s to the nearest integer, ties to even
// q is that of the exact quotient: x * (1 / s) is off by at most 127 * 2^-22 = 3e-5 (the reciprocal by one unit), so its
// nearest integer can be the wrong one of two where the quotient lies that close to the middle. The remainder x - q s tells:
// it is a whole multiple of the smaller of both spacings and little over s / 2, hence exact in one fma (x one binade
// under s = 2^k is the exception, and there the product with 1 / s = 2^-k is exact); under s / 2, q is right.
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
template <int EK, int CTRL>
__device__ __forceinline__ uint32_t absmax_dpp(uint32_t m) {
  return absmax_join<EK>(m, (uint32_t)__builtin_amdgcn_update_dpp((int)m, (int)m, CTRL, 0xf, 0xf, false));
}
// Over the LPR (16 to 64) lanes of a row, on every lane: within 16 by data-parallel moves (the lane opposite in two, four,
// eight, sixteen), across them by the row and half swaps.
template <int EK, int LPR>
__device__ __forceinline__ uint32_t absmax_lanes(uint32_t m) {
  m = absmax_dpp<EK, 0xb1>(m);
  m = absmax_dpp<EK, 0x4e>(m);
  m = absmax_dpp<EK, 0x141>(m);
  m = absmax_dpp<EK, 0x140>(m);
  if constexpr (LPR >= 32) {
    const auto s = __builtin_amdgcn_permlane16_swap(m, m, false, false);
    m = absmax_join<EK>((uint32_t)s[0], (uint32_t)s[1]);
  }
  if constexpr (LPR == 64) {
    const auto s = __builtin_amdgcn_permlane32_swap(m, m, false, false);
    m = absmax_join<EK>((uint32_t)s[0], (uint32_t)s[1]);
  }
  return m;
}
// The row's scale (NaN where it holds an infinity or a NaN) and what its elements are multiplied by first.
template <int EK>
__device__ __forceinline__ void row_scale(uint32_t m, float& s, float& inv) {
  float amax;
  if constexpr (EK == EK_F32) amax = __uint_as_float(m);
  else amax = el_to_f32<EK>(max(m & 0xffffu, m >> 16));
  const bool fine = amax < INFINITY;
  // the quotient's bits have a period of 7, so it keeps 2^-7 of a step away from the middle of two floats: rounding the
  // 64-bit product is rounding the quotient
  s = fmaxf((float)((double)amax * (1.0 / 127.0)), 1.1754943508e-38f);
  inv = fine ? __builtin_amdgcn_rcpf(s) : 0.f;
  if (!fine) s = __uint_as_float(0x7fc00000u);
}
// The integers of a chunk's elements, 4 to a word; inv = 0: zeros.
template <int EK>
__device__ __forceinline__ void chunk_to_int8(const u32x4& w, float s, float inv, uint32_t* out) {
  constexpr int V = El<EK>::V;
  constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: added, the sum's lowest bits are the nearest integer
  float v[V], y[V], rem[V], most = 0.f;
  chunk_widen<EK>(w, v);
  const float half = 0.5f * s;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    y[e] = fmaf(v[e], inv, kRound);
    rem[e] = fmaf(kRound - y[e], s, v[e]);
    most = fmaxf(most, fabsf(rem[e]));
  }
  if (most >= half)  // (rare: a tie, or a product on the wrong side)
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (fabsf(rem[e]) > half || (fabsf(rem[e]) == half && (__float_as_uint(y[e]) & 1u))) y[e] += copysignf(1.0f, rem[e]);
#pragma unroll
  for (int g = 0; g < V / 4; ++g) {
    const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(y[4 * g + 1]), __float_as_uint(y[4 * g]), 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(y[4 * g + 3]), __float_as_uint(y[4 * g + 2]), 0x04000c0cu);
    out[g] = inv == 0.f ? 0u : lo | hi;
  }
}

// lik_quantize_int8; `stream`: rows are read past the caches. Alone that is the faster way (1,030,001 rows of 128 fp16 there
// and back 137 against 153 us when the way back took 74); in front of a product that reads its integers from the caches the slower one (124 against 119).
int quantize_rows_int8(const void* x, int64_t x_stride, int32_t dtype, int64_t rows, int32_t dim, int8_t* out,
                       int64_t out_stride, float* scale, bool stream, hipStream_t s);

}  // namespace enc
}  // namespace lik
