// Device helpers shared by the encoder operators (layer norm, gated
// feed-forward block, attention).
#pragma once
#include "lik_common.h"

namespace lik {
namespace enc {

// Element types of the encoder operators: 16-bit ones as the MFMA operands
// name them, fp32 for the layer norm.
template <int EK>
struct El {
  static constexpr int B = EK == EK_F32 ? 4 : 2;  // bytes
  static constexpr int V = 16 / B;                // elements of a 16-byte chunk
};

template <int EK>
__device__ __forceinline__ float el_to_f32(uint32_t bits) {
  if constexpr (EK == EK_F32) return __uint_as_float(bits);
  else if constexpr (EK == EK_F16) return f16_to_f32((uint16_t)bits);
  else return __uint_as_float(bits << 16);
}
template <int EK>
__device__ __forceinline__ uint32_t f32_to_el(float x) {
  if constexpr (EK == EK_F32) return __float_as_uint(x);
  else if constexpr (EK == EK_F16) return f32_to_f16_bits(x);
  else return f32_to_bf16_bits(x);
}
// two floats as packed 16-bit elements
template <int EK>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (EK == EK_F16) {
    const f16x2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
  } else {
    const bf16x2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
}
template <int EK>
__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b) {
  if constexpr (EK == EK_F16) {
    a = f16_to_f32((uint16_t)(w & 0xffffu));
    b = f16_to_f32((uint16_t)(w >> 16));
  } else {
    a = bf16lo_to_f32(w);
    b = bf16hi_to_f32(w);
  }
}

// c plus f times the two packed elements, in fp32 (one instruction, rounded once; subnormals are kept)
template <int EK>
__device__ __forceinline__ float add2(uint32_t w, float c, float f = 1.0f) {
  if constexpr (EK == EK_F16)
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), f16x2{(_Float16)f, (_Float16)f}, c, false);
  else
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), bf16x2{(__bf16)f, (__bf16)f}, c, false);
}

constexpr uint32_t kOob = 0xfffffff0u;  // a lane offset outside every buffer: the load returns (or writes to LDS) zeros

// Raw buffer descriptor of `bytes` bytes from base (both wave-uniform).
__device__ __forceinline__ u32x4 raw_desc(const void* base, uint32_t bytes) {
  const uint64_t b = (uint64_t)base;
  return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)b),
               (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(b >> 32) & 0xffffu),
               (uint32_t)__builtin_amdgcn_readfirstlane(bytes), 0x00020000u};
}
__device__ __forceinline__ uint32_t sat32(int64_t n) {  // buffer sizes: 0 .. just under the lane offset kOob
  return n <= 0 ? 0u : n > 0xffffff00ll ? 0xffffff00u : (uint32_t)n;
}

// 64 lanes x 16 bytes from memory to LDS at `lds` (wave-uniform, lane i's bytes
// at lds + 16 i). Inline asm: the compiler would wait for every such load before
// any later LDS read; here the caller waits (vmcnt) and places the barrier. M0
// holds the LDS address and is restored.
__device__ __forceinline__ void dma16(uint32_t lds, uint32_t voff, const u32x4& desc) {
  uint32_t saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"  // an M0 write needs one wait state before an LDS DMA reads it
      "buffer_load_dwordx4 %2, %3, 0 offen lds\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(desc)
      : "memory");
}
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}

// Transposing LDS read: in each group of 16 lanes, lane i names 4 consecutive
// 16-bit elements of row i / 4 (columns 4 (i % 4) ..); lane j gets column j of
// the four rows.
__device__ __forceinline__ u32x2 lds_tr(uint32_t addr) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(
      u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(uintptr_t)addr));
}
__device__ __forceinline__ u32x4 lds_b128(uint32_t addr) {
  return *(__attribute__((address_space(3))) const u32x4*)(uintptr_t)addr;
}

template <int EK>
__device__ __forceinline__ f32x16 mfma16(const f32x16& c, const u32x4& a, const u32x4& b) {
  return mfma32<EK>(c, &a, &b);
}

// Four consecutive elements of accumulator quads 2 j and 2 j + 1, as 16-bit pairs, to eight consecutive ones a lane
// (the wavefront's halves exchange): half h then holds elements 16 j + 8 h + 0..7.
__device__ __forceinline__ u32x4 join_halves(uint32_t a0, uint32_t a1, uint32_t b0, uint32_t b1) {
  const auto s0 = __builtin_amdgcn_permlane32_swap(a0, b0, false, false);
  const auto s1 = __builtin_amdgcn_permlane32_swap(a1, b1, false, false);
  return u32x4{(uint32_t)s0[0], (uint32_t)s1[0], (uint32_t)s0[1], (uint32_t)s1[1]};
}
// On every lane.
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) x = fmaxf(x, __shfl_xor(x, s));
  return x;
}

// The workgroups of one XCD (round-robin by block index) get a contiguous range of tiles.
__device__ __forceinline__ uint32_t xcd_tile(uint32_t id, uint32_t n) {
  const uint32_t x = id & 7u, per = n >> 3, extra = n & 7u;
  return x * per + (x < extra ? x : extra) + (id >> 3);
}

inline size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }
inline char* align256(void* p) { return (char*)(((uintptr_t)p + 255) & ~(uintptr_t)255); }

}  // namespace enc
}  // namespace lik
