// Layer norm with an optional residual sum, forward and backward.
//
//   s = round(x + residual)  (the type of x; s = x without a residual)
//   mean = sum s / d,  rstd = 1 / sqrt(sum (s - mean)^2 / d + eps)
//   y = (s - mean) rstd w + b
// backward, with u = (s - mean) rstd and c = gy w:
//   gx = rstd (c - mean(c) - u mean(c u)) + gs,  gw = sum_rows gy u,  gb = sum_rows gy
//
// Bound by HBM: every row is read once and stays in registers between the two
// sums and the output (a group of LPR lanes holds a row, NV 16-byte chunks a
// lane), all arithmetic in fp32. The backward's groups walk many rows with
// the weight gradients of their columns in registers; a workgroup adds its
// groups' in LDS and writes one slice of partial sums, and a second kernel
// adds the slices in a fixed order (no atomics: the same bits every time).
// Measured (a large copy: 5.15 TB/s): 38400 x 768 bf16 with the residual sum, forward 43 us (5.5 TB/s of the four
// arrays), backward 53 + 5 us (4.4); 32961 x 1027 fp32, forward 51 us (5.3), backward 79 + 6 us (5.1).
#include "lik_enc.h"

namespace lik {
namespace enc {
namespace {

struct NormP {
  const char* x;
  const char* r;  // residual; null: none
  const void* w;
  const void* b;  // null: none
  char* y;
  char* s;        // stored sum; null without a residual
  float* stat;    // [rows][2] mean, rstd; null: not kept
  const char* gy;
  const char* gs;  // gradient of the stored sum; null: none
  char* gx;
  float* part;     // [workgroups][2][d] partial sums of gw and gb
  int64_t rows, x_sr, r_sr, gy_sr, gs_sr;  // row strides in bytes
  int d;
  int wf32;  // weights are fp32 (else the type of x)
  float eps;
};

// One lane's chunk c of a row: V elements from column c * V. TAIL: the chunk may
// reach past d (only a lane's last one can), zeros there.
// Rows may start on any element: the 16-byte access is left to the hardware.
template <int EK, bool NT, bool TAIL>
__device__ __forceinline__ void load_chunk(const char* row, int c, int d, float* v) {
  constexpr int V = El<EK>::V, B = El<EK>::B;
  const int e0 = c * V;
  if (!TAIL || e0 + V <= d) {
    typedef u32x4 __attribute__((aligned(2))) u32x4_u;
    const u32x4 t = NT ? (u32x4)__builtin_nontemporal_load((const u32x4_u*)(row + (int64_t)e0 * B))
                       : (u32x4) * (const u32x4_u*)(row + (int64_t)e0 * B);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (EK == EK_F32) v[i] = __uint_as_float(t[i]);
      else unpack2<EK>(t[i], v[2 * i], v[2 * i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      v[i] = 0.f;
      if (e0 + i < d) {
        if constexpr (EK == EK_F32) v[i] = ((const float*)row)[e0 + i];
        else v[i] = el_to_f32<EK>(((const uint16_t*)row)[e0 + i]);
      }
    }
  }
}
template <int EK, bool TAIL>
__device__ __forceinline__ void store_chunk(char* row, int c, int d, const float* v) {
  constexpr int V = El<EK>::V, B = El<EK>::B;
  const int e0 = c * V;
  if (!TAIL || e0 + V <= d) {
    typedef u32x4 __attribute__((aligned(2))) u32x4_u;
    u32x4 t;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (EK == EK_F32) t[i] = __float_as_uint(v[i]);
      else t[i] = pack2<EK>(v[2 * i], v[2 * i + 1]);
    }
    *(u32x4_u*)(row + (int64_t)e0 * B) = t;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (e0 + i < d) {
        if constexpr (EK == EK_F32) ((float*)row)[e0 + i] = v[i];
        else ((uint16_t*)row)[e0 + i] = (uint16_t)f32_to_el<EK>(v[i]);
      }
  }
}
// V weights from column c * V, in the type of x or fp32
template <int EK, bool TAIL>
__device__ __forceinline__ void load_weights(const void* w, bool wf32, int c, int d, float* v) {
  constexpr int V = El<EK>::V;
  if (EK == EK_F32 || wf32) {
#pragma unroll
    for (int h = 0; h < V / 4; ++h) load_chunk<EK_F32, false, TAIL>((const char*)w, c * (V / 4) + h, d, v + 4 * h);
  } else {
    load_chunk<EK, false, TAIL>((const char*)w, c, d, v);
  }
}
// f(j, last): the chunks of a lane; only the last one can reach past the row.
template <int NV, typename F>
__device__ __forceinline__ void each_chunk(F f) {
#pragma unroll
  for (int j = 0; j < NV - 1; ++j) f(j, std::false_type{});
  f(NV - 1, std::true_type{});
}
// A row's chunks into v, zeros past d.
template <int EK, int LPR, int NV>
__device__ __forceinline__ void load_row(const char* row, int lane, int d, float (*v)[El<EK>::V]) {
  each_chunk<NV>([&](int j, auto last) { load_chunk<EK, true, decltype(last)::value>(row, j * LPR + lane, d, v[j]); });
}
template <int EK, int LPR, int NV>
__device__ __forceinline__ void store_row(char* row, int lane, int d, const float (*v)[El<EK>::V]) {
  each_chunk<NV>([&](int j, auto last) { store_chunk<EK, decltype(last)::value>(row, j * LPR + lane, d, v[j]); });
}

template <int CTRL>
__device__ __forceinline__ float dpp_add(float a) {
  const int x = __builtin_bit_cast(int, a);
  return a + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(x, x, CTRL, 0xf, 0xf, false));
}
// Sum of a over the LPR lanes of a row, on every lane: within 16 lanes by data-parallel moves (each lane adds the
// one opposite it), across them by the row and half swaps. LPR = 256: the four wavefronts meet in LDS (s_red has
// 2 slots of 4 floats, used in turn).
template <int LPR>
__device__ __forceinline__ float row_sum(float a, float* s_red, int slot) {
  a = dpp_add<0xb1>(a);   // lanes 1, 0, 3, 2 of each four
  a = dpp_add<0x4e>(a);   // lanes 2, 3, 0, 1
  a = dpp_add<0x141>(a);  // mirrored in eight
  a = dpp_add<0x140>(a);  // mirrored in sixteen
  if constexpr (LPR >= 32) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(a), false, false);
    a = __uint_as_float((uint32_t)s[0]) + __uint_as_float((uint32_t)s[1]);
  }
  if constexpr (LPR >= 64) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(a), false, false);
    a = __uint_as_float((uint32_t)s[0]) + __uint_as_float((uint32_t)s[1]);
  }
  if constexpr (LPR == 256) {
    const int wv = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) s_red[slot * 4 + wv] = a;
    __syncthreads();
    a = (s_red[slot * 4] + s_red[slot * 4 + 1]) + (s_red[slot * 4 + 2] + s_red[slot * 4 + 3]);
  }
  return a;
}

template <int EK, int LPR, int NV>
__global__ void __launch_bounds__(256) layer_norm_kernel(const NormP p) {
  constexpr int V = El<EK>::V, RPW = 256 / LPR;
  __shared__ float s_red[8];
  const int g = threadIdx.x / LPR, lane = threadIdx.x % LPR;
  const float inv_d = 1.0f / (float)p.d;
  // (LPR = 256: one row a workgroup, so every thread takes part in each barrier)
  for (int64_t row = (int64_t)blockIdx.x * RPW + g; row < p.rows; row += (int64_t)gridDim.x * RPW) {
    float v[NV][V];
    load_row<EK, LPR, NV>(p.x + row * p.x_sr, lane, p.d, v);
    if (p.r) {
      float t[NV][V];
      load_row<EK, LPR, NV>(p.r + row * p.r_sr, lane, p.d, t);
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) v[j][i] = el_to_f32<EK>(f32_to_el<EK>(v[j][i] + t[j][i]));
      store_row<EK, LPR, NV>(p.s + row * (int64_t)p.d * El<EK>::B, lane, p.d, v);
    }
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) sum += v[j][i];
    const float mean = row_sum<LPR>(sum, s_red, 0) * inv_d;
    float sq = 0.f;
    each_chunk<NV>([&](int j, auto last) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float t = !decltype(last)::value || (j * LPR + lane) * V + i < p.d ? v[j][i] - mean : 0.f;
        sq = fmaf(t, t, sq);
      }
    });
    const float rstd = 1.0f / sqrtf(row_sum<LPR>(sq, s_red, 1) * inv_d + p.eps);
    if (p.stat && lane == 0) {
      p.stat[2 * row] = mean;
      p.stat[2 * row + 1] = rstd;
    }
    each_chunk<NV>([&](int j, auto last) {
      constexpr bool TAIL = decltype(last)::value;
      const int c = j * LPR + lane;
      float w[V], b[V];
      load_weights<EK, TAIL>(p.w, p.wf32, c, p.d, w);
      if (p.b) load_weights<EK, TAIL>(p.b, p.wf32, c, p.d, b);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float u = (v[j][i] - mean) * rstd;
        w[i] = p.b ? fmaf(u, w[i], b[i]) : u * w[i];
      }
      store_chunk<EK, TAIL>(p.y + row * (int64_t)p.d * El<EK>::B, c, p.d, w);
    });
    if constexpr (LPR == 256) __syncthreads();
  }
}

// Workgroups of the backward a CU: what the registers of NV chunks of V values allow.
template <int EK, int NV>
constexpr int kBwdWgs = NV * El<EK>::V <= 24 ? 3 : 2;

template <int EK, int LPR, int NV>
__global__ void __launch_bounds__(256, (kBwdWgs<EK, NV>)) layer_norm_bwd_kernel(const NormP p) {
  constexpr int V = El<EK>::V, RPW = 256 / LPR;
  __shared__ float s_red[8];
  extern __shared__ float s_col[];  // [2][LPR * NV * V] column sums of the workgroup (LPR < 256)
  const int g = threadIdx.x / LPR, lane = threadIdx.x % LPR;
  const float inv_d = 1.0f / (float)p.d;
  float gw[NV][V], gb[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) gw[j][i] = gb[j][i] = 0.f;
  for (int64_t row = (int64_t)blockIdx.x * RPW + g; row < p.rows; row += (int64_t)gridDim.x * RPW) {
    float v[NV][V], t[NV][V];
    load_row<EK, LPR, NV>(p.x + row * p.x_sr, lane, p.d, v);
    load_row<EK, LPR, NV>(p.gy + row * p.gy_sr, lane, p.d, t);
    const float mean = p.stat[2 * row], rstd = p.stat[2 * row + 1];
    float c1 = 0.f, c2 = 0.f;
    each_chunk<NV>([&](int j, auto last) {
      float w[V];
      load_weights<EK, decltype(last)::value>(p.w, p.wf32, j * LPR + lane, p.d, w);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        // past d: t = 0, so neither sum nor gradient sees the value of u
        const float u = (v[j][i] - mean) * rstd;
        gw[j][i] = fmaf(t[j][i], u, gw[j][i]);
        gb[j][i] += t[j][i];
        t[j][i] *= w[i];
        c1 += t[j][i];
        c2 = fmaf(t[j][i], u, c2);
        v[j][i] = u;
      }
    });
    c1 = row_sum<LPR>(c1, s_red, 0) * inv_d;
    c2 = row_sum<LPR>(c2, s_red, 1) * inv_d;
    each_chunk<NV>([&](int j, auto last) {
      constexpr bool TAIL = decltype(last)::value;
      const int c = j * LPR + lane;
      float o[V];
      if (p.gs) load_chunk<EK, true, TAIL>(p.gs + row * p.gs_sr, c, p.d, o);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float q = rstd * (t[j][i] - c1 - v[j][i] * c2);
        o[i] = p.gs ? o[i] + q : q;
      }
      store_chunk<EK, TAIL>(p.gx + row * (int64_t)p.d * El<EK>::B, c, p.d, o);
    });
    if constexpr (LPR == 256) __syncthreads();
  }
  float* out = p.part + (int64_t)blockIdx.x * 2 * p.d;
  if constexpr (LPR == 256) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int e = (j * LPR + lane) * V + i;
        if (e < p.d) {
          out[e] = gw[j][i];
          out[p.d + e] = gb[j][i];
        }
      }
  } else {
    constexpr int W = LPR * NV * V;
    for (int k = 0; k < RPW; ++k) {  // the groups in turn, so that the order of the sums is fixed
      if (g == k)
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const int e = (j * V + i) * LPR + lane;  // lane-major: no bank conflicts
            s_col[e] = k ? s_col[e] + gw[j][i] : gw[j][i];
            s_col[W + e] = k ? s_col[W + e] + gb[j][i] : gb[j][i];
          }
      __syncthreads();
    }
    for (int e = threadIdx.x; e < p.d; e += 256) {
      const int c = e / V, at = ((c / LPR) * V + e % V) * LPR + c % LPR;
      out[e] = s_col[at];
      out[p.d + e] = s_col[W + at];
    }
  }
}

// gw[e] / gb[e]: the sum of the workgroups' slices. 64 columns a workgroup,
// its 16 wavefronts each add every 16th slice, then their sums in order.
template <int EK>
__global__ void __launch_bounds__(1024) norm_grads_kernel(const float* part, int slices, int d, int wf32, void* gw,
                                                          void* gb) {
  __shared__ float s[16][64];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int e = blockIdx.x * 64 + lane;  // column of [gw, gb]
  float a = 0.f;
  if (e < 2 * d)
#pragma unroll 8
    for (int k = wv; k < slices; k += 16) a += part[(int64_t)k * 2 * d + e];
  s[wv][lane] = a;
  __syncthreads();
  if (wv == 0 && e < 2 * d) {
    for (int k = 1; k < 16; ++k) a += s[k][lane];
    void* out = e < d ? gw : gb;
    const int at = e < d ? e : e - d;
    if (out) {
      if (EK == EK_F32 || wf32) ((float*)out)[at] = a;
      else ((uint16_t*)out)[at] = (uint16_t)f32_to_el<EK>(a);
    }
  }
}

constexpr int kNormMaxDim = 8192;  // 256 lanes x 32 values in registers
constexpr int kNormBwdMost = 3 * 256;  // workgroups of the backward: one round of the CUs

// slices: the workgroups whose partial sums a backward leaves.
template <int EK, bool BWD, int LPR, int NV>
int launch_norm_one(const NormP& p, hipStream_t s, int& slices) {
  const int64_t rpw = 256 / LPR, need = (p.rows + rpw - 1) / rpw;  // steps of the whole call
  int64_t wgs = need < (1 << 20) ? need : (1 << 20);
  if constexpr (BWD) {
    // one round of the CUs, the steps dealt out evenly (a partial round of workgroups or steps leaves CUs idle:
    // 38400 x 768 bf16 58 us against 73 with 768 workgroups of 6 or 7 steps)
    const int64_t most = 256 * kBwdWgs<EK, NV>, each = (need + most - 1) / most;
    wgs = (need + each - 1) / each;
    slices = (int)wgs;
    const uint32_t lds = LPR == 256 ? 0u : (uint32_t)(2 * LPR * NV * El<EK>::V * 4);
    launch_kernel(layer_norm_bwd_kernel<EK, LPR, NV>, dim3((unsigned)wgs), dim3(256), lds, s, p);
  } else {
    launch_kernel(layer_norm_kernel<EK, LPR, NV>, dim3((unsigned)wgs), dim3(256), 0u, s, p);
  }
  return hipGetLastError() == hipSuccess ? LIK_OK : LIK_ERR_LAUNCH;
}

// Lanes of a row: the fewest that hold it in up to four 16-byte chunks each
// (more rows per wavefront and shorter sums), in up to 32 values each for the
// longer rows. NV = chunks / lanes rounded up, so that only a lane's last chunk can
// reach past the row.
int norm_lanes(int chunks, int v) {
  return chunks <= 64 ? 16 : chunks <= 128 ? 32 : chunks <= 64 * 32 / v ? 64 : 256;
}
template <int EK, bool BWD, int LPR, int LO, int HI>
int launch_norm_nv(const NormP& p, int nv, hipStream_t s, int& slices) {
  if constexpr (LO < HI) {
    if (nv > LO) return launch_norm_nv<EK, BWD, LPR, LO + 1, HI>(p, nv, s, slices);
  }
  return launch_norm_one<EK, BWD, LPR, LO>(p, s, slices);
}

template <int EK, bool BWD>
int launch_norm(const NormP& p, hipStream_t s, int& slices) {
  constexpr int V = El<EK>::V, MOST = 32 / V;
  const int chunks = (p.d + V - 1) / V;
  const int lpr = norm_lanes(chunks, V), nv = (chunks + lpr - 1) / lpr;
  if (lpr == 16) return launch_norm_nv<EK, BWD, 16, 1, 4>(p, nv, s, slices);
  if (lpr == 32) return launch_norm_nv<EK, BWD, 32, 3, 4>(p, nv, s, slices);
  if (lpr == 64) return launch_norm_nv<EK, BWD, 64, 3, MOST>(p, nv, s, slices);
  return launch_norm_nv<EK, BWD, 256, MOST / 4 + 1, MOST>(p, nv, s, slices);
}

// d and the types in range
int norm_check(int32_t dtype, int32_t wdtype, int64_t rows, int64_t d) {
  if (dtype != LIK_BF16 && dtype != LIK_F16 && dtype != LIK_F32) return LIK_ERR_UNSUPPORTED;
  if (wdtype != dtype && wdtype != LIK_F32) return LIK_ERR_UNSUPPORTED;
  if (rows < 0 || d < 1) return LIK_ERR_INVALID;
  return d <= kNormMaxDim ? LIK_OK : LIK_ERR_UNSUPPORTED;
}

// every array (null: not there) starts on one of its elements
template <typename... P>
bool on_element(int64_t size, P... p) {
  return (... && ((uintptr_t)p % (uintptr_t)size == 0));
}

template <bool BWD>
int norm_run(const NormP& p, int32_t dtype, hipStream_t s, int& slices) {
  if (dtype == LIK_BF16) return launch_norm<EK_BF16, BWD>(p, s, slices);
  if (dtype == LIK_F16) return launch_norm<EK_F16, BWD>(p, s, slices);
  return launch_norm<EK_F32, BWD>(p, s, slices);
}

}  // namespace
}  // namespace enc
}  // namespace lik

using namespace lik;
using namespace lik::enc;

extern "C" {

int lik_layer_norm(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, int32_t dtype,
                   int64_t rows, int32_t dim, const void* weight, const void* bias, int32_t weight_dtype, float eps,
                   void* y, void* sum, float* stats, lik_stream_t stream) {
  if (const int rc = norm_check(dtype, weight_dtype, rows, dim)) return rc;
  if (rows == 0) return LIK_OK;
  if (!x || !weight || !y || (residual && !sum)) return LIK_ERR_INVALID;
  const int64_t e = dtype == LIK_F32 ? 4 : 2, we = weight_dtype == LIK_F32 ? 4 : 2;
  if (!on_element(e, x, residual, y, sum) || !on_element(we, weight, bias) || !on_element(4, stats))
    return LIK_ERR_UNSUPPORTED;
  NormP p{};
  p.x = (const char*)x;
  p.x_sr = x_stride * e;
  p.r = (const char*)residual;
  p.r_sr = residual_stride * e;
  p.rows = rows;
  p.d = dim;
  p.w = weight;
  p.b = bias;
  p.wf32 = weight_dtype == LIK_F32;
  p.eps = eps;
  p.y = (char*)y;
  p.s = (char*)sum;
  p.stat = stats;
  int none = 0;
  return norm_run<false>(p, dtype, (hipStream_t)stream, none);
}

size_t lik_layer_norm_backward_workspace_size(int32_t dtype, int64_t rows, int32_t dim) {
  if (norm_check(dtype, dtype, rows, dim) != LIK_OK || rows == 0) return 0;
  const int64_t wgs = rows < kNormBwdMost ? rows : kNormBwdMost;  // (at least a row each)
  return (size_t)wgs * 2 * (size_t)dim * 4 + 256;
}

int lik_layer_norm_backward(const void* grad_y, int64_t grad_y_stride, const void* grad_sum, int64_t grad_sum_stride,
                            const void* sum, int64_t sum_stride, const float* stats, int32_t dtype, int64_t rows,
                            int32_t dim, const void* weight, int32_t weight_dtype, void* grad_x, void* grad_weight,
                            void* grad_bias, void* workspace, size_t workspace_bytes, lik_stream_t stream) {
  if (const int rc = norm_check(dtype, weight_dtype, rows, dim)) return rc;
  if (rows == 0) return grad_weight || grad_bias ? LIK_ERR_INVALID : LIK_OK;  // the weights' would stay unwritten
  if (!grad_y || !sum || !stats || !weight || !grad_x) return LIK_ERR_INVALID;
  if (!workspace || workspace_bytes < lik_layer_norm_backward_workspace_size(dtype, rows, dim))
    return LIK_ERR_WORKSPACE;
  const int64_t e = dtype == LIK_F32 ? 4 : 2, we = weight_dtype == LIK_F32 ? 4 : 2;
  if (!on_element(e, grad_y, grad_sum, sum, grad_x) || !on_element(we, weight, grad_weight, grad_bias) ||
      !on_element(4, stats))
    return LIK_ERR_UNSUPPORTED;
  NormP p{};
  p.x = (const char*)sum;
  p.x_sr = sum_stride * e;
  p.gy = (const char*)grad_y;
  p.gy_sr = grad_y_stride * e;
  p.gs = (const char*)grad_sum;
  p.gs_sr = grad_sum_stride * e;
  p.rows = rows;
  p.d = dim;
  p.w = weight;
  p.wf32 = weight_dtype == LIK_F32;
  p.stat = const_cast<float*>(stats);
  p.gx = (char*)grad_x;
  p.part = (float*)align256(workspace);
  const hipStream_t s = (hipStream_t)stream;
  int slices = 0;
  if (const int rc = norm_run<true>(p, dtype, s, slices)) return rc;
  if (grad_weight || grad_bias) {
    const dim3 grid((unsigned)((2 * dim + 63) / 64)), block(1024);
    if (dtype == LIK_BF16)
      launch_kernel(norm_grads_kernel<EK_BF16>, grid, block, 0u, s, p.part, slices, dim, p.wf32, grad_weight, grad_bias);
    else if (dtype == LIK_F16)
      launch_kernel(norm_grads_kernel<EK_F16>, grid, block, 0u, s, p.part, slices, dim, p.wf32, grad_weight, grad_bias);
    else
      launch_kernel(norm_grads_kernel<EK_F32>, grid, block, 0u, s, p.part, slices, dim, p.wf32, grad_weight, grad_bias);
    if (hipGetLastError() != hipSuccess) return LIK_ERR_LAUNCH;
  }
  return LIK_OK;
}

}  // extern "C"
