// Token vectors as 8-bit integers with a scale each, and back (the definition: lik_int8.h).
//
// Bound by HBM: a row stays in the registers of its lanes between the maximum and the conversion, so each
// element is read once and one byte written; rows past 16384 elements (fp32: 8192) are read twice, the second
// time from L2. Measured: 1,030,001 rows of 128 fp16 to integers 67 us (6.0 TB/s), back 68 us (5.9); 44801 rows of 1152 bf16 to
// integers 29 us (5.3); 32961 rows of 1027 fp32, which start off 16 bytes, 40 us (4.2) and 27 us (6.2).
#include "lik_int8.h"

namespace lik {
namespace enc {
namespace {

struct QuantP {
  const char* x;
  int64_t x_ld;  // bytes
  int64_t rows;
  int dim, end;  // end: bytes of a row that are written
  int8_t* out;
  int64_t out_ld;
  float* scale;
  bool stream;
};

template <int V>
__device__ __forceinline__ void store_int8(int8_t* row, int e, int end, const uint32_t* w) {
  typedef uint32_t __attribute__((aligned(1))) u32_u;
  typedef u32x2 __attribute__((aligned(1))) u32x2_u;
  if (e + V <= end) {
    if constexpr (V == 8) *(u32x2_u*)(row + e) = u32x2{w[0], w[1]};
    else *(u32_u*)(row + e) = w[0];
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (e + i < end) row[e + i] = (int8_t)(w[i / 4] >> (i % 4 * 8));
}

// LPR lanes a row with NV chunks each in registers, U rows at once. Only a lane's last chunk can reach past the row.
// NT: rows are read past the caches.
template <int EK, int LPR, int NV, int U, bool NT>
__global__ void __launch_bounds__(256) quantize_kernel(const QuantP p) {
  constexpr int V = El<EK>::V, RPW = 64 / LPR;
  const int lane = threadIdx.x % LPR, g = threadIdx.x % 64 / LPR;
  const int whole = p.dim / V;
  const int64_t first = (threadIdx.x / 64) * (RPW * U) + g, step = (int64_t)gridDim.x * (4 * RPW * U);
  for (int64_t b = (int64_t)blockIdx.x * (4 * RPW * U); b < p.rows; b += step) {
    const int64_t r0 = b + first;
    u32x4 w[U][NV];
    // every lane loads: rows and chunks past the end name the last ones
    if (whole)
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          typedef u32x4 __attribute__((aligned(2))) u32x4_u;
          const int64_t r = r0 + u * RPW < p.rows ? r0 + u * RPW : p.rows - 1;
          const int c = j * LPR + lane;
          const u32x4_u* at = (const u32x4_u*)(p.x + r * p.x_ld) + (j < NV - 1 || c < whole ? c : whole - 1);
          if constexpr (NT) w[u][j] = __builtin_nontemporal_load(at);
          else w[u][j] = *at;
        }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if ((NV - 1) * LPR + lane >= whole) w[u][NV - 1] = u32x4{0u, 0u, 0u, 0u};
    if (p.dim % V && (NV - 1) * LPR + lane == whole) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r0 + u * RPW < p.rows) chunk_load<EK>(p.x + (r0 + u * RPW) * p.x_ld, whole * V, p.dim, w[u][NV - 1]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < NV; ++j) m = absmax_bits<EK>(w[u][j], m);
      m = absmax_lanes<EK, LPR>(m);
      float s, inv;
      row_scale<EK>(m, s, inv);
      const int64_t r = r0 + u * RPW;
      if (r >= p.rows) continue;
      if (lane == 0) p.scale[r] = s;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        uint32_t q[V / 4];
        chunk_to_int8<EK>(w[u][j], s, inv, q);
        store_int8<V>(p.out + r * p.out_ld, (j * LPR + lane) * V, p.end, q);
      }
    }
  }
}

// Wider rows: a workgroup each, NV chunks a thread in registers.
template <int EK, int NV, bool NT>
__global__ void __launch_bounds__(256) quantize_row_kernel(const QuantP p) {
  constexpr int V = El<EK>::V;
  typedef u32x4 __attribute__((aligned(2))) u32x4_u;
  __shared__ uint32_t s_m[4];
  const int whole = p.dim / V;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const char* row = p.x + r * p.x_ld;
    u32x4 w[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = j * 256 + (int)threadIdx.x;
      const u32x4_u* at = (const u32x4_u*)row + (c < whole ? c : whole - 1);
      if constexpr (NT) w[j] = __builtin_nontemporal_load(at);
      else w[j] = *at;
    }
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = j * 256 + (int)threadIdx.x;
      if (c >= whole) w[j] = u32x4{0u, 0u, 0u, 0u};
      if (p.dim % V && c == whole) chunk_load<EK>(row, c * V, p.dim, w[j]);
      m = absmax_bits<EK>(w[j], m);
    }
    m = absmax_lanes<EK, 64>(m);
    if (threadIdx.x % 64 == 0) s_m[threadIdx.x / 64] = m;
    __syncthreads();
    m = absmax_join<EK>(absmax_join<EK>(s_m[0], s_m[1]), absmax_join<EK>(s_m[2], s_m[3]));
    float s, inv;
    row_scale<EK>(m, s, inv);
    if (threadIdx.x == 0) p.scale[r] = s;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      uint32_t q[V / 4];
      chunk_to_int8<EK>(w[j], s, inv, q);
      store_int8<V>(p.out + r * p.out_ld, (j * 256 + (int)threadIdx.x) * V, p.end, q);
    }
    __syncthreads();  // (s_m is the next row's)
  }
}

// Wider still: read twice.
template <int EK>
__global__ void __launch_bounds__(256) quantize_wide_kernel(const QuantP p) {
  constexpr int V = El<EK>::V;
  __shared__ uint32_t s_m[4];
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const char* row = p.x + r * p.x_ld;
    u32x4 w;
    uint32_t m = 0;
    for (int e = threadIdx.x * V; e < p.dim; e += 256 * V) {
      chunk_load<EK>(row, e, p.dim, w);
      m = absmax_bits<EK>(w, m);
    }
    m = absmax_lanes<EK, 64>(m);
    if (threadIdx.x % 64 == 0) s_m[threadIdx.x / 64] = m;
    __syncthreads();
    m = absmax_join<EK>(absmax_join<EK>(s_m[0], s_m[1]), absmax_join<EK>(s_m[2], s_m[3]));
    float s, inv;
    row_scale<EK>(m, s, inv);
    if (threadIdx.x == 0) p.scale[r] = s;
    for (int e = threadIdx.x * V; e < p.end; e += 256 * V) {
      uint32_t q[V / 4];
      chunk_load<EK>(row, e, p.dim, w);
      chunk_to_int8<EK>(w, s, inv, q);
      store_int8<V>(p.out + r * p.out_ld, e, p.end, q);
    }
    __syncthreads();  // (s_m is the next row's)
  }
}

// (a launch has less than 2^32 threads)
unsigned groups(int64_t want) { return (unsigned)(want < (1 << 22) ? want : 1 << 22); }
template <int EK, int LPR, int NV, int U>
void launch_rows(const QuantP& p, hipStream_t s) {
  const int64_t per = 4 * (64 / LPR) * U;
  const dim3 grid(groups((p.rows + per - 1) / per));
  if (p.stream) launch_kernel(quantize_kernel<EK, LPR, NV, U, true>, grid, dim3(256), 0u, s, p);
  else launch_kernel(quantize_kernel<EK, LPR, NV, U, false>, grid, dim3(256), 0u, s, p);
}
template <int EK, int NV>
void launch_row(const QuantP& p, hipStream_t s) {
  if (p.stream) launch_kernel(quantize_row_kernel<EK, NV, true>, dim3(groups(p.rows)), dim3(256), 0u, s, p);
  else launch_kernel(quantize_row_kernel<EK, NV, false>, dim3(groups(p.rows)), dim3(256), 0u, s, p);
}
template <int EK>
int launch_quantize(const QuantP& p, hipStream_t s) {
  const int ch = (p.end + El<EK>::V - 1) / El<EK>::V;
  // the fewest chunks a lane: all but its last are whole. Few rows: a wavefront each (32 rows of 768 bf16: 3.5 us, two
  // rows a wavefront 4.2 us)
  if (p.rows <= 1024 && ch <= 64) launch_rows<EK, 64, 1, 1>(p, s);
  else if (p.rows <= 1024 && ch <= 128) launch_rows<EK, 64, 2, 1>(p, s);
  else if (ch <= 16) launch_rows<EK, 16, 1, 4>(p, s);
  else if (ch <= 32) launch_rows<EK, 16, 2, 2>(p, s);
  else if (ch <= 48) launch_rows<EK, 16, 3, 1>(p, s);
  else if (ch <= 64) launch_rows<EK, 16, 4, 1>(p, s);
  else if (ch <= 96) launch_rows<EK, 32, 3, 1>(p, s);
  else if (ch <= 128) launch_rows<EK, 32, 4, 1>(p, s);
  else if (ch <= 192) launch_rows<EK, 64, 3, 1>(p, s);
  else if (ch <= 256) launch_rows<EK, 64, 4, 1>(p, s);
  else if (ch <= 320) launch_rows<EK, 64, 5, 1>(p, s);
  else if (ch <= 384) launch_rows<EK, 64, 6, 1>(p, s);
  else if (ch <= 448) launch_rows<EK, 64, 7, 1>(p, s);
  else if (ch <= 512) launch_rows<EK, 64, 8, 1>(p, s);
  else if (ch <= 1024) launch_row<EK, 4>(p, s);
  else if (ch <= 2048) launch_row<EK, 8>(p, s);
  else launch_kernel(quantize_wide_kernel<EK>, dim3(groups(p.rows)), dim3(256), 0u, s, p);
  return hipGetLastError() == hipSuccess ? LIK_OK : LIK_ERR_LAUNCH;
}

struct DequantP {
  const int8_t* x;
  int64_t x_ld, rows;
  const float* scale;
  int dim;
  char* out;
};

// LPR lanes a row, U rows and NC chunks of V elements at once, so that neighbouring lanes write neighbouring 16 bytes.
// (A thread with 16 elements of its own instead: 32961 x 1027 fp32 58 us, now 27; stores past the caches: 1,030,001 rows of 128 fp16
// there and back 188 us instead of 154, both with the rows read through the caches.) The product is rounded to fp32, then
// to the output's type: half a step of it and 2^-24. A single rounding would differ in 6 of 100,000 fp16 values.
template <int EK, int LPR, int NC, int U>
__global__ void __launch_bounds__(256) dequantize_kernel(const DequantP p) {
  constexpr int B = El<EK>::B, V = El<EK>::V, RPW = 64 / LPR, W = V / 4;
  typedef uint32_t __attribute__((aligned(1))) u32_u;
  typedef u32x2 __attribute__((aligned(1))) u32x2_u;
  const int lane = threadIdx.x % LPR, g = threadIdx.x % 64 / LPR, whole = p.dim / V;
  const int64_t first = (threadIdx.x / 64) * (RPW * U) + g, step = (int64_t)gridDim.x * (4 * RPW * U);
  for (int64_t b = (int64_t)blockIdx.x * (4 * RPW * U); b < p.rows; b += step) {
    const int64_t r0 = b + first;
    float s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) s[u] = p.scale[r0 + u * RPW < p.rows ? r0 + u * RPW : p.rows - 1];
    for (int c0 = 0; c0 < whole; c0 += LPR * NC) {
      uint32_t w[U][NC][W];
      // every lane loads: rows and chunks past the end name the last ones
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < NC; ++j) {
          const int64_t r = r0 + u * RPW < p.rows ? r0 + u * RPW : p.rows - 1;
          const int c = c0 + j * LPR + lane;
          const int8_t* in = p.x + r * p.x_ld + (c < whole ? c : whole - 1) * V;
          if constexpr (W == 2) {
            const u32x2 t = *(const u32x2_u*)in;
            w[u][j][0] = t[0];
            w[u][j][1] = t[1];
          } else {
            w[u][j][0] = *(const u32_u*)in;
          }
        }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < NC; ++j) {
          const int c = c0 + j * LPR + lane;
          float v[V];
#pragma unroll
          for (int k = 0; k < V; ++k) v[k] = s[u] * (float)(int8_t)(w[u][j][k / 4] >> (k % 4 * 8));
          if (r0 + u * RPW < p.rows && c < whole)
            chunk_store<EK, true>(p.out + (r0 + u * RPW) * ((int64_t)p.dim * B), c * V, p.dim, chunk_narrow<EK>(v));
        }
    }
    if (whole * V + lane < p.dim)  // (V <= LPR)
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r0 + u * RPW < p.rows) {
          const int64_t r = r0 + u * RPW;
          const int e = whole * V + lane;
          const float v = s[u] * (float)p.x[r * p.x_ld + e];
          if constexpr (EK == EK_F32) ((float*)p.out)[r * p.dim + e] = v;
          else ((uint16_t*)p.out)[r * p.dim + e] = (uint16_t)f32_to_el<EK>(v);
        }
  }
}
template <int EK>
int launch_dequantize(const DequantP& p, hipStream_t s) {
  const int ch = (p.dim + El<EK>::V - 1) / El<EK>::V;
  if (ch <= 32)  // 4 rows a wavefront, 4 times
    launch_kernel(dequantize_kernel<EK, 16, 1, 4>, dim3(groups((p.rows + 63) / 64)), dim3(256), 0u, s, p);
  else  // a wavefront each
    launch_kernel(dequantize_kernel<EK, 64, 4, 1>, dim3(groups((p.rows + 3) / 4)), dim3(256), 0u, s, p);
  return hipGetLastError() == hipSuccess ? LIK_OK : LIK_ERR_LAUNCH;
}

int rows_check(int32_t dtype, int64_t rows, int32_t dim) {
  if (dtype != LIK_BF16 && dtype != LIK_F16 && dtype != LIK_F32) return LIK_ERR_UNSUPPORTED;
  if (rows < 0 || dim < 1) return LIK_ERR_INVALID;
  if (dim > (1 << 24) || rows > (1ll << 40)) return LIK_ERR_UNSUPPORTED;
  return LIK_OK;
}

}  // namespace

int quantize_rows_int8(const void* x, int64_t x_stride, int32_t dtype, int64_t rows, int32_t dim, int8_t* out,
                       int64_t out_stride, float* scale, bool stream, hipStream_t s) {
  if (const int rc = rows_check(dtype, rows, dim)) return rc;
  if (rows == 0) return LIK_OK;
  if (!x || !out || !scale || out_stride < dim) return LIK_ERR_INVALID;
  const int eb = dtype == LIK_F32 ? 4 : 2;
  if ((uintptr_t)x % eb || (uintptr_t)scale % 4) return LIK_ERR_UNSUPPORTED;
  if ((const void*)out == x) return LIK_ERR_INVALID;  // (a row's integers lie where others' elements do)
  const int64_t end = (dim + 15) / 16 * 16;
  const QuantP p{(const char*)x, x_stride * eb, rows, dim, (int)(end < out_stride ? end : out_stride), out, out_stride,
                 scale, stream};
  switch (dtype) {
    case LIK_BF16: return launch_quantize<EK_BF16>(p, s);
    case LIK_F16: return launch_quantize<EK_F16>(p, s);
    default: return launch_quantize<EK_F32>(p, s);
  }
}

}  // namespace enc
}  // namespace lik

using namespace lik;
using namespace lik::enc;

extern "C" {

int lik_quantize_int8(const void* x, int64_t x_stride, int32_t dtype, int64_t rows, int32_t dim, int8_t* out,
                      int64_t out_stride, float* scale, lik_stream_t stream) {
  return quantize_rows_int8(x, x_stride, dtype, rows, dim, out, out_stride, scale, true, (hipStream_t)stream);
}

int lik_dequantize_int8(const int8_t* x, int64_t x_stride, const float* scale, int32_t dtype, int64_t rows, int32_t dim,
                        void* out, lik_stream_t stream) {
  if (const int rc = rows_check(dtype, rows, dim)) return rc;
  if (rows == 0) return LIK_OK;
  if (!x || !out || !scale) return LIK_ERR_INVALID;
  if ((uintptr_t)out % (dtype == LIK_F32 ? 4 : 2) || (uintptr_t)scale % 4) return LIK_ERR_UNSUPPORTED;
  if (out == (const void*)x) return LIK_ERR_INVALID;
  const DequantP p{x, x_stride, rows, scale, dim, (char*)out};
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case LIK_BF16: return launch_dequantize<EK_BF16>(p, s);
    case LIK_F16: return launch_dequantize<EK_F16>(p, s);
    default: return launch_dequantize<EK_F32>(p, s);
  }
}

}  // extern "C"
