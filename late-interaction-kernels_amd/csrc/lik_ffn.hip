// Gated feed-forward block: y = (act(x Wg^T) * (x Wu^T)) Wo^T + residual, and
// its gradients. Wg and Wu are the first and the last `hidden` rows of w_in.
//
// Five matrix products on one tile kernel, out[m][n] = sum_k A(m, k) B(n, k):
//   forward   h = act(x Wg^T) * (x Wu^T)   A, B along k;  gate and up rows of one
//                                          column meet in one lane's registers
//             y = h Wo^T + residual        A, B along k
//   backward  dh = gy Wo                   B across k; the epilogue turns dh into
//             dg = dh u act'(g), du = dh act(g), side by side as [rows][2 hidden]
//             dx = [dg du] [Wg; Wu]        B across k
//             dw_in = [dg du]^T x, dw_out = gy^T h   A and B across k, k = rows
// Sums over k are fp32 (MFMA accumulators, fp32 partial sums where k is split). h, dg and du are rounded
// once to the 16-bit type, as the next product's operands have to be. g and u are kept for the backward so
// that dg and du carry next to no other rounding, at any size: of bf16 calls the upper 20 bits of the fp32 value
// (12 significant bits against the 8 of dg and du), of fp16 calls fp32.
// fp16 has no range for dg and du of any gy (nor for large inputs): they are held s times, s the power of two that brings a
// bound of theirs to 2^14 .. 2^15, d max|gy| max|Wo| max(|u| max|act'|, |act(g)|), and dx and dw_in are scaled back. The last factor
// comes from the forward, a value a kept block; a kernel finds the others. The bound is some 2^7 to 2^12 above the largest
// elements, which leaves 17 powers of two of normal numbers below those.
#include "lik_act.h"

namespace lik {
namespace enc {
namespace {

enum { EPI_STORE = 0, EPI_GLU = 1, EPI_GLU_BWD = 2 };

struct GemmP {
  const char* a;  // A(m, k): m * a_ld + k, or across k: k * a_ld + m (elements of 2 bytes)
  const char* b;
  int64_t a_ld, b_ld;  // bytes
  int m, n, k;
  int tiles_n, full;   // the first `full` tiles are one workgroup's each,
  int tail, splits;    // the `tail` others are `splits` workgroups' each,
  int k_per;           // of k_per (a multiple of 64) of k
  float* part;         // their sums [tail][splits][a tile in the accumulators' order]
  char* out;           // [m][n] 16-bit, row stride out_ld bytes; EPI_GLU_BWD: [m][2 hidden]
  int64_t out_ld;
  const char* res;     // EPI_STORE: added before the rounding; null: none
  int64_t res_ld;
  char* gu;            // EPI_GLU: kept g and u (null: not kept), KeptBlock; EPI_GLU_BWD: read
  int hidden;
  int act;
  float* bound;        // fp16, EPI_GLU with gu: [blocks][2] largest factors of dg and du (blocks of 16 columns: one each)
  const float* scale;  // fp16, null: 1. EPI_GLU_BWD: dg and du are held as many times; EPI_STORE: the sums are multiplied by it
};

// One operand's tile of T rows (m or n) by 64 k in LDS, 128 bytes a row of T:
// along k: [T][64], 8 chunks a row; across k: [64][T], T / 8 chunks a row.
constexpr int BK = 64;

template <int T, bool X, int NW>
struct Stage {
  static constexpr int BYTES = T * BK * 2;
  static constexpr int NI = BYTES / 1024 / NW;  // 1 KB loads of a wavefront
  static_assert(BYTES % (1024 * NW) == 0 && T % 128 == 0, "");

  // 16-byte chunk c of row r lies at chunk c ^ swz(r), so that reads cover the 64 banks evenly: along
  // k 16 consecutive rows (two to 256 bytes) at one chunk; across k (rows of whole 256 bytes) four
  // consecutive rows at 64 bytes each.
  __device__ __forceinline__ static int swz(int r) { return X ? (r & 3) << 2 : (r >> 1) & 7; }
  // Lane offsets of the wavefront's loads from the tile's origin, kOob past the matrix' edge.
  // `rows`: rows (along k) or columns (across k) the tile has; glu: rows 32..63 of each 64 are up rows.
  __device__ __forceinline__ static void offsets(uint32_t* off, int wv, int lane, int64_t ld, int rows, bool glu,
                                                 int hidden) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int slot = (wv * NI + i) * 64 + lane;
      if constexpr (X) {
        const int r = slot / (T / 8), c = (slot % (T / 8)) ^ swz(r);
        off[i] = c * 8 < rows ? (uint32_t)(r * ld + c * 16) : kOob;
      } else {
        const int r = slot / 8, c = (slot % 8) ^ swz(r);
        const int at = glu ? (r / 64) * 32 + r % 32 : r;
        off[i] = at < rows ? (uint32_t)((at + (glu && (r & 32) ? (int64_t)hidden : 0)) * ld + c * 16) : kOob;
      }
    }
  }
  // load i of a step of which k_left k exist (at most BK)
  __device__ __forceinline__ static void issue(uint32_t lds, const uint32_t* off, int i, int wv, int lane,
                                               const u32x4& desc, int k_left) {
    uint32_t o = off[i];
    if (k_left < BK) {
      const int slot = (wv * NI + i) * 64 + lane;
      if constexpr (X) {
        if (slot / (T / 8) >= k_left) o = kOob;
      } else {
        if (((slot % 8) ^ swz(slot / 8)) * 8 >= k_left) o = kOob;
      }
    }
    dma16(lds + (wv * NI + i) * 1024, o, desc);
  }
  // Lane addresses (from the buffer's origin) of the wavefront's MFMA operands: block j is 32 rows from
  // row0 + 32 j, row0 a multiple of 32; lane l has row l % 32, k = 16 ks + 8 (l / 32) + 0..7.
  // Along k: one 16-byte read, a[ks]. Across k: two transposing reads (k + 0..3, k + 4..7), a[j].
  __device__ __forceinline__ static void bases(uint32_t* a, int row0, int lane) {
    const int h = lane >> 5;
    if constexpr (X) {
      const int i = lane & 15, k = 8 * h + (i >> 2);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int col = row0 + 32 * j + (lane & 16) + 4 * (i & 3);
        a[j] = k * (T * 2) + (((col >> 3) ^ swz(k)) << 4) + ((col & 4) << 1);
      }
    } else {
      const int r = row0 + (lane & 31);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) a[ks] = r * 128 + (((ks * 2 + h) ^ swz(r)) << 4);
    }
  }
  __device__ __forceinline__ static u32x4 frag(const uint32_t* a, uint32_t lds, int j, int ks) {
    if constexpr (X) {
      const u32x2 lo = lds_tr(a[j] + lds + ks * 16 * (T * 2)), hi = lds_tr(a[j] + lds + (ks * 16 + 4) * (T * 2));
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    } else {
      return lds_b128(a[ks] + lds + j * 32 * 128);
    }
  }
};

// The inverse of join_halves.
__device__ __forceinline__ u32x4 split_halves(const u32x4& x) {
  const auto s0 = __builtin_amdgcn_permlane32_swap(x[0], x[2], false, false);
  const auto s1 = __builtin_amdgcn_permlane32_swap(x[1], x[3], false, false);
  return u32x4{(uint32_t)s0[0], (uint32_t)s1[0], (uint32_t)s0[1], (uint32_t)s1[1]};
}
template <int EK>
__device__ __forceinline__ void unpack8(const u32x4& x, float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) unpack2<EK>(x[i], v[2 * i], v[2 * i + 1]);
}

// The kept g and u: blocks of 32 rows by 32 hidden columns [rows / 32][hidden / 32], each as the accumulators lie, so that a
// wavefront writes and reads whole KB. bf16: of g, then of u, two KB of 16-bit pieces (quads 0 and 1, 2 and 3 of a lane), then one KB
// with the last 4 bits of both in a byte. fp16: the four quads of g, then of u.
template <int EK>
constexpr int kKeptBlock = EK == EK_BF16 ? 5120 : 8192;
// A lane's 16 bytes in the first KB of the block of row m and column n (multiples of 32 but for the lane's part of m).
template <int EK>
__device__ __forceinline__ char* kept_at(const GemmP& p, int m, int n, int h) {
  const int64_t block = (int64_t)(m >> 5) * ((p.hidden + 31) >> 5) + (n >> 5);
  return p.gu + block * kKeptBlock<EK> + ((m & 31) + 32 * h) * 16;
}
// Bound of |act'|: gelu 1.13, silu 1.10.
constexpr float kSlopeMost = 1.25f;
__device__ __forceinline__ float max_finite(float big, float x) {  // (rows that are not finite are NaN at any scale)
  const float a = fabsf(x);
  return a < INFINITY ? fmaxf(big, a) : big;
}
// The upper 20 bits of an fp32 value (rounded to nearest): 16 of them, and 4 in a nibble of the byte that g and u share.
__device__ __forceinline__ uint32_t round20(float x) { return __float_as_uint(x) + 0x800u; }
__device__ __forceinline__ uint32_t pack_upper(uint32_t a, uint32_t b) {  // upper halves of a and b
  return __builtin_amdgcn_perm(b, a, 0x07060302u);
}
__device__ __forceinline__ uint32_t low_byte(uint32_t g, uint32_t u) { return ((g >> 12) & 0xfu) | ((u >> 8) & 0xf0u); }

// What the epilogue of a 32 x 32 block reads: the residual, or g and u.
template <int EK, int EPI>
struct Extra {
  u32x4 x[EPI == EPI_GLU_BWD ? (EK == EK_BF16 ? 5 : 8) : 2];
};
// Lane (l32, h) of a block's accumulators holds m = l32 and n = 8 q + 4 h + e of quad q, element e. The block
// starts at column n (a hidden column for both GLU epilogues); columns come in groups of 8.
template <int EK, int EPI>
__device__ __forceinline__ void load_extra(const GemmP& p, Extra<EK, EPI>& ex, int m, int n, int h) {
  if constexpr (EPI == EPI_STORE) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      ex.x[j] = u32x4{0u, 0u, 0u, 0u};
      const int c = n + 16 * j + 8 * h;
      if (p.res && m < p.m && c < p.n) ex.x[j] = *(const u32x4*)(p.res + m * p.res_ld + c * 2);
    }
  } else if constexpr (EPI == EPI_GLU_BWD) {
    constexpr int N = EK == EK_BF16 ? 5 : 8;
    if (m - (m & 31) < p.m && n < p.hidden) {
      const char* at = kept_at<EK>(p, m, n, h);
#pragma unroll
      for (int i = 0; i < N; ++i) ex.x[i] = *(const u32x4*)(at + i * 1024);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) ex.x[i] = u32x4{0u, 0u, 0u, 0u};
    }
  }
}
// c0: the block's sums (EPI_GLU: of the gate), c1: EPI_GLU only, the up projection's.
// NJ: groups of 16 columns.
template <int EK, int EPI, int NJ = 2>
__device__ __forceinline__ void finish_block(const GemmP& p, const f32x16& c0, const f32x16& c1,
                                             const Extra<EK, EPI>& ex, int m, int n, int h) {
  float scale = 1.0f, bound = 0.f;
  if constexpr (EK == EK_F16 && EPI != EPI_GLU)
    if (p.scale) scale = *p.scale;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {  // quads 2 j, 2 j + 1: 16 columns
    const int c = n + 16 * j + 8 * h;
    const bool on = m < p.m && c < (EPI == EPI_STORE ? p.n : p.hidden);
    if constexpr (EPI == EPI_STORE) {
      float v[8];
      unpack8<EK>(split_halves(ex.x[j]), v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = EK == EK_F16 ? fmaf(c0[8 * j + e], scale, v[e]) : v[e] + c0[8 * j + e];
      const u32x4 o =
          join_halves(pack2<EK>(v[0], v[1]), pack2<EK>(v[2], v[3]), pack2<EK>(v[4], v[5]), pack2<EK>(v[6], v[7]));
      if (on) *(u32x4*)(p.out + m * p.out_ld + c * 2) = o;
    } else if constexpr (EPI == EPI_GLU) {
      float g[8], v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] = c0[8 * j + e];
      act8<false>(p.act, g, v, nullptr);
      if constexpr (EK == EK_F16)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          bound = max_finite(max_finite(bound, v[e]), kSlopeMost * c1[8 * j + e]);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= c1[8 * j + e];
      const u32x4 o =
          join_halves(pack2<EK>(v[0], v[1]), pack2<EK>(v[2], v[3]), pack2<EK>(v[4], v[5]), pack2<EK>(v[6], v[7]));
      if (on) *(u32x4*)(p.out + m * p.out_ld + c * 2) = o;
      if (p.gu && m - (m & 31) < p.m && n < p.hidden) {
        const int part = NJ == 1 ? (n >> 4) & 1 : j;  // (blocks of 16 columns are halves)
        char* at = kept_at<EK>(p, m, n, h);
        if constexpr (EK == EK_BF16) {
          u32x4 kg, ku;
          u32x2 low = {0u, 0u};
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const uint32_t g0 = round20(c0[8 * j + e]), g1 = round20(c0[8 * j + e + 1]);
            const uint32_t u0 = round20(c1[8 * j + e]), u1 = round20(c1[8 * j + e + 1]);
            kg[e / 2] = pack_upper(g0, g1);
            ku[e / 2] = pack_upper(u0, u1);
            low[e / 4] |= (low_byte(g0, u0) | low_byte(g1, u1) << 8) << (e % 4 * 8);
          }
          *(u32x4*)(at + part * 1024) = kg;
          *(u32x4*)(at + 2048 + part * 1024) = ku;
          *(u32x2*)(at + 4096 + part * 8) = low;
        } else {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int e = 8 * j + 4 * q;
            *(f32x4*)(at + (2 * part + q) * 1024) = f32x4{c0[e], c0[e + 1], c0[e + 2], c0[e + 3]};
            *(f32x4*)(at + 4096 + (2 * part + q) * 1024) = f32x4{c1[e], c1[e + 1], c1[e + 2], c1[e + 3]};
          }
        }
      }
    } else {
      float g[8], u[8], dg[8], du[8];
      if constexpr (EK == EK_BF16) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t kg = ex.x[j][e / 2], ku = ex.x[2 + j][e / 2], low = ex.x[4][2 * j + e / 4] >> (e % 4 * 8);
          g[e] = __uint_as_float((e % 2 ? kg & 0xffff0000u : kg << 16) | (low & 0xfu) << 12);
          u[e] = __uint_as_float((e % 2 ? ku & 0xffff0000u : ku << 16) | (low & 0xf0u) << 8);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          g[e] = __uint_as_float(ex.x[2 * j + e / 4][e % 4]);
          u[e] = __uint_as_float(ex.x[4 + 2 * j + e / 4][e % 4]);
        }
      }
      float a[8], slope[8];
      act8<true>(p.act, g, a, slope);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float dh = EK == EK_F16 ? c0[8 * j + e] * scale : c0[8 * j + e];
        du[e] = dh * a[e];
        dg[e] = dh * u[e] * slope[e];
      }
      const u32x4 og = join_halves(pack2<EK>(dg[0], dg[1]), pack2<EK>(dg[2], dg[3]), pack2<EK>(dg[4], dg[5]),
                                   pack2<EK>(dg[6], dg[7]));
      const u32x4 ou = join_halves(pack2<EK>(du[0], du[1]), pack2<EK>(du[2], du[3]), pack2<EK>(du[4], du[5]),
                                   pack2<EK>(du[6], du[7]));
      if (on) {
        char* o = p.out + m * p.out_ld + c * 2;
        *(u32x4*)o = og;
        *(u32x4*)(o + (int64_t)p.hidden * 2) = ou;
      }
    }
  }
  if constexpr (EK == EK_F16 && EPI == EPI_GLU)
    if (p.gu && m - (m & 31) < p.m && n < p.hidden) {
      bound = wave_max(bound);
      const int64_t block = (int64_t)(m >> 5) * ((p.hidden + 31) >> 5) + (n >> 5);
      if ((m & 31) + h == 0) {
        if (NJ == 1) p.bound[2 * block + ((n >> 4) & 1)] = bound;
        else *(f32x2*)(p.bound + 2 * block) = f32x2{bound, 0.f};
      }
    }
}

// fp16: the largest finite |gy|, |Wo| and forward's factor, a workgroup's share: part[3][gridDim.x]. Bound by reading
// them once, with too little in flight: 40 MB of 16480 rows (1024, 2816) 16 us with 1024 workgroups, 28 with 256.
struct BoundP {
  const char *g, *w;  // [rows][d], [d][f]
  int64_t g_ld, w_ld, rows;
  int d, f;
  const float* factor;  // [blocks][2]
  int64_t blocks;
  float* part;
  float* scale;  // s, 1 / s
};
__device__ __forceinline__ float rows_max(const char* at, int64_t ld, int64_t rows, int d) {
  typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
  const int chunks = d / 8;
  int lpr = 1;  // lanes of a row
  while (lpr < chunks && lpr < 64) lpr *= 2;
  const int c0 = (int)threadIdx.x % lpr, step = 256 / lpr;
  i16x2 top = {0, 0};
  for (int64_t r = (int64_t)blockIdx.x * step + threadIdx.x / lpr; r < rows; r += (int64_t)gridDim.x * step)
#pragma unroll 4
    for (int c = c0; c < chunks; c += lpr) {
      const u32x4 x = *(const u32x4*)(at + r * ld + c * 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const i16x2 a = __builtin_bit_cast(i16x2, x[i] & 0x7fff7fffu);
        const i16x2 finite = (a - i16x2{0x7c00, 0x7c00}) >> 15;  // -1; infinities and NaN: 0
        top = __builtin_elementwise_max(top, a & finite);
      }
    }
  return f16_to_f32((uint16_t)(top[0] > top[1] ? top[0] : top[1]));
}
__global__ void __launch_bounds__(256) bound_kernel(const BoundP p) {
  __shared__ float s_big[3][4];
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, cols = (p.f + 31) / 32;
  float big[3] = {rows_max(p.g, p.g_ld, p.rows, p.d), rows_max(p.w, p.w_ld, p.d, p.f), 0.f};
  for (int64_t b = (int64_t)blockIdx.x * 256 + tid; b < p.blocks; b += (int64_t)gridDim.x * 256) {
    const f32x2 x = *(const f32x2*)(p.factor + 2 * b);
    big[2] = fmaxf(big[2], x[0]);
    if ((int)(b % cols) * 32 + 16 < p.f) big[2] = fmaxf(big[2], x[1]);
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    big[i] = wave_max(big[i]);
    if (lane == 0) s_big[i][wv] = big[i];
  }
  __syncthreads();
  if (tid < 3)
    p.part[tid * gridDim.x + blockIdx.x] = fmaxf(fmaxf(s_big[tid][0], s_big[tid][1]), fmaxf(s_big[tid][2], s_big[tid][3]));
}
constexpr int kBoundWgs = 1024;
__global__ void __launch_bounds__(64) scale_kernel(const BoundP p) {
  float bound = (float)p.d;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    float x = 0.f;
#pragma unroll
    for (int k = 0; k < kBoundWgs / 64; ++k) x = fmaxf(x, p.part[i * kBoundWgs + k * 64 + threadIdx.x]);
    bound *= wave_max(x);
  }
  int e = 15;  // where nothing is: s = 1
  if (bound > 0.f) frexpf(bound, &e);  // bound < 2^e
  const int up = e < -85 ? 100 : 15 - e;
  if (threadIdx.x == 0) {
    p.scale[0] = ldexpf(1.0f, up);
    p.scale[1] = ldexpf(1.0f, -up);
  }
}

// Measured at 256 x 256: a step of 64 k takes 1.7 to 1.8 us with all CUs busy, 1.2 PFLOP/s (a library product of
// 8192^3 reaches 1.25 to 1.3: the chip's power bounds both; LDS reads have no bank conflicts and L2 serves the
// loads at 24 bytes a clock and CU). A round's first loads and its epilogue, about 8 us, run under nothing, since a
// tile takes a whole CU: that is a third of a round at 768 k. 16480 rows (1024, 2816) bf16: gate and up 220 us with the
// activation and 325 MB written, dh 184 us with 418 MB read and written, dx 161 + 12 us, dw_in and dw_out 273 + 24 us,
// the output projection 100 + 12 us.
// A workgroup of WM x WN wavefronts owns a TM x TN tile and walks k in steps of 64 (whole 128-byte lines of
// either layout), four k steps of 16 each; the operands of one are read from LDS while the one before is
// multiplied. A has three LDS buffers and B two (all 160 KB at 256 x 256): before a step's last k step its
// buffers have been read, there the next step's are waited for and B's loads of the step after it start;
// A's start one k step later and are in flight across the wait, so that requests never run dry.
template <int EK, bool XA, bool XB, int TM, int TN, int WM, int WN, int EPI>
__global__ void __launch_bounds__(WM* WN * 64) gemm_kernel(const GemmP p) {
  constexpr int NW = WM * WN, MB = TM / WM / 32, NB = TN / WN / 32;
  using SA = Stage<TM, XA, NW>;
  using SB = Stage<TN, XB, NW>;
  constexpr bool GLU = EPI == EPI_GLU;
  __shared__ __attribute__((aligned(1024))) char s_tile[3 * SA::BYTES + 2 * SB::BYTES];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wv % WM, wn = wv / WM;
  const bool whole = (int)blockIdx.x < p.full;
  const int at = (int)blockIdx.x - p.full, split = whole ? 0 : at / p.tail;
  const uint32_t t = whole ? xcd_tile(blockIdx.x, (uint32_t)p.full) : (uint32_t)(p.full + at % p.tail);
  const int tm = (int)(t / (uint32_t)p.tiles_n), tn = (int)(t % (uint32_t)p.tiles_n);
  const int m0 = tm * TM, n0 = GLU ? tn * (TN / 2) : tn * TN;  // GLU: n0 counts hidden columns
  const int k0 = split * p.k_per, k1 = whole || k0 + p.k_per > p.k ? p.k : k0 + p.k_per;
  const int steps = (k1 - k0 + BK - 1) / BK;

  uint32_t offa[SA::NI], offb[SB::NI];
  SA::offsets(offa, wv, lane, p.a_ld, p.m - m0, false, 0);
  SB::offsets(offb, wv, lane, p.b_ld, (GLU ? p.hidden : p.n) - n0, GLU, p.hidden);
  const uint32_t lds0 = lds_addr(s_tile);
  uint32_t ra[4], rb[4];
  SA::bases(ra, wm * (TM / WM), lane);
  SB::bases(rb, wn * (TN / WN), lane);
  // A's loads of step i go into buffer i % 3, B's into i % 2; a step past the end loads nothing but counts alike
  const uint32_t ldb = lds0 + 3 * SA::BYTES;
  auto k_of = [&](int i) { return k0 + i * BK; };
  auto desc_a = [&](int i) {
    const int64_t k = k_of(i);
    return raw_desc(XA ? p.a + k * p.a_ld + (int64_t)m0 * 2 : p.a + (int64_t)m0 * p.a_ld + k * 2,
                    k < k1 ? 0xffffff00u : 0u);
  };
  auto desc_b = [&](int i) {
    const int64_t k = k_of(i);
    return raw_desc(XB ? p.b + k * p.b_ld + (int64_t)n0 * 2 : p.b + (int64_t)n0 * p.b_ld + k * 2,
                    k < k1 ? 0xffffff00u : 0u);
  };
  u32x4 fa[2][MB], fb[2][NB];
  auto read = [&](int set, uint32_t la, uint32_t lb, int ks, int j) {
    if (j < MB) fa[set][j] = SA::frag(ra, la, j, ks);
    else fb[set][j - MB] = SB::frag(rb, lb, j - MB, ks);
  };

  f32x16 acc[NB][MB];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j) acc[i][j] = f32x16{};
  // One k step: the MFMAs of operand set `set`, and spread between them the reads of the other set
  // (k step ks of buffers la, lb) and `loads` loads.
  auto k_step = [&](auto SET, uint32_t la, uint32_t lb, int ks, auto LOADS, auto load) {
    constexpr int set = decltype(SET)::value;
    constexpr int S = NB * MB, R = MB + NB, OPS = R + decltype(LOADS)::value;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      acc[s / MB][s % MB] = mfma16<EK>(acc[s / MB][s % MB], fb[set][s / MB], fa[set][s % MB]);
#pragma unroll
      for (int o = s * OPS / S; o < (s + 1) * OPS / S; ++o) {
        if (o < R) read(set ^ 1, la, lb, ks, o);
        else load(o - R);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  using std::integral_constant;
  constexpr integral_constant<int, 0> S0{}, NONE{};
  constexpr integral_constant<int, 1> S1{};
  constexpr integral_constant<int, SA::NI> LA{};
  constexpr integral_constant<int, SB::NI> LB{};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const u32x4 da = desc_a(i), db = desc_b(i);
#pragma unroll
    for (int j = 0; j < SA::NI; ++j) SA::issue(lds0 + i * SA::BYTES, offa, j, wv, lane, da, k1 - k_of(i));
#pragma unroll
    for (int j = 0; j < SB::NI; ++j) SB::issue(ldb + i * SB::BYTES, offb, j, wv, lane, db, k1 - k_of(i));
  }
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(SA::NI + SB::NI) : "memory");
#pragma unroll
  for (int j = 0; j < MB + NB; ++j) read(0, lds0, ldb, 0, j);
  uint32_t a0 = lds0, a1 = lds0 + SA::BYTES, a2 = lds0 + 2 * SA::BYTES, b0 = ldb, b1 = ldb + SB::BYTES;
  for (int i = 0; i < steps; ++i) {
    const int left = k1 - k_of(i + 2);
    const u32x4 da = desc_a(i + 2), db = desc_b(i + 2);
    k_step(S0, a0, b0, 1, LA, [&](int j) { SA::issue(a2, offa, j, wv, lane, da, left); });
    k_step(S1, a0, b0, 2, NONE, [&](int) {});
    k_step(S0, a0, b0, 3, NONE, [&](int) {});
    // the next step's buffers are complete, and every wavefront has read all of this step's
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(SA::NI) : "memory");
    k_step(S1, a1, b1, 0, LB, [&](int j) { SB::issue(b0, offb, j, wv, lane, db, left); });
    const uint32_t a = a0, b = b0;
    a0 = a1, a1 = a2, a2 = a;
    b0 = b1, b1 = b;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load is in flight to LDS when the workgroup ends

  if (!whole) {
    float* out = p.part + (((int64_t)(at % p.tail) * p.splits + split) * NW + wv) * (NB * MB * 1024) + lane * 4;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < MB; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *(f32x4*)(out + ((i * MB + j) * 4 + q) * 256) =
              f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    return;
  }
  const int l32 = lane & 31, h = lane >> 5;
  constexpr int PAIR = GLU ? 2 : 1;  // column blocks of one output block
#pragma unroll
  for (int j = 0; j < MB; ++j) {
    const int m = m0 + wm * (TM / WM) + j * 32 + l32, n = n0 + wn * (TN / WN / PAIR);
    // a row's loads before its first store (g and u of fp16 calls take twice the registers: block by block)
    constexpr int AHEAD = EK == EK_F16 && EPI == EPI_GLU_BWD ? 1 : NB / PAIR;
#pragma unroll
    for (int i0 = 0; i0 < NB / PAIR; i0 += AHEAD) {
      Extra<EK, EPI> ex[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) load_extra<EK, EPI>(p, ex[i], m, n + (i0 + i) * 32, h);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        finish_block<EK, EPI>(p, acc[(i0 + i) * PAIR][j], acc[(i0 + i) * PAIR + PAIR - 1][j], ex[i], m,
                              n + (i0 + i) * 32, h);
    }
  }
}

// The tail's epilogue: a workgroup adds the splits of one block of every wavefront in order.
template <int EK, int TM, int TN, int WM, int WN, int EPI>
__global__ void __launch_bounds__(WM* WN * 64) gemm_finish_kernel(const GemmP p) {
  constexpr int NW = WM * WN, MB = TM / WM / 32, NB = TN / WN / 32, PAIR = EPI == EPI_GLU ? 2 : 1;
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, wm = wv % WM, wn = wv / WM, h = lane >> 5;
  int u = (int)blockIdx.x;
  const int j = u % MB;
  u /= MB;
  const int i = u % (NB / PAIR) * PAIR;
  u /= NB / PAIR;
  const int t = p.full + u, tm = t / p.tiles_n, tn = t % p.tiles_n;
  const int m = tm * TM + wm * (TM / WM) + j * 32 + (lane & 31);
  const int n = tn * (TN / PAIR) + wn * (TN / WN / PAIR) + i / PAIR * 32;
  Extra<EK, EPI> ex;
  load_extra<EK, EPI>(p, ex, m, n, h);
  f32x16 c[PAIR];
#pragma unroll
  for (int b = 0; b < PAIR; ++b) c[b] = f32x16{};
  const float* in = p.part + ((int64_t)u * p.splits * NW + wv) * (NB * MB * 1024) + lane * 4;
#pragma unroll 2
  for (int s = 0; s < p.splits; ++s, in += NW * NB * MB * 1024)
#pragma unroll
    for (int b = 0; b < PAIR; ++b)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 x = *(const f32x4*)(in + (((i + b) * MB + j) * 4 + q) * 256);
#pragma unroll
        for (int e = 0; e < 4; ++e) c[b][4 * q + e] += x[e];
      }
  finish_block<EK, EPI>(p, c[0], c[PAIR - 1], ex, m, n, h);
}

// Few rows: the weights are read once for all of them and little else happens, so the call is bound by the latency of
// a launch and of one chain of loads: 32 rows (768, 1152) 6 + 7.5 us against 30 + 31 us by 256 x 256 tiles. A workgroup owns 32 weight rows (EPI_GLU: 16 gate and the 16 up rows of the same columns,
// which meet in one lane's accumulators) and 32 MB rows of x, its eight wavefronts an eighth of k each: operands
// go from memory to registers as they lie, the eight sums meet in LDS and are added in order.
template <int EK, int EPI, int MB>
__global__ void __launch_bounds__(512) few_rows_kernel(const GemmP p) {
  constexpr int NW = 8, U = 6;
  __shared__ __attribute__((aligned(16))) float s_sum[NW][MB][4][64][4];
  const int lane = threadIdx.x & 63, l32 = lane & 31, h = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = (int)blockIdx.x * (EPI == EPI_GLU ? 16 : 32);
  const int n = EPI == EPI_GLU ? n0 + (l32 & 15) : n0 + l32;
  // rows from n0 on, whose address is 64 bits wide: all rows together can pass a lane's 32-bit offset
  const int row = EPI == EPI_GLU && l32 >= 16 ? p.hidden + (l32 & 15) : l32;
  const uint32_t boff = n < (EPI == EPI_GLU ? p.hidden : p.n) ? (uint32_t)(row * p.b_ld) : kOob;
  uint32_t aoff[MB];
#pragma unroll
  for (int j = 0; j < MB; ++j) aoff[j] = j * 32 + l32 < p.m ? (uint32_t)((j * 32 + l32) * p.a_ld) : kOob;
  const __amdgpu_buffer_rsrc_t rb =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p.b + n0 * p.b_ld), (short)0, (int)0xffffff00u, 0x00020000);
  const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<char*>(p.a), (short)0, (int)0xffffff00u, 0x00020000);
  f32x16 acc[MB];
#pragma unroll
  for (int j = 0; j < MB; ++j) acc[j] = f32x16{};
  const int all = (p.k + 15) / 16, per = (all + NW - 1) / NW;
  const int end = (wv + 1) * per < all ? (wv + 1) * per : all;
  for (int ks = wv * per; ks < end; ks += U) {
    u32x4 fb[U], fa[U][MB];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = (ks + u) * 16 + 8 * h;
      const bool on = ks + u < end && e < p.k;
      fb[u] = __builtin_amdgcn_raw_buffer_load_b128(rb, on && boff != kOob ? boff + e * 2 : kOob, 0, 0);
#pragma unroll
      for (int j = 0; j < MB; ++j)
        fa[u][j] = __builtin_amdgcn_raw_buffer_load_b128(ra, on && aoff[j] != kOob ? aoff[j] + e * 2 : kOob, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < MB; ++j) acc[j] = mfma16<EK>(acc[j], fb[u], fa[u][j]);
  }
#pragma unroll
  for (int j = 0; j < MB; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *(f32x4*)s_sum[wv][j][q][lane] = f32x4{acc[j][4 * q], acc[j][4 * q + 1], acc[j][4 * q + 2], acc[j][4 * q + 3]};
  __syncthreads();
  if (wv >= MB) return;
  const int m = wv * 32 + l32;
  Extra<EK, EPI> ex;
  load_extra<EK, EPI>(p, ex, m, n0, h);
  f32x16 c = {};
#pragma unroll
  for (int w = 0; w < NW; ++w)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4 x = *(const f32x4*)s_sum[w][wv][q][lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) c[4 * q + e] += x[e];
    }
  if constexpr (EPI == EPI_GLU) {
    f32x16 up = {};
#pragma unroll
    for (int e = 0; e < 8; ++e) up[e] = c[8 + e];
    finish_block<EK, EPI, 1>(p, c, up, ex, m, n0, h);
  } else {
    finish_block<EK, EPI>(p, c, c, ex, m, n0, h);
  }
}

constexpr int kCUs = 256;
// Whether few_rows_kernel takes one of the forward's products: m rows by n weight rows of length k. Both
// products together, few_rows_kernel against the 128 x 128 tiles: (768, 1152) 32 rows 13 against 20 us, 64 rows 17
// against 20, 128 rows 25 against 20; (1024, 2624) 32 rows 20 against 25, 64 rows 28 against 25.
bool few_rows(int64_t m, int64_t n, int64_t k) { return m <= 32 || (m <= 64 && n * k <= (1 << 21)); }

template <int EK, int EPI>
int launch_few_rows(const GemmP& p, hipStream_t s) {
  const unsigned nb = EPI == EPI_GLU ? (p.hidden + 15) / 16 : (p.n + 31) / 32;
  if (p.m <= 32)
    launch_kernel(few_rows_kernel<EK, EPI, 1>, dim3(nb), dim3(512), 0u, s, p);
  else
    launch_kernel(few_rows_kernel<EK, EPI, 2>, dim3(nb), dim3(512), 0u, s, p);
  return hipGetLastError() == hipSuccess ? LIK_OK : LIK_ERR_LAUNCH;
}

// Tiles of 256 x 256 (eight wavefronts, all of a CU's LDS) read the least for their work; tiles of 128 x 128 (four
// wavefronts, two workgroups a CU) give four times as many workgroups where there are few. Tiles run in rounds of
// the CUs. What is left after the whole rounds would take another round on a few CUs; instead k of each of those
// tiles is split over several workgroups, whose fp32 sums a second kernel adds. The choice takes the least of
// the costs in us, as measured: a step of 64 k, a round's start and epilogue, and for split tiles the second
// launch and the partial sums written and read at about 4.5 TB/s.
struct Shape {
  int tile, tiles_n, full, tail, splits, k_per;
  double cost;
};
Shape tile_shape(int tile, int64_t m, int64_t n, int64_t k) {
  const bool big = tile == 256;
  const int64_t tn = (n + tile - 1) / tile, tiles = (m + tile - 1) / tile * tn, steps = (k + BK - 1) / BK;
  const int64_t slots = big ? kCUs : 2 * kCUs;
  const double start = big ? 8.0 : 5.0;
  const auto step = [&](int64_t wgs) { return big ? 1.8 : wgs > kCUs ? 1.2 : 0.7; };
  const int64_t whole = tiles / slots * slots, left = tiles - whole;
  Shape s{tile, (int)tn, (int)tiles, 0, 1, (int)(steps * BK), 0.0};
  const double rounds = whole / slots * (steps * step(slots) + start);
  s.cost = rounds + (left ? steps * step(left) + start : 0.0);
  if (left == 0) return s;
  for (int64_t sp = 2; sp <= steps / 2 && left * sp <= 4 * slots; ++sp) {
    const int64_t per = (steps + sp - 1) / sp;
    if ((steps + per - 1) / per != sp) continue;
    const double cost = rounds + (step(left * sp) * per + start) * ((left * sp + slots - 1) / slots) + 8 +
                        left * sp * tile * tile * 8 / 4.5e6;
    if (cost < s.cost) s = {tile, (int)tn, (int)whole, (int)left, (int)sp, (int)(per * BK), cost};
  }
  return s;
}
// n: columns of the tiles' B operand (EPI_GLU: gate and up)
Shape gemm_shape(int64_t m, int64_t n, int64_t k) {
  const Shape a = tile_shape(256, m, n, k), b = tile_shape(128, m, n, k);
  return a.cost <= b.cost ? a : b;
}
size_t part_bytes(const Shape& s) { return (size_t)s.tail * s.splits * s.tile * s.tile * 4; }
int64_t glu_columns(int64_t hidden) { return (hidden + 31) / 32 * 64; }  // (blocks of 32 gate and 32 up columns)

template <int EK, bool XA, bool XB, int EPI, int T>
int launch_tiles(const GemmP& p, hipStream_t s) {
  constexpr int WM = T / 64, WN = 2;
  const int groups = p.full + p.tail * p.splits;
  launch_kernel(gemm_kernel<EK, XA, XB, T, T, WM, WN, EPI>, dim3((unsigned)groups), dim3(WM * WN * 64), 0u, s, p);
  if (hipGetLastError() != hipSuccess) return LIK_ERR_LAUNCH;
  if (p.tail) {
    constexpr int blocks = T / WM / 32 * (T / WN / 32) / (EPI == EPI_GLU ? 2 : 1);
    launch_kernel(gemm_finish_kernel<EK, T, T, WM, WN, EPI>, dim3((unsigned)(p.tail * blocks)), dim3(WM * WN * 64), 0u, s, p);
    if (hipGetLastError() != hipSuccess) return LIK_ERR_LAUNCH;
  }
  return LIK_OK;
}
template <int EK, bool XA, bool XB, int EPI>
int launch_gemm(GemmP p, float* part, hipStream_t s) {
  if constexpr (!XA && !XB)
    if (few_rows(p.m, EPI == EPI_GLU ? 2ll * p.hidden : p.n, p.k)) return launch_few_rows<EK, EPI>(p, s);
  const Shape sh = gemm_shape(p.m, EPI == EPI_GLU ? glu_columns(p.hidden) : p.n, p.k);
  p.tiles_n = sh.tiles_n;
  p.full = sh.full;
  p.tail = sh.tail;
  p.splits = sh.splits;
  p.k_per = sh.k_per;
  p.part = part;
  return sh.tile == 256 ? launch_tiles<EK, XA, XB, EPI, 256>(p, s) : launch_tiles<EK, XA, XB, EPI, 128>(p, s);
}

size_t most(size_t a, size_t b) { return a > b ? a : b; }
size_t ffn_ws(int64_t rows, int d, int f) {
  return most(part_bytes(gemm_shape(rows, glu_columns(f), d)), part_bytes(gemm_shape(rows, d, f))) + 256;
}

struct FfnBwdWs {  // dg and du come first
  size_t bound, part, total;
};
FfnBwdWs ffn_bwd_ws(int64_t rows, int d, int f) {
  FfnBwdWs w;
  w.bound = align256((size_t)rows * 2 * f * 2);
  w.part = w.bound + align256((3 * kBoundWgs + 2) * 4);
  w.total = w.part + 256 +
            most(most(part_bytes(gemm_shape(rows, f, d)), part_bytes(gemm_shape(rows, d, 2 * f))),
                 most(part_bytes(gemm_shape(2 * f, d, rows)), part_bytes(gemm_shape(d, f, rows))));
  return w;
}

int64_t kept_blocks(int64_t rows, int f) { return ((rows + 31) / 32) * ((f + 31) / 32); }
// (fp16: the forward's factors after the blocks)
float* kept_bound(void* gu, int64_t rows, int f) { return (float*)((char*)gu + kept_blocks(rows, f) * kKeptBlock<EK_F16>); }

int ffn_check(int32_t dtype, int64_t rows, int32_t d, int32_t f, int32_t act) {
  if (dtype != LIK_BF16 && dtype != LIK_F16) return LIK_ERR_UNSUPPORTED;
  if (rows < 0 || d < 8 || f < 8 || act < ACT_GELU || act > ACT_SILU) return LIK_ERR_INVALID;
  // 16-byte chunks of k; rows of weights and tokens within a 32-bit tile offset
  if (d % 8 || f % 8 || d > (1 << 20) || f > (1 << 20) || rows > 0x7fffff00) return LIK_ERR_UNSUPPORTED;
  const int64_t most_n = (2ll * f > d ? 2ll * f : d) / 128 + 1;  // workgroups of a launch, in 31 bits
  if ((rows / 128 + 1) * most_n > (1 << 30)) return LIK_ERR_UNSUPPORTED;
  return LIK_OK;
}
// 16-byte rows; a tile of 256, and `more` rows before it, within a lane's 32-bit offset
bool rows16(const void* p, int64_t stride, int64_t more = 0) {
  return (uintptr_t)p % 16 == 0 && stride % 8 == 0 && stride >= 0 && stride <= (1 << 21) &&
         (more + 256) * stride * 2 < 0xfff00000ll;
}

template <int EK>
int ffn_forward(const void* x, int64_t x_ld, int64_t rows, int d, int f, const void* w_in, int64_t wi_ld,
                const void* w_out, int64_t wo_ld, const void* res, int64_t res_ld, int act, void* out, void* h,
                void* gu, float* part, hipStream_t s) {
  GemmP p{};
  p.act = act;
  p.hidden = f;
  p.m = (int)rows;
  p.a = (const char*)x;
  p.a_ld = x_ld * 2;
  p.b = (const char*)w_in;
  p.b_ld = wi_ld * 2;
  p.n = f;
  p.k = d;
  p.out = (char*)h;
  p.out_ld = (int64_t)f * 2;
  p.gu = (char*)gu;
  if (EK == EK_F16 && gu) p.bound = kept_bound(gu, rows, f);
  if (const int rc = launch_gemm<EK, false, false, EPI_GLU>(p, part, s)) return rc;
  p.a = (const char*)h;
  p.a_ld = (int64_t)f * 2;
  p.b = (const char*)w_out;
  p.b_ld = wo_ld * 2;
  p.n = d;
  p.k = f;
  p.out = (char*)out;
  p.out_ld = (int64_t)d * 2;
  p.res = (const char*)res;
  p.res_ld = res_ld * 2;
  return launch_gemm<EK, false, false, EPI_STORE>(p, part, s);
}

template <int EK>
int ffn_backward(const void* g, int64_t g_ld, const void* x, int64_t x_ld, int64_t rows, int d, int f,
                 const void* w_in, int64_t wi_ld, const void* w_out, int64_t wo_ld, const void* h, const void* gu,
                 int act, void* gx, void* gw_in, void* gw_out, char* ws, hipStream_t s) {
  const FfnBwdWs w = ffn_bwd_ws(rows, d, f);
  char* dgu = ws;
  float* part = (float*)(ws + w.part);
  GemmP p{};
  p.act = act;
  p.hidden = f;
  if (gx || gw_in) {
    p.m = (int)rows;
    p.a = (const char*)g;
    p.a_ld = g_ld * 2;
    p.b = (const char*)w_out;
    p.b_ld = wo_ld * 2;
    p.n = f;
    p.k = d;
    p.out = dgu;
    p.out_ld = (int64_t)f * 4;
    p.gu = (char*)const_cast<void*>(gu);
    if (EK == EK_F16) {
      float* at = (float*)(ws + w.bound);
      const BoundP b{(const char*)g, (const char*)w_out, g_ld * 2, wo_ld * 2, rows, d, f, kept_bound(p.gu, rows, f),
                     kept_blocks(rows, f), at, at + 3 * kBoundWgs};
      launch_kernel(bound_kernel, dim3(kBoundWgs), dim3(256), 0u, s, b);
      if (hipGetLastError() != hipSuccess) return LIK_ERR_LAUNCH;
      launch_kernel(scale_kernel, dim3(1), dim3(64), 0u, s, b);
      if (hipGetLastError() != hipSuccess) return LIK_ERR_LAUNCH;
      p.scale = b.scale;
    }
    if (const int rc = launch_gemm<EK, false, true, EPI_GLU_BWD>(p, part, s)) return rc;
    if (p.scale) ++p.scale;  // 1 / s
  }
  if (gx) {
    p.a = dgu;
    p.a_ld = (int64_t)f * 4;
    p.b = (const char*)w_in;
    p.b_ld = wi_ld * 2;
    p.n = d;
    p.k = 2 * f;
    p.out = (char*)gx;
    p.out_ld = (int64_t)d * 2;
    if (const int rc = launch_gemm<EK, false, true, EPI_STORE>(p, part, s)) return rc;
  }
  p.k = (int)rows;
  if (gw_in) {
    p.m = 2 * f;
    p.n = d;
    p.a = dgu;
    p.a_ld = (int64_t)f * 4;
    p.b = (const char*)x;
    p.b_ld = x_ld * 2;
    p.out = (char*)gw_in;
    p.out_ld = (int64_t)d * 2;
    if (const int rc = launch_gemm<EK, true, true, EPI_STORE>(p, part, s)) return rc;
  }
  if (gw_out) {
    p.scale = nullptr;
    p.m = d;
    p.n = f;
    p.a = (const char*)g;
    p.a_ld = g_ld * 2;
    p.b = (const char*)h;
    p.b_ld = (int64_t)f * 2;
    p.out = (char*)gw_out;
    p.out_ld = (int64_t)f * 2;
    if (const int rc = launch_gemm<EK, true, true, EPI_STORE>(p, part, s)) return rc;
  }
  return LIK_OK;
}

}  // namespace
}  // namespace enc
}  // namespace lik

using namespace lik;
using namespace lik::enc;

extern "C" {

size_t lik_gated_ffn_workspace_size(int32_t dtype, int64_t rows, int32_t dim, int32_t hidden) {
  if (ffn_check(dtype, rows, dim, hidden, ACT_GELU) != LIK_OK || rows == 0) return 0;
  return ffn_ws(rows, dim, hidden);
}

size_t lik_gated_ffn_kept_size(int32_t dtype, int64_t rows, int32_t dim, int32_t hidden) {
  if (ffn_check(dtype, rows, dim, hidden, ACT_GELU) != LIK_OK) return 0;
  return (size_t)kept_blocks(rows, hidden) * (dtype == LIK_BF16 ? kKeptBlock<EK_BF16> : kKeptBlock<EK_F16> + 8);
}

int lik_gated_ffn(const void* x, int64_t x_stride, int32_t dtype, int64_t rows, int32_t dim, int32_t hidden,
                  const void* w_in, int64_t w_in_stride, const void* w_out, int64_t w_out_stride, const void* residual,
                  int64_t residual_stride, int32_t activation, void* out, void* hidden_act, void* gate_up,
                  void* workspace, size_t workspace_bytes, lik_stream_t stream) {
  if (const int rc = ffn_check(dtype, rows, dim, hidden, activation)) return rc;
  if (rows == 0) return LIK_OK;
  if (!x || !w_in || !w_out || !out || !hidden_act) return LIK_ERR_INVALID;
  if (!rows16(x, x_stride) || !rows16(w_in, w_in_stride, hidden) || !rows16(w_out, w_out_stride) || !rows16(out, 0) ||
      !rows16(hidden_act, 0) || !rows16(gate_up, 0) || (residual && !rows16(residual, residual_stride)))
    return LIK_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < ffn_ws(rows, dim, hidden)) return LIK_ERR_WORKSPACE;
  const auto fn = dtype == LIK_BF16 ? ffn_forward<EK_BF16> : ffn_forward<EK_F16>;
  return fn(x, x_stride, rows, dim, hidden, w_in, w_in_stride, w_out, w_out_stride, residual, residual_stride,
            activation, out, hidden_act, gate_up, (float*)align256(workspace), (hipStream_t)stream);
}

size_t lik_gated_ffn_backward_workspace_size(int32_t dtype, int64_t rows, int32_t dim, int32_t hidden) {
  if (ffn_check(dtype, rows, dim, hidden, ACT_GELU) != LIK_OK || rows == 0) return 0;
  return ffn_bwd_ws(rows, dim, hidden).total;
}

int lik_gated_ffn_backward(const void* grad, int64_t grad_stride, const void* x, int64_t x_stride, int32_t dtype,
                           int64_t rows, int32_t dim, int32_t hidden, const void* w_in, int64_t w_in_stride,
                           const void* w_out, int64_t w_out_stride, const void* hidden_act, const void* gate_up,
                           int32_t activation, void* grad_x, void* grad_w_in, void* grad_w_out, void* workspace,
                           size_t workspace_bytes, lik_stream_t stream) {
  if (const int rc = ffn_check(dtype, rows, dim, hidden, activation)) return rc;
  if (rows == 0) return LIK_ERR_INVALID;  // the gradients of the weights would stay unwritten
  if (!grad || !x || !w_in || !w_out || !hidden_act || !gate_up) return LIK_ERR_INVALID;
  if (!rows16(grad, grad_stride) || !rows16(x, x_stride) || !rows16(w_in, w_in_stride, hidden) ||
      !rows16(w_out, w_out_stride) || !rows16(hidden_act, 0) || !rows16(gate_up, 0) || !rows16(grad_x, 0) ||
      !rows16(grad_w_in, 0) || !rows16(grad_w_out, 0))
    return LIK_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < lik_gated_ffn_backward_workspace_size(dtype, rows, dim, hidden))
    return LIK_ERR_WORKSPACE;
  const auto fn = dtype == LIK_BF16 ? ffn_backward<EK_BF16> : ffn_backward<EK_F16>;
  return fn(grad, grad_stride, x, x_stride, rows, dim, hidden, w_in, w_in_stride, w_out, w_out_stride, hidden_act,
            gate_up, activation, grad_x, grad_w_in, grad_w_out, align256(workspace), (hipStream_t)stream);
}

}  // extern "C"
