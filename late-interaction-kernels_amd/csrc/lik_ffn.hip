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
// Sums over k are fp32 (MFMA accumulators, fp32 partial sums where k is split).
// h, dg and du are rounded once to the 16-bit type, as the next product's operands
// have to be; g and u are kept in fp32 for the backward, so that dg and du carry no
// second rounding.
#include "lik_enc.h"

namespace lik {
namespace enc {
namespace {

enum { ACT_GELU = 0, ACT_GELU_TANH = 1, ACT_SILU = 2 };
enum { EPI_STORE = 0, EPI_GLU = 1, EPI_GLU_BWD = 2, EPI_PART = 3 };

struct GemmP {
  const char* a;  // A(m, k): m * a_ld + k, or across k: k * a_ld + m (elements of 2 bytes)
  const char* b;
  int64_t a_ld, b_ld;  // bytes
  int m, n, k;
  int k_per;           // k of one split (a multiple of 64)
  int tiles_m, tiles_n, splits;
  char* out;           // [m][n] 16-bit, row stride out_ld bytes; EPI_PART: fp32 [split][m][n]
  int64_t out_ld;
  const char* res;     // EPI_STORE: added before the rounding; null: none
  int64_t res_ld;
  float* gu;           // EPI_GLU: [m][2 hidden] kept g and u (null: not kept); EPI_GLU_BWD: read
  int hidden;
  int act;
};

// act(x) and its derivative
template <bool SLOPE>
__device__ __forceinline__ float act_of(int act, float x, float& slope) {
  if (act == ACT_SILU) {
    const float s = 1.0f / (1.0f + __expf(-x));
    if (SLOPE) slope = s * (1.0f + x * (1.0f - s));
    return x * s;
  }
  if (act == ACT_GELU_TANH) {
    // (1 + tanh u) / 2 = sigmoid(2 u), u = sqrt(2 / pi) (x + 0.044715 x^3)
    const float x2 = x * x;
    const float s = 1.0f / (1.0f + __expf(-1.5957691216f * x * fmaf(0.044715f, x2, 1.0f)));
    if (SLOPE) slope = s * (1.0f + x * (1.0f - s) * 1.5957691216f * fmaf(0.134145f, x2, 1.0f));
    return x * s;
  }
  const float cdf = 0.5f * (1.0f + erff(x * 0.70710678118f));
  if (SLOPE) slope = fmaf(x, 0.39894228040f * __expf(-0.5f * x * x), cdf);
  return x * cdf;
}

// One operand's tile of T rows (m or n) by 64 k in LDS, 128 bytes a row of T:
// along k: [T][64], 8 chunks a row; across k: [64][T], T / 8 chunks a row.
template <int T, bool X, int NW>
struct Stage {
  static constexpr int BYTES = T * 128;
  static constexpr int NI = T / 8 / NW;  // 1 KB loads of a wavefront
  static_assert(T % (8 * NW) == 0, "");

  // Lane offsets of the wavefront's loads from the tile's origin, kOob past the matrix' edge.
  // `rows`: rows (along k) or columns (across k) the tile has; glu: rows 32..63 of each 64 are up rows.
  __device__ __forceinline__ static void offsets(uint32_t* off, int wv, int lane, int64_t ld, int rows, bool glu,
                                                 int hidden) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int slot = (wv * NI + i) * 64 + lane;
      if constexpr (X) {
        const int r = slot / (T / 8), c = (slot % (T / 8)) ^ lds_swz(r);
        off[i] = c * 8 < rows ? (uint32_t)(r * ld + c * 16) : kOob;
      } else {
        const int r = slot / 8, c = (slot % 8) ^ lds_swz(r);
        const int at = glu ? (r / 64) * 32 + r % 32 : r;
        off[i] = at < rows ? (uint32_t)((at + (glu && (r & 32) ? (int64_t)hidden : 0)) * ld + c * 16) : kOob;
      }
    }
  }
  // k_left: k of this step that exist (at most 64)
  __device__ __forceinline__ static void issue(uint32_t lds, const uint32_t* off, int wv, int lane, const char* base,
                                               uint32_t bytes, int k_left) {
    const u32x4 desc = raw_desc(base, bytes);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      uint32_t o = off[i];
      const int slot = (wv * NI + i) * 64 + lane;
      if constexpr (X) {
        if (k_left < 64 && slot / (T / 8) >= k_left) o = kOob;
      } else {
        if (k_left < 64 && (int)((slot % 8) ^ lds_swz(slot / 8)) * 8 >= k_left) o = kOob;
      }
      dma16(lds + (wv * NI + i) * 1024, o, desc);
    }
  }
  // MFMA operand of 32 rows from row0, k step ks (16 k): lane l has row l % 32, k = 8 (l / 32) + 0..7.
  __device__ __forceinline__ static u32x4 frag(uint32_t lds, int row0, int ks, int lane) {
    if constexpr (X) {
      const int i = lane & 15, h = lane >> 5;
      const int col = row0 + 16 * ((lane >> 4) & 1) + 4 * (i & 3);
      const int k0 = ks * 16 + 8 * h + (i >> 2);
      const u32x2 lo = lds_tr(lds + k0 * (T * 2) + (((col >> 3) ^ lds_swz(k0)) << 4) + ((col & 4) << 1));
      const u32x2 hi = lds_tr(lds + (k0 + 4) * (T * 2) + (((col >> 3) ^ lds_swz(k0 + 4)) << 4) + ((col & 4) << 1));
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    } else {
      const int r = row0 + (lane & 31), c = ks * 2 + (lane >> 5);
      return lds_b128(lds + r * 128 + ((c ^ lds_swz(r)) << 4));
    }
  }
};

// Four consecutive n of accumulator quads 2j and 2j + 1, as 16-bit pairs, to
// eight consecutive n per lane (the wavefront's halves exchange): lane half h
// then holds n = 16 j + 8 h + 0..7 of its m.
__device__ __forceinline__ u32x4 join_halves(uint32_t a0, uint32_t a1, uint32_t b0, uint32_t b1) {
  const auto s0 = __builtin_amdgcn_permlane32_swap(a0, b0, false, false);
  const auto s1 = __builtin_amdgcn_permlane32_swap(a1, b1, false, false);
  return u32x4{(uint32_t)s0[0], (uint32_t)s1[0], (uint32_t)s0[1], (uint32_t)s1[1]};
}

template <int EK, bool XA, bool XB, int TM, int TN, int WM, int WN, int EPI>
__global__ void __launch_bounds__(WM* WN * 64) gemm_kernel(const GemmP p) {
  constexpr int NW = WM * WN, MB = TM / WM / 32, NB = TN / WN / 32;
  using SA = Stage<TM, XA, NW>;
  using SB = Stage<TN, XB, NW>;
  constexpr bool GLU = EPI == EPI_GLU;
  __shared__ __attribute__((aligned(1024))) char s_tile[2][SA::BYTES + SB::BYTES];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wv % WM, wn = wv / WM;
  uint32_t t = xcd_tile(blockIdx.x, gridDim.x);
  const int split = (int)(t / (uint32_t)(p.tiles_m * p.tiles_n));
  t %= (uint32_t)(p.tiles_m * p.tiles_n);
  const int tm = (int)(t / (uint32_t)p.tiles_n), tn = (int)(t % (uint32_t)p.tiles_n);
  const int m0 = tm * TM, n0 = GLU ? tn * (TN / 2) : tn * TN;  // GLU: n0 counts hidden columns
  const int k0 = split * p.k_per, k1 = k0 + p.k_per < p.k ? k0 + p.k_per : p.k;

  uint32_t offa[SA::NI], offb[SB::NI];
  SA::offsets(offa, wv, lane, p.a_ld, p.m - m0, false, 0);
  SB::offsets(offb, wv, lane, p.b_ld, (GLU ? p.hidden : p.n) - n0, GLU, p.hidden);
  const uint32_t lds0 = lds_addr(s_tile[0]), lds1 = lds_addr(s_tile[1]);
  auto issue = [&](uint32_t lds, int k) {
    const int left = k1 - k;
    if constexpr (XA) SA::issue(lds, offa, wv, lane, p.a + (int64_t)k * p.a_ld + (int64_t)m0 * 2, 0xffffff00u, left);
    else SA::issue(lds, offa, wv, lane, p.a + (int64_t)m0 * p.a_ld + (int64_t)k * 2, 0xffffff00u, left);
    if constexpr (XB)
      SB::issue(lds + SA::BYTES, offb, wv, lane, p.b + (int64_t)k * p.b_ld + (int64_t)n0 * 2, 0xffffff00u, left);
    else
      SB::issue(lds + SA::BYTES, offb, wv, lane, p.b + (int64_t)n0 * p.b_ld + (int64_t)k * 2, 0xffffff00u, left);
  };

  f32x16 acc[NB][MB];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j) acc[i][j] = f32x16{};
  issue(lds0, k0);
  int buf = 0;
  for (int k = k0; k < k1; k += 64, buf ^= 1) {
    // this step's tile is complete, and every wavefront is done with the other buffer
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const uint32_t lds = buf ? lds1 : lds0;
    if (k + 64 < k1) issue(buf ? lds0 : lds1, k + 64);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      u32x4 fa[MB], fb[NB];
#pragma unroll
      for (int j = 0; j < MB; ++j) fa[j] = SA::frag(lds, wm * (TM / WM) + j * 32, ks, lane);
#pragma unroll
      for (int i = 0; i < NB; ++i) fb[i] = SB::frag(lds + SA::BYTES, wn * (TN / WN) + i * 32, ks, lane);
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < MB; ++j) acc[i][j] = mfma16<EK>(acc[i][j], fb[i], fa[j]);
    }
  }

  // Epilogue. Lane (l32, h) of acc[i][j] holds m = l32 and n = 8 q + 4 h + e of quad q, element e.
  const int l32 = lane & 31, h = lane >> 5;
#pragma unroll
  for (int j = 0; j < MB; ++j) {
    const int m = m0 + wm * (TM / WM) + j * 32 + l32;
    if constexpr (EPI == EPI_STORE) {
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
          const int n = n0 + wn * (TN / WN) + i * 32 + 8 * q;  // this pair of quads: 16 columns
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = acc[i][j][q * 4 + e];
          if (p.res) {
            // the lane's own quads: columns n + 4 h and n + 8 + 4 h
#pragma unroll
            for (int u = 0; u < 2; ++u)
              if (m < p.m && n + 8 * u < p.n) {
                const u32x2 r = *(const u32x2*)(p.res + m * p.res_ld + (n + 8 * u + 4 * h) * 2);
                float a, b;
                unpack2<EK>(r[0], a, b);
                v[4 * u] += a;
                v[4 * u + 1] += b;
                unpack2<EK>(r[1], a, b);
                v[4 * u + 2] += a;
                v[4 * u + 3] += b;
              }
          }
          const u32x4 o = join_halves(pack2<EK>(v[0], v[1]), pack2<EK>(v[2], v[3]), pack2<EK>(v[4], v[5]),
                                      pack2<EK>(v[6], v[7]));
          if (m < p.m && n + 8 * h < p.n) *(u32x4*)(p.out + m * p.out_ld + (n + 8 * h) * 2) = o;
        }
    } else if constexpr (EPI == EPI_PART) {
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = n0 + wn * (TN / WN) + i * 32 + 8 * q + 4 * h;
          const f32x4 o = {acc[i][j][q * 4], acc[i][j][q * 4 + 1], acc[i][j][q * 4 + 2], acc[i][j][q * 4 + 3]};
          if (m < p.m && n < p.n) *(f32x4*)(p.out + (((int64_t)split * p.m + m) * p.n + n) * 4) = o;
        }
    } else if constexpr (EPI == EPI_GLU) {
      static_assert(EPI != EPI_GLU || NB % 2 == 0, "gate and up blocks in pairs");
#pragma unroll
      for (int i = 0; i < NB; i += 2)
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
          const int f = n0 + wn * (TN / WN / 2) + (i / 2) * 32 + 8 * q;
          float v[8], none;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            v[e] = act_of<false>(p.act, acc[i][j][q * 4 + e], none) * acc[i + 1][j][q * 4 + e];
          if (p.gu) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
              if (m < p.m && f + 8 * u < p.hidden) {
                float* g = p.gu + (int64_t)m * 2 * p.hidden + f + 8 * u + 4 * h;
                const int s = (q + u) * 4;
                *(f32x4*)g = f32x4{acc[i][j][s], acc[i][j][s + 1], acc[i][j][s + 2], acc[i][j][s + 3]};
                *(f32x4*)(g + p.hidden) =
                    f32x4{acc[i + 1][j][s], acc[i + 1][j][s + 1], acc[i + 1][j][s + 2], acc[i + 1][j][s + 3]};
              }
          }
          const u32x4 o = join_halves(pack2<EK>(v[0], v[1]), pack2<EK>(v[2], v[3]), pack2<EK>(v[4], v[5]),
                                      pack2<EK>(v[6], v[7]));
          if (m < p.m && f + 8 * h < p.hidden) *(u32x4*)(p.out + m * p.out_ld + (f + 8 * h) * 2) = o;
        }
    } else {
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
          const int f = n0 + wn * (TN / WN) + i * 32 + 8 * q;
          float dg[8], du[8];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            f32x4 g = {}, up = {};
            if (m < p.m && f + 8 * u < p.hidden) {
              const float* at = p.gu + (int64_t)m * 2 * p.hidden + f + 8 * u + 4 * h;
              g = *(const f32x4*)at;
              up = *(const f32x4*)(at + p.hidden);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float dh = acc[i][j][(q + u) * 4 + e];
              float slope;
              du[4 * u + e] = dh * act_of<true>(p.act, g[e], slope);
              dg[4 * u + e] = dh * up[e] * slope;
            }
          }
          const u32x4 og = join_halves(pack2<EK>(dg[0], dg[1]), pack2<EK>(dg[2], dg[3]), pack2<EK>(dg[4], dg[5]),
                                       pack2<EK>(dg[6], dg[7]));
          const u32x4 ou = join_halves(pack2<EK>(du[0], du[1]), pack2<EK>(du[2], du[3]), pack2<EK>(du[4], du[5]),
                                       pack2<EK>(du[6], du[7]));
          if (m < p.m && f + 8 * h < p.hidden) {
            char* o = p.out + m * p.out_ld + (f + 8 * h) * 2;
            *(u32x4*)o = og;
            *(u32x4*)(o + (int64_t)p.hidden * 2) = ou;
          }
        }
    }
  }
}

// out = the sum of the splits' fp32 partial sums, rounded once; four elements a thread.
template <int EK>
__global__ void __launch_bounds__(256) sum_parts_kernel(const float* part, int splits, int64_t n4, char* out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n4) return;
  f32x4 a = *(const f32x4*)(part + i * 4);
  for (int s = 1; s < splits; ++s) {
    const f32x4 b = *(const f32x4*)(part + ((int64_t)s * n4 + i) * 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] += b[e];
  }
  *(u32x2*)(out + i * 8) = u32x2{pack2<EK>(a[0], a[1]), pack2<EK>(a[2], a[3])};
}

constexpr int kTM = 256, kTN = 256;

template <int EK, bool XA, bool XB, int EPI>
int launch_gemm(GemmP p, hipStream_t s) {
  const int n = EPI == EPI_GLU ? 2 * p.hidden : p.n;
  p.tiles_m = (p.m + kTM - 1) / kTM;
  p.tiles_n = EPI == EPI_GLU ? (p.hidden + kTN / 2 - 1) / (kTN / 2) : (n + kTN - 1) / kTN;
  launch_kernel(gemm_kernel<EK, XA, XB, kTM, kTN, 4, 2, EPI>, dim3((unsigned)(p.tiles_m * p.tiles_n * p.splits)),
                dim3(512), 0u, s, p);
  return hipGetLastError() == hipSuccess ? LIK_OK : LIK_ERR_LAUNCH;
}

// Weight gradients have few tiles and a long k (the rows): k is split so that the
// tiles fill the 256 CUs, in steps of 64 k.
struct Splits {
  int splits, k_per;
};
Splits weight_splits(int m, int n, int64_t k) {
  const int tiles = ((m + kTM - 1) / kTM) * ((n + kTN - 1) / kTN);
  int64_t want = 256 / tiles;
  const int64_t most = (k + 511) / 512;
  if (want > most) want = most;
  if (want < 1) want = 1;
  const int64_t per = ((k + want - 1) / want + 63) / 64 * 64;
  return {(int)((k + per - 1) / per), (int)per};
}

template <int EK>
int weight_grad(GemmP p, char* out, float* part, hipStream_t s) {
  const Splits sp = weight_splits(p.m, p.n, p.k);
  p.splits = sp.splits;
  p.k_per = sp.k_per;
  if (sp.splits == 1) {
    p.out = out;
    p.out_ld = (int64_t)p.n * 2;
    return launch_gemm<EK, true, true, EPI_STORE>(p, s);
  }
  p.out = (char*)part;
  if (const int rc = launch_gemm<EK, true, true, EPI_PART>(p, s)) return rc;
  const int64_t n4 = (int64_t)p.m * p.n / 4;
  launch_kernel(sum_parts_kernel<EK>, dim3((unsigned)((n4 + 255) / 256)), dim3(256), 0u, s, (const float*)part,
                sp.splits, n4, out);
  return hipGetLastError() == hipSuccess ? LIK_OK : LIK_ERR_LAUNCH;
}

struct FfnBwdWs {
  size_t dgu, part, total;
};
FfnBwdWs ffn_bwd_ws(int64_t rows, int d, int f) {
  FfnBwdWs w;
  w.dgu = 0;
  const Splits a = weight_splits(2 * f, d, rows), b = weight_splits(d, f, rows);
  const size_t pa = a.splits > 1 ? (size_t)a.splits * 2 * f * d * 4 : 0;
  const size_t pb = b.splits > 1 ? (size_t)b.splits * d * f * 4 : 0;
  w.part = align256((size_t)rows * 2 * f * 2);
  w.total = w.part + (pa > pb ? pa : pb) + 256;
  return w;
}

int ffn_check(int32_t dtype, int64_t rows, int32_t d, int32_t f, int32_t act) {
  if (dtype != LIK_BF16 && dtype != LIK_F16) return LIK_ERR_UNSUPPORTED;
  if (rows < 0 || d < 8 || f < 8 || act < ACT_GELU || act > ACT_SILU) return LIK_ERR_INVALID;
  // 16-byte chunks of k; rows of weights and tokens within a 32-bit tile offset
  if (d % 8 || f % 8 || d > (1 << 20) || f > (1 << 20) || rows > 0x7fffff00) return LIK_ERR_UNSUPPORTED;
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
                float* gu, hipStream_t s) {
  GemmP p{};
  p.splits = 1;
  p.act = act;
  p.hidden = f;
  p.m = (int)rows;
  p.a = (const char*)x;
  p.a_ld = x_ld * 2;
  p.b = (const char*)w_in;
  p.b_ld = wi_ld * 2;
  p.n = f;
  p.k = p.k_per = d;
  p.out = (char*)h;
  p.out_ld = (int64_t)f * 2;
  p.gu = gu;
  if (const int rc = launch_gemm<EK, false, false, EPI_GLU>(p, s)) return rc;
  p.a = (const char*)h;
  p.a_ld = (int64_t)f * 2;
  p.b = (const char*)w_out;
  p.b_ld = wo_ld * 2;
  p.n = d;
  p.k = p.k_per = f;
  p.out = (char*)out;
  p.out_ld = (int64_t)d * 2;
  p.res = (const char*)res;
  p.res_ld = res_ld * 2;
  return launch_gemm<EK, false, false, EPI_STORE>(p, s);
}

template <int EK>
int ffn_backward(const void* g, int64_t g_ld, const void* x, int64_t x_ld, int64_t rows, int d, int f,
                 const void* w_in, int64_t wi_ld, const void* w_out, int64_t wo_ld, const void* h, const float* gu,
                 int act, void* gx, void* gw_in, void* gw_out, char* ws, hipStream_t s) {
  const FfnBwdWs w = ffn_bwd_ws(rows, d, f);
  char* dgu = ws + w.dgu;
  float* part = (float*)(ws + w.part);
  GemmP p{};
  p.splits = 1;
  p.act = act;
  p.hidden = f;
  if (gx || gw_in) {
    p.m = (int)rows;
    p.a = (const char*)g;
    p.a_ld = g_ld * 2;
    p.b = (const char*)w_out;
    p.b_ld = wo_ld * 2;
    p.n = f;
    p.k = p.k_per = d;
    p.out = dgu;
    p.out_ld = (int64_t)f * 4;
    p.gu = const_cast<float*>(gu);
    if (const int rc = launch_gemm<EK, false, true, EPI_GLU_BWD>(p, s)) return rc;
  }
  if (gx) {
    p.a = dgu;
    p.a_ld = (int64_t)f * 4;
    p.b = (const char*)w_in;
    p.b_ld = wi_ld * 2;
    p.n = d;
    p.k = p.k_per = 2 * f;
    p.out = (char*)gx;
    p.out_ld = (int64_t)d * 2;
    if (const int rc = launch_gemm<EK, false, true, EPI_STORE>(p, s)) return rc;
  }
  p.k = (int)rows;
  if (gw_in) {
    p.m = 2 * f;
    p.n = d;
    p.a = dgu;
    p.a_ld = (int64_t)f * 4;
    p.b = (const char*)x;
    p.b_ld = x_ld * 2;
    if (const int rc = weight_grad<EK>(p, (char*)gw_in, part, s)) return rc;
  }
  if (gw_out) {
    p.m = d;
    p.n = f;
    p.a = (const char*)g;
    p.a_ld = g_ld * 2;
    p.b = (const char*)h;
    p.b_ld = (int64_t)f * 2;
    if (const int rc = weight_grad<EK>(p, (char*)gw_out, part, s)) return rc;
  }
  return LIK_OK;
}

}  // namespace
}  // namespace enc
}  // namespace lik

using namespace lik;
using namespace lik::enc;

extern "C" {

int lik_gated_ffn(const void* x, int64_t x_stride, int32_t dtype, int64_t rows, int32_t dim, int32_t hidden,
                  const void* w_in, int64_t w_in_stride, const void* w_out, int64_t w_out_stride, const void* residual,
                  int64_t residual_stride, int32_t activation, void* out, void* hidden_act, float* gate_up,
                  lik_stream_t stream) {
  if (const int rc = ffn_check(dtype, rows, dim, hidden, activation)) return rc;
  if (rows == 0) return LIK_OK;
  if (!x || !w_in || !w_out || !out || !hidden_act) return LIK_ERR_INVALID;
  if (!rows16(x, x_stride) || !rows16(w_in, w_in_stride, hidden) || !rows16(w_out, w_out_stride) || !rows16(out, 0) ||
      !rows16(hidden_act, 0) || !rows16(gate_up, 0) || (residual && !rows16(residual, residual_stride)))
    return LIK_ERR_UNSUPPORTED;
  const auto fn = dtype == LIK_BF16 ? ffn_forward<EK_BF16> : ffn_forward<EK_F16>;
  return fn(x, x_stride, rows, dim, hidden, w_in, w_in_stride, w_out, w_out_stride, residual, residual_stride,
            activation, out, hidden_act, gate_up, (hipStream_t)stream);
}

size_t lik_gated_ffn_backward_workspace_size(int32_t dtype, int64_t rows, int32_t dim, int32_t hidden) {
  if (ffn_check(dtype, rows, dim, hidden, ACT_GELU) != LIK_OK || rows == 0) return 0;
  return ffn_bwd_ws(rows, dim, hidden).total;
}

int lik_gated_ffn_backward(const void* grad, int64_t grad_stride, const void* x, int64_t x_stride, int32_t dtype,
                           int64_t rows, int32_t dim, int32_t hidden, const void* w_in, int64_t w_in_stride,
                           const void* w_out, int64_t w_out_stride, const void* hidden_act, const float* gate_up,
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
