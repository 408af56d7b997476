// Attention, backward. With p from the scores and the kept statistics,
//   dv_j = sum_i p_ij g_i,  ds_ij = p_ij (g_i v_j - delta_i),  delta_i = sum_d g_i o_i
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i
// Two kernels, each with the sums of its own rows in registers: one walks the keys for
// the gradient of q, one the queries (of every head that shares the key head) for
// those of k and v. Both compute the scores and g v again: seven products where
// one kernel with the gradient of q in memory would take five, but no atomics (the
// same bits every time) and no fp32 gradient of q to clear, add to and convert.
// 16 causal sequences of 1030 rows, 16 heads over 4 of 128, bf16: 184 us (567 TFLOP/s of its three products) and
// 237 us (587, four), two wavefronts a SIMD at 226 and 250 registers, bound by the chain from scores to
// probabilities to products inside a wavefront. Sequences of 129 to 320 keys have one kernel for all three: 128 passages of 50 to 300
// rows, 12 heads of 64: 155 us, the two 88 and 93.
// p and ds are rounded once to the 16-bit type, as the products' operands have to be. fp16 has no range for either: p is
// held 2^14 times (2^-28 is still a normal number), and ds 2^14 gs times, gs the power of two that brings the bound
// |g v - delta| <= 2 dim max|g| max|v| to 1 .. 2 (of a wavefront's queries; of a key head's): nothing passes 2^15, and the
// largest elements, some 2^6 under the bound, keep 20 powers of two below them. The sums are scaled back.
#include "lik_attn.h"

namespace lik {
namespace enc {
namespace {

// log2 of what p is held times
template <int EK>
constexpr float kLiftP = EK == EK_F16 ? 14.0f : 0.0f;
template <int EK>
constexpr float kUnliftP = EK == EK_F16 ? 1.0f / 16384 : 1.0f;
// A pair's probability from its score and the query's L, 2^kLiftP times. L is taken off the score first, not inside the
// exponent: c L past 2^11 or so is spaced too widely for that (scores of 1e5 gave gradients 1% off), and one more
// instruction costs less than asking for it.
template <int EK>
__device__ __forceinline__ float pair_p(const AttP& p, float s, float l) {
  return __builtin_amdgcn_exp2f(EK == EK_F16 ? fmaf(s - l, p.c, kLiftP<EK>) : (s - l) * p.c);
}
// gs from the largest |g| and |v| (1 where one is zero)
__device__ __forceinline__ float scale_for(float g, float v, int dim) {
  const float bound = 2.0f * (float)dim * g * v;
  if (!(bound > 0.f)) return 1.0f;
  int e;
  frexpf(bound, &e);  // bound = m 2^e, m in 1/2 .. 1
  return ldexpf(2.0f, -e);
}
// The largest finite |x| of N chunks of fp16 elements: rows that are not finite are NaN in the end, at any scale.
template <int N>
__device__ __forceinline__ float max_finite(const u32x4* x) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  u16x2 m = {0, 0};
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, x[k][i] & 0x7fff7fffu));
  uint32_t top = m[0] > m[1] ? m[0] : m[1];
  if (__ballot(top >= 0x7c00u) != 0) {  // infinities or NaN: one by one
    top = 0;
    for (int k = 0; k < N; ++k)
      for (int i = 0; i < 8; ++i) {
        const uint32_t a = (x[k][i / 2] >> (16 * (i % 2))) & 0x7fffu;
        if (a < 0x7c00u && a > top) top = a;
      }
  }
  return f16_to_f32((uint16_t)top);
}

// fp16: the largest |v| of 128 keys of a key head. One read of the values: 17 MB (16 x 1030 rows, 4 heads of 128) 6 us.
__global__ void __launch_bounds__(256) attention_vmax_kernel(const AttP p) {
  __shared__ float s_big[4];
  const int tid = threadIdx.x, kv_heads = p.heads / p.group;
  const int tile = (int)(blockIdx.x % (unsigned)p.k_tiles);
  const unsigned t = blockIdx.x / (unsigned)p.k_tiles;
  const int kvh = (int)(t % (unsigned)kv_heads), seq = (int)(t / (unsigned)kv_heads);
  const Span ks = span_of(p.cu_k, p.k_rows, p.k_len, seq);
  const char* base = p.v.data + (p.cu_k ? ks.row * p.v.sl : seq * p.v.sn) + kvh * p.v.sh;
  const int chunks = p.dim / 8;
  u32x4 x[8];  // (at most 16 chunks a row)
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int i = j * 256 + tid, pos = tile * 128 + i / chunks;
    x[j] = u32x4{0u, 0u, 0u, 0u};
    if (i < 128 * chunks && pos < ks.len && (!p.km || p.km[seq * p.km_sn + pos * p.km_sl] != 0))
      x[j] = *(const u32x4*)(base + pos * p.v.sl + i % chunks * 16);
  }
  const float big = wave_max(max_finite<8>(x));
  if ((tid & 63) == 0) s_big[tid >> 6] = big;
  __syncthreads();
  if (tid == 0) p.vmax[blockIdx.x] = fmaxf(fmaxf(s_big[0], s_big[1]), fmaxf(s_big[2], s_big[3]));
}
// A key head's largest |v| (all lanes of a wavefront).
__device__ __forceinline__ float head_vmax(const AttP& p, int seq, int kvh, int lane) {
  const float* at = p.vmax + ((int64_t)seq * (p.heads / p.group) + kvh) * p.k_tiles;
  float big = 0.f;
  for (int i = lane; i < p.k_tiles; i += 64) big = fmaxf(big, at[i]);
  return wave_max(big);
}

// delta of the lane's query, whose g is in columns (on: it has one; else 0), and the largest |g| for fp16. row: its first
// element in the output.
template <int EK, int DC>
__device__ __forceinline__ float row_delta(const AttP& p, const u32x4* gf, int64_t row, bool on, float& big, int lane) {
  u32x4 of[Dim<DC>::KS];
  load_cols<DC>(of, on ? p.out + row * 2 : nullptr, p.dim, lane);
  float d = 0.f;
#pragma unroll
  for (int k = 0; k < Dim<DC>::KS; ++k) {
    const int e = k * 16 + 8 * (lane >> 5);
    u32x2 low = {0u, 0u};
    if (on && e < p.dim) low = *(const u32x2*)(p.low + row + e);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float g[2], o[2];
      unpack2<EK>(gf[k][i / 2], g[0], g[1]);
      unpack2<EK>(of[k][i / 2], o[0], o[1]);
      d = fmaf(g[i % 2], with_low<EK>(o[i % 2], low[i / 4], i % 4), d);
    }
  }
  if constexpr (EK == EK_F16) big = fmaxf(big, max_finite<Dim<DC>::KS>(gf));
  return d + swap_half(d);
}

// Gradients of the lane's key (kon: it is kept) to memory, from their sums; those of a key that no kept query sees are zeros.
// Its pairs added p = 0 times what the rows hold, which is no zero where a kept key or its value is not finite: then (and only
// then) the queries' statistics (`lse`, [heads of the group][q_total], the sequence's first row) are asked. at: the row's byte in
// both; kpos < klen: it exists.
template <int EK, int DC>
__device__ __forceinline__ void store_key(const AttP& p, f32x16* dk, f32x16* dv, float fk, int64_t at, bool kon, int kpos,
                                          int klen, const float* lse, int qlen, int lane) {
  if (!kon)  // (their lanes ran on zero rows)
#pragma unroll
    for (int d = 0; d < DC; ++d) dk[d] = dv[d] = f32x16{};
  float odd = store_cols<EK, DC>(p.gk + at, dk, fk, p.dim, lane, kpos < klen) +
              store_cols<EK, DC>(p.gv + at, dv, kUnliftP<EK>, p.dim, lane, kpos < klen);
  odd += swap_half(odd);
  bool seen = odd == 0.f;
  if (__ballot(!seen) == 0) return;
  for (int h = 0; h < p.group; ++h)
    for (int q0 = 0; q0 < qlen && __ballot(!seen) != 0; q0 += 64) {  // a lane a query, then a lane a key
      const uint64_t have = __ballot(q0 + lane < qlen && lse[(int64_t)h * p.q_total + q0 + lane] != INFINITY);
      const int lo = p.right == kNone || kpos - p.right < q0 ? 0 : kpos - p.right - q0;
      const int hi = p.left == kNone || kpos + p.left > q0 + 63 ? 63 : kpos + p.left - q0;
      if (lo <= 63 && hi >= 0) seen = seen || (have & (~0ull << lo) & (~0ull >> (63 - hi))) != 0;
    }
  const int e = 8 * (lane >> 5);  // (the lane's own 16 bytes, written above)
  for (int d = e; d < p.dim; d += 16)
    if (!seen && kpos < klen) {
      *(u32x4*)(p.gk + at + d * 2) = u32x4{0u, 0u, 0u, 0u};
      *(u32x4*)(p.gv + at + d * 2) = u32x4{0u, 0u, 0u, 0u};
    }
}

// Gradient of q: the forward's walk over the keys (K rows also by transposing
// reads, V rows in LDS), dq^T[d][query] += K^T ds^T. Its queries' delta, which the other kernel reads, comes
// from the same registers.
template <int EK, int DC>
__global__ void __launch_bounds__(256, 2) attention_dq_kernel(const AttP p) {
  using D = Dim<DC>;
  __shared__ __attribute__((aligned(1024))) char s_tile[2][2 * D::TILE];
  __shared__ int s_kept[2];
  __shared__ float s_big[4];
  extern __shared__ uint32_t s_bits[];
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int item = work_item(p);
  if (item < 0) return;
  uint32_t t = (uint32_t)item;
  const int tile = (int)(t % (uint32_t)p.tiles);
  t /= (uint32_t)p.tiles;
  const int head = (int)(t % (uint32_t)p.heads), seq = (int)(t / (uint32_t)p.heads);
  const int kvh = head / p.group;
  const Span qs = span_of(p.cu_q, p.q_rows, p.q_len, seq), ks = span_of(p.cu_k, p.k_rows, p.k_len, seq);
  const int q0 = tile * 128;
  if (p.gq) clear_uncovered(p, item, p.cu_q, p.q_rows, p.heads * p.dim / 8, p.gq);
  float* gmax = EK == EK_F16 ? p.gmax + ((int64_t)seq * p.heads + head) * p.q_tiles + tile : nullptr;
  if (q0 >= qs.len) {
    if (EK == EK_F16 && tid == 0) *gmax = 0.f;
    return;
  }

  u32x4 qf[D::KS], gf[D::KS];
  const char* qbase = p.q.data + (p.cu_q ? qs.row * p.q.sl : seq * p.q.sn) + head * p.q.sh;
  const char* gbase = p.g.data + (p.cu_q ? qs.row * p.g.sl : seq * p.g.sn) + head * p.g.sh;
  float big = 0.f;
  const int qpos = q0 + wv * 32 + l32;  // the lane's query
  const int64_t at = (int64_t)head * p.q_total + qs.row + qpos;
  const float lse = qpos < qs.len ? p.lse[at] : INFINITY;
  const bool on = lse != INFINITY;  // +inf: past the end, masked, or without a key
  load_cols<DC>(qf, on ? qbase + qpos * p.q.sl : nullptr, p.dim, lane);
  load_cols<DC>(gf, on ? gbase + qpos * p.g.sl : nullptr, p.dim, lane);
  const int64_t row = ((qs.row + qpos) * p.heads + head) * p.dim;
  const float delta = row_delta<EK, DC>(p, gf, row, on, big, lane);
  if (qpos < qs.len && lane < 32) p.delta[at] = delta;
  const bool any = __ballot(on) != 0;  // this wavefront has a query
  float gs = 1.0f;  // of this wavefront's queries
  if constexpr (EK == EK_F16) {
    big = wave_max(big);
    if (lane == 0) s_big[wv] = big;
    gs = scale_for(big, head_vmax(p, seq, kvh, lane), p.dim);
    __syncthreads();
    if (tid == 0) *gmax = fmaxf(fmaxf(s_big[0], s_big[1]), fmaxf(s_big[2], s_big[3]));
  }

  int klen = ks.len;
  bool holes = false;
  if (p.km) {
    const Kept kept = scan_mask(s_bits, p.km + seq * p.km_sn, p.km_sl, klen, s_kept);
    klen = kept.extent;
    holes = kept.holes;
  }
  const int q_end = (q0 + 128 < qs.len ? q0 + 128 : qs.len) - 1;
  const int kb = p.left == kNone || q0 - p.left < 0 ? 0 : (q0 - p.left) & ~63;
  int ke = p.right == kNone || (int64_t)q_end + p.right + 1 >= klen ? klen : q_end + p.right + 1;
  if (__syncthreads_or(any) == 0 || !p.gq) ke = kb;

  const char* kbase = p.k.data + (p.cu_k ? ks.row * p.k.sl : seq * p.k.sn) + kvh * p.k.sh;
  const char* vbase = p.v.data + (p.cu_k ? ks.row * p.v.sl : seq * p.v.sn) + kvh * p.v.sh;
  const Rows<DC> krows(p.k.sl, p.dim, wv, lane), vrows(p.v.sl, p.dim, wv, lane);
  const Frags<DC> frags(lane);
  const uint32_t lds[2] = {lds_addr(s_tile[0]), lds_addr(s_tile[1])};
  auto issue = [&](uint32_t at, int kt) {
    const uint32_t* bits = holes ? s_bits + (kt >> 5) : nullptr;
    krows.issue(at, kbase + kt * p.k.sl, klen - kt, bits, wv, lane);
    vrows.issue(at + D::TILE, vbase + kt * p.v.sl, klen - kt, bits, wv, lane);
  };

  const Window win(p);
  f32x16 acc[DC];
#pragma unroll
  for (int d = 0; d < DC; ++d) acc[d] = f32x16{};
  const int wq0 = q0 + wv * 32, wq1 = wq0 + 31;  // the wavefront's queries
  if (kb < ke) issue(lds[0], kb);
  int buf = 0;
  for (int kt = kb; kt < ke; kt += 64, buf ^= 1) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (kt + 64 < ke) issue(buf ? lds[0] : lds[1], kt + 64);
    if (!any || (p.right != kNone && kt > wq1 + p.right) || (p.left != kNone && kt + 63 < wq0 - p.left)) continue;
    const uint32_t at = buf ? lds[1] : lds[0];
    const bool whole = kt + 64 <= klen && !holes && (p.right == kNone || kt + 63 <= wq0 + p.right) &&
                       (p.left == kNone || kt >= wq1 - p.left);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f32x16 s = {}, dp = {};
#pragma unroll
      for (int k = 0; k < D::KS; ++k) {
        const u32x4 kf = frags.row(at, u * 32, k);
        const u32x4 vf = frags.row(at + D::TILE, u * 32, k);
        s = mfma16<EK>(s, kf, qf[k]);
        dp = mfma16<EK>(dp, vf, gf[k]);
      }
      if (!whole)
        mask_scores(s, kt + u * 32, klen, holes ? s_bits : nullptr, win.on,
                    kt + u * 32 + 4 * (lane >> 5) - qpos + win.back, win.reach, lane);
      u32x4 df[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = pair_p<EK>(p, s[i], lse);
        s[i] = e * (EK == EK_F16 ? (dp[i] - delta) * gs : dp[i] - delta);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) df[k][e] = pack2<EK>(s[k * 8 + 2 * e], s[k * 8 + 2 * e + 1]);
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int d = 0; d < DC; ++d) {
          const u32x4 kf = frags.col(at, u * 32 + k * 16, d);
          acc[d] = mfma16<EK>(acc[d], kf, df[k]);
        }
    }
  }
  if (!p.gq) return;
  if (!on)  // no gradient, whatever the keys and values hold (their lanes ran on zero rows)
#pragma unroll
    for (int d = 0; d < DC; ++d) acc[d] = f32x16{};
  store_cols<EK, DC>(p.gq + ((qs.row + qpos) * p.heads + head) * p.dim * 2, acc, p.scale * kUnliftP<EK> / gs, p.dim, lane,
                     qpos < qs.len);
}

// Masked keys under a causal order or a window leave single queries without a key: their statistics say which. (Without
// either, a mask leaves all queries without one or none. Longer sequences' bits do not fit LDS: there the rows are read.)
__host__ __device__ __forceinline__ bool by_statistic(const AttP& p) {
  return p.km && (p.left != kNone || p.right != kNone) && p.q_len <= kMaskMost;
}

// Gradients of k and v: a wavefront owns 32 keys as MFMA columns and walks the queries of the group's
// heads, QT at a time, K in registers. For head dims over 32 V's rows stay in LDS, which leaves room for three
// wavefronts a SIMD up to 64 (262 -> 252 us for the training step on 128 passages) and for two above, where a
// step is 32 queries (455 -> 258 us of this kernel for 16 x 1030 causal rows, 16 / 4 heads of 128).
//   P[query][key] from S = Q K^T;  dv^T[d][key] += G^T P;  dp = G V^T;  dk^T[d][key] += Q^T ds
template <int EK, int DC>
__global__ void __launch_bounds__(256, DC <= 2 ? 3 : 2) attention_dkv_kernel(const AttP p) {
  using D = Dim<DC>;
  constexpr bool VL = DC > 1;  // V in LDS
  constexpr int QT = DC > 2 ? 32 : 64, TILE = D::PITCH * QT;
  __shared__ __attribute__((aligned(1024))) char s_tile[2][2 * TILE];
  __shared__ __attribute__((aligned(1024))) char s_v[VL ? 2 * D::TILE : 16];
  __shared__ __attribute__((aligned(16))) float s_stat[2][2][QT];  // L and delta
  __shared__ int s_kept[2];
  __shared__ float s_big[4];
  extern __shared__ uint32_t s_bits[];
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kv_heads = p.heads / p.group;
  const int item = work_item(p);
  if (item < 0) return;
  uint32_t t = (uint32_t)item;
  const int tile = (int)(t % (uint32_t)p.tiles);
  t /= (uint32_t)p.tiles;
  const int kvh = (int)(t % (uint32_t)kv_heads), seq = (int)(t / (uint32_t)kv_heads);
  const Span qs = span_of(p.cu_q, p.q_rows, p.q_len, seq), ks = span_of(p.cu_k, p.k_rows, p.k_len, seq);
  const int k0 = tile * 128;
  clear_uncovered(p, item, p.cu_k, p.k_rows, kv_heads * p.dim / 8, p.gk);
  clear_uncovered(p, item, p.cu_k, p.k_rows, kv_heads * p.dim / 8, p.gv);
  if (k0 >= ks.len) return;
  float gs = 1.0f;
  if constexpr (EK == EK_F16) {
    const float* gm = p.gmax + ((int64_t)seq * p.heads + kvh * p.group) * p.q_tiles;
    float big = 0.f;
    for (int i = tid; i < p.group * p.q_tiles; i += 256) big = fmaxf(big, gm[i]);
    big = wave_max(big);
    if (lane == 0) s_big[wv] = big;
    __syncthreads();
    gs = scale_for(fmaxf(fmaxf(s_big[0], s_big[1]), fmaxf(s_big[2], s_big[3])), head_vmax(p, seq, kvh, lane), p.dim);
  }

  u32x4 kf[D::KS], vf[VL ? 1 : D::KS];
  const char* kbase = p.k.data + (p.cu_k ? ks.row * p.k.sl : seq * p.k.sn) + kvh * p.k.sh;
  const char* vbase = p.v.data + (p.cu_k ? ks.row * p.v.sl : seq * p.v.sn) + kvh * p.v.sh;
  const int kpos = k0 + wv * 32 + l32;  // the lane's key
  const bool kon = kpos < ks.len && (!p.km || p.km[seq * p.km_sn + kpos * p.km_sl] != 0);
  load_cols<DC>(kf, kon ? kbase + kpos * p.k.sl : nullptr, p.dim, lane);
  if constexpr (!VL) load_cols<DC>(vf, kon ? vbase + kpos * p.v.sl : nullptr, p.dim, lane);
  const bool any = __ballot(kon) != 0;
  if constexpr (VL) {  // (what masked rows hold stays in their own columns)
    const Rows<DC> vrows(p.v.sl, p.dim, wv, lane);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      vrows.issue(lds_addr(s_v) + i * D::TILE, vbase + (k0 + 64 * i) * p.v.sl, ks.len - k0 - 64 * i, nullptr, wv, lane);
  }

  // Queries that keep no key are not read: what their rows of q and g hold would meet p = 0 in the products, which is no
  // zero for infinities and NaN.
  int qlen = qs.len;
  if (p.left != kNone && (int64_t)ks.len + p.left < qlen) qlen = ks.len + p.left;  // (the window ends before the last ones)
  bool holes = false;
  if (p.qm || by_statistic(p)) {
    const float* lse = p.lse + (int64_t)kvh * p.group * p.q_total + qs.row;
    const Kept kept = by_statistic(p) ? scan_kept(s_bits, qlen, s_kept,
                                                  [&](int t) {
                                                    bool on = false;
                                                    for (int h = 0; h < p.group; ++h)
                                                      on = on || lse[h * p.q_total + t] != INFINITY;
                                                    return on;
                                                  })
                                      : scan_mask(s_bits, p.qm + seq * p.qm_sn, p.qm_sl, qlen, s_kept);
    qlen = kept.extent;
    holes = kept.holes;
  }
  // queries that keep one of these keys: key - right <= query <= key + left
  const int k_end = (k0 + 128 < ks.len ? k0 + 128 : ks.len) - 1;
  const int qb = p.right == kNone || k0 - p.right < 0 ? 0 : (k0 - p.right) & ~63;
  int qe = p.left == kNone || (int64_t)k_end + p.left + 1 >= qlen ? qlen : k_end + p.left + 1;
  if (__syncthreads_or(any) == 0) qe = qb;
  const int steps = qe > qb ? (qe - qb + QT - 1) / QT : 0;  // of one head

  const Rows<DC, QT> qrows(p.q.sl, p.dim, wv, lane), grows(p.g.sl, p.dim, wv, lane);
  const Frags<DC> frags(lane);
  const uint32_t lds[2] = {lds_addr(s_tile[0]), lds_addr(s_tile[1])};
  const char* q0 = p.q.data + (p.cu_q ? qs.row * p.q.sl : seq * p.q.sn);
  const char* g0 = p.g.data + (p.cu_q ? qs.row * p.g.sl : seq * p.g.sn);
  auto issue = [&](uint32_t at, int head, int qt) {
    const uint32_t* bits = holes ? s_bits + (qt >> 5) : nullptr;
    qrows.issue(at, q0 + head * p.q.sh + qt * p.q.sl, qlen - qt, bits, wv, lane);
    grows.issue(at + TILE, g0 + head * p.g.sh + qt * p.g.sl, qlen - qt, bits, wv, lane);
  };
  // threads 0..QT - 1: a query's L (+inf past the end: p = 0), QT..2 QT - 1: its delta
  auto stat = [&](int head, int qt) {
    float x = 0.f;
    if (tid < 2 * QT) {
      const int pos = qt + tid % QT;
      const int64_t at = (int64_t)head * p.q_total + qs.row + pos;
      x = pos < qlen ? (tid < QT ? p.lse[at] : p.delta[at]) : tid < QT ? INFINITY : 0.f;
    }
    return x;
  };

  // a query keeps a key where 0 <= query - key + ahead <= reach
  const int ahead = p.right == kNone ? 0x3fffffff : p.right;
  const uint32_t reach = (uint32_t)ahead + (p.left == kNone ? 0x3fffffffu : (uint32_t)p.left);
  f32x16 dk[DC], dv[DC];
#pragma unroll
  for (int d = 0; d < DC; ++d) dk[d] = dv[d] = f32x16{};
  const int wk0 = k0 + wv * 32, wk1 = wk0 + 31;  // the wavefront's keys
  const int total = steps * p.group;
  int head = kvh * p.group, qt = qb;
  if (total) {
    const float x = stat(head, qt);
    issue(lds[0], head, qt);
    if (tid < 2 * QT) s_stat[0][tid / QT][tid % QT] = x;
  }
  int buf = 0;
  for (int it = 0; it < total; ++it, buf ^= 1) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const int now = qt;
    qt += QT;
    if (qt >= qe) {
      qt = qb;
      ++head;
    }
    float next = 0.f;
    if (it + 1 < total) {
      next = stat(head, qt);
      issue(buf ? lds[0] : lds[1], head, qt);
    }
    const bool skip = !any || (p.left != kNone && now > wk1 + p.left) || (p.right != kNone && now + QT - 1 < wk0 - p.right);
    if (!skip) {
      const uint32_t at = buf ? lds[1] : lds[0];
      const bool whole =
          (p.left == kNone || now + QT - 1 <= wk0 + p.left) && (p.right == kNone || now >= wk1 - p.right);
#pragma unroll
      for (int u = 0; u < QT / 32; ++u) {
        f32x16 s = {}, dp = {};
#pragma unroll
        for (int k = 0; k < D::KS; ++k) {
          const u32x4 qf = frags.row(at, u * 32, k);
          const u32x4 gf = frags.row(at + TILE, u * 32, k);
          s = mfma16<EK>(s, qf, kf[k]);
          dp = mfma16<EK>(dp, gf, VL ? frags.row(lds_addr(s_v), wv * 32, k) : vf[VL ? 0 : k]);
        }
        if (!whole)
          mask_scores(s, 0, 64, nullptr, true, now + u * 32 + 4 * (lane >> 5) - kpos + ahead, reach, lane);
        u32x4 pf[2], df[2];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x4 ls = *(const f32x4*)&s_stat[buf][0][u * 32 + 8 * q + 4 * (lane >> 5)];
          const f32x4 dl = *(const f32x4*)&s_stat[buf][1][u * 32 + 8 * q + 4 * (lane >> 5)];
          float e[4], ds[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            e[i] = pair_p<EK>(p, s[q * 4 + i], ls[i]);
            const float x = dp[q * 4 + i] - dl[i];
            ds[i] = e[i] * (EK == EK_F16 ? x * gs : x);
          }
          pf[q / 2][(q % 2) * 2] = pack2<EK>(e[0], e[1]);
          pf[q / 2][(q % 2) * 2 + 1] = pack2<EK>(e[2], e[3]);
          df[q / 2][(q % 2) * 2] = pack2<EK>(ds[0], ds[1]);
          df[q / 2][(q % 2) * 2 + 1] = pack2<EK>(ds[2], ds[3]);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int d = 0; d < DC; ++d) {
            const u32x4 gc = frags.col(at + TILE, u * 32 + k * 16, d);
            const u32x4 qc = frags.col(at, u * 32 + k * 16, d);
            dv[d] = mfma16<EK>(dv[d], gc, pf[k]);
            dk[d] = mfma16<EK>(dk[d], qc, df[k]);
          }
      }
    }
    if (it + 1 < total && tid < 2 * QT) s_stat[buf ^ 1][tid / QT][tid % QT] = next;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // V's loads where there was no step
  const int64_t at = ((ks.row + kpos) * kv_heads + kvh) * p.dim * 2;
  store_key<EK, DC>(p, dk, dv, p.scale * kUnliftP<EK> / gs, at, kon, kpos, ks.len,
                    p.lse + (int64_t)kvh * p.group * p.q_total + qs.row, qs.len, lane);
}

// All gradients of sequences of up to 32 KW keys in one pass: five products and one read of the rows, no sum in memory. A
// workgroup has a key head. KW wavefronts own 32 keys each, as above (K and V in registers), and walk the queries 32 at a time; their
// ds goes through LDS to DC more wavefronts with a block of 32 head dims each: dq^T[d][query] = K^T ds^T of the step before, over all
// keys at once. The queries' statistics come first, by all wavefronts (one wait for memory, and the rows are in L2 for the walk):
// up to kShortRows of them, all heads of the group together.
// 128 passages of 50 to 300 rows padded to 300, 12 heads of 64, bf16: 155 us, about 80 of them the reads and writes around the walk (65
// at the copy rate; a workgroup of 12 wavefronts at 162 registers fills a CU, so its walk overlaps no other's loads), the rest the steps.
constexpr int kShortRows = 2048;
template <int EK, int DC, int KW>
__global__ void __launch_bounds__((KW + DC) * 64, (KW + DC + 3) / 4) attention_grads_kernel(const AttP p) {
  using D = Dim<DC>;
  constexpr int T = (KW + DC) * 64, TILE = 32 * D::PITCH, DS = 32 * 64;
  __shared__ __attribute__((aligned(1024))) char s_k[KW * TILE];
  __shared__ __attribute__((aligned(1024))) char s_tile[3][2 * TILE];
  __shared__ __attribute__((aligned(1024))) char s_ds[2][KW * DS];  // [key][query], 16-byte chunks exchanged by (key / 4) % 4
  __shared__ __attribute__((aligned(16))) float s_lse[kShortRows], s_delta[kShortRows];  // L and delta, 32 a step
  __shared__ float s_big[2][KW + DC];  // |g|, |v|
  __shared__ int s_blocks, s_last;
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, h = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kv_heads = p.heads / p.group;
  const int item = work_item(p);
  if (item < 0) return;
  const int kvh = item % kv_heads, seq = item / kv_heads;
  const Span qs = span_of(p.cu_q, p.q_rows, p.q_len, seq), ks = span_of(p.cu_k, p.k_rows, p.k_len, seq);
  if (p.gq) clear_uncovered(p, item, p.cu_q, p.q_rows, p.heads * p.dim / 8, p.gq);
  clear_uncovered(p, item, p.cu_k, p.k_rows, kv_heads * p.dim / 8, p.gk);
  clear_uncovered(p, item, p.cu_k, p.k_rows, kv_heads * p.dim / 8, p.gv);
  if (tid == 0) s_blocks = s_last = 0;
  __syncthreads();

  const int head0 = kvh * p.group, most = (qs.len + 31) / 32;
  const char* const q0 = p.q.data + (p.cu_q ? qs.row * p.q.sl : seq * p.q.sn);
  const char* const g0 = p.g.data + (p.cu_q ? qs.row * p.g.sl : seq * p.g.sn);
  // +inf: past the end, masked, or without a key
  auto lse_of = [&](int head, int pos) {
    return pos < qs.len ? p.lse[(int64_t)head * p.q_total + qs.row + pos] : INFINITY;
  };
  // the wavefront's keys; rows that are none or masked are zeros
  const bool keys = wv < KW;
  const int kpos = wv * 32 + l32;
  // (what the first loads wait for, at once)
  const bool kon = keys && kpos < ks.len && (!p.km || p.km[seq * p.km_sn + kpos * p.km_sl] != 0);
  float lse = wv < most * p.group ? lse_of(head0 + wv / most, wv % most * 32 + l32) : INFINITY;
  const float lse0 = wv < 4 ? lse_of(head0, wv * 8 + lane / 8) : INFINITY;

  // Q and G of 32 queries, by four wavefronts; rows without a statistic are not read
  const bool loads = wv < 4;
  const Rows<DC, 32, 4> qrows(p.q.sl, p.dim, wv & 3, lane), grows(p.g.sl, p.dim, wv & 3, lane);
  auto issue = [&](int buf, int head, int qt, float lse) {
    const bool on = lse != INFINITY;
    const uint32_t at = lds_addr(s_tile[buf]) + wv * 1024;
    dma16(at, on ? qrows.off[0] : kOob, raw_desc(q0 + head * p.q.sh + qt * p.q.sl, 0xffffff00u));
    dma16(at + TILE, on ? grows.off[0] : kOob, raw_desc(g0 + head * p.g.sh + qt * p.g.sl, 0xffffff00u));
  };
  if (loads) issue(0, head0, 0, lse0);
  const char* kbase = p.k.data + (p.cu_k ? ks.row * p.k.sl : seq * p.k.sn) + kvh * p.k.sh;
  const char* vbase = p.v.data + (p.cu_k ? ks.row * p.v.sl : seq * p.v.sn) + kvh * p.v.sh;
  u32x4 kf[D::KS], vf[D::KS];
  load_cols<DC>(kf, kon ? kbase + kpos * p.k.sl : nullptr, p.dim, lane);
  load_cols<DC>(vf, kon ? vbase + kpos * p.v.sl : nullptr, p.dim, lane);
  const bool any = __ballot(kon) != 0;
  if (any && lane == 0) atomicMax(&s_blocks, wv + 1);

  float gs = 1.0f, big = 0.f;
  for (int it = wv; it < most * p.group;) {
    const int head = head0 + it / most, qt = it % most * 32, pos = qt + l32;
    const bool on = lse != INFINITY;
    const int64_t row = ((qs.row + pos) * p.heads + head) * p.dim;
    u32x4 gf[D::KS];
    load_cols<DC>(gf, on ? g0 + head * p.g.sh + pos * p.g.sl : nullptr, p.dim, lane);
    const float d = row_delta<EK, DC>(p, gf, row, on, big, lane);
    if (lane < 32) {
      s_lse[it * 32 + l32] = lse;
      s_delta[it * 32 + l32] = d;
    }
    if (__ballot(on) && lane == 0) atomicMax(&s_last, qt + 32);
    it += KW + DC;
    if (it < most * p.group) lse = lse_of(head0 + it / most, it % most * 32 + l32);
  }
  if constexpr (EK == EK_F16) {
    const float vbig = wave_max(max_finite<D::KS>(vf));
    big = wave_max(big);
    if (lane == 0) {
      s_big[0][wv] = big;
      s_big[1][wv] = vbig;
    }
  }
  if (keys)
#pragma unroll
    for (int k = 0; k < D::KS; ++k)
      *(u32x4*)(s_k + kpos * D::PITCH + (((2 * k + h) ^ D::swz(l32)) << 4)) = kf[k];
  __syncthreads();
  const int blocks = (s_blocks + 1) & ~1;  // of 32 keys, read in pairs
  int qe = s_last < qs.len ? s_last : qs.len;  // queries to walk: a window ends before the last one
  if (p.left != kNone && (int64_t)ks.len + p.left < qe) qe = ks.len + p.left;
  if (!blocks) qe = 0;
  const int steps = (qe + 31) / 32, total = steps * p.group;
  if constexpr (EK == EK_F16) {
    float vbig = big = 0.f;
#pragma unroll
    for (int w = 0; w < KW + DC; ++w) {
      big = fmaxf(big, s_big[0][w]);
      vbig = fmaxf(vbig, s_big[1][w]);
    }
    gs = scale_for(big, vbig, p.dim);
  }

  struct Pos {
    int head, qt;
  };
  auto after = [&](Pos a) { return a.qt + 32 < qe ? Pos{a.head, a.qt + 32} : Pos{a.head + 1, 0}; };
  const Frags<DC> frags(lane);
  if (keys) {
    // a query keeps a key where 0 <= query - key + ahead <= reach
    const int ahead = p.right == kNone ? 0x3fffffff : p.right;
    const uint32_t reach = (uint32_t)ahead + (p.left == kNone ? 0x3fffffffu : (uint32_t)p.left);
    const int wk0 = wv * 32, wk1 = wk0 + 31;
    const uint32_t kept = kon ? 0xffffffffu : 0u;
    f32x16 dk[DC], dv[DC];
#pragma unroll
    for (int d = 0; d < DC; ++d) dk[d] = dv[d] = f32x16{};
    auto issue_step = [&](int buf, Pos a) {
      issue(buf, a.head, a.qt, s_lse[(a.head - head0) * most * 32 + a.qt + wv * 8 + lane / 8]);
    };
    Pos now = {head0, 0}, ahead2 = after(now);
    if (loads && total > 1) issue_step(1, ahead2);
    int buf = 0;
    for (int it = 0; it < total; ++it, buf = buf == 2 ? 0 : buf + 1) {
      if (it + 1 < total) asm volatile("s_waitcnt vmcnt(2) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      ahead2 = after(ahead2);
      if (loads && it + 2 < total) issue_step(buf ? buf - 1 : 2, ahead2);
      const int qt = now.qt, stat = (now.head - head0) * most * 32 + qt;
      now = after(now);
      if (wv >= blocks) continue;
      char* const ds_row = s_ds[it & 1] + kpos * 64 + 8 * h;
      u32x4 pf[2], df[2] = {};
      if (any && (p.left == kNone || qt <= wk1 + p.left) && (p.right == kNone || qt + 31 >= wk0 - p.right)) {
        const uint32_t at = lds_addr(s_tile[buf]);
        f32x16 s = {}, dp = {};
#pragma unroll
        for (int k = 0; k < D::KS; ++k) {
          s = mfma16<EK>(s, frags.row(at, 0, k), kf[k]);
          dp = mfma16<EK>(dp, frags.row(at + TILE, 0, k), vf[k]);
        }
        if ((p.left != kNone && qt + 31 > wk0 + p.left) || (p.right != kNone && qt < wk1 - p.right))
          mask_scores(s, 0, 64, nullptr, true, qt + 4 * h - kpos + ahead, reach, lane);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x4 ls = *(const f32x4*)&s_lse[stat + 8 * q + 4 * h];
          const f32x4 dl = *(const f32x4*)&s_delta[stat + 8 * q + 4 * h];
          float e[4], ds[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            e[i] = pair_p<EK>(p, s[q * 4 + i], ls[i]);
            const float x = dp[q * 4 + i] - dl[i];
            ds[i] = e[i] * (EK == EK_F16 ? x * gs : x);
          }
          pf[q / 2][(q % 2) * 2] = pack2<EK>(e[0], e[1]);
          pf[q / 2][(q % 2) * 2 + 1] = pack2<EK>(e[2], e[3]);
          df[q / 2][(q % 2) * 2] = pack2<EK>(ds[0], ds[1]) & kept;
          df[q / 2][(q % 2) * 2 + 1] = pack2<EK>(ds[2], ds[3]) & kept;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int d = 0; d < DC; ++d) {
            dv[d] = mfma16<EK>(dv[d], frags.col(at + TILE, k * 16, d), pf[k]);
            dk[d] = mfma16<EK>(dk[d], frags.col(at, k * 16, d), df[k]);
          }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *(u32x2*)(ds_row + ((q ^ ((l32 >> 2) & 3)) << 4)) = u32x2{df[q / 2][(q % 2) * 2], df[q / 2][(q % 2) * 2 + 1]};
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const int64_t at = ((ks.row + kpos) * kv_heads + kvh) * p.dim * 2;
    store_key<EK, DC>(p, dk, dv, p.scale * kUnliftP<EK> / gs, at, kon, kpos, ks.len,
                      p.lse + (int64_t)head0 * p.q_total + qs.row, qs.len, lane);
  } else {
    const int block = wv - KW;  // of 32 head dims
    // transposing reads of ds: lane l has query l % 32 of keys row0 + 4 (l / 32) + {0..3, 8..11}, as Frags::col
    const int i16 = lane & 15, col = (lane & 16) + 4 * (i16 & 3), c0 = 4 * h + (i16 >> 2);
    const uint32_t lo = c0 * 64 + (((col >> 3) ^ ((c0 >> 2) & 3)) << 4) + ((col & 4) << 1);
    const uint32_t hi = (c0 + 8) * 64 + (((col >> 3) ^ (((c0 + 8) >> 2) & 3)) << 4) + ((col & 4) << 1);
    Pos before = {head0, 0};
    for (int it = 0; it <= total; ++it) {
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (it && p.gq) {
        const uint32_t at = lds_addr(s_ds[(it - 1) & 1]), kt = lds_addr(s_k);
        f32x16 acc = {};
        for (int b = 0; b < blocks; b += 2)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t d = at + b * DS + k * 1024;
            const u32x2 x = lds_tr(d + lo), y = lds_tr(d + hi);
            acc = mfma16<EK>(acc, frags.col(kt + b * TILE, k * 16, block), u32x4{x[0], x[1], y[0], y[1]});
          }
        const int pos = before.qt + l32;
        // queries without a statistic: no gradient, whatever the keys hold
        if (s_lse[(before.head - head0) * most * 32 + pos] == INFINITY) acc = f32x16{};
        store_cols<EK, 1>(p.gq + (((qs.row + pos) * p.heads + before.head) * p.dim + block * 32) * 2, &acc,
                          p.scale * kUnliftP<EK> / gs, p.dim - block * 32, lane, pos < qs.len);
        before = after(before);
      }
    }
  }
  if (p.gq) {  // queries after the last step have none of the keys
    const int chunks = p.group * p.dim / 8;
    for (int i = tid; i < (qs.len - steps * 32) * chunks; i += T) {
      const int64_t row = (qs.row + steps * 32 + i / chunks) * p.heads + head0;
      *(u32x4*)(p.gq + row * p.dim * 2 + i % chunks * 16) = u32x4{0u, 0u, 0u, 0u};
    }
  }
}

// One kernel for all gradients: 129 to 320 keys (up to 128 the two kernels have more workgroups a CU: 128 passages of 128 rows 160 us, one
// kernel 171; a key head more than one of these is one tile of theirs), if a workgroup's walk is short or there are enough
// of them (4 key heads of 63 steps: 111 us, two kernels 71; 192 of 32: 82 and 101; 256 of 64: 178 and 232). Where k and v need no
// gradient the first of the two kernels alone is faster.
bool one_pass(const AttP& p) {
  const int64_t steps = (p.q_len + 31) / 32 * p.group;
  return p.gk && p.k_len > 128 && p.k_len <= 320 && steps * 32 <= kShortRows &&
         (steps <= 32 || (int64_t)p.n * (p.heads / p.group) >= 192);
}
template <int EK, int DC, int KW>
int launch_grads(AttP p, hipStream_t s) {
  const unsigned grid = work_grid(p, (int64_t)p.n * (p.heads / p.group), 1);
  if (!grid) return LIK_ERR_UNSUPPORTED;
  launch_kernel(attention_grads_kernel<EK, DC, KW>, dim3(grid), dim3((KW + DC) * 64), 0u, s, p);
  return hipGetLastError() == hipSuccess ? LIK_OK : LIK_ERR_LAUNCH;
}

template <int EK, int DC>
int launch_backward(AttP p, hipStream_t s) {
  if constexpr (DC <= 2) {
    if (one_pass(p)) {
      if (p.k_len <= 192) return launch_grads<EK, DC, 6>(p, s);
      return launch_grads<EK, DC, 10>(p, s);
    }
  }
  if constexpr (EK == EK_F16) {
    const int64_t tiles = (int64_t)p.n * (p.heads / p.group) * p.k_tiles;
    if (tiles > 0x3fffffff) return LIK_ERR_UNSUPPORTED;
    launch_kernel(attention_vmax_kernel, dim3((unsigned)tiles), dim3(256), 0u, s, p);
    if (hipGetLastError() != hipSuccess) return LIK_ERR_LAUNCH;
  }
  p.tiles = p.q_tiles;
  unsigned grid = work_grid(p, (int64_t)p.tiles * p.n * p.heads, (int64_t)p.tiles * p.group);
  if (!grid) return LIK_ERR_UNSUPPORTED;
  launch_kernel(attention_dq_kernel<EK, DC>, dim3(grid), dim3(256), p.km ? mask_words(p.k_len) * 4 : 0u, s, p);
  if (hipGetLastError() != hipSuccess) return LIK_ERR_LAUNCH;
  p.tiles = p.k_tiles;
  const int64_t wgs = (int64_t)p.n * (p.heads / p.group) * p.tiles;
  if (!p.gk) return LIK_OK;
  grid = work_grid(p, wgs, p.tiles);
  if (!grid) return LIK_ERR_UNSUPPORTED;
  launch_kernel(attention_dkv_kernel<EK, DC>, dim3(grid), dim3(256),
                p.qm || by_statistic(p) ? mask_words(p.q_len) * 4 : 0u, s, p);
  return hipGetLastError() == hipSuccess ? LIK_OK : LIK_ERR_LAUNCH;
}

template <int EK>
int run_backward(const AttP& p, hipStream_t s) {
  if (p.dim <= 32) return launch_backward<EK, 1>(p, s);
  if (p.dim <= 64) return launch_backward<EK, 2>(p, s);
  if (p.dim <= 96) return launch_backward<EK, 3>(p, s);
  return launch_backward<EK, 4>(p, s);
}

int tiles128(int64_t len) { return (int)((len + 127) / 128); }
size_t gmax_bytes(const AttP& p) { return align256((size_t)p.n * p.heads * tiles128(p.q_len) * 4); }
size_t backward_ws(const AttP& p) {
  return align256((size_t)p.q_total * p.heads * 4) + gmax_bytes(p) +
         (size_t)p.n * (p.heads / p.group) * tiles128(p.k_len) * 4 + 256;
}

}  // namespace
}  // namespace enc
}  // namespace lik

using namespace lik;
using namespace lik::enc;

extern "C" {

size_t lik_attention_backward_workspace_size(const lik_attention_t* a) {
  AttP p{};
  int rc;
  return attention_shape(a, p, rc) ? backward_ws(p) : 0;
}

int lik_attention_backward(const lik_attention_t* a, const void* out, const float* lse, const int8_t* out_low,
                           const void* grad,
                           int64_t grad_stride_n, int64_t grad_stride_l, int64_t grad_stride_h, void* grad_q,
                           void* grad_k, void* grad_v, void* workspace, size_t workspace_bytes, lik_stream_t stream) {
  AttP p{};
  int rc;
  const bool queries = attention_shape(a, p, rc);
  if (rc != LIK_OK) return rc;
  const hipStream_t s = (hipStream_t)stream;
  if (!grad_k != !grad_v) return LIK_ERR_INVALID;
  if ((uintptr_t)grad_q % 16 || (uintptr_t)grad_k % 16 || (uintptr_t)grad_v % 16) return LIK_ERR_UNSUPPORTED;
  if (!queries || a->k_len == 0) {  // no kernel comes by the keys
    const int64_t keys = a->cu_k ? a->k_rows : a->n * a->k_len;
    rc = clear_rows(grad_k, keys, a->kv_heads, a->dim, s);
    if (rc == LIK_OK) rc = clear_rows(grad_v, keys, a->kv_heads, a->dim, s);
    if (rc == LIK_OK) rc = clear_rows(grad_q, p.q_total, a->heads, a->dim, s);
    return rc;
  }
  if (!out || !lse || !out_low || !grad) return LIK_ERR_INVALID;
  if (!att_rows_ok(grad, grad_stride_n, grad_stride_l, grad_stride_h) || (uintptr_t)out % 16 || (uintptr_t)out_low % 16)
    return LIK_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < backward_ws(p)) return LIK_ERR_WORKSPACE;
  char* ws = align256(workspace);
  p.delta = (float*)ws;
  p.gmax = (float*)(ws + align256((size_t)p.q_total * p.heads * 4));
  p.out = (char*)const_cast<void*>(out);
  p.lse = const_cast<float*>(lse);
  p.low = const_cast<int8_t*>(out_low);
  p.vmax = (float*)((char*)p.gmax + gmax_bytes(p));
  p.q_tiles = tiles128(p.q_len);
  p.k_tiles = tiles128(p.k_len);
  p.g = {(const char*)grad, grad_stride_n * 2, grad_stride_l * 2, grad_stride_h * 2};
  p.gq = (char*)grad_q;
  p.gk = (char*)grad_k;
  p.gv = (char*)grad_v;
  return a->dtype == LIK_BF16 ? run_backward<EK_BF16>(p, s) : run_backward<EK_F16>(p, s);
}

}  // extern "C"
