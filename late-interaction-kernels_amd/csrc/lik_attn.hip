// Attention, forward. One pass over the keys with the running maximum and sum of
// the softmax; the layout of the products is described in lik_attn.h.
//
// Bounds, measured with 256 padded sequences of 12 heads of 64 (a call among others): up to 128 tokens the rows' reads and
// writes (50 us, 4.0 TB/s), at 1024 the softmax's vector instructions beside the MFMAs (1042 us, 790 TFLOP/s; per 32 x 64 scores
// 512 clocks of MFMA and about 1000 of vector work, four wavefronts a SIMD). Between them tiles that a sequence does not fill:
// 50 to 300 tokens 105 us (63 at the copy rate). The statistic of training calls (STAT) adds 2 to 3%.
#include "lik_attn.h"

namespace lik {
namespace enc {
namespace {

// The reference maximum only moves when a score passes it by more than 2^kRise, and probabilities are 2^kLift
// times those to that reference. bf16: up to 256 instead of 1, which no rounding sees, and the output is rescaled less often. fp16: up
// to 2^15; what is 2^-26 of a row's largest is still a normal number (2^-14) and what is 2^-36 is not dropped, so the
// weights of many such keys are not lost (a lift of 0 dropped them under 2^-25).
template <int EK>
constexpr float kRise = EK == EK_F16 ? 3.0f : 8.0f;
template <int EK>
constexpr float kLift = EK == EK_F16 ? 12.0f : 0.0f;

// One step of the softmax on 32 NU scores of a lane's column: s to probabilities, packed as MFMA operands in pf;
// top, sum and the output so far follow the running maximum. The sum is that of the rounded probabilities, which are the
// output's weights: whatever the values have in common comes out exact. (With the sum before the rounding the output was off
// by the weights' missing share of it, and delta = g o against g v with it: gradients of q and k over values of 16 +- 1 were
// 2 roundoffs off.) STAT: `whole` is the sum before the rounding, for the statistic that the gradients' probabilities come from.
template <int EK, int DC, int NU, bool STAT>
__device__ __forceinline__ void softmax_step(f32x16 (&s)[NU], f32x16 (&o)[DC], float& top, float& sum, float& whole, float c,
                                             u32x4 (&pf)[2 * NU]) {
  float m = s[0][0];
#pragma unroll
  for (int u = 0; u < NU; ++u)
#pragma unroll
    for (int i = 0; i < 16; ++i) m = fmaxf(m, s[u][i]);
  m = fmaxf(m, swap_half(m));
  if (__ballot(fmaf(m, c, -kRise<EK>) > top * c) != 0) {
    const float up = fmaxf(m, top);
    const float alpha = up == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((top - up) * c);
    top = up;
    sum *= alpha;
    if constexpr (STAT) whole *= alpha;
#pragma unroll
    for (int d = 0; d < DC; ++d) o[d] *= alpha;
  }
  float mc = top == -INFINITY ? 0.f : fmaf(top, c, -kLift<EK>);
  // A large reference is spaced too widely to be taken off inside the exponent (2^11: by 2^-12; 3e9: by 2^8): off the
  // scores first.
  if (__ballot(fabsf(mc) > 2048.0f) != 0) {
    const float off = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[u][i] -= off;
    mc = -kLift<EK>;
  }
#pragma unroll
  for (int u = 0; u < NU; ++u)
#pragma unroll
    for (int i = 0; i < 16; ++i) s[u][i] = __builtin_amdgcn_exp2f(fmaf(s[u][i], c, -mc));
  if constexpr (STAT) {
    float add[2] = {};
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) add[i % 2] += s[u][i];
    whole += add[0] + add[1];
  }
  float add[2] = {};
#pragma unroll
  for (int k = 0; k < 2 * NU; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      pf[k][e] = pack2<EK>(s[k / 2][(k % 2) * 8 + 2 * e], s[k / 2][(k % 2) * 8 + 2 * e + 1]);
      add[e % 2] = add2<EK>(pf[k][e], add[e % 2]);
    }
  sum += add[0] + add[1];
}

// One split's share of a row's output: its mean of the values in fp32, and its statistic.
template <int DC>
__device__ __forceinline__ void store_part(const AttP& p, int split, int64_t row, int head, const f32x16 (&o)[DC],
                                           float inv, float lse, int lane) {
  if (lane < 32) p.part_lse[((int64_t)split * p.heads + head) * p.q_total + row] = lse;
  float* at = p.part_o + (((int64_t)split * p.q_total + row) * p.heads + head) * p.dim;
#pragma unroll
  for (int d = 0; d < DC; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int e = d * 32 + 8 * q + 4 * (lane >> 5);
      if (e < p.dim)
        *(f32x4*)(at + e) =
            f32x4{o[d][q * 4] * inv, o[d][q * 4 + 1] * inv, o[d][q * 4 + 2] * inv, o[d][q * 4 + 3] * inv};
    }
}

// What a wavefront does with 64 keys: K rows at kl and V rows at vl in LDS, its 32 queries in qf.
//   scores  S^T[key][query] = K Q^T   (K rows from LDS, Q in registers)
//   output  O^T[d][query]  += V^T P^T (V by transposing LDS reads, P as it lies)
// whole: every pair is kept; else the arguments of mask_scores.
template <int EK, int DC, bool STAT>
__device__ __forceinline__ void attend_tile(const Frags<DC>& frags, uint32_t kl, uint32_t vl,
                                            const u32x4 (&qf)[Dim<DC>::KS], f32x16 (&o)[DC], float& top, float& sum,
                                            float& stat, float c, bool whole, int kt, int klen, const uint32_t* bits, bool window,
                                            int first, uint32_t reach, int lane) {
  f32x16 s[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    s[u] = f32x16{};
#pragma unroll
    for (int k = 0; k < Dim<DC>::KS; ++k) s[u] = mfma16<EK>(s[u], frags.row(kl, u * 32, k), qf[k]);
  }
  if (!whole) {
#pragma unroll
    for (int u = 0; u < 2; ++u) mask_scores(s[u], kt + u * 32, klen, bits, window, first + u * 32, reach, lane);
  }
  u32x4 pf[4];
  softmax_step<EK, DC, 2, STAT>(s, o, top, sum, stat, c, pf);
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int d = 0; d < DC; ++d) o[d] = mfma16<EK>(o[d], frags.col(vl, k * 16, d), pf[k]);
}

// A wavefront's finished queries to memory. on: the lane's row exists, q_on: its mask keeps it.
// whole: the sum of the probabilities before their rounding (or sum again).
template <int EK, int DC>
__device__ __forceinline__ void store_rows(const AttP& p, int split, int64_t row, int head, f32x16 (&o)[DC], float top,
                                           float sum, float whole, bool on, bool q_on, int lane) {
  const float total = sum + swap_half(sum), stat = whole + swap_half(whole);
  const bool kept = q_on && total != 0.f;
  const float inv = kept ? 1.0f / total : 0.f;
  const float lse = kept ? fmaf(__builtin_amdgcn_logf(stat) - kLift<EK>, p.inv_c, top) : INFINITY;
  if (!kept)  // a masked row's sums hold what the values hold: not zero times that
#pragma unroll
    for (int d = 0; d < DC; ++d) o[d] = f32x16{};
  if (p.splits > 1) {
    if (on) store_part<DC>(p, split, row, head, o, inv, kept ? lse : -INFINITY, lane);
    return;
  }
  if (p.lse && on && lane < 32) p.lse[(int64_t)head * p.q_total + row] = lse;
  store_cols<EK, DC>(p.out + (row * p.heads + head) * p.dim * 2, o, inv, p.dim, lane, on);
  if (p.low) store_low<EK, DC>(p.low + (row * p.heads + head) * p.dim, o, inv, p.dim, lane, on);
}

// A workgroup of four wavefronts owns 128 queries of one head, a wavefront 32 of them as MFMA columns, and
// walks the keys that any of them keeps, 64 at a time, in two LDS buffers: the next tile is loaded while this one
// is used.
template <int EK, int DC, bool STAT>
__global__ void __launch_bounds__(256, DC <= 2 ? 4 : 2) attention_kernel(const AttP p) {
  using D = Dim<DC>;
  __shared__ __attribute__((aligned(1024))) char s_tile[2][2 * D::TILE];
  __shared__ int s_kept[2];
  extern __shared__ uint32_t s_bits[];
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int item = work_item(p);
  if (item < 0) return;
  uint32_t t = (uint32_t)item;
  const int split = (int)(t % (uint32_t)p.splits);
  t /= (uint32_t)p.splits;
  const int tile = (int)(t % (uint32_t)p.tiles);
  t /= (uint32_t)p.tiles;
  const int head = (int)(t % (uint32_t)p.heads), seq = (int)(t / (uint32_t)p.heads);
  const int kvh = head / p.group;
  const Span qs = span_of(p.cu_q, p.q_rows, p.q_len, seq), ks = span_of(p.cu_k, p.k_rows, p.k_len, seq);
  const int q0 = tile * 128;
  if (p.splits == 1) clear_uncovered(p, item, p.cu_q, p.q_rows, p.heads * p.dim / 8, p.out);
  if (q0 >= qs.len) return;  // (all threads)

  const char* kbase = p.k.data + (p.cu_k ? ks.row * p.k.sl : seq * p.k.sn) + kvh * p.k.sh;
  const char* vbase = p.v.data + (p.cu_k ? ks.row * p.v.sl : seq * p.v.sn) + kvh * p.v.sh;
  const Rows<DC> krows(p.k.sl, p.dim, wv, lane), vrows(p.v.sl, p.dim, wv, lane);
  const Frags<DC> frags(lane);
  const uint32_t lds[2] = {lds_addr(s_tile[0]), lds_addr(s_tile[1])};
  int klen = ks.len;
  bool holes = false;
  auto issue = [&](uint32_t at, int kt) {
    const uint32_t* bits = holes ? s_bits + (kt >> 5) : nullptr;
    krows.issue(at, kbase + kt * p.k.sl, klen - kt, bits, wv, lane);
    vrows.issue(at + D::TILE, vbase + kt * p.v.sl, klen - kt, bits, wv, lane);
  };

  // The first tile's loads start before the keep bits are known (and again without the masked rows, if there
  // are any): a short sequence's time is a chain of such latencies.
  const int q_end = (q0 + 128 < qs.len ? q0 + 128 : qs.len) - 1;  // last query of the workgroup
  int kb = p.left == kNone || q0 - p.left < 0 ? 0 : (q0 - p.left) & ~63;
  int ke = p.right == kNone || (int64_t)q_end + p.right + 1 >= klen ? klen : q_end + p.right + 1;
  if (p.splits > 1) {  // this split's share
    const int tiles = ke > kb ? (ke - kb + 63) / 64 : 0, per = (tiles + p.splits - 1) / p.splits;
    kb += split * per * 64;
    ke = kb + per * 64 < ke ? kb + per * 64 : ke;
  }
  if (kb < ke) issue(lds[0], kb);
  const int qpos = q0 + wv * 32 + l32;  // the lane's query
  const bool qon = qpos < qs.len && (!p.qm || p.qm[seq * p.qm_sn + qpos * p.qm_sl] != 0);
  u32x4 qf[D::KS];
  const char* qbase = p.q.data + (p.cu_q ? qs.row * p.q.sl : seq * p.q.sn) + head * p.q.sh;
  load_cols<DC>(qf, qon ? qbase + qpos * p.q.sl : nullptr, p.dim, lane);
  const bool any = __ballot(qon) != 0;  // this wavefront has a query

  if (p.km) {
    const Kept kept = scan_mask(s_bits, p.km + seq * p.km_sn, p.km_sl, klen, s_kept);
    klen = kept.extent;
    holes = kept.holes;
    ke = ke < klen ? ke : klen;
    if ((holes || (klen < ks.len && klen < kb + 64)) && kb < ke) {  // masked rows have to read as zeros
      asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
      issue(lds[0], kb);
    }
  }
  if (__syncthreads_or(any) == 0) ke = kb;  // no query of this tile is kept

  const Window win(p);
  f32x16 o[DC];
  float top = -INFINITY, sum = 0.f, stat = 0.f;
#pragma unroll
  for (int d = 0; d < DC; ++d) o[d] = f32x16{};
  const int wq0 = q0 + wv * 32, wq1 = wq0 + 31;  // the wavefront's queries
  int buf = 0;
  for (int kt = kb; kt < ke; kt += 64, buf ^= 1) {
    // this tile is complete, and every wavefront is done with the other buffer
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (kt + 64 < ke) issue(buf ? lds[0] : lds[1], kt + 64);
    if (!any || (p.right != kNone && kt > wq1 + p.right) || (p.left != kNone && kt + 63 < wq0 - p.left)) continue;
    const uint32_t at = buf ? lds[1] : lds[0];
    const bool whole = kt + 64 <= klen && !holes && (p.right == kNone || kt + 63 <= wq0 + p.right) &&
                       (p.left == kNone || kt >= wq1 - p.left);
    attend_tile<EK, DC, STAT>(frags, at, at + D::TILE, qf, o, top, sum, stat, p.c, whole, kt, klen, holes ? s_bits : nullptr, win.on,
                        kt + 4 * (lane >> 5) - qpos + win.back, win.reach, lane);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load is in flight to LDS when the workgroup ends
  store_rows<EK, DC>(p, split, qs.row + qpos, head, o, top, sum, STAT ? stat : sum, qpos < qs.len, qon, lane);
}

// Few queries over long keys: bound by reading K and V once, so every key head's queries (all heads of the
// group, up to 32 QB rows) are one wavefront's MFMA columns, and every wavefront has keys of its own: 32 at a
// time through two private LDS buffers, no barrier, 4 to 8 KB in flight for each of K and V. A wavefront's keys
// are a split; attention_join_kernel adds them. 4 sequences of 5000 to 8192 keys, one query, 16 heads over 4 of 128,
// fp16: 16 + 6 us (54 MB, 10.5 us at the copy rate; 47 + 7 us by attention_kernel, a wavefront of four at work and every
// query head reading the keys).
template <int EK, int DC, int QB>
__global__ void __launch_bounds__(256, DC <= 2 ? 2 : 1) attention_rows_kernel(const AttP p) {
  using D = Dim<DC>;
  constexpr int TILE = 32 * D::PITCH, NI = 2 * TILE / 1024;
  __shared__ __attribute__((aligned(1024))) char s_ring[4][2][2 * TILE];
  __shared__ int s_kept[2];
  extern __shared__ uint32_t s_bits[];
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int item = work_item(p);
  if (item < 0) return;
  const int wsplits = p.splits / 4, kv_heads = p.heads / p.group;
  uint32_t t = (uint32_t)item;
  const int ws = (int)(t % (uint32_t)wsplits);
  t /= (uint32_t)wsplits;
  const int kvh = (int)(t % (uint32_t)kv_heads), seq = (int)(t / (uint32_t)kv_heads);
  const Span qs = span_of(p.cu_q, p.q_rows, p.q_len, seq), ks = span_of(p.cu_k, p.k_rows, p.k_len, seq);
  const int split = ws * 4 + wv, steps = (ks.len + 31) / 32, per = (steps + p.splits - 1) / p.splits;
  const int first = ws * 4 * per * 32, kb = split * per * 32;  // the workgroup's first key, the wavefront's
  const int last = first + 4 * per * 32 < ks.len ? first + 4 * per * 32 : ks.len;
  int ke = kb + per * 32 < ks.len ? kb + per * 32 : ks.len;

  const char* kbase = p.k.data + (p.cu_k ? ks.row * p.k.sl : seq * p.k.sn) + kvh * p.k.sh;
  const char* vbase = p.v.data + (p.cu_k ? ks.row * p.v.sl : seq * p.v.sn) + kvh * p.v.sh;
  const Rows<DC, 32, 1> krows(p.k.sl, p.dim, 0, lane), vrows(p.v.sl, p.dim, 0, lane);
  const Frags<DC> frags(lane);
  const uint32_t lds[2] = {lds_addr(s_ring[wv][0]), lds_addr(s_ring[wv][1])};
  bool holes = false;
  auto issue = [&](uint32_t at, int kt) {
    const uint32_t* bits = holes ? s_bits + ((kt - first) >> 5) : nullptr;
    krows.issue(at, kbase + kt * p.k.sl, ke - kt, bits, 0, lane);
    vrows.issue(at + TILE, vbase + kt * p.v.sl, ke - kt, bits, 0, lane);
  };
  if (!p.km) {
    if (kb < ke) issue(lds[0], kb);
    if (kb + 32 < ke) issue(lds[1], kb + 32);
  }
  // column c: row c % q_len of head c / q_len of the group
  int row[QB], head[QB];
  bool on[QB];
  u32x4 qf[QB][D::KS];
  const char* qbase = p.q.data + (p.cu_q ? qs.row * p.q.sl : seq * p.q.sn);
#pragma unroll
  for (int b = 0; b < QB; ++b) {
    const int c = b * 32 + l32;
    row[b] = c % (int)p.q_len;
    head[b] = kvh * p.group + c / (int)p.q_len;
    on[b] = c < p.group * (int)p.q_len && row[b] < qs.len;
    const bool q_on = on[b] && (!p.qm || p.qm[seq * p.qm_sn + row[b] * p.qm_sl] != 0);
    load_cols<DC>(qf[b], q_on ? qbase + row[b] * p.q.sl + head[b] * p.q.sh : nullptr, p.dim, lane);
    if (!q_on) row[b] = -1 - row[b];  // written as a row without keys
  }
  if (p.km) {  // the workgroup's own keys' bits
    const Kept kept = scan_mask(s_bits, p.km + seq * p.km_sn + first * p.km_sl, p.km_sl, last > first ? last - first : 0,
                                s_kept);
    holes = kept.holes;
    ke = ke < first + kept.extent ? ke : first + kept.extent;
    if (kb < ke) issue(lds[0], kb);
    if (kb + 32 < ke) issue(lds[1], kb + 32);
  }

  f32x16 o[QB][DC];
  float top[QB], sum[QB], stat[QB];
#pragma unroll
  for (int b = 0; b < QB; ++b) {
    top[b] = -INFINITY;
    sum[b] = stat[b] = 0.f;
#pragma unroll
    for (int d = 0; d < DC; ++d) o[b][d] = f32x16{};
  }
  int buf = 0;
  for (int kt = kb; kt < ke; kt += 32, buf ^= 1) {
    // this tile is complete (the next one's loads, if there is one, are younger)
    if (kt + 32 < ke) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NI) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const uint32_t at = buf ? lds[1] : lds[0];
    f32x16 s[QB][1];
#pragma unroll
    for (int b = 0; b < QB; ++b) s[b][0] = f32x16{};
#pragma unroll
    for (int k = 0; k < D::KS; ++k) {
      const u32x4 kf = frags.row(at, 0, k);
#pragma unroll
      for (int b = 0; b < QB; ++b) s[b][0] = mfma16<EK>(s[b][0], kf, qf[b][k]);
    }
    u32x4 pf[QB][2];
#pragma unroll
    for (int b = 0; b < QB; ++b) {
      if (holes || kt + 32 > ke)
        mask_scores(s[b][0], kt - first, ke - first, holes ? s_bits : nullptr, false, 0, 0u, lane);
      softmax_step<EK, DC, 1, true>(s[b], o[b], top[b], sum[b], stat[b], p.c, pf[b]);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int d = 0; d < DC; ++d) {
        const u32x4 vf = frags.col(at + TILE, k * 16, d);
#pragma unroll
        for (int b = 0; b < QB; ++b) o[b][d] = mfma16<EK>(o[b][d], vf, pf[b][k]);
      }
    if (kt + 64 < ke) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this buffer has been read
      issue(at, kt + 64);
    }
  }
#pragma unroll
  for (int b = 0; b < QB; ++b) {
    const float total = sum[b] + swap_half(sum[b]), whole = stat[b] + swap_half(stat[b]);
    const bool kept = row[b] >= 0 && total != 0.f;
    if (!kept)  // (as in store_rows)
#pragma unroll
      for (int d = 0; d < DC; ++d) o[b][d] = f32x16{};
    if (on[b])
      store_part<DC>(p, split, qs.row + (row[b] < 0 ? -1 - row[b] : row[b]), head[b], o[b], kept ? 1.0f / total : 0.f,
                     kept ? fmaf(__builtin_amdgcn_logf(whole) - kLift<EK>, p.inv_c, top[b]) : -INFINITY, lane);
  }
}

// Joins the splits of a row: sum_s 2^(c (L_s - L)) o_s. A wavefront a row and head: its lanes take the splits'
// statistics, then two elements each.
template <int EK>
__global__ void __launch_bounds__(256) attention_join_kernel(const AttP p) {
  __shared__ float s_w[4][64];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int64_t rh = (int64_t)blockIdx.x * 4 + wv;
  const int64_t row = rh / p.heads;
  const int head = (int)(rh % p.heads);
  if (row >= p.q_total) return;
  if (p.cu_q && (row < p.cu_q[0] || row >= p.cu_q[p.n])) {  // in no sequence
    if (lane * 8 < p.dim) *(u32x4*)(p.out + (rh * p.dim + lane * 8) * 2) = u32x4{0u, 0u, 0u, 0u};
    return;
  }
  // (at most 64 splits)
  const float l = lane < p.splits ? p.part_lse[((int64_t)lane * p.heads + head) * p.q_total + row] : -INFINITY;
  float top = l;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) top = max_nan(top, __shfl_xor(top, s));
  const float w = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((l - top) * p.c);
  float total = w;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) total += __shfl_xor(total, s);
  const float inv = top == -INFINITY ? 0.f : 1.0f / total;
  if (p.lse && lane == 0)
    p.lse[(int64_t)head * p.q_total + row] = top == -INFINITY ? INFINITY : fmaf(__builtin_amdgcn_logf(total), p.inv_c, top);
  s_w[wv][lane] = w * inv;  // (a wavefront reads only what it wrote itself)
  __builtin_amdgcn_wave_barrier();
  const int e = 4 * (lane & 31);
  if (e >= p.dim) return;
  f32x4 a = {};
  const float* in = p.part_o + rh * p.dim + e;
  const int64_t step = p.q_total * p.heads * p.dim;
#pragma unroll 4
  for (int s = lane >> 5; s < p.splits; s += 2) {  // the halves take the even and the odd splits
    const f32x4 x = *(const f32x4*)(in + s * step);
    const float ws = s_w[wv][s];
#pragma unroll
    for (int k = 0; k < 4; ++k) a[k] = fmaf(ws, x[k], a[k]);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) a[k] += swap_half(a[k]);
  if (lane < 32) {
    *(u32x2*)(p.out + (rh * p.dim + e) * 2) = u32x2{pack2<EK>(a[0], a[1]), pack2<EK>(a[2], a[3])};
    if (p.low) *(uint32_t*)(p.low + rh * p.dim + e) = low_bytes<EK>(a[0], a[1], a[2], a[3]);
  }
}

// Splits of the keys. Up to 64 rows a key head and no window: attention_rows_kernel may take the call, whose
// workgroups fill the CUs once (LDS: two a CU up to head dim 64, else one), a wavefront 64 keys at least. It writes at
// least four fp32 shares of each row and reads them again, for reading the keys once: shared heads, where the shares are at
// most a third of the keys' and values' bytes (12 k_len each row); heads of their own, only where the key heads alone do not
// fill the CUs and rows are few for the keys. us of both kernels, this one first: 16 / 4 heads of 128, 300 keys, 512
// sequences, 1 query 90 and 203, 16 queries 219 and 210 (1000 keys 365 and 554); 12 heads of 64, 1000 keys, 1 query, 24
// sequences 21 and 25, 48 sequences 34 and 27; 512 sequences of 64 queries and 300 keys 375 and 122, without 1.6 GB of shares.
// More rows: where the tiles of queries do not fill the 256 CUs and the keys are long, down to 256 keys a split.
void forward_shape(AttP& p) {
  p.tiles = (int)((p.q_len + 127) / 128);
  const bool window = p.left != kNone || p.right != kNone;
  const int64_t rows = p.q_len * p.group, units = (int64_t)p.n * (p.heads / p.group), slots = p.dim <= 64 ? 512 : 256;
  p.few = !window && rows <= 64 && p.k_len >= 256 &&
          (p.group > 1 ? 12 * rows <= p.k_len : units <= slots && p.k_len >= 512 && 48 * rows <= p.k_len);
  int64_t s;
  if (p.few) {
    s = slots / units;
    const int64_t most = (p.k_len + 255) / 256;
    if (s > most) s = most;
    if (s > 16) s = 16;
    if (s < 1) s = 1;
    if (s < 2 && p.k_len > 1 << 17) s = 2;  // (a workgroup's keep bits, beside 128 KB of tiles)
    p.splits = 4 * (int)s;
    return;
  }
  const int64_t wgs = (int64_t)p.n * p.heads * p.tiles;
  s = p.left != kNone && p.right != kNone ? 1 : 512 / wgs;  // (a window is short)
  if (s > p.k_len / 256) s = p.k_len / 256;
  if (s > 64) s = 64;
  p.splits = s < 2 ? 1 : (int)s;
}
size_t forward_ws(const AttP& p) {
  if (p.splits < 2) return 0;
  return align256((size_t)p.splits * p.q_total * p.heads * p.dim * 4) +
         align256((size_t)p.splits * p.q_total * p.heads * 4) + 256;
}

template <int EK, int DC>
int launch_forward(AttP p, hipStream_t s) {
  if (p.few) {
    const int64_t per = p.splits / 4, steps = ((p.k_len + 31) / 32 + p.splits - 1) / p.splits;
    const uint32_t bits = p.km ? mask_words(4 * 32 * steps) * 4 : 0u;  // a workgroup's keys
    const unsigned grid = work_grid(p, per * p.n * (p.heads / p.group), per);
    if (!grid) return LIK_ERR_UNSUPPORTED;
    if (p.q_len * p.group <= 32)
      launch_kernel(attention_rows_kernel<EK, DC, 1>, dim3(grid), dim3(256), bits, s, p);
    else
      launch_kernel(attention_rows_kernel<EK, DC, 2>, dim3(grid), dim3(256), bits, s, p);
  } else {
    const int64_t per = (int64_t)p.tiles * p.splits;
    const unsigned grid = work_grid(p, per * p.n * p.heads, per * p.group);
    if (!grid) return LIK_ERR_UNSUPPORTED;
    const auto kernel = p.lse || p.splits > 1 ? attention_kernel<EK, DC, true> : attention_kernel<EK, DC, false>;
    launch_kernel(kernel, dim3(grid), dim3(256), p.km ? mask_words(p.k_len) * 4 : 0u, s, p);
  }
  if (hipGetLastError() != hipSuccess) return LIK_ERR_LAUNCH;
  if (p.splits > 1) {
    const int64_t m = p.q_total * p.heads;
    launch_kernel(attention_join_kernel<EK>, dim3((unsigned)((m + 3) / 4)), dim3(256), 0u, s, p);
    if (hipGetLastError() != hipSuccess) return LIK_ERR_LAUNCH;
  }
  return LIK_OK;
}

template <int EK>
int run_forward(const AttP& p, hipStream_t s) {
  if (p.dim <= 32) return launch_forward<EK, 1>(p, s);
  if (p.dim <= 64) return launch_forward<EK, 2>(p, s);
  if (p.dim <= 96) return launch_forward<EK, 3>(p, s);
  return launch_forward<EK, 4>(p, s);
}

__global__ void __launch_bounds__(256) clear_kernel(u32x4* at, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    at[i] = u32x4{0u, 0u, 0u, 0u};
}

}  // namespace

int clear_rows(void* data, int64_t rows, int heads, int dim, hipStream_t s) {
  const int64_t n = rows * heads * dim / 8;
  if (!data || n <= 0) return LIK_OK;
  const int64_t wgs = (n + 255) / 256;
  launch_kernel(clear_kernel, dim3((unsigned)(wgs < 4096 ? wgs : 4096)), dim3(256), 0u, s, (u32x4*)data, n);
  return hipGetLastError() == hipSuccess ? LIK_OK : LIK_ERR_LAUNCH;
}

bool attention_shape(const lik_attention_t* a, AttP& p, int& rc) {
  rc = LIK_ERR_INVALID;
  if (!a || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads || a->dim < 1 || a->n < 0 || a->q_len < 0 ||
      a->k_len < 0 || !(a->scale > 0.f) || !(a->scale < INFINITY) || !a->cu_q != !a->cu_k || a->left < -1 || a->right < -1)
    return false;
  if (a->cu_q && (a->q_mask || a->k_mask || a->q_rows < 0 || a->k_rows < 0)) return false;
  rc = LIK_ERR_UNSUPPORTED;
  if ((a->dtype != LIK_BF16 && a->dtype != LIK_F16) || a->dim % 8 || a->dim > 128 || a->q_len > (1 << 30) ||
      a->k_len > (1 << 30) || a->n > 0x7fffffff)
    return false;
  if ((a->k_mask && a->k_len > kMaskMost) || (a->q_mask && a->q_len > kMaskMost)) return false;
  p.q_total = a->cu_q ? a->q_rows : a->n * a->q_len;
  rc = LIK_OK;
  if (a->n == 0 || p.q_total == 0 || a->q_len == 0) return false;
  const bool keys = (a->cu_k ? a->k_rows : a->n * a->k_len) > 0;
  if (!a->q || (keys && (!a->k || !a->v))) {
    rc = LIK_ERR_INVALID;
    return false;
  }
  if (!att_rows_ok(a->q, a->q_stride_n, a->q_stride_l, a->q_stride_h) ||
      !att_rows_ok(a->k, a->k_stride_n, a->k_stride_l, a->k_stride_h) ||
      !att_rows_ok(a->v, a->v_stride_n, a->v_stride_l, a->v_stride_h)) {
    rc = LIK_ERR_UNSUPPORTED;
    return false;
  }
  p.q = {(const char*)a->q, a->q_stride_n * 2, a->q_stride_l * 2, a->q_stride_h * 2};
  p.k = {(const char*)a->k, a->k_stride_n * 2, a->k_stride_l * 2, a->k_stride_h * 2};
  p.v = {(const char*)a->v, a->v_stride_n * 2, a->v_stride_l * 2, a->v_stride_h * 2};
  p.cu_q = a->cu_q;
  p.cu_k = a->cu_k;
  p.q_rows = a->q_rows;
  p.k_rows = a->k_rows;
  p.qm = a->q_mask;
  p.km = a->k_mask;
  p.qm_sn = a->q_mask_stride_n;
  p.qm_sl = a->q_mask_stride_l;
  p.km_sn = a->k_mask_stride_n;
  p.km_sl = a->k_mask_stride_l;
  p.q_len = a->q_len;
  p.k_len = a->k_len;
  p.n = (int)a->n;
  p.heads = a->heads;
  p.group = a->heads / a->kv_heads;
  p.dim = a->dim;
  p.left = a->left < 0 || a->left >= (1 << 30) ? kNone : a->left;
  p.right = a->right < 0 || a->right >= (1 << 30) ? kNone : a->right;
  p.scale = a->scale;
  p.c = a->scale * 1.4426950408889634f;
  p.inv_c = 1.0f / p.c;
  return true;
}

}  // namespace enc
}  // namespace lik

using namespace lik;
using namespace lik::enc;

extern "C" {

size_t lik_attention_workspace_size(const lik_attention_t* a) {
  AttP p{};
  int rc;
  if (!attention_shape(a, p, rc)) return 0;
  forward_shape(p);
  return forward_ws(p);
}

int lik_attention(const lik_attention_t* a, void* out, float* lse, int8_t* out_low, void* workspace, size_t workspace_bytes,
                  lik_stream_t stream) {
  AttP p{};
  int rc;
  const bool queries = attention_shape(a, p, rc);
  if (rc != LIK_OK) return rc;
  if (!out && p.q_total > 0) return LIK_ERR_INVALID;
  if ((uintptr_t)out % 16 || (uintptr_t)out_low % 16) return LIK_ERR_UNSUPPORTED;
  if (!queries) return clear_rows(out, p.q_total, a->heads, a->dim, (hipStream_t)stream);
  forward_shape(p);
  if (p.splits > 1) {
    if (!workspace || workspace_bytes < forward_ws(p)) return LIK_ERR_WORKSPACE;
    char* ws = align256(workspace);
    p.part_o = (float*)ws;
    p.part_lse = (float*)(ws + align256((size_t)p.splits * p.q_total * p.heads * p.dim * 4));
  }
  p.out = (char*)out;
  p.lse = lse;
  p.low = out_low;
  return a->dtype == LIK_BF16 ? run_forward<EK_BF16>(p, (hipStream_t)stream)
                              : run_forward<EK_F16>(p, (hipStream_t)stream);
}

}  // extern "C"
