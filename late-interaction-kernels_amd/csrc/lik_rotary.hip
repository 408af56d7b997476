// Rotary positions: the pairs (a, b) of a head's first 2 * pairs elements are turned by the token's position,
//   theta = position * frequency_i,  (a, b) -> amplitude (a cos theta - b sin theta, b cos theta + a sin theta),
// pair i being elements (i, i + pairs) or (2 i, 2 i + 1); the other elements are copied. The gradient is the
// same map with -theta.
//
// Bound by HBM: every element is read once and written once. A workgroup owns T consecutive tokens and holds
// their cosines and sines in LDS, since all heads of q and of k share them. theta is taken in turns and
// reduced to less than one in 64 bits (an fp32 angle of position 10^5 is off by 0.004), sine and cosine of
// what is left are fp32, and so is the turn; it is rounded once.
#include "lik_enc.h"

namespace lik {
namespace enc {
namespace {

struct RotP {
  struct Rows {
    const char* x;
    char* y;            // [rows][heads][dim]
    int64_t sn, sl, sh;  // bytes
    int heads;
  } t[2];               // q, k
  int64_t rows, len;    // token row = sequence * len + l (packed: l)
  const void* pos;      // null: counted
  int64_t pos_sn, pos_sl;
  const int32_t* cu;    // packed
  int n_seqs;
  int64_t offset;
  const void* freq;
  bool pos64, freq64;
  int pairs, dim;
  int tokens;           // of a workgroup
  float amp, sign;
};

constexpr int kMostTokens = 32, kTable = 2048;  // tokens and cosines of a workgroup

template <int EK, bool INTER>
__global__ void __launch_bounds__(256) rotary_kernel(const RotP p) {
  constexpr int V = El<EK>::V;
  __shared__ double s_pos[kMostTokens];
  __shared__ int s_on[kMostTokens];
  __shared__ int64_t s_at[2][kMostTokens];
  __shared__ f32x2 s_cs[kTable];
  const int tid = threadIdx.x;
  for (int64_t row0 = (int64_t)blockIdx.x * p.tokens; row0 < p.rows; row0 += (int64_t)gridDim.x * p.tokens) {
    const int tokens = (int)(p.rows - row0 < p.tokens ? p.rows - row0 : p.tokens);

    if (tid < tokens) {
      const int64_t row = row0 + tid;
      int64_t seq = 0, l = row;
      if (!p.cu) {
        seq = row / p.len;
        l = row - seq * p.len;
      }
      s_at[0][tid] = seq * p.t[0].sn + l * p.t[0].sl;
      s_at[1][tid] = seq * p.t[1].sn + l * p.t[1].sl;
      int64_t pos = l + p.offset;
      int on = 1;
      if (p.pos) {
        const int64_t i = seq * p.pos_sn + l * p.pos_sl;
        pos = p.pos64 ? ((const int64_t*)p.pos)[i] : ((const int32_t*)p.pos)[i];
      } else if (p.cu) {  // the last sequence that starts at or before the row
        int lo = -1, hi = p.n_seqs + 1;
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (p.cu[mid] <= row) lo = mid;
          else hi = mid;
        }
        on = lo >= 0 && lo < p.n_seqs;
        if (on) pos = row - p.cu[lo] + p.offset;
      }
      s_pos[tid] = (double)pos;
      s_on[tid] = on;
    }
    __syncthreads();
    for (int i = tid; i < tokens * p.pairs; i += 256) {
      const int t = i / p.pairs, j = i - t * p.pairs;
      const double f = p.freq64 ? ((const double*)p.freq)[j] : (double)((const float*)p.freq)[j];
      const double turns = s_pos[t] * (f * 0.15915494309189533577);
      float s, c;
      sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
      s_cs[i] = f32x2{p.amp * c, p.amp * p.sign * s};
    }
    __syncthreads();

    // a chunk: V pairs, or V of the elements behind them
    const int rot = (p.pairs + V - 1) / V, rest = (p.dim - 2 * p.pairs + V - 1) / V;
    const int chunks = rot + rest, heads = p.t[0].heads + p.t[1].heads;
    for (int i = tid; i < tokens * heads * chunks; i += 256) {
      const int t = i / (heads * chunks), r = i - t * (heads * chunks);
      int head = r / chunks;
      const int c = r - head * chunks;
      const int which = head >= p.t[0].heads;
      const RotP::Rows& x = p.t[which];
      if (which) head -= p.t[0].heads;
      const char* in = x.x + s_at[which][t] + head * x.sh;
      char* out = x.y + ((row0 + t) * x.heads + head) * ((int64_t)p.dim * El<EK>::B);
      u32x4 wa, wb;
      if (c >= rot) {
        const int e = 2 * p.pairs + (c - rot) * V;
        chunk_load<EK>(in, e, p.dim, wa);
        if (!s_on[t]) wa = u32x4{0u, 0u, 0u, 0u};
        chunk_store<EK>(out, e, p.dim, wa);
        continue;
      }
      const int j = c * V;
      const int ea = INTER ? 2 * j : j, eb = INTER ? 2 * j + V : j + p.pairs;
      const int enda = INTER ? 2 * p.pairs : p.pairs, endb = 2 * p.pairs;
      chunk_load<EK>(in, ea, enda, wa);
      chunk_load<EK>(in, eb, endb, wb);
      float v[2 * V], y[2 * V];
      chunk_widen<EK>(wa, v);
      chunk_widen<EK>(wb, v + V);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const f32x2 cs = s_cs[t * p.pairs + (j + k < p.pairs ? j + k : 0)];
        const int ia = INTER ? 2 * k : k, ib = INTER ? 2 * k + 1 : V + k;
        y[ia] = fmaf(v[ia], cs[0], -v[ib] * cs[1]);
        y[ib] = fmaf(v[ib], cs[0], v[ia] * cs[1]);
      }
      wa = chunk_narrow<EK>(y);
      wb = chunk_narrow<EK>(y + V);
      if (!s_on[t]) wa = wb = u32x4{0u, 0u, 0u, 0u};
      chunk_store<EK>(out, ea, enda, wa);
      chunk_store<EK>(out, eb, endb, wb);
    }
    __syncthreads();  // (the arrays are the next tokens')
  }
}

template <int EK>
int launch_rotary(const RotP& p, bool inter, hipStream_t s) {
  const int64_t want = (p.rows + p.tokens - 1) / p.tokens;
  const unsigned groups = (unsigned)(want < (1 << 22) ? want : 1 << 22);  // (a launch has less than 2^32 threads)
  if (inter)
    launch_kernel(rotary_kernel<EK, true>, dim3(groups), dim3(256), 0u, s, p);
  else
    launch_kernel(rotary_kernel<EK, false>, dim3(groups), dim3(256), 0u, s, p);
  return hipGetLastError() == hipSuccess ? LIK_OK : LIK_ERR_LAUNCH;
}

}  // namespace
}  // namespace enc
}  // namespace lik

using namespace lik;
using namespace lik::enc;

extern "C" int lik_rotary(const lik_rotary_t* a, void* q_out, void* k_out, lik_stream_t stream) {
  if (!a) return LIK_ERR_INVALID;
  if (a->dtype != LIK_BF16 && a->dtype != LIK_F16 && a->dtype != LIK_F32) return LIK_ERR_UNSUPPORTED;
  if (a->n < 0 || a->len < 0 || a->heads < 0 || a->kv_heads < 0 || a->dim < 1 || a->pairs < 1 ||
      a->pairs > a->dim / 2 || (a->positions && a->cu_seqlens) || (!a->frequencies))
    return LIK_ERR_INVALID;
  if ((a->positions && a->position_bits != 32 && a->position_bits != 64) ||
      (a->frequency_bits != 32 && a->frequency_bits != 64))
    return LIK_ERR_INVALID;
  if (a->dim > 1024 || a->heads > (1 << 16) || a->kv_heads > (1 << 16) || a->n > 0x7ffffffe) return LIK_ERR_UNSUPPORTED;
  const int64_t most = (int64_t)1 << 40;
  if (a->len > most || (!a->cu_seqlens && a->n > most / (a->len > 0 ? a->len : 1))) return LIK_ERR_UNSUPPORTED;
  const int eb = a->dtype == LIK_F32 ? 4 : 2;
  const int heads = a->q ? a->heads : 0, kv = a->k ? a->kv_heads : 0;
  RotP p{};
  p.rows = a->cu_seqlens ? a->len : a->n * a->len;
  if (p.rows == 0 || heads + kv == 0) return LIK_OK;
  if ((heads && !q_out) || (kv && !k_out)) return LIK_ERR_INVALID;
  if ((uintptr_t)a->q % eb || (uintptr_t)a->k % eb || (uintptr_t)q_out % eb || (uintptr_t)k_out % eb ||
      (uintptr_t)a->frequencies % (a->frequency_bits / 8) || (uintptr_t)a->cu_seqlens % 4 ||
      (a->positions && (uintptr_t)a->positions % (a->position_bits / 8)))
    return LIK_ERR_UNSUPPORTED;
  p.t[0] = {(const char*)a->q, (char*)q_out, a->q_stride_n * eb, a->q_stride_l * eb, a->q_stride_h * eb, heads};
  p.t[1] = {(const char*)a->k, (char*)k_out, a->k_stride_n * eb, a->k_stride_l * eb, a->k_stride_h * eb, kv};
  p.len = a->len;
  p.pos = a->positions;
  p.pos_sn = a->position_stride_n;
  p.pos_sl = a->position_stride_l;
  p.cu = a->cu_seqlens;
  p.n_seqs = (int)a->n;
  p.offset = a->offset;
  p.freq = a->frequencies;
  p.pos64 = a->position_bits == 64;
  p.freq64 = a->frequency_bits == 64;
  p.pairs = a->pairs;
  p.dim = a->dim;
  p.amp = a->amplitude;
  p.sign = a->inverse ? -1.0f : 1.0f;
  p.tokens = kMostTokens;
  while (p.tokens > 1 && (p.tokens * p.pairs > kTable || p.rows < 1024 * p.tokens)) p.tokens /= 2;
  hipStream_t s = (hipStream_t)stream;
  switch (a->dtype) {
    case LIK_BF16: return launch_rotary<EK_BF16>(p, a->interleaved != 0, s);
    case LIK_F16: return launch_rotary<EK_F16>(p, a->interleaved != 0, s);
    default: return launch_rotary<EK_F32>(p, a->interleaved != 0, s);
  }
}
