// Rotary positions: the pairs (a, b) of a head's first 2 * pairs elements are turned by the token's position,
//   theta = position * frequency_i,  (a, b) -> amplitude (a cos theta - b sin theta, b cos theta + a sin theta),
// pair i being elements (i, i + pairs) or (2 i, 2 i + 1); the other elements are copied. The gradient is the
// same map with -theta.
//
// Bound by HBM: every element is read once and written once. A workgroup owns T consecutive tokens and holds
// their cosines and sines in LDS, since all heads of q and of k share them. theta is taken in turns and
// reduced to less than one in 64 bits (an fp32 angle of position 10^5 is off by 0.004), sine and cosine of
// what is left are fp32, and so is the turn; it is rounded once. Measured (a large copy: 5.03 TB/s): 44928 packed
// tokens of 24 heads of 64, bf16, 55 us (5.0 TB/s); 16480 tokens of 20 heads of 128 of which a half is turned 36 us
// (4.7); 20000 of 16 heads of 96 fp32, a quarter turned, interleaved 49 us (5.0); one query of 32 tokens 3.5 us.
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
  int rot, items;       // items of a head: of pairs, all
  int tokens;           // of a workgroup
  float amp, sign;
};

constexpr int kMostTokens = 32, kTable = 2048;  // tokens and cosines of a workgroup

// WHOLE: no chunk is taken to pieces (there are V pairs at least, and no elements behind them or V at least).
template <int EK, bool INTER, bool WHOLE>
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

    // An item: two chunks, of V pairs or of the elements behind them (lanes of both kinds take the same way).
    const int heads = p.t[0].heads + p.t[1].heads, items = tokens * heads * p.items;
    for (int i = tid; i < items; i += 256) {
      const int th = i / p.items, c = i - th * p.items, t = th / heads;
      int head = th - t * heads;
      const bool is_k = head >= p.t[0].heads;
      if (is_k) head -= p.t[0].heads;
      const char* in = is_k ? p.t[1].x + s_at[1][t] + head * p.t[1].sh : p.t[0].x + s_at[0][t] + head * p.t[0].sh;
      char* out = (is_k ? p.t[1].y : p.t[0].y) +
                  ((row0 + t) * (is_k ? p.t[1].heads : p.t[0].heads) + head) * ((int64_t)p.dim * El<EK>::B);
      const bool turned = c < p.rot;
      // the first pair. WHOLE: the last chunk of a kind ends where its elements do and shares some with the one before
      const int j = WHOLE && turned && c * V > p.pairs - V ? p.pairs - V : c * V;
      int ea = turned ? (INTER ? 2 * j : j) : 2 * p.pairs + (c - p.rot) * 2 * V;
      int eb = turned && !INTER ? j + p.pairs : ea + V;
      if (WHOLE && !turned) {
        ea = ea < p.dim - V ? ea : p.dim - V;
        eb = eb < p.dim - V ? eb : p.dim - V;
      }
      const int enda = turned ? (INTER ? 2 * p.pairs : p.pairs) : p.dim, endb = turned ? 2 * p.pairs : p.dim;
      u32x4 wa, wb = {0u, 0u, 0u, 0u};
      chunk_load<EK, WHOLE>(in, ea, enda, wa);
      if (WHOLE || eb < endb) chunk_load<EK, WHOLE>(in, eb, endb, wb);
      float v[2 * V], y[2 * V];
      chunk_widen<EK>(wa, v);
      chunk_widen<EK>(wb, v + V);
      const int at = t * p.pairs + (turned ? j : 0);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const f32x2 cs = s_cs[WHOLE || j + k < p.pairs ? at + k : at];
        const int ia = INTER ? 2 * k : k, ib = INTER ? 2 * k + 1 : V + k;
        y[ia] = fmaf(v[ia], cs[0], -v[ib] * cs[1]);
        y[ib] = fmaf(v[ib], cs[0], v[ia] * cs[1]);
      }
      const u32x4 ya = chunk_narrow<EK>(y), yb = chunk_narrow<EK>(y + V);
      const bool on = s_on[t];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        wa[k] = !on ? 0u : turned ? ya[k] : wa[k];
        wb[k] = !on ? 0u : turned ? yb[k] : wb[k];
      }
      chunk_store<EK, WHOLE>(out, ea, enda, wa);
      if (WHOLE || eb < endb) chunk_store<EK, WHOLE>(out, eb, endb, wb);
    }
    __syncthreads();  // (the arrays are the next tokens')
  }
}

template <int EK, bool INTER>
int launch_rotary(RotP p, hipStream_t s) {
  constexpr int V = El<EK>::V;
  const int rest = p.dim - 2 * p.pairs;
  p.rot = (p.pairs + V - 1) / V;
  p.items = p.rot + (rest + 2 * V - 1) / (2 * V);
  // Three items a thread: more tokens a workgroup leave some CUs a workgroup more than others (44928 tokens of 24 heads of
  // 64, bf16: 8 tokens 55 us, 16 58 us, 32 61 us). Few rows: as many workgroups as there can be.
  const int64_t per = (int64_t)(p.t[0].heads + p.t[1].heads) * p.items;
  p.tokens = 1;
  while (p.tokens < kMostTokens && p.tokens * per < 768 && 2 * p.tokens * p.pairs <= kTable && p.rows >= 2048 * p.tokens)
    p.tokens *= 2;
  const int64_t want = (p.rows + p.tokens - 1) / p.tokens;
  const unsigned groups = (unsigned)(want < (1 << 22) ? want : 1 << 22);  // (a launch has less than 2^32 threads)
  if (p.pairs >= V && (rest == 0 || rest >= V))
    launch_kernel(rotary_kernel<EK, INTER, true>, dim3(groups), dim3(256), 0u, s, p);
  else
    launch_kernel(rotary_kernel<EK, INTER, false>, dim3(groups), dim3(256), 0u, s, p);
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
  // (elements near a chunk's end are read by two threads)
  if ((heads && (q_out == a->q || q_out == a->k)) || (kv && (k_out == a->k || k_out == a->q)) ||
      (heads && kv && q_out == k_out))
    return LIK_ERR_INVALID;
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
  hipStream_t s = (hipStream_t)stream;
  switch (a->dtype) {
    case LIK_BF16: return a->interleaved ? launch_rotary<EK_BF16, true>(p, s) : launch_rotary<EK_BF16, false>(p, s);
    case LIK_F16: return a->interleaved ? launch_rotary<EK_F16, true>(p, s) : launch_rotary<EK_F16, false>(p, s);
    default: return a->interleaved ? launch_rotary<EK_F32, true>(p, s) : launch_rotary<EK_F32, false>(p, s);
  }
}
