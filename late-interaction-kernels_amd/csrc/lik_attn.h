// What the attention kernels share: parameters, the sequences and their masks,
// tiles of rows in LDS.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i k_j) / sum over the kept j
// A pair (i, j) of one sequence is kept where both masks keep its rows and
// i - left <= j <= i + right. A row without a kept key gives o = 0 and no gradient.
//
// Every product is a 32 x 32 MFMA whose columns are the rows that a wavefront owns
// (queries in the forward and the gradient of q, keys in the gradients of k and v)
// and whose rows are the other side's, streamed through LDS 64 at a time. A lane
// then holds 16 scores of ONE column: maximum and sum of the softmax are in-lane plus
// one exchange between the wavefront's halves, and the probabilities, rounded and
// packed, are the next product's operand as they lie (the accumulator's order of
// rows only permutes that product's sum, and the transposing LDS reads of the other
// operand follow the same order).
#pragma once
#include "lik_enc.h"

namespace lik {
namespace enc {

struct AttRows {  // rows of one operand: byte strides
  const char* data;
  int64_t sn, sl, sh;
};

struct AttP {
  AttRows q, k, v, g;  // g: gradient of the output
  const int32_t *cu_q, *cu_k;
  int64_t q_rows, k_rows;  // packed: rows in memory
  const int8_t *qm, *km;
  int64_t qm_sn, qm_sl, km_sn, km_sl;
  int64_t q_len, k_len, q_total;  // q_total: rows of the output per head
  int n, heads, group, dim;       // group: query heads of one key head
  int left, right;                // INT32_MAX: unbounded
  float scale, c, inv_c;          // c = scale log2 e
  char* out;                      // [q_total][heads][dim]
  int8_t* low;                    // what the output's rounding took off, by element (below); null: not kept
  float* lse;                     // [heads][q_total]: L with p = 2^(c (q k - L)), log2(sum 2^(c q k)) / c; +inf where nothing is kept
  float* delta;                   // [heads][q_total]: sum_d g o
  char *gq, *gk, *gv;             // contiguous gradients
  float* gmax;                    // fp16: [sequence][head][q tile]: largest |g|
  float* vmax;                    // fp16: [sequence][key head][k tile]: largest |v|
  int q_tiles, k_tiles;           // backward: tiles of 128 rows of a sequence
  float* part_o;                  // forward split over keys: [split][q_total][heads][dim] fp32
  float* part_lse;                // [split][heads][q_total]: L of a split's keys; -inf where none is kept
  int splits, tiles;              // q tiles (k tiles) of a sequence
  bool few;                       // forward: attention_rows_kernel
  int chunk, wgs;                 // workgroups: `chunk` in a row go to one XCD; wgs of them have work
};

constexpr int kNone = 0x7fffffff;

// Work item of this workgroup, or -1. Items of one key head share its keys in their XCD's L2 (workgroups go to the
// XCDs in turn), so `chunk` items in a row go to one XCD; the chunks go round, because sequences differ in length.
__device__ __forceinline__ int work_item(const AttP& p) {
  const int x = (int)blockIdx.x & 7, j = (int)blockIdx.x >> 3;
  const int64_t w = (int64_t)(j / p.chunk) * 8 * p.chunk + x * p.chunk + j % p.chunk;
  return w < p.wgs ? (int)w : -1;
}
// A chunk is a key head's items, but at least eight chunks go to every XCD. Returns the grid (0: too large).
inline unsigned work_grid(AttP& p, int64_t wgs, int64_t per_key_head) {
  if (wgs > 0x3fffffff) return 0;
  int64_t c = (wgs + 63) / 64;
  if (c > per_key_head) c = per_key_head;
  if (c < 1) c = 1;
  p.chunk = (int)c;
  p.wgs = (int)wgs;
  return (unsigned)((wgs + 8 * c - 1) / (8 * c) * 8 * c);
}

// A sequence's rows: first row, length.
struct Span {
  int64_t row;
  int len;
};
__device__ __forceinline__ Span span_of(const int32_t* cu, int64_t rows, int64_t len, int i) {
  if (!cu) return {i * len, (int)len};
  // offsets outside the rows in memory are cut off
  int64_t a = cu[i], b = cu[i + 1];
  a = a < 0 ? 0 : a > rows ? rows : a;
  b = b < a ? a : b > rows ? rows : b;
  const int64_t l = b - a < len ? b - a : len;
  return {a, (int)l};
}

// Zeros in the packed rows of `out` ([rows][16-byte chunks of a row]) that belong to no sequence, a share by each work item's
// workgroup. (Called beside span_of: the offsets arrive together.)
__device__ __forceinline__ void clear_uncovered(const AttP& p, int item, const int32_t* cu, int64_t rows, int row_chunks,
                                                char* out) {
  if (!cu) return;
  int64_t first = cu[0], end = cu[p.n];
  first = first < 0 ? 0 : first > rows ? rows : first;
  end = end < first ? first : end > rows ? rows : end;
  const int64_t front = first * row_chunks, chunks = front + (rows - end) * row_chunks;
  if (chunks == 0) return;
  for (int64_t i = (int64_t)item * blockDim.x + threadIdx.x; i < chunks; i += (int64_t)p.wgs * blockDim.x)
    *(u32x4*)(out + (i < front ? i : end * row_chunks + i - front) * 16) = u32x4{0u, 0u, 0u, 0u};
}

// Keep bits of len tokens (kept(t): whether token t is) into LDS, 32 tokens a word, by all 256 threads; returns the
// last kept token + 1 and whether a token before it is dropped.
struct Kept {
  int extent;
  bool holes;
};
template <typename F>
__device__ __forceinline__ Kept scan_kept(uint32_t* bits, int len, int* s_kept, F kept) {
  const int tid = threadIdx.x;
  if (tid < 2) s_kept[tid] = 0;
  __syncthreads();
  int last = 0, count = 0;
  for (int t0 = 0; t0 < len; t0 += 256) {
    const int t = t0 + tid;
    const bool on = t < len && kept(t);
    const uint64_t b = __ballot(on);
    if ((tid & 63) == 0) {
      bits[t >> 5] = (uint32_t)b;
      bits[(t >> 5) + 1] = (uint32_t)(b >> 32);
      count += __popcll(b);
      if (b) last = t + 64 - __clzll(b);
    }
  }
  if ((tid & 63) == 0) {
    atomicMax(&s_kept[0], last);
    atomicAdd(&s_kept[1], count);
  }
  __syncthreads();
  return {s_kept[0], s_kept[1] != s_kept[0]};
}
__device__ __forceinline__ Kept scan_mask(uint32_t* bits, const int8_t* mask, int64_t stride, int len, int* s_kept) {
  return scan_kept(bits, len, s_kept, [=](int t) { return mask[t * stride] != 0; });
}
// words of keep bits that are written for len tokens
inline uint32_t mask_words(int64_t len) { return (uint32_t)((len + 255) / 256 * 8); }
constexpr int64_t kMaskMost = 1 << 18;  // tokens whose keep bits fit LDS beside the tiles

// The kernels' sizes by the head dimension: k steps of 16, blocks of 32, bytes of a row in LDS.
template <int DC>
struct Dim {
  static constexpr int KS = DC * 2, DB = DC, PITCH = DC <= 2 ? 128 : 256;
  static constexpr int SPR = PITCH / 16, TILE = 64 * PITCH;
  // 16-byte chunk c of row r lies at chunk c ^ swz(r): 16 consecutive rows at one chunk (row-wise reads)
  // cover the 64 banks, and so do any four rows of an aligned group at 64 bytes each (transposing reads).
  __device__ __forceinline__ static int swz(int r) {
    return PITCH == 128 ? ((r & 2) << 1) | ((r >> 2) & 3) : ((r & 3) << 2) | ((r >> 2) & 3);
  }
};

// N rows of one operand into LDS by NW wavefronts (wv: which of them this is); row r at r * PITCH, chunks swizzled. The lane offsets
// within a tile are kept; rows that do not exist (limit) or are not kept (bits, null: all are) read as zeros.
template <int DC, int N = 64, int NW = 4>
struct Rows {
  using D = Dim<DC>;
  static constexpr int NI = N * D::PITCH / 1024 / NW;
  uint32_t off[NI];
  __device__ __forceinline__ Rows(int64_t ld, int dim, int wv, int lane) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int slot = (wv * NI + i) * 64 + lane, r = slot / D::SPR, c = (slot % D::SPR) ^ D::swz(r);
      off[i] = c * 8 < dim ? (uint32_t)r * (uint32_t)ld + c * 16 : kOob;
    }
  }
  __device__ __forceinline__ void issue(uint32_t lds, const char* base, int limit, const uint32_t* bits, int wv,
                                        int lane) const {
    const u32x4 desc = raw_desc(base, 0xffffff00u);
    if (limit >= N && !bits) {
#pragma unroll
      for (int i = 0; i < NI; ++i) dma16(lds + (wv * NI + i) * 1024, off[i], desc);
    } else {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int r = ((wv * NI + i) * 64 + lane) / D::SPR;
        bool on = r < limit;
        if (bits) on = on && ((bits[r >> 5] >> (r & 31)) & 1u);
        dma16(lds + (wv * NI + i) * 1024, on ? off[i] : kOob, desc);
      }
    }
  }
};
// Lane addresses of the MFMA operands in a tile (tiles start on 1 KB): the swizzle makes the k step (row-wise)
// and the block of 32 columns (across) an exclusive or, everything else an immediate offset.
// row(): rows row0 .. row0 + 31, elements 16 ks + 8 (lane / 32) ..
// col(): lane l has element 32 db + l % 32 of rows row0 + 4 (l / 32) + {0..3, 8..11}, the order in which
// accumulators hold rows (row0 a multiple of 16).
template <int DC>
struct Frags {
  using D = Dim<DC>;
  uint32_t r, lo, hi;
  __device__ __forceinline__ explicit Frags(int lane) {
    const int l32 = lane & 31, h = lane >> 5, i = lane & 15, col = (lane & 16) + 4 * (i & 3), c0 = 4 * h + (i >> 2);
    r = l32 * D::PITCH + ((h ^ D::swz(l32)) << 4);
    lo = c0 * D::PITCH + (((col >> 3) ^ D::swz(c0)) << 4) + ((col & 4) << 1);
    hi = (c0 + 8) * D::PITCH + (((col >> 3) ^ D::swz(c0 + 8)) << 4) + ((col & 4) << 1);
  }
  __device__ __forceinline__ u32x4 row(uint32_t tile, int row0, int ks) const {
    return lds_b128(((tile + r) ^ (ks << 5)) + row0 * D::PITCH);
  }
  __device__ __forceinline__ u32x4 col(uint32_t tile, int row0, int db) const {
    const u32x2 a = lds_tr(((tile + lo) ^ (db << 6)) + row0 * D::PITCH);
    const u32x2 b = lds_tr(((tile + hi) ^ (db << 6)) + row0 * D::PITCH);
    return u32x4{a[0], a[1], b[0], b[1]};
  }
};
// This lane's column operand of a row in memory (null: zeros): elements 16 ks + 8 (lane / 32) ..
template <int DC>
__device__ __forceinline__ void load_cols(u32x4* f, const char* row, int dim, int lane) {
#pragma unroll
  for (int ks = 0; ks < Dim<DC>::KS; ++ks) {
    const int e = ks * 16 + 8 * (lane >> 5);
    f[ks] = row && e < dim ? *(const u32x4*)(row + e * 2) : u32x4{0u, 0u, 0u, 0u};
  }
}

// other half's value of x
__device__ __forceinline__ float swap_half(float x) {
  const uint32_t b = __float_as_uint(x);
  const auto s = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return __uint_as_float((threadIdx.x & 32) ? (uint32_t)s[0] : (uint32_t)s[1]);
}

__device__ __forceinline__ constexpr int acc_row(int i) { return 8 * (i / 4) + i % 4; }

// Sets the scores of a 32 x 32 block that are not kept to -inf. In this lane element i is row
// t + 4 (lane / 32) + acc_row(i) of the streamed side. end: rows from there on are none; bits (null: all are
// kept): their keep bits; window: element i is kept where 0 <= first + acc_row(i) <= span.
__device__ __forceinline__ void mask_scores(f32x16& s, int t, int end, const uint32_t* bits, bool window, int first,
                                            uint32_t span, int lane) {
  const int h4 = 4 * (lane >> 5);
  if (window) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = (uint32_t)(first + acc_row(i)) <= span ? s[i] : -INFINITY;
  }
  if (bits && t < end) {
    const uint32_t w = bits[t >> 5] >> h4;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = (w & (1u << acc_row(i))) ? s[i] : -INFINITY;
  }
  if (t + 32 > end) {
    const int left = end - t - h4;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = acc_row(i) < left ? s[i] : -INFINITY;
  }
}

// The output's rounding error as a byte: the difference of the fp32 results' bits before and after the
// rounding, in steps of 2^LOW fp32 units (256 steps from half a unit of the 16-bit type below to half above).
// delta = sum_d g o cancels against g v in the backward pass: with the byte o is as good as fp32 there.
template <int EK>
constexpr int kLow = EK == EK_F16 ? 5 : 8;
template <int EK>
__device__ __forceinline__ uint32_t low_byte1(float o) {  // in byte 1
  const int most = 1 << (kLow<EK> + 7);
  const int d = (int)(__float_as_uint(o) - __float_as_uint(el_to_f32<EK>(f32_to_el<EK>(o)))) + (1 << (kLow<EK> - 1));
  return (uint32_t)(d < -most ? -most : d > most - 1 ? most - 1 : d) << (8 - kLow<EK>);
}
template <int EK>
__device__ __forceinline__ uint32_t low_bytes(float a, float b, float c, float d) {
  const uint32_t ab = __builtin_amdgcn_perm(low_byte1<EK>(b), low_byte1<EK>(a), 0x0c0c0501u);
  return __builtin_amdgcn_perm(low_byte1<EK>(d), low_byte1<EK>(c), 0x05010c0cu) | ab;
}
// The value again, to a 256th of its rounding error (k: which byte of low).
template <int EK>
__device__ __forceinline__ float with_low(float r, uint32_t low, int k) {
  const int byte = (int)(low << (24 - 8 * k)) >> 24;
  return __uint_as_float(__float_as_uint(r) + (uint32_t)(byte << kLow<EK>));
}

// One column's DB x 32 elements times f to its row in memory (dim elements). Returns 0, or NaN if one of the lane's is
// not finite.
template <int EK, int DC>
__device__ __forceinline__ float store_cols(char* row, const f32x16* acc, float f, int dim, int lane, bool on) {
  float odd[2] = {};
#pragma unroll
  for (int db = 0; db < DC; ++db)
#pragma unroll
    for (int q = 0; q < 4; q += 2) {
      const f32x16& a = acc[db];
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = pack2<EK>(a[q * 4 + 2 * i] * f, a[q * 4 + 2 * i + 1] * f);
        odd[i % 2] = add2<EK>(w[i], odd[i % 2], 0.f);
      }
      const u32x4 o = join_halves(w[0], w[1], w[2], w[3]);
      const int e = db * 32 + 8 * q + 8 * (lane >> 5);
      if (on && e < dim) *(u32x4*)(row + e * 2) = o;
    }
  return odd[0] + odd[1];
}
// The same elements' bytes.
template <int EK, int DC>
__device__ __forceinline__ void store_low(int8_t* row, const f32x16* acc, float f, int dim, int lane, bool on) {
#pragma unroll
  for (int db = 0; db < DC; ++db)
#pragma unroll
    for (int q = 0; q < 4; q += 2) {
      const f32x16& a = acc[db];
      const auto s = __builtin_amdgcn_permlane32_swap(
          low_bytes<EK>(a[q * 4] * f, a[q * 4 + 1] * f, a[q * 4 + 2] * f, a[q * 4 + 3] * f),
          low_bytes<EK>(a[q * 4 + 4] * f, a[q * 4 + 5] * f, a[q * 4 + 6] * f, a[q * 4 + 7] * f), false, false);
      const int e = db * 32 + 8 * q + 8 * (lane >> 5);
      if (on && e < dim) *(u32x2*)(row + e) = u32x2{(uint32_t)s[0], (uint32_t)s[1]};
    }
}

// The window as one unsigned test: a key is kept where 0 <= key - query + back <= reach.
struct Window {
  bool on;
  int back;
  uint32_t reach;
  __device__ __forceinline__ explicit Window(const AttP& p)
      : on(p.left != kNone || p.right != kNone), back(p.left == kNone ? 0x3fffffff : p.left),
        reach((uint32_t)back + (p.right == kNone ? 0x3fffffffu : (uint32_t)p.right)) {}
};

// 16-byte rows; 64 of them within a lane's 32-bit offset
inline bool att_rows_ok(const void* d, int64_t sn, int64_t sl, int64_t sh) {
  return (uintptr_t)d % 16 == 0 && sn % 8 == 0 && sl % 8 == 0 && sh % 8 == 0 && sl >= 0 && sl < (1 << 24);  // (64 rows of up to 2^25 bytes)
}
// Checks the arguments that both directions share and fills the parameters; false: there is no query (rc is LIK_OK: what
// the call writes are zeros), or rc is an error.
bool attention_shape(const lik_attention_t* a, AttP& p, int& rc);
// Zeros in the rows of an output or gradient (null: not wanted).
int clear_rows(void* data, int64_t rows, int heads, int dim, hipStream_t s);

}  // namespace enc
}  // namespace lik
