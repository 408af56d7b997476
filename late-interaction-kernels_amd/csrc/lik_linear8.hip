// Linear layer on 8-bit integers: y = act(sx_m sw_n sum_k x w + b_n) (times the up half) + residual.
//
// x rows carry a scale each (quantised here from 16- or 32-bit rows, or given), weight rows another. The sums are
// exact 32-bit integers (in <= 131071: 2^14 a product), everything after them is fp32, rounded once.
#include "lik_act.h"
#include "lik_int8.h"

namespace lik {
namespace enc {
namespace {

typedef int i32x16 __attribute__((ext_vector_type(16)));

struct LinP {
  const char* a;  // tokens: int8 rows (few rows: of any type)
  const char* b;  // weight: int8 rows; GLU: gate rows, then up rows
  int64_t a_ld, b_ld;  // bytes
  int m, n, k;         // n: columns of the output
  int tiles_n, full;   // the first `full` tiles are one workgroup's each,
  int tail, splits;    // the `tail` others are `splits` workgroups' each,
  int k_per;           // of k_per of k
  int* part;           // their sums [tail][splits][a tile in the accumulators' order]
  const float* sx;
  const float* sw;
  const char* bias;    // null: none
  bool bias32;         // fp32 (else the output's type)
  const char* res;     // of the output's type; null: none
  int64_t res_ld;
  char* out;           // [m][n]
  int act;             // -1: none
};

__device__ __forceinline__ i32x16 mfma_i8(const i32x16& c, const u32x4& a, const u32x4& b) {
  return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

// What a lane of a 32 x 32 block needs of its columns, n = 8 q + 4 h + e of quad q, element e: weight scale and bias.
struct Cols {
  f32x4 s[4], b[4];
};
template <int OK>
__device__ __forceinline__ f32x4 load4(const char* p, bool f32, int n, int end) {
  typedef f32x4 __attribute__((aligned(4))) f32x4_u;
  typedef u32x2 __attribute__((aligned(2))) u32x2_u;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (OK == EK_F32 || f32) {
    if (n + 4 <= end) return *(const f32x4_u*)(p + (int64_t)n * 4);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < end) v[e] = ((const float*)p)[n + e];
  } else if constexpr (OK != EK_F32) {
    if (n + 4 <= end) {
      const u32x2 w = *(const u32x2_u*)(p + (int64_t)n * 2);
      float a, b, c, d;
      unpack2<OK>(w[0], a, b);
      unpack2<OK>(w[1], c, d);
      return f32x4{a, b, c, d};
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < end) v[e] = el_to_f32<OK>(((const uint16_t*)p)[n + e]);
  }
  return v;
}
// n: the block's first column, `more`: rows of the weight before it (the up half: n hidden ones)
template <int OK>
__device__ __forceinline__ void load_cols(const LinP& p, Cols& c, int n, int more, int h) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    c.s[q] = load4<EK_F32>((const char*)(p.sw + more), true, n + 8 * q + 4 * h, p.n);
    c.b[q] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (p.bias)
      c.b[q] = load4<OK>(p.bias + (int64_t)more * (OK == EK_F32 || p.bias32 ? 4 : 2), p.bias32, n + 8 * q + 4 * h, p.n);
  }
}

// Residual of a lane's columns as they are stored: 16-bit outputs 16 j + 8 h + 0..7 (a chunk each), fp32 8 q + 4 h + 0..3.
template <int OK>
constexpr int kResChunks = OK == EK_F32 ? 4 : 2;
template <int OK>
struct Res {
  u32x4 x[kResChunks<OK>];
};
template <int OK>
__device__ __forceinline__ void load_res(const LinP& p, Res<OK>& r, int m, int n, int h) {
#pragma unroll
  for (int j = 0; j < kResChunks<OK>; ++j) {
    r.x[j] = u32x4{0u, 0u, 0u, 0u};
    const int c = OK == EK_F32 ? n + 8 * j + 4 * h : n + 16 * j + 8 * h;
    if (p.res && m < p.m && c < p.n) chunk_load<OK>(p.res + m * p.res_ld, c, p.n, r.x[j]);
  }
}

__device__ __forceinline__ void activate(int act, float* v) {
  if (act < 0) return;
  float y[8];
  act8<false>(act, v, y, nullptr);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = y[e];
}

// Lane (m, h) of a block's sums: c0 (GLU: of the gate), c1 (GLU: of the up half); NJ: groups of 16 columns.
template <int OK, bool GLU, int NJ = 2>
__device__ __forceinline__ void finish_block(const LinP& p, const i32x16& c0, const i32x16& c1, const Cols& w0,
                                             const Cols& w1, const Res<OK>& r, float sx, int m, int n, int h) {
  char* row = p.out + m * ((int64_t)p.n * El<OK>::B);
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      v[e] = fmaf((float)c0[8 * j + e], sx * w0.s[2 * j + e / 4][e % 4], w0.b[2 * j + e / 4][e % 4]);
    activate(p.act, v);
    if constexpr (GLU)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        v[e] *= fmaf((float)c1[8 * j + e], sx * w1.s[2 * j + e / 4][e % 4], w1.b[2 * j + e / 4][e % 4]);
    if constexpr (OK == EK_F32) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int c = n + 16 * j + 8 * q + 4 * h;
        u32x4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = __float_as_uint(v[4 * q + e] + __uint_as_float(r.x[2 * j + q][e]));
        if (m < p.m && c < p.n) chunk_store<OK>(row, c, p.n, o);
      }
    } else {
      const int c = n + 16 * j + 8 * h;
      if (p.res) {  // in the accumulators' order
        const auto s0 = __builtin_amdgcn_permlane32_swap(r.x[j][0], r.x[j][2], false, false);
        const auto s1 = __builtin_amdgcn_permlane32_swap(r.x[j][1], r.x[j][3], false, false);
        const u32x4 x = {(uint32_t)s0[0], (uint32_t)s1[0], (uint32_t)s0[1], (uint32_t)s1[1]};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float a, b;
          unpack2<OK>(x[i], a, b);
          v[2 * i] += a;
          v[2 * i + 1] += b;
        }
      }
      const u32x4 o =
          join_halves(pack2<OK>(v[0], v[1]), pack2<OK>(v[2], v[3]), pack2<OK>(v[4], v[5]), pack2<OK>(v[6], v[7]));
      if (m < p.m && c < p.n) chunk_store<OK>(row, c, p.n, o);
    }
  }
}

// A tile's rows in LDS: BK = 64 bytes of k each, 4 chunks of 16; chunk c of row r lies at chunk c ^ ((r >> 2) & 3), so
// that 16 consecutive rows at one chunk cover the 64 banks.
constexpr int BK = 64;
template <int T, int NW>
struct Stage {
  static constexpr int BYTES = T * BK;
  static constexpr int NI = BYTES / 1024 / NW;  // 1 KB loads of a wavefront
  static_assert(BYTES % (1024 * NW) == 0, "");
  __device__ __forceinline__ static int swz(int r) { return (r >> 2) & 3; }
  // Lane offsets of the wavefront's loads from the tile's origin; glu: rows 32..63 of each 64 are up rows.
  __device__ __forceinline__ static void offsets(uint32_t* off, int wv, int lane, int64_t ld, int rows, bool glu,
                                                 int hidden) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int slot = (wv * NI + i) * 64 + lane, r = slot / 4, c = (slot % 4) ^ swz(r);
      const int at = glu ? (r / 64) * 32 + r % 32 : r;
      off[i] = at < rows ? (uint32_t)((at + (glu && (r & 32) ? (int64_t)hidden : 0)) * ld + c * 16) : kOob;
    }
  }
  __device__ __forceinline__ static void issue(uint32_t lds, const uint32_t* off, int i, int wv, int lane,
                                               const u32x4& desc, int k_left) {
    uint32_t o = off[i];
    if (k_left < BK) {
      const int slot = (wv * NI + i) * 64 + lane;
      if (((slot % 4) ^ swz(slot / 4)) * 16 >= k_left) o = kOob;
    }
    dma16(lds + (wv * NI + i) * 1024, o, desc);
  }
  // Lane addresses of MFMA operands: lane l has row row0 + l % 32, k = 32 ks + 16 (l / 32) + 0..15.
  __device__ __forceinline__ static void bases(uint32_t* a, int row0, int lane) {
    const int r = row0 + (lane & 31), h = lane >> 5;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) a[ks] = r * BK + (((ks * 2 + h) ^ swz(r)) << 4);
  }
  __device__ __forceinline__ static u32x4 frag(const uint32_t* a, uint32_t lds, int j, int ks) {
    return lds_b128(a[ks] + lds + j * 32 * BK);
  }
};

// A workgroup of WM x WN wavefronts owns a TM x TN tile and walks k in steps of 64 bytes, NS of them in LDS: the
// loads of step i + NS - 1 start while step i is multiplied.
template <int OK, bool GLU, int TM, int TN, int WM, int WN, int NS, int OCC>
__global__ void __launch_bounds__(WM* WN * 64) __attribute__((amdgpu_waves_per_eu(OCC, OCC)))
linear8_kernel(const LinP p) {
  constexpr int NW = WM * WN, MB = TM / WM / 32, NB = TN / WN / 32, PAIR = GLU ? 2 : 1;
  using SA = Stage<TM, NW>;
  using SB = Stage<TN, NW>;
  constexpr int SBYTES = SA::BYTES + SB::BYTES, NI = SA::NI + SB::NI;
  __shared__ __attribute__((aligned(1024))) char s_tile[NS * SBYTES];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wv % WM, wn = wv / WM;
  const bool whole = (int)blockIdx.x < p.full;
  const int at = (int)blockIdx.x - p.full, split = whole ? 0 : at / p.tail;
  const uint32_t t = whole ? xcd_tile(blockIdx.x, (uint32_t)p.full) : (uint32_t)(p.full + at % p.tail);
  const int tm = (int)(t / (uint32_t)p.tiles_n), tn = (int)(t % (uint32_t)p.tiles_n);
  const int m0 = tm * TM, n0 = tn * (TN / PAIR);
  const int k0 = split * p.k_per, k1 = whole || k0 + p.k_per > p.k ? p.k : k0 + p.k_per;
  const int steps = (k1 - k0 + BK - 1) / BK;

  uint32_t offa[SA::NI], offb[SB::NI];
  SA::offsets(offa, wv, lane, p.a_ld, p.m - m0, false, 0);
  SB::offsets(offb, wv, lane, p.b_ld, p.n - n0, GLU, p.n);
  const uint32_t lds0 = lds_addr(s_tile);
  uint32_t ra[2], rb[2];
  SA::bases(ra, wm * (TM / WM), lane);
  SB::bases(rb, wn * (TN / WN), lane);
  const char* a_at = p.a + (int64_t)m0 * p.a_ld;
  const char* b_at = p.b + (int64_t)n0 * p.b_ld;
  // a step past the end loads nothing but counts alike
  auto desc = [&](const char* at0, int i) {
    const int k = k0 + i * BK;
    return raw_desc(at0 + k, k < k1 ? 0xffffff00u : 0u);
  };
  u32x4 fa[2][MB], fb[2][NB];
  auto read = [&](int set, uint32_t lds, int ks, int j) {
    if (j < MB) fa[set][j] = SA::frag(ra, lds, j, ks);
    else fb[set][j - MB] = SB::frag(rb, lds + SA::BYTES, j - MB, ks);
  };
  auto issue = [&](int j, uint32_t lds, const u32x4& da, const u32x4& db, int left) {
    if (j < SA::NI) SA::issue(lds, offa, j, wv, lane, da, left);
    else SB::issue(lds + SA::BYTES, offb, j - SA::NI, wv, lane, db, left);
  };

  i32x16 acc[NB][MB];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j) acc[i][j] = i32x16{};
  // The MFMAs of operand set `set`, and spread between them the reads of the other set and `loads` loads.
  auto k_step = [&](auto SET, uint32_t lds, int ks, auto LOADS, auto load) {
    constexpr int set = decltype(SET)::value;
    constexpr int S = NB * MB, R = MB + NB, OPS = R + decltype(LOADS)::value;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      acc[s / MB][s % MB] = mfma_i8(acc[s / MB][s % MB], fb[set][s / MB], fa[set][s % MB]);
#pragma unroll
      for (int o = s * OPS / S; o < (s + 1) * OPS / S; ++o) {
        if (o < R) read(set ^ 1, lds, ks, o);
        else load(o - R);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  using std::integral_constant;
  constexpr integral_constant<int, 0> S0{}, NONE{};
  constexpr integral_constant<int, 1> S1{};
  constexpr integral_constant<int, NI> ALL{};
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) {
    const u32x4 da = desc(a_at, i), db = desc(b_at, i);
#pragma unroll
    for (int j = 0; j < NI; ++j) issue(j, lds0 + i * SBYTES, da, db, k1 - k0 - i * BK);
  }
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NS - 2) * NI) : "memory");
#pragma unroll
  for (int j = 0; j < MB + NB; ++j) read(0, lds0, 0, j);
  uint32_t cur = lds0, next = lds0 + SBYTES, into = lds0 + (NS - 1) * SBYTES;
  for (int i = 0; i < steps; ++i) {
    const u32x4 da = desc(a_at, i + NS - 1), db = desc(b_at, i + NS - 1);
    const int left = k1 - k0 - (i + NS - 1) * BK;
    k_step(S0, cur, 1, ALL, [&](int j) { issue(j, into, da, db, left); });
    // the next step is complete in LDS, and every wavefront has read all of this one
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NS - 2) * NI) : "memory");
    k_step(S1, next, 0, NONE, [&](int) {});
    into = cur;
    cur = next;
    next = next == lds0 + (NS - 1) * SBYTES ? lds0 : next + SBYTES;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load is in flight to LDS when the workgroup ends

  if (!whole) {
    int* out = p.part + (((int64_t)(at % p.tail) * p.splits + split) * NW + wv) * (NB * MB * 1024) + lane * 4;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < MB; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *(i32x4*)(out + ((i * MB + j) * 4 + q) * 256) =
              i32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    return;
  }
  const int l32 = lane & 31, h = lane >> 5;
  float sx[MB];
#pragma unroll
  for (int j = 0; j < MB; ++j) {
    const int m = m0 + wm * (TM / WM) + j * 32 + l32;
    sx[j] = m < p.m ? p.sx[m] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < NB; i += PAIR) {
    const int n = n0 + wn * (TN / WN / PAIR) + i / PAIR * 32;
    Cols w0, w1;
    load_cols<OK>(p, w0, n, 0, h);
    if (GLU) load_cols<OK>(p, w1, n, p.n, h);
#pragma unroll
    for (int j = 0; j < MB; ++j) {
      const int m = m0 + wm * (TM / WM) + j * 32 + l32;
      Res<OK> r;
      load_res<OK>(p, r, m, n, h);
      finish_block<OK, GLU>(p, acc[i][j], acc[i + PAIR - 1][j], w0, w1, r, sx[j], m, n, h);
    }
  }
}

// The tail's epilogue: a workgroup adds the splits of one block of every wavefront.
template <int OK, bool GLU, int TM, int TN, int WM, int WN>
__global__ void __launch_bounds__(WM* WN * 64) linear8_finish_kernel(const LinP p) {
  constexpr int NW = WM * WN, MB = TM / WM / 32, NB = TN / WN / 32, PAIR = GLU ? 2 : 1;
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, wm = wv % WM, wn = wv / WM, h = lane >> 5;
  int u = (int)blockIdx.x;
  const int j = u % MB;
  u /= MB;
  const int i = u % (NB / PAIR) * PAIR;
  u /= NB / PAIR;
  const int t = p.full + u, tm = t / p.tiles_n, tn = t % p.tiles_n;
  const int m = tm * TM + wm * (TM / WM) + j * 32 + (lane & 31);
  const int n = tn * (TN / PAIR) + wn * (TN / WN / PAIR) + i / PAIR * 32;
  Res<OK> r;
  load_res<OK>(p, r, m, n, h);
  Cols w0, w1;
  load_cols<OK>(p, w0, n, 0, h);
  if (GLU) load_cols<OK>(p, w1, n, p.n, h);
  i32x16 c[PAIR];
#pragma unroll
  for (int b = 0; b < PAIR; ++b) c[b] = i32x16{};
  const int* in = p.part + ((int64_t)u * p.splits * NW + wv) * (NB * MB * 1024) + lane * 4;
#pragma unroll 2
  for (int s = 0; s < p.splits; ++s, in += NW * NB * MB * 1024)
#pragma unroll
    for (int b = 0; b < PAIR; ++b)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const i32x4 x = *(const i32x4*)(in + (((i + b) * MB + j) * 4 + q) * 256);
#pragma unroll
        for (int e = 0; e < 4; ++e) c[b][4 * q + e] += x[e];
      }
  finish_block<OK, GLU>(p, c[0], c[PAIR - 1], w0, w1, r, m < p.m ? p.sx[m] : 0.f, m, n, h);
}

// Few rows: the weight is read once for all of them. A workgroup owns 32 weight rows (GLU: 16 gate and the 16 up rows of
// the same columns, which meet in one lane's accumulators) and all 32 MB rows of x, its eight wavefronts an eighth of k
// each: operands go from memory to registers as they lie, the eight sums meet in LDS. Rows that are no integers yet
// are quantised on the way, by every workgroup for itself: the wavefronts' maxima meet in LDS first. (XK: EK_FP8
// stands for 8-bit integers.)
constexpr int kInt8 = EK_FP8;
template <int XK, int OK, bool GLU, int MB>
__global__ void __launch_bounds__(512) few_rows8_kernel(const LinP p) {
  constexpr int NW = 8, U = XK == EK_F32 ? 2 : 4;
  constexpr int XB = XK == kInt8 ? 1 : XK == EK_F32 ? 4 : 2;  // bytes of an element
  constexpr int XC = XB;                                      // 16-byte chunks of 16 elements
  __shared__ __attribute__((aligned(16))) int s_sum[NW][MB][4][64][4];
  __shared__ uint32_t s_max[NW][MB * 32];
  const int lane = threadIdx.x & 63, l32 = lane & 31, h = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = (int)blockIdx.x * (GLU ? 16 : 32);
  const int n = GLU ? n0 + (l32 & 15) : n0 + l32;
  const char* wrow = p.b + (int64_t)(GLU && l32 >= 16 ? n + p.n : n) * p.b_ld;
  const bool won = n < p.n;
  const int k16 = (p.k + 15) / 16 * 16;
  i32x16 acc[MB];
#pragma unroll
  for (int j = 0; j < MB; ++j) acc[j] = i32x16{};
  const int all = (p.k + 31) / 32, per = (all + NW - 1) / NW, first = wv * per;
  const int end = first + per < all ? first + per : all;
  u32x4 fb[U], x[U][MB][XC];
  auto load_x = [&](int ks) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < MB; ++j) {
        const int e = (ks + u) * 32 + 16 * h, m = j * 32 + l32;
        const bool on = ks + u < end && m < p.m;
#pragma unroll
        for (int c = 0; c < XC; ++c) {
          x[u][j][c] = u32x4{0u, 0u, 0u, 0u};
          if constexpr (XK == kInt8) {
            if (on && e < k16) x[u][j][c] = *(const u32x4*)(p.a + m * p.a_ld + e);
          } else {
            const int at = e + c * El<XK>::V;
            if (on && at < p.k) chunk_load<XK>(p.a + m * p.a_ld, at, p.k, x[u][j][c]);
          }
        }
      }
  };
  auto load_w = [&](int ks) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = (ks + u) * 32 + 16 * h;
      fb[u] = u32x4{0u, 0u, 0u, 0u};
      if (won && ks + u < end && e < k16) fb[u] = *(const u32x4*)(wrow + e);
    }
  };
  float sx[MB], inv[MB];
  load_w(first);
  if constexpr (XK != kInt8) {
    uint32_t top[MB];
#pragma unroll
    for (int j = 0; j < MB; ++j) top[j] = 0;
    // from the last steps to the first, which stay in registers
    for (int ks = first + (per - 1) / U * U; ks >= first; ks -= U) {
      load_x(ks);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < MB; ++j)
#pragma unroll
          for (int c = 0; c < XC; ++c) top[j] = absmax_bits<XK>(x[u][j][c], top[j]);
    }
#pragma unroll
    for (int j = 0; j < MB; ++j) {
      top[j] = absmax_join<XK>(top[j], (uint32_t)__shfl_xor((int)top[j], 32));
      if (h == 0) s_max[wv][j * 32 + l32] = top[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < MB; ++j) {
#pragma unroll
      for (int w = 0; w < NW; ++w) top[j] = absmax_join<XK>(top[j], s_max[w][j * 32 + l32]);
      row_scale<XK>(top[j], sx[j], inv[j]);
    }
  } else {
    load_x(first);
#pragma unroll
    for (int j = 0; j < MB; ++j) sx[j] = j * 32 + l32 < p.m ? p.sx[j * 32 + l32] : 0.f;
  }
  for (int ks = first; ks < end; ks += U) {
    if (ks != first) {
      load_w(ks);
      load_x(ks);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < MB; ++j) {
        u32x4 q;
        if constexpr (XK == kInt8) {
          q = x[u][j][0];
        } else {
          constexpr int W = El<XK>::V / 4;  // words of a chunk's integers
#pragma unroll
          for (int c = 0; c < XC; ++c) {
            uint32_t w[W];
            chunk_to_int8<XK>(x[u][j][c], sx[j], inv[j], w);
#pragma unroll
            for (int i = 0; i < W; ++i) q[c * W + i] = w[i];
          }
        }
        acc[j] = mfma_i8(acc[j], fb[u], q);
      }
  }
#pragma unroll
  for (int j = 0; j < MB; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *(i32x4*)s_sum[wv][j][q][lane] = i32x4{acc[j][4 * q], acc[j][4 * q + 1], acc[j][4 * q + 2], acc[j][4 * q + 3]};
  __syncthreads();
  if (wv >= MB) return;
  const int m = wv * 32 + l32;
  float s = sx[0];
#pragma unroll
  for (int j = 1; j < MB; ++j) s = wv == j ? sx[j] : s;
  Res<OK> r;
  load_res<OK>(p, r, m, n0, h);
  Cols w0, w1;
  load_cols<OK>(p, w0, n0, 0, h);
  if (GLU) load_cols<OK>(p, w1, n0, p.n, h);
  i32x16 c = {};
#pragma unroll
  for (int w = 0; w < NW; ++w)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const i32x4 v = *(const i32x4*)s_sum[w][wv][q][lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) c[4 * q + e] += v[e];
    }
  if constexpr (GLU) {
    i32x16 up = {};
#pragma unroll
    for (int e = 0; e < 8; ++e) up[e] = c[8 + e];
    finish_block<OK, GLU, 1>(p, c, up, w0, w1, r, s, m, n0, h);
  } else {
    finish_block<OK, GLU>(p, c, c, w0, w1, r, s, m, n0, h);
  }
}

constexpr int kCUs = 256;
bool few_rows(int64_t m) { return m <= 64; }

struct Shape {
  bool large;
  int tiles_n, full, tail, splits, k_per;
};
// n: rows of the weight's tiles
Shape shape_of(int64_t m, int64_t n, int64_t k, bool glu) {
  const bool large = (m + 255) / 256 * ((n + 127) / 128) >= kCUs;
  const int64_t tm = large ? 256 : glu ? 64 : 128, tn = large || glu ? 128 : 64;
  const int64_t cols = (n + tn - 1) / tn;
  return Shape{large, (int)cols, (int)((m + tm - 1) / tm * cols), 0, 1, (int)k};
}
int64_t glu_rows(int64_t n) { return (n + 31) / 32 * 64; }  // (blocks of 32 gate and 32 up rows)
size_t part_bytes(const Shape& s) { return (size_t)s.tail * s.splits * (s.large ? 256 * 128 : 128 * 64) * 4; }

template <int OK, bool GLU, int TM, int TN, int NS, int OCC>
int launch_tiles(const LinP& p, hipStream_t s) {
  const int groups = p.full + p.tail * p.splits;
  launch_kernel(linear8_kernel<OK, GLU, TM, TN, 2, 2, NS, OCC>, dim3((unsigned)groups), dim3(256), 0u, s, p);
  if (hipGetLastError() != hipSuccess) return LIK_ERR_LAUNCH;
  if (p.tail) {
    constexpr int blocks = TM / 64 * (TN / 64) / (GLU ? 2 : 1);
    launch_kernel(linear8_finish_kernel<OK, GLU, TM, TN, 2, 2>, dim3((unsigned)(p.tail * blocks)), dim3(256), 0u, s, p);
    if (hipGetLastError() != hipSuccess) return LIK_ERR_LAUNCH;
  }
  return LIK_OK;
}
template <int OK, bool GLU>
int launch_gemm(LinP p, int* part, hipStream_t s) {
  const Shape sh = shape_of(p.m, GLU ? glu_rows(p.n) : p.n, p.k, GLU);
  p.tiles_n = sh.tiles_n;
  p.full = sh.full;
  p.tail = sh.tail;
  p.splits = sh.splits;
  p.k_per = sh.k_per;
  p.part = part;
  if (sh.large) return launch_tiles<OK, GLU, 256, 128, 3, 2>(p, s);
  // (a wavefront has 32 columns of a 128 x 64 tile: gate and up blocks need 64)
  if constexpr (GLU) return launch_tiles<OK, GLU, 64, 128, 3, 3>(p, s);
  else return launch_tiles<OK, GLU, 128, 64, 3, 3>(p, s);
}

template <int XK, int OK, bool GLU>
int launch_few(const LinP& p, hipStream_t s) {
  const unsigned nb = GLU ? (p.n + 15) / 16 : (p.n + 31) / 32;
  if (p.m <= 32)
    launch_kernel(few_rows8_kernel<XK, OK, GLU, 1>, dim3(nb), dim3(512), 0u, s, p);
  else
    launch_kernel(few_rows8_kernel<XK, OK, GLU, 2>, dim3(nb), dim3(512), 0u, s, p);
  return hipGetLastError() == hipSuccess ? LIK_OK : LIK_ERR_LAUNCH;
}

template <int OK, bool GLU>
int run(const lik_linear_int8_t* a, LinP p, char* ws, hipStream_t s) {
  if (few_rows(a->rows)) switch (a->x_dtype) {
      case LIK_BF16: return launch_few<EK_BF16, OK, GLU>(p, s);
      case LIK_F16: return launch_few<EK_F16, OK, GLU>(p, s);
      case LIK_F32: return launch_few<EK_F32, OK, GLU>(p, s);
      default: return launch_few<kInt8, OK, GLU>(p, s);
    }
  if (a->x_dtype != LIK_INT8) {
    const int64_t k16 = ((int64_t)p.k + 15) / 16 * 16;
    int8_t* x8 = (int8_t*)ws;
    ws += align256((size_t)(p.m * k16));
    float* sx = (float*)ws;
    ws += align256((size_t)p.m * 4);
    if (const int rc = lik_quantize_int8(a->x, a->x_stride, a->x_dtype, a->rows, a->in, x8, k16, sx, (lik_stream_t)s))
      return rc;
    p.a = (const char*)x8;
    p.a_ld = k16;
    p.sx = sx;
  }
  return launch_gemm<OK, GLU>(p, (int*)ws, s);
}

constexpr int64_t kFar = 0xfff00000ll;  // bytes that a lane's 32-bit offset reaches
int linear_check(const lik_linear_int8_t* a) {
  const auto is_float = [](int32_t t) { return t == LIK_BF16 || t == LIK_F16 || t == LIK_F32; };
  if (!is_float(a->out_dtype) || !(is_float(a->x_dtype) || a->x_dtype == LIK_INT8)) return LIK_ERR_UNSUPPORTED;
  if (a->rows < 0 || a->in < 1 || a->out_features < 1 || a->activation < -1 || a->activation > ACT_SILU)
    return LIK_ERR_INVALID;
  if (a->bias && a->bias_dtype != a->out_dtype && a->bias_dtype != LIK_F32) return LIK_ERR_UNSUPPORTED;
  if (a->in > 131071 || a->rows > 0x7fffff00 || a->out_features > (1 << 24)) return LIK_ERR_UNSUPPORTED;
  const int64_t groups = ((a->rows + 63) / 64) * ((2ll * a->out_features + 63) / 64);
  return groups < (1 << 24) ? LIK_OK : LIK_ERR_UNSUPPORTED;  // (a launch has less than 2^32 threads)
}
size_t linear_ws(const lik_linear_int8_t* a) {
  if (few_rows(a->rows)) return 0;
  const Shape sh = shape_of(a->rows, a->gated ? glu_rows(a->out_features) : a->out_features, a->in, a->gated != 0);
  size_t b = part_bytes(sh);
  if (a->x_dtype != LIK_INT8)
    b += align256((size_t)(a->rows * (((int64_t)a->in + 15) / 16 * 16))) + align256((size_t)a->rows * 4);
  return b ? b + 256 : 0;
}

}  // namespace
}  // namespace enc
}  // namespace lik

using namespace lik;
using namespace lik::enc;

extern "C" {

size_t lik_linear_int8_workspace_size(const lik_linear_int8_t* a) {
  if (!a || linear_check(a) != LIK_OK || a->rows == 0) return 0;
  return linear_ws(a);
}

int lik_linear_int8(const lik_linear_int8_t* a, void* out, void* workspace, size_t workspace_bytes,
                    lik_stream_t stream) {
  if (!a) return LIK_ERR_INVALID;
  if (const int rc = linear_check(a)) return rc;
  if (a->rows == 0) return LIK_OK;
  const bool int8 = a->x_dtype == LIK_INT8;
  if (!a->x || !a->weight || !a->weight_scale || !out || (int8 && !a->x_scale)) return LIK_ERR_INVALID;
  const int ob = a->out_dtype == LIK_F32 ? 4 : 2, xb = int8 ? 16 : a->x_dtype == LIK_F32 ? 4 : 2;
  if ((uintptr_t)a->x % xb || (uintptr_t)out % ob || (uintptr_t)a->weight_scale % 4 || (uintptr_t)a->x_scale % 4 ||
      (uintptr_t)a->residual % ob || (a->bias && (uintptr_t)a->bias % (a->bias_dtype == LIK_F32 ? 4 : 2)))
    return LIK_ERR_UNSUPPORTED;
  // 16-byte chunks of integers; a tile's rows within a lane's 32-bit offset
  if ((uintptr_t)a->weight % 16 || a->weight_stride % 16 || a->weight_stride < 0 ||
      ((a->gated ? a->out_features : 0) + 256ll) * a->weight_stride >= kFar)
    return LIK_ERR_UNSUPPORTED;
  if (int8 && (a->in % 16 || a->x_stride % 16 || a->x_stride < 0 || 256 * a->x_stride >= kFar))
    return LIK_ERR_UNSUPPORTED;
  if (workspace_bytes < linear_ws(a) || (!workspace && linear_ws(a))) return LIK_ERR_WORKSPACE;
  LinP p{};
  p.a = (const char*)a->x;
  p.a_ld = a->x_stride * (int8 ? 1 : xb);
  p.b = (const char*)a->weight;
  p.b_ld = a->weight_stride;
  p.m = (int)a->rows;
  p.n = a->out_features;
  p.k = a->in;
  p.sx = a->x_scale;
  p.sw = a->weight_scale;
  p.bias = (const char*)a->bias;
  p.bias32 = a->bias_dtype == LIK_F32;
  p.res = (const char*)a->residual;
  p.res_ld = a->residual_stride * ob;
  p.out = (char*)out;
  p.act = a->activation;
  char* ws = workspace ? align256(workspace) : nullptr;
  hipStream_t s = (hipStream_t)stream;
  switch (a->out_dtype) {
    case LIK_BF16: return a->gated ? run<EK_BF16, true>(a, p, ws, s) : run<EK_BF16, false>(a, p, ws, s);
    case LIK_F16: return a->gated ? run<EK_F16, true>(a, p, ws, s) : run<EK_F16, false>(a, p, ws, s);
    default: return a->gated ? run<EK_F32, true>(a, p, ws, s) : run<EK_F32, false>(a, p, ws, s);
  }
}

}  // extern "C"
