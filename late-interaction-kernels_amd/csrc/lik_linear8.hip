// Linear layer on 8-bit integers: y = act(sx_m sw_n sum_k x w + b_n) (times the up half) + residual.
//
// x rows carry a scale each (quantised here from 16- or 32-bit rows, or given), weight rows another. The sums are
// exact 32-bit integers (in <= 131071: 2^14 a product), everything after them is fp32, rounded once.
//
// Bound by the matrix cores' power at long k (8192^3: 478 us, 2.3 POP/s, 2.9 on zeros; a library product 2.05), by launch
// latency and one chain of loads for few rows, by epilogues in between: a tile of 256 x 256 takes 0.95 us a step of 64 k and about
// 2 us at its end, 12 steps at 768 features.
#include "lik_act.h"
#include "lik_int8.h"

#include <utility>

namespace lik {
namespace enc {
namespace {

typedef int i32x16 __attribute__((ext_vector_type(16)));

struct LinP {
  const char* a;  // tokens: int8 rows (few rows: of any type)
  const char* b;  // weight: int8 rows; GLU: gate rows, then up rows
  int64_t a_ld, b_ld;  // bytes
  int m, n, k;         // n: columns of the output
  int tiles_n, tiles;  // tiles of a row of them, all
  const float* sx;
  const float* sw;
  const char* bias;    // null: none
  bool bias32;         // fp32 (else the output's type)
  const char* res;     // of the output's type; null: none
  int64_t res_ld;
  char* out;           // [m][n]
  bool rows16;         // whose rows start on 16 bytes, 256 of them within a lane's 32-bit offset
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
template <int OK>
__device__ __forceinline__ void store4(char* row, int n, int end, const float* v) {
  typedef u32x4 __attribute__((aligned(4))) u32x4_u;
  typedef u32x2 __attribute__((aligned(2))) u32x2_u;
  if (n + 4 <= end) {
    if constexpr (OK == EK_F32)
      *(u32x4_u*)(row + (int64_t)n * 4) =
          u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
    else
      *(u32x2_u*)(row + (int64_t)n * 2) = u32x2{pack2<OK>(v[0], v[1]), pack2<OK>(v[2], v[3])};
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n + e < end) {
      if constexpr (OK == EK_F32) ((float*)row)[n + e] = v[e];
      else ((uint16_t*)row)[n + e] = (uint16_t)f32_to_el<OK>(v[e]);
    }
}
// n: the block's first column, `more`: rows of the weight before it (the up half: n hidden ones). Of its two groups of 16
// columns those from g on, ng of them (here and below).
__device__ __forceinline__ void load_scales(const LinP& p, f32x4* s, int n, int more, int h, int g, int ng) {
#pragma unroll
  for (int q = 2 * g; q < 2 * (g + ng); ++q) s[q] = load4<EK_F32>((const char*)(p.sw + more), true, n + 8 * q + 4 * h, p.n);
}
template <int OK>
__device__ __forceinline__ void load_cols(const LinP& p, Cols& c, int n, int more, int h, int g, int ng) {
  load_scales(p, c.s, n, more, h, g, ng);
#pragma unroll
  for (int q = 2 * g; q < 2 * (g + ng); ++q) {
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
// Column of chunk j of a lane, from the block's first.
template <int OK>
__device__ __forceinline__ int chunk_column(int j, int h) {
  return OK == EK_F32 ? 8 * j + 4 * h : 16 * j + 8 * h;
}
template <int OK>
__device__ __forceinline__ void load_res(const LinP& p, Res<OK>& r, int m, int n, int h, int g = 0, int ng = 2) {
  constexpr int C = kResChunks<OK> / 2;
#pragma unroll
  for (int j = C * g; j < C * (g + ng); ++j) {
    r.x[j] = u32x4{0u, 0u, 0u, 0u};
    const int c = n + chunk_column<OK>(j, h);
    if (p.res && m < p.m && c < p.n) chunk_load<OK>(p.res + m * p.res_ld, c, p.n, r.x[j]);
  }
}

template <int OK>
__device__ __forceinline__ void activate(int act, float* v) {
  if (act < 0) return;
  float y[8];
  if constexpr (OK == EK_F32) act8_f32(act, v, y);
  else act8<false>(act, v, y, nullptr);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = y[e];
}

// A sum is scaled as (sum * sx) * sw + b: the scales' own product may leave fp32's range where the result does not (1e-25 and
// 1e-18: under 2^-126, which keeps a few bits; 1e20 and 1e20: an infinity, which a sum of zero makes NaN). The first product
// is exact or normal, and finite unless sx is past 2^96 (sums reach 2^31). Such a token gives 2^64 of its scale to the
// weights': near_scale for the token, lift_scales for copies of the weights' scales (past 2^63 the largest float will do: a
// sum other than zero makes either infinite). Kernels ask once whether a wavefront has such rows, so that all others do without.
__device__ __forceinline__ bool far_scale(float sx) { return fabsf(sx) > 0x1p96f; }
__device__ __forceinline__ uint64_t far_rows(float sx) { return __builtin_amdgcn_ballot_w64(far_scale(sx)); }
__device__ __forceinline__ float near_scale(float sx) { return far_scale(sx) ? sx * 0x1p-64f : sx; }
template <int NQ>
__device__ __forceinline__ void lift_scales(f32x4* sw, bool far) {
#pragma unroll
  for (int e = 0; e < 4 * NQ; ++e) {
    const float w = sw[e / 4][e % 4], a = fabsf(w);
    if (far) sw[e / 4][e % 4] = a > 0x1p63f && a < INFINITY ? copysignf(0x1.fffffep127f, w) : w * 0x1p64f;
  }
}

// Weight scales and biases of a lane's columns in 16 of a block: two quads.
struct Cols8 {
  f32x4 s[2], b[2];
};
// Lane (m, h) of 16 columns' sums, c0 (GLU: of the gate) and c1 (GLU: of the up half), as it stores them: 16-byte
// chunks, one or (fp32) two; r: the residual's.
template <int OK, bool GLU, bool RES>
__device__ __forceinline__ void group_outputs(const LinP& p, const int* c0, const int* c1, const Cols8& w0,
                                              const Cols8& w1, const u32x4* r, float sx, u32x4* out) {
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = fmaf((float)c0[e] * sx, w0.s[e / 4][e % 4], w0.b[e / 4][e % 4]);
  activate<OK>(p.act, v);
  if constexpr (GLU)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= fmaf((float)c1[e] * sx, w1.s[e / 4][e % 4], w1.b[e / 4][e % 4]);
  if constexpr (OK == EK_F32) {
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e / 4][e % 4] = __float_as_uint(RES ? v[e] + __uint_as_float(r[e / 4][e % 4]) : v[e]);
  } else {
    if constexpr (RES) {  // in the accumulators' order
      const auto s0 = __builtin_amdgcn_permlane32_swap(r[0][0], r[0][2], false, false);
      const auto s1 = __builtin_amdgcn_permlane32_swap(r[0][1], r[0][3], false, false);
      const u32x4 x = {(uint32_t)s0[0], (uint32_t)s1[0], (uint32_t)s0[1], (uint32_t)s1[1]};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float a, b;
        unpack2<OK>(x[i], a, b);
        v[2 * i] += a;
        v[2 * i + 1] += b;
      }
    }
    out[0] = join_halves(pack2<OK>(v[0], v[1]), pack2<OK>(v[2], v[3]), pack2<OK>(v[4], v[5]), pack2<OK>(v[6], v[7]));
  }
}
template <int OK, bool GLU>
__device__ __forceinline__ void finish_block(const LinP& p, const i32x16& c0, const i32x16& c1, const Cols& w0, const Cols& w1,
                                             const Res<OK>& r, float sx, int m, int n, int h, int g0, int ng) {
  constexpr int C = kResChunks<OK> / 2;  // chunks of a group
  char* row = p.out + m * ((int64_t)p.n * El<OK>::B);
#pragma unroll
  for (int g = g0; g < g0 + ng; ++g) {
    int a0[8], a1[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) a0[e] = c0[8 * g + e], a1[e] = c1[8 * g + e];
    u32x4 o[C];
    group_outputs<OK, GLU, true>(p, a0, a1, Cols8{{w0.s[2 * g], w0.s[2 * g + 1]}, {w0.b[2 * g], w0.b[2 * g + 1]}},
                           Cols8{{w1.s[2 * g], w1.s[2 * g + 1]}, {w1.b[2 * g], w1.b[2 * g + 1]}}, r.x + C * g, sx, o);
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int c = n + chunk_column<OK>(C * g + j, h);
      if (m < p.m && c < p.n) chunk_store<OK>(row, c, p.n, o[j]);
    }
  }
}

// A tile's rows in LDS: BK = 64 bytes of k each, 4 chunks of 16; chunk c of row r lies at chunk c ^ ((r >> 2) & 3), so
// that 16 consecutive rows at one chunk cover the 64 banks.
constexpr int BK = 64;
template <int T, int NW>
struct Stage {
  static constexpr int BYTES = T * BK, LOADS = BYTES / 1024;  // loads of 1 KB: a wavefront's are wv, wv + NW, ..
  static constexpr int NI = (LOADS + NW - 1) / NW;
  static_assert(BYTES % 1024 == 0, "");
  __device__ __forceinline__ static int swz(int r) { return (r >> 2) & 3; }
  // Lane offsets of the wavefront's loads from the tile's origin; glu: rows 32..63 of each 64 are up rows.
  __device__ __forceinline__ static void offsets(uint32_t* off, int wv, int lane, int64_t ld, int rows, bool glu,
                                                 int hidden) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int slot = (i * NW + wv) * 64 + lane, r = slot / 4, c = (slot % 4) ^ swz(r);
      const int at = glu ? (r / 64) * 32 + r % 32 : r;
      off[i] = r < T && at < rows ? (uint32_t)((at + (glu && (r & 32) ? (int64_t)hidden : 0)) * ld + c * 16) : kOob;
    }
  }
  // `spare`: 1 KB for a wavefront's load past the tile (all wavefronts count as many)
  __device__ __forceinline__ static void issue(uint32_t lds, const uint32_t* off, int i, int wv, int lane,
                                               const u32x4& desc, int k_left, uint32_t spare) {
    uint32_t o = off[i];
    if (k_left < BK) {
      const int slot = (i * NW + wv) * 64 + lane;
      if (((slot % 4) ^ swz(slot / 4)) * 16 >= k_left) o = kOob;
    }
    dma16((i + 1) * NW <= LOADS || i * NW + wv < LOADS ? lds + (i * NW + wv) * 1024 : spare, o, desc);
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

// Too few tiles for the walk below: a workgroup of WM x WN wavefronts owns a TM x TN tile and goes along k in steps of 64 bytes, NS of
// them in LDS: the loads of step i + NS - 1 start while step i is multiplied. Tiles of 256 x 128 where those fill the CUs (16481 rows of
// integers 768 -> 768 21 us), else of 128 x 64 (300 rows of bf16 768 -> 2304 10.3 us with their quantising), gated 64 x 128.
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
  const uint32_t t = xcd_tile(blockIdx.x, (uint32_t)p.tiles);
  const int tm = (int)(t / (uint32_t)p.tiles_n), tn = (int)(t % (uint32_t)p.tiles_n);
  const int m0 = tm * TM, n0 = tn * (TN / PAIR);
  const int steps = (p.k + BK - 1) / BK;
  const int l32 = lane & 31, h = lane >> 5;
  float sx[MB];  // (first of all loads, which are waited for in order)
#pragma unroll
  for (int j = 0; j < MB; ++j) {
    const int m = m0 + wm * (TM / WM) + j * 32 + l32;
    sx[j] = m < p.m ? p.sx[m] : 0.f;
  }

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
    return raw_desc(at0 + i * BK, i < steps ? 0xffffff00u : 0u);
  };
  u32x4 fa[2][MB], fb[2][NB];
  auto read = [&](int set, uint32_t lds, int ks, int j) {
    if (j < MB) fa[set][j] = SA::frag(ra, lds, j, ks);
    else fb[set][j - MB] = SB::frag(rb, lds + SA::BYTES, j - MB, ks);
  };
  auto issue = [&](int j, uint32_t lds, const u32x4& da, const u32x4& db, int left) {
    if (j < SA::NI) SA::issue(lds, offa, j, wv, lane, da, left, 0);
    else SB::issue(lds + SA::BYTES, offb, j - SA::NI, wv, lane, db, left, 0);
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
    for (int j = 0; j < NI; ++j) issue(j, lds0 + i * SBYTES, da, db, p.k - i * BK);
  }
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NS - 2) * NI) : "memory");
#pragma unroll
  for (int j = 0; j < MB + NB; ++j) read(0, lds0, 0, j);
  uint32_t cur = lds0, next = lds0 + SBYTES, into = lds0 + (NS - 1) * SBYTES;
  for (int i = 0; i < steps; ++i) {
    const u32x4 da = desc(a_at, i + NS - 1), db = desc(b_at, i + NS - 1);
    const int left = p.k - (i + NS - 1) * BK;
    k_step(S0, cur, 1, ALL, [&](int j) { issue(j, into, da, db, left); });
    // the next step is complete in LDS, and every wavefront has read all of this one
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NS - 2) * NI) : "memory");
    k_step(S1, next, 0, NONE, [&](int) {});
    into = cur;
    cur = next;
    next = next == lds0 + (NS - 1) * SBYTES ? lds0 : next + SBYTES;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load is in flight to LDS when the workgroup ends

  uint64_t far = 0;
#pragma unroll
  for (int j = 0; j < MB; ++j) {
    far |= far_rows(sx[j]);
    sx[j] = near_scale(sx[j]);
  }
  constexpr int NG = GLU && OK == EK_F32 ? 1 : 2;  // groups of columns at once, as many as the registers hold scales and biases of
#pragma unroll
  for (int i = 0; i < NB; i += PAIR)
#pragma unroll
    for (int g = 0; g < 2; g += NG) {
      const int n = n0 + wn * (TN / WN / PAIR) + i / PAIR * 32;
      Cols w0, w1;
      load_cols<OK>(p, w0, n, 0, h, g, NG);
      if (GLU) load_cols<OK>(p, w1, n, p.n, h, g, NG);
#pragma unroll
      for (int j = 0; j < MB; ++j) {
        const int m = m0 + wm * (TM / WM) + j * 32 + l32;
        if (__builtin_expect(far != 0, false)) {  // (loaded again: the last rows' may be lifted)
          const bool lift = m < p.m && far_scale(p.sx[m]);
          load_scales(p, w0.s, n, 0, h, g, NG);
          lift_scales<2 * NG>(w0.s + 2 * g, lift);
          if (GLU) {
            load_scales(p, w1.s, n, p.n, h, g, NG);
            lift_scales<2 * NG>(w1.s + 2 * g, lift);
          }
        }
        Res<OK> r;
        load_res<OK>(p, r, m, n, h, g, NG);
        finish_block<OK, GLU>(p, acc[i][j], acc[i + PAIR - 1][j], w0, w1, r, sx[j], m, n, h, g, NG);
      }
    }
}

constexpr int64_t kFar = 0xfff00000ll;      // bytes that a lane's 32-bit offset reaches
constexpr uint32_t kNoRow = 0xfff80000u;    // a lane offset past them, also with a block's place in a tile's row added

// f(0), f(1), .. f(N - 1) as constants
template <typename F, int... I>
__device__ __forceinline__ void each_of(std::integer_sequence<int, I...>, F f) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void each(F f) {
  each_of(std::make_integer_sequence<int, N>{}, f);
}

// Many tiles: a workgroup per CU walks over its tiles of 256 x TN without a break. The loads run NS - 1 steps ahead,
// over the tiles' ends; of a finished tile's outputs some are stored at once and DEF 16-byte stores a lane wait in
// registers for the next tile's steps, so that the writes of all CUs do not come in bursts with nothing else to do.
// The waits count: a step waits for its own loads only, with all younger loads and stores in flight. So every
// store is issued whatever its lanes hold (a lane without an output names an offset out of range), and column
// edges, which store element by element, wait for everything (44801 x 768 -> 2305 184 us). Two workgroups a CU with tiles of 256 x 128
// instead fall into step and do not overlap. 44801 rows 768 -> 2304 fp16 99 to 103 us by card (256 x 128 tiles: 134), 1152 -> 768 with a
// residual 66 to 84 us by what is in the caches (98), 16480 rows 1024 -> 2 x 2816 with silu 112 to 116 us (125).
template <int OK, bool GLU, bool RES, int TN, int DEF>
__global__ void __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) linear8_stream_kernel(const LinP p) {
  constexpr int TM = 256, NW = 8, WM = 4, WN = 2, NS = 4;
  constexpr int MB = TM / WM / 32, NB = TN / WN / 32, PAIR = GLU ? 2 : 1;
  constexpr int PER = OK == EK_F32 ? 4 : 2;           // stores of a block
  constexpr int ALL = NB / PAIR * MB * PER, NOW = ALL - DEF;  // stores of a tile, and those at once
  using SA = Stage<TM, NW>;
  using SB = Stage<TN, NW>;
  constexpr int SBYTES = SA::BYTES + SB::BYTES, NI = SA::NI + SB::NI;  // loads of a step
  constexpr bool SPARE = SB::LOADS % NW != 0;
  __shared__ __attribute__((aligned(1024))) char s_tile[NS * SBYTES + (SPARE ? 1024 : 0)];
  __shared__ float s_sx[2][TM];
  __shared__ __attribute__((aligned(16))) float s_sw[2][TN], s_b[2][TN];
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, h = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wv % WM, wn = wv / WM;
  const int steps = (p.k + BK - 1) / BK;
  // tiles of this workgroup: t, t + stride, ..: its XCD's share, dealt round its workgroups
  const uint32_t x = blockIdx.x & 7u, per = (uint32_t)p.tiles >> 3, extra = (uint32_t)p.tiles & 7u;
  const int end = (int)(x * per + (x < extra ? x : extra) + per + (x < extra ? 1 : 0));
  const int stride = ((int)gridDim.x - (int)x + 7) / 8;
  int t = end - (int)(per + (x < extra ? 1 : 0)) + (int)(blockIdx.x >> 3);
  if (t >= end) return;

  const uint32_t lds0 = lds_addr(s_tile), spare = lds0 + NS * SBYTES;
  uint32_t ra[2], rb[2];
  SA::bases(ra, wm * (TM / WM), lane);
  SB::bases(rb, wn * (TN / WN), lane);
  // the loads' own place: tile lt, step ls of it
  int lt = t, ls = 0;
  uint32_t offa[SA::NI], offb[SB::NI], into = lds0;
  const char *la, *lb;
  auto seek = [&]() {
    const int tm = lt / p.tiles_n, m0 = tm * TM, n0 = (lt - tm * p.tiles_n) * (TN / PAIR);
    SA::offsets(offa, wv, lane, p.a_ld, p.m - m0, false, 0);
    SB::offsets(offb, wv, lane, p.b_ld, p.n - n0, GLU, p.n);
    la = p.a + (int64_t)m0 * p.a_ld;
    lb = p.b + (int64_t)n0 * p.b_ld;
  };
  u32x4 da, db;
  int left;
  auto aim = [&]() {  // past the last tile nothing is loaded, but counted alike
    const uint32_t size = lt < end ? 0xffffff00u : 0u;
    da = raw_desc(la + ls * BK, size);
    db = raw_desc(lb + ls * BK, size);
    left = p.k - ls * BK;
  };
  auto issue = [&](int j) {
    if (j < SA::NI) SA::issue(into, offa, j, wv, lane, da, left, spare);
    else SB::issue(into + SA::BYTES, offb, j - SA::NI, wv, lane, db, left, spare);
  };
  auto advance = [&]() {
    into = into == lds0 + (NS - 1) * SBYTES ? lds0 : into + SBYTES;
    if (++ls == steps) {
      ls = 0;
      lt += stride;
      if (lt < end) seek();
    }
  };
  // weight scales, biases and token scales of a tile, one or two values a thread; as they come, since whatever is done
  // with a loaded value waits for all that is in flight
  float col0 = 0.f;
  uint32_t col1 = 0;
  auto load_tile_cols = [&](int tile) {
    const int tm = tile / p.tiles_n, m0 = tm * TM, n0 = (tile - tm * p.tiles_n) * (TN / PAIR);
    if (tid < TM) {
      col0 = m0 + tid < p.m ? p.sx[m0 + tid] : 0.f;
    } else if (tid - TM < TN) {
      const int r = tid - TM, n = n0 + (GLU ? r / 64 * 32 + r % 32 : r);
      const int at = GLU && (r & 32) ? n + p.n : n;
      col0 = n < p.n ? p.sw[at] : 0.f;
      col1 = 0;
      if (p.bias && n < p.n) {
        if (OK == EK_F32 || p.bias32) col1 = ((const uint32_t*)p.bias)[at];
        else col1 = ((const uint16_t*)p.bias)[at];
      }
    }
  };
  auto keep_tile_cols = [&](int buf) {
    if (tid < TM) s_sx[buf][tid] = col0;
    else if (tid - TM < TN) {
      s_sw[buf][tid - TM] = col0;
      s_b[buf][tid - TM] = OK == EK_F32 || p.bias32 ? __uint_as_float(col1) : el_to_f32<OK>(col1);
    }
  };

  u32x4 fa[2][MB], fb[2][NB];
  auto read = [&](int set, uint32_t lds, int ks, int j) {
    if (j < MB) fa[set][j] = SA::frag(ra, lds, j, ks);
    else fb[set][j - MB] = SB::frag(rb, lds + SA::BYTES, j - MB, ks);
  };
  i32x16 acc[NB][MB];
  auto k_step = [&](auto SET, uint32_t lds, int ks, auto EXTRA, auto extra_op) {
    constexpr int set = decltype(SET)::value;
    constexpr int S = NB * MB, R = MB + NB, OPS = R + decltype(EXTRA)::value;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      acc[s / MB][s % MB] = mfma_i8(acc[s / MB][s % MB], fb[set][s / MB], fa[set][s % MB]);
#pragma unroll
      for (int o = s * OPS / S; o < (s + 1) * OPS / S; ++o) {
        if (o < R) read(set ^ 1, lds, ks, o);
        else extra_op(o - R);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  using std::integral_constant;
  constexpr integral_constant<int, 0> S0{}, NONE{};
  constexpr integral_constant<int, 1> S1{};
  constexpr integral_constant<int, NI> LOADS{};

  u32x4 later[DEF ? DEF : 1];  // deferred outputs,
  uint32_t out_off[MB][2];     // their rows' lane offsets
  __amdgpu_buffer_rsrc_t out_desc = __builtin_amdgcn_make_buffer_rsrc(p.out, (short)0, 0, 0x00020000);
#pragma unroll
  for (int d = 0; d < (DEF ? DEF : 1); ++d) later[d] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < MB; ++j) out_off[j][0] = out_off[j][1] = kNoRow;
  // Streamed past the caches where that is faster (44801 x 768 -> 2304 with its quantising launch: fp16 120 against 139 us;
  // 20000 rows to fp32: 92 against 84; with a residual no difference).
  constexpr int NT = OK == EK_F32 || RES ? 0 : 2;
  // Store O of a tile, of block (O / PER / MB, O / PER % MB): 16 rows (the block's first or last) of 64 bytes, so that the
  // chunks of two lanes that are 16 apart have changed places. The block's place is part of the lane's offset and no scalar
  // register: a 16-byte store reads its last registers up to two wait states after it is issued, the compiler counts those
  // for stores with a constant offset only, and with a register a conversion right behind one went to memory in its place.
  auto put = [&](auto O, const u32x4& v) {
    constexpr int o = decltype(O)::value, g = o % PER, j = o / PER % MB, i = o / PER / MB;
    __builtin_amdgcn_raw_buffer_store_b128(v, out_desc, out_off[j][g & 1] + (i * 32 * El<OK>::B + g / 2 * 64), 0, NT);
  };

  load_tile_cols(t);
  keep_tile_cols(0);
  seek();
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) {
    aim();
#pragma unroll
    for (int j = 0; j < NI; ++j) issue(j);
    advance();
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
  for (int j = 0; j < MB + NB; ++j) read(0, lds0, 0, j);
  uint32_t cur = lds0, next = lds0 + SBYTES;
  // One step of 64 k; AT: which one of the tile, while its stores matter. Younger than the loads that it waits for
  // (which started NS - 2 steps before) are the loads of NS - 2 steps, the deferred stores of those steps that are
  // of this tile, and the stores at once of the tile before if they came in between.
  auto step = [&](auto AT) {
    constexpr int at = decltype(AT)::value, from = at > NS - 2 ? at - (NS - 2) : 0, to = at < DEF ? at : DEF;
    constexpr int young = (NS - 2) * NI + (at < NS - 2 ? NOW : 0) + (to > from ? to - from : 0);
    aim();
    k_step(S0, cur, 1, LOADS, issue);
    // the next step is complete in LDS, and every wavefront has read all of this one
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(young < 63 ? young : 63) : "memory");
    k_step(S1, next, 0, NONE, [&](int) {});
    if constexpr (at < DEF) put(integral_constant<int, NOW + at>{}, later[at]);
    advance();
    cur = next;
    next = next == lds0 + (NS - 1) * SBYTES ? lds0 : next + SBYTES;
  };
  constexpr int HEAD = DEF + NS - 2;  // steps that know of stores

  for (int buf = 0;; buf ^= 1) {
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < MB; ++j) acc[i][j] = i32x16{};
    const int after = t + stride;
    if (after < end) load_tile_cols(after);
    const int tm = t / p.tiles_n, m0 = tm * TM, n0 = (t - tm * p.tiles_n) * (TN / PAIR);
    each<HEAD>([&](auto I) {
      if (decltype(I)::value < steps) step(I);
    });
    for (int i = HEAD; i < steps; ++i) step(integral_constant<int, HEAD>{});
    if (steps < DEF)
      each<DEF>([&](auto I) {
        if (decltype(I)::value >= steps) put(integral_constant<int, NOW + decltype(I)::value>{}, later[decltype(I)::value]);
      });

    // the residual's blocks are asked for one ahead
    constexpr int RB = RES ? 2 : 1;
    Res<OK> res[RB][MB];
    auto ask_res = [&](auto I) {
      constexpr int i = decltype(I)::value;
#pragma unroll
      for (int j = 0; j < MB; ++j)
        load_res<OK>(p, res[i % RB][j], m0 + wm * (TM / WM) + j * 32 + l32, n0 + wn * (TN / WN / PAIR) + i * 32, h);
    };
    if constexpr (RES) ask_res(S0);
    const bool edge = !p.rows16 || n0 + TN / PAIR > p.n;
    const int64_t out_ld = (int64_t)p.n * El<OK>::B;
    out_desc = __builtin_amdgcn_make_buffer_rsrc(p.out + m0 * out_ld + n0 * El<OK>::B, (short)0, (int)kFar, 0x00020000);
    float sx[MB];
    uint64_t far = 0;
#pragma unroll
    for (int j = 0; j < MB; ++j) {
      const int r = wm * (TM / WM) + j * 32 + l32;
      far |= far_rows(s_sx[buf][r]);
      sx[j] = near_scale(s_sx[buf][r]);
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int ro = wm * (TM / WM) + j * 32 + g * 16 + (lane & 15);
        out_off[j][g] = edge || m0 + ro >= p.m
                            ? kNoRow
                            : (uint32_t)(ro * out_ld + wn * (TN / WN / PAIR) * El<OK>::B + (lane & 16) * 2 + h * 16);
      }
    }
    each<NB / PAIR>([&](auto I) {
      constexpr int i = decltype(I)::value, C = PER / 2;
      const int n = n0 + wn * (TN / WN / PAIR) + i * 32;
      if constexpr (RES && i + 1 < NB / PAIR) ask_res(integral_constant<int, i + 1>{});
      u32x4 o[MB][PER];
      each<2>([&](auto G) {
        constexpr int g = decltype(G)::value;
        Cols8 w0, w1;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int at = wn * (TN / WN) + i * PAIR * 32 + 16 * g + 8 * q + 4 * h;
          w0.s[q] = *(const f32x4*)&s_sw[buf][at];
          w0.b[q] = *(const f32x4*)&s_b[buf][at];
          if (GLU) w1.s[q] = *(const f32x4*)&s_sw[buf][at + 32], w1.b[q] = *(const f32x4*)&s_b[buf][at + 32];
        }
        each<MB>([&](auto J) {
          constexpr int j = decltype(J)::value;
          if (__builtin_expect(far != 0, false)) {  // (loaded again: the last rows' may be lifted)
            const bool lift = far_scale(s_sx[buf][wm * (TM / WM) + j * 32 + l32]);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int at = wn * (TN / WN) + i * PAIR * 32 + 16 * g + 8 * q + 4 * h;
              w0.s[q] = *(const f32x4*)&s_sw[buf][at];
              if (GLU) w1.s[q] = *(const f32x4*)&s_sw[buf][at + 32];
            }
            lift_scales<2>(w0.s, lift);
            if (GLU) lift_scales<2>(w1.s, lift);
          }
          int a0[8], a1[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) a0[e] = acc[i * PAIR][j][8 * g + e], a1[e] = acc[i * PAIR + PAIR - 1][j][8 * g + e];
          group_outputs<OK, GLU, RES>(p, a0, a1, w0, w1, res[i % RB][j].x + C * g, sx[j], o[j] + C * g);
          if (edge) {
            const int m = m0 + wm * (TM / WM) + j * 32 + l32;
#pragma unroll
            for (int k = 0; k < C; ++k) {
              const int c = n + chunk_column<OK>(g * C + k, h);
              if (m < p.m && c < p.n) chunk_store<OK>(p.out + m * out_ld, c, p.n, o[j][g * C + k]);
            }
          }
          // two chunks are whole: the block's last 16 rows of the first and its first 16 of the second change places
          if constexpr (C == 2 || g == 1) {
            constexpr int k0 = C == 2 ? 2 * g : 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const auto s2 = __builtin_amdgcn_permlane16_swap(o[j][k0][e], o[j][k0 + 1][e], false, false);
              o[j][k0][e] = (uint32_t)s2[0];
              o[j][k0 + 1][e] = (uint32_t)s2[1];
            }
            each<2>([&](auto K) {
              constexpr int k = k0 + decltype(K)::value, at = (i * MB + j) * PER + k;
              if constexpr (at < NOW) put(integral_constant<int, at>{}, o[j][k]);
              else later[at - NOW] = o[j][k];
            });
          }
          __builtin_amdgcn_sched_barrier(0);
        });
      });
    });
    if (edge) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (after >= end) break;
    keep_tile_cols(buf ^ 1);
    t = after;
#pragma unroll
    for (int j = 0; j < MB + NB; ++j) read(0, cur, 0, j);  // (again: they need no registers meanwhile)
  }
  if (DEF)
    each<DEF>([&](auto I) {
      put(integral_constant<int, NOW + decltype(I)::value>{}, later[decltype(I)::value]);
    });
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load is in flight to LDS when the workgroup ends
}

// Few rows: the weight is read once for all of them. A workgroup owns 16 weight rows (GLU: 8 gate and the 8 up rows of
// the same columns) and all of up to 16 MB rows of x, its eight wavefronts an eighth of k each: operands go from memory
// to registers as they lie, the eight sums meet in LDS. Rows that are no integers yet are quantised on the way, by every
// workgroup for itself: the wavefronts' maxima meet in LDS first. 768 -> 2304 features of integers: 1 row 3.1 us, 32 rows 3.8, 64
// rows 4.8 (32 weight rows a workgroup: 32 rows 9.8 us with quantising, now 7.3); 4096 -> 4096: 5.2, 8.4, 12.2.
constexpr int kInt8 = 8;  // XK: 8-bit integers, next to the element types
template <int XK, int OK, bool GLU, int MB>
__global__ void __launch_bounds__(512) few_rows8_kernel(const LinP p) {
  constexpr int NW = 8, U = XK == kInt8 ? 4 : XK == EK_F32 ? 1 : 2;
  constexpr int XC = XK == kInt8 ? 1 : XK == EK_F32 ? 4 : 2;  // 16-byte chunks of 16 elements of x
  __shared__ __attribute__((aligned(16))) int s_sum[NW][MB][64][4];
  __shared__ uint32_t s_max[NW][MB * 16];
  const int lane = threadIdx.x & 63, l16 = lane & 15, quad = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = (int)blockIdx.x * (GLU ? 8 : 16);
  const int n = n0 + (GLU ? l16 & 7 : l16);
  const char* wrow = p.b + (int64_t)(GLU && l16 >= 8 ? n + p.n : n) * p.b_ld;
  const bool won = n < p.n;
  const int k16 = (p.k + 15) / 16 * 16;
  const int all = (p.k + 63) / 64, per = (all + NW - 1) / NW, first = wv * per;
  const int end = first + per < all ? first + per : all;
  // what the epilogue reads comes meanwhile: four columns of one row a lane
  const int m = wv * 16 + l16, c = n0 + 4 * quad;
  const bool last = wv < MB && m < p.m && (!GLU || quad < 2) && c < p.n;
  f32x4 s0 = {}, b0 = {}, s1 = {}, b1 = {}, res = {};
  i32x4 acc[MB];
#pragma unroll
  for (int j = 0; j < MB; ++j) acc[j] = i32x4{0, 0, 0, 0};
  u32x4 fb[U], x[U][MB][XC];
  auto load_w = [&](int ks) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = (ks + u) * 64 + 16 * quad;
      fb[u] = u32x4{0u, 0u, 0u, 0u};
      if (won && ks + u < end && e < k16) fb[u] = *(const u32x4*)(wrow + e);
    }
  };
  auto load_x = [&](int ks) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < MB; ++j) {
        const int e = (ks + u) * 64 + 16 * quad, row = j * 16 + l16;
        const bool on = ks + u < end && row < p.m;
#pragma unroll
        for (int i = 0; i < XC; ++i) {
          x[u][j][i] = u32x4{0u, 0u, 0u, 0u};
          if constexpr (XK == kInt8) {
            if (on && e < k16) x[u][j][i] = *(const u32x4*)(p.a + row * p.a_ld + e);
          } else {
            constexpr int V = El<XK>::V;
            if (on && e + (i + 1) * V <= p.k) chunk_load<XK, true>(p.a + row * p.a_ld, e + i * V, p.k, x[u][j][i]);
          }
        }
      }
    if constexpr (XK != kInt8) {  // the row's end: after all whole loads, since each of these is waited for
      constexpr int V = El<XK>::V;
      if (p.k % V != 0 && ks <= p.k / 64 && ks + U > p.k / 64)
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < MB; ++j)
#pragma unroll
            for (int i = 0; i < XC; ++i) {
              const int e = (ks + u) * 64 + 16 * quad + i * V, row = j * 16 + l16;
              if (ks + u < end && row < p.m && e < p.k && e + V > p.k)
                chunk_load<XK>(p.a + row * p.a_ld, e, p.k, x[u][j][i]);
            }
    }
  };
  auto load_last = [&]() {
    if (!last) return;
    s0 = load4<EK_F32>((const char*)p.sw, true, c, p.n);
    if (GLU) s1 = load4<EK_F32>((const char*)(p.sw + p.n), true, c, p.n);
    if (p.bias) {
      b0 = load4<OK>(p.bias, p.bias32, c, p.n);
      if (GLU) b1 = load4<OK>(p.bias + (int64_t)p.n * (OK == EK_F32 || p.bias32 ? 4 : 2), p.bias32, c, p.n);
    }
    if (p.res) res = load4<OK>(p.res + m * p.res_ld, false, c, p.n);
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
      if (ks == first) load_last();
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < MB; ++j)
#pragma unroll
          for (int i = 0; i < XC; ++i) top[j] = absmax_bits<XK>(x[u][j][i], top[j]);
    }
#pragma unroll
    for (int j = 0; j < MB; ++j) {
      const auto s16 = __builtin_amdgcn_permlane16_swap(top[j], top[j], false, false);
      top[j] = absmax_join<XK>((uint32_t)s16[0], (uint32_t)s16[1]);
      const auto s32 = __builtin_amdgcn_permlane32_swap(top[j], top[j], false, false);
      top[j] = absmax_join<XK>((uint32_t)s32[0], (uint32_t)s32[1]);
      if (quad == 0) s_max[wv][j * 16 + l16] = top[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < MB; ++j) {
#pragma unroll
      for (int w = 0; w < NW; ++w) top[j] = absmax_join<XK>(top[j], s_max[w][j * 16 + l16]);
      row_scale<XK>(top[j], sx[j], inv[j]);
    }
  } else {
    load_x(first);
    load_last();
#pragma unroll
    for (int j = 0; j < MB; ++j) sx[j] = j * 16 + l16 < p.m ? p.sx[j * 16 + l16] : 0.f;
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
          for (int i = 0; i < XC; ++i) {
            uint32_t w[W];
            chunk_to_int8<XK>(x[u][j][i], sx[j], inv[j], w);
#pragma unroll
            for (int e = 0; e < W; ++e) q[i * W + e] = w[e];
          }
        }
        // lane l: weight row (x row) l % 16, k = 16 (l / 16) + 0..15; sums of x row l % 16, weight rows 4 (l / 16) + 0..3
        acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, fb[u]), __builtin_bit_cast(i32x4, q),
                                                       acc[j], 0, 0, 0);
      }
  }
#pragma unroll
  for (int j = 0; j < MB; ++j) *(i32x4*)s_sum[wv][j][lane] = acc[j];
  __syncthreads();
  if (!last) return;
  float s = sx[0];
#pragma unroll
  for (int j = 1; j < MB; ++j) s = wv == j ? sx[j] : s;
  i32x4 sum = {0, 0, 0, 0}, up = {0, 0, 0, 0};
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    sum += *(const i32x4*)s_sum[w][wv][lane];
    if (GLU) up += *(const i32x4*)s_sum[w][wv][lane + 32];
  }
  lift_scales<1>(&s0, far_scale(s));
  if (GLU) lift_scales<1>(&s1, far_scale(s));
  s = near_scale(s);
  float v[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = v[e + 4] = fmaf((float)sum[e] * s, s0[e], b0[e]);
  activate<OK>(p.act, v);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (GLU) v[e] *= fmaf((float)up[e] * s, s1[e], b1[e]);
    v[e] += res[e];
  }
  store4<OK>(p.out + m * ((int64_t)p.n * El<OK>::B), c, p.n, v);
}

constexpr int kCUs = 256;
bool few_rows(int64_t m) { return m <= 64; }
// Whether few_rows8_kernel quantises its rows itself: each workgroup does it for all of them, which costs more than a
// launch of its own where there is much (768 to 2304 features: 1 row 4.1 us, 32 rows 7.3 against 3.5 + 3.8 in two launches, 64
// rows 10.3 against 3.6 + 4.8; 32 rows of 1152 10.2 against 3.5 + 4.2).
bool quantise_within(int64_t m, int64_t k) { return (m <= 16 ? 16 : m <= 32 ? 32 : 64) * k <= 32 * 1024; }

struct Shape {
  // 256, 192: tiles of 256 x as many, walked, where those of 256 x 256 fill the CUs. A round of 192 takes 0.78 of one of 256 at
  // short k and 0.82 at longer (integers to bf16: 51200 x 768 -> 2304 120 us by 8 rounds of 256, 124 by 10 of 192; 88064 x 768 ->
  // 1536 135 by 9, 143 by 11; 56320 x 768 -> 1152 73 by 5, 73 by 6; 56320 x 768 -> 1536 94 by 6, 91 by 7; with k = 384 the same
  // four 85 and 80, 98 and 93, 54 and 50, 67 and 61, and 88064 x 384 -> 1152 73 by 7, 76 by 9). A residual's registers leave only
  // 192. 1: 256 x 128, where those fill the CUs; 0: 128 x 64 (gated: 64 x 128)
  int tile;
  int64_t tiles_n, tiles;
};
// n: rows of the weight's tiles
Shape shape_of(int64_t m, int64_t n, int64_t k, bool glu, bool res) {
  const int64_t rt = (m + 255) / 256;
  const auto rounds = [&](int64_t tn) { return (rt * ((n + tn - 1) / tn) + kCUs - 1) / kCUs; };
  int tile = rt * ((n + 127) / 128) >= kCUs ? 1 : 0;
  if (rt * ((n + 255) / 256) >= kCUs && !(glu && res))
    tile = glu || (!res && 100 * rounds(256) <= (k > 512 ? 82 : 78) * rounds(192)) ? 256 : 192;
  const int64_t tm = tile ? 256 : glu ? 64 : 128, tn = tile > 1 ? tile : tile || glu ? 128 : 64;
  const int64_t cols = (n + tn - 1) / tn, tiles = (m + tm - 1) / tm * cols;
  return Shape{tile, cols, tiles};
}
int64_t glu_rows(int64_t n) { return (n + 31) / 32 * 64; }  // (blocks of 32 gate and 32 up rows)

template <int OK, bool GLU, int TM, int TN, int NS, int OCC>
int launch_tiles(const LinP& p, hipStream_t s) {
  launch_kernel(linear8_kernel<OK, GLU, TM, TN, 2, 2, NS, OCC>, dim3((unsigned)p.tiles), dim3(256), 0u, s, p);
  return hipGetLastError() == hipSuccess ? LIK_OK : LIK_ERR_LAUNCH;
}
template <int OK, bool GLU, bool RES>
int launch_stream(const LinP& p, int tile, hipStream_t s) {
  // Deferred stores: with a residual they change nothing (44801 x 1152 -> 768 105 us either way), its reads are what takes the time.
  constexpr int DEF = RES ? 0 : 8;
  const unsigned groups = p.tiles < kCUs ? p.tiles : kCUs;
  if constexpr (!GLU)
    if (tile == 192) {
      launch_kernel(linear8_stream_kernel<OK, GLU, RES, 192, DEF>, dim3(groups), dim3(512), 0u, s, p);
      return hipGetLastError() == hipSuccess ? LIK_OK : LIK_ERR_LAUNCH;
    }
  if constexpr (!RES)
    launch_kernel(linear8_stream_kernel<OK, GLU, RES, 256, DEF>, dim3(groups), dim3(512), 0u, s, p);
  return hipGetLastError() == hipSuccess ? LIK_OK : LIK_ERR_LAUNCH;
}
template <int OK, bool GLU>
int launch_gemm(LinP p, hipStream_t s) {
  const Shape sh = shape_of(p.m, GLU ? glu_rows(p.n) : p.n, p.k, GLU, p.res != nullptr);
  p.tiles_n = (int)sh.tiles_n;
  p.tiles = (int)sh.tiles;
  if constexpr (!GLU)
    if (sh.tile > 1 && p.res) return launch_stream<OK, GLU, true>(p, sh.tile, s);
  if (sh.tile > 1) return launch_stream<OK, GLU, false>(p, sh.tile, s);
  if (sh.tile) return launch_tiles<OK, GLU, 256, 128, 3, 2>(p, s);
  // (a wavefront has 32 columns of a 128 x 64 tile: gate and up blocks need 64)
  if constexpr (GLU) return launch_tiles<OK, GLU, 64, 128, 3, 3>(p, s);
  else return launch_tiles<OK, GLU, 128, 64, 3, 3>(p, s);
}

template <int XK, int OK, bool GLU>
int launch_few(const LinP& p, hipStream_t s) {
  const unsigned nb = GLU ? (p.n + 7) / 8 : (p.n + 15) / 16;
  if (p.m <= 16)
    launch_kernel(few_rows8_kernel<XK, OK, GLU, 1>, dim3(nb), dim3(512), 0u, s, p);
  else if (p.m <= 32)
    launch_kernel(few_rows8_kernel<XK, OK, GLU, 2>, dim3(nb), dim3(512), 0u, s, p);
  else
    launch_kernel(few_rows8_kernel<XK, OK, GLU, 4>, dim3(nb), dim3(512), 0u, s, p);
  return hipGetLastError() == hipSuccess ? LIK_OK : LIK_ERR_LAUNCH;
}

template <int OK, bool GLU>
int run(const lik_linear_int8_t* a, LinP p, char* ws, hipStream_t s) {
  const bool few = few_rows(a->rows);
  if (few && a->x_dtype != LIK_INT8 && quantise_within(a->rows, a->in)) switch (a->x_dtype) {
      case LIK_BF16: return launch_few<EK_BF16, OK, GLU>(p, s);
      case LIK_F16: return launch_few<EK_F16, OK, GLU>(p, s);
      default: return launch_few<EK_F32, OK, GLU>(p, s);
    }
  if (a->x_dtype != LIK_INT8) {
    const int64_t k16 = ((int64_t)p.k + 15) / 16 * 16;
    int8_t* x8 = (int8_t*)ws;
    ws += align256((size_t)(p.m * k16));
    float* sx = (float*)ws;
    ws += align256((size_t)p.m * 4);
    if (const int rc = quantize_rows_int8(a->x, a->x_stride, a->x_dtype, a->rows, a->in, x8, k16, sx, false, s)) return rc;
    p.a = (const char*)x8;
    p.a_ld = k16;
    p.sx = sx;
  }
  return few ? launch_few<kInt8, OK, GLU>(p, s) : launch_gemm<OK, GLU>(p, s);
}

int linear_check(const lik_linear_int8_t* a) {
  const auto is_float = [](int32_t t) { return t == LIK_BF16 || t == LIK_F16 || t == LIK_F32; };
  if (!is_float(a->out_dtype) || !(is_float(a->x_dtype) || a->x_dtype == LIK_INT8)) return LIK_ERR_UNSUPPORTED;
  if (a->rows < 0 || a->in < 1 || a->out_features < 1 || a->activation < -1 || a->activation > ACT_SILU)
    return LIK_ERR_INVALID;
  if (a->bias && a->bias_dtype != a->out_dtype && a->bias_dtype != LIK_F32) return LIK_ERR_UNSUPPORTED;
  // (131072 integers: the caller's 131071 or fewer and zeros)
  if (a->in > (a->x_dtype == LIK_INT8 ? 131072 : 131071) || a->rows > 0x7fffff00 || a->out_features > (1 << 24)) return LIK_ERR_UNSUPPORTED;
  // a launch has less than 2^32 threads; walked tiles are counted in 31 bits
  const Shape sh = shape_of(a->rows, a->gated ? glu_rows(a->out_features) : a->out_features, a->in, a->gated != 0, a->residual);
  return few_rows(a->rows) || sh.tiles < (sh.tile > 1 ? 1ll << 30 : 1ll << 24) ? LIK_OK : LIK_ERR_UNSUPPORTED;
}
// Rows quantised in a launch of their own: the integers, then the scales.
size_t linear_ws(const lik_linear_int8_t* a) {
  if (a->x_dtype == LIK_INT8 || (few_rows(a->rows) && quantise_within(a->rows, a->in))) return 0;
  return align256((size_t)(a->rows * (((int64_t)a->in + 15) / 16 * 16))) + align256((size_t)a->rows * 4) + 256;
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
  if (out == a->x || out == (const void*)a->weight) return LIK_ERR_INVALID;
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
  p.rows16 = (uintptr_t)out % 16 == 0 && (int64_t)p.n * ob % 16 == 0 && 256ll * p.n * ob < kFar;
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
