// Rotary positions, and K and V quantized into the pages of a cache and read back (gfx950).
//
// All three are bound by HBM: every value is read once and written once, and a row of D elements is
// held by CG = D/8 adjacent lanes, 8 elements (16 bytes of 16-bit values, 8 bytes of codes) each. No row
// waits for another, so there is no LDS and no loop: as many waves as a CU holds hide the latency.
// Measured (a large copy reaches 4.9 TB/s read and written): 2.3 million rotated rows of 128 fp16 values
// 203 us, 5.8 TB/s; 128 thousand rows of K and V written in 23 us, 4.4 TB/s, and read back in 19 us, 5.3
// TB/s; 262 thousand rows read in 33 us, 6.1 TB/s. The smallest calls take 3 to 5 us, the rest of their
// time is the launch.
//
// A cache page holds 64 tokens of every K/V head: K8 and V8 (pages, H, 64, D) codes, SK and SV (pages,
// H, 64) fp32. Position p of sequence b lies in page table[b][p / 64], row p % 64. A page number
// outside the pool, like a position beyond the table's row, names no page: nothing is written there
// and zeros are read.
#include "sage_device.h"
#include "sage_launch.h"

namespace sage {
namespace {

constexpr int THREADS = 256;

// The page row of position p (of one head) in rows of the pool, or -1 where there is no page.
__device__ __forceinline__ int64_t pool_row(const int* __restrict__ table, int64_t max_pages,
                                            int64_t num_pages, int64_t H, int64_t h, int64_t p) {
  if (p < 0 || p >= max_pages * NPAD) return -1;
  const int page = table[p / NPAD];
  if (page < 0 || page >= num_pages) return -1;
  return ((int64_t)page * H + h) * NPAD + p % NPAD;
}

// A thread's place in a (B, N, H) set of rows: `inner` is the dimension that adjacent rows differ in,
// the one along which the caller's rows are closer in memory.
struct Unit {
  u32 b, n, h;
};
__device__ __forceinline__ Unit unit_of(u32 u, u32 N, u32 H, bool heads_inner) {
  const u32 inner = heads_inner ? H : N, outer = heads_inner ? N : H;
  const u32 t = u / inner, i = u - t * inner, b = t / outer, o = t - b * outer;
  return {b, heads_inner ? o : i, heads_inner ? i : o};
}

// ---------------------------------------------------------------------------------------------
// Rotary positions. A pair (a, b) becomes (a c - b s, b c + a s), in fp32 with a rounding for each
// product and one for their sum (no fused multiply-add, so that the bits do not depend on the
// compiler's choice), then one to the output type where there is one.
// ---------------------------------------------------------------------------------------------
struct Rotary {
  const float* table;   // (rows, R): R/2 cosines, then R/2 sines; null: no rotation
  int64_t rows;
  const int* positions;
  int64_t p_sb;         // elements between two sequences' positions
  int R;                // rotated columns, a multiple of 16
  int interleaved;      // pairs (2i, 2i + 1), else (i, i + R/2)
  int inverse;          // by the negative angle: the transposed rotation, its gradient
};

// The cosines and sines of this lane's 8 columns. cs[e] and sn[e] belong to column 8cg + e; the sine
// carries the sign with which the pair's other column enters.
__device__ __forceinline__ void rotary_angles(const Rotary& r, int64_t b, int64_t n, int cg,
                                              float (&cs)[8], float (&sn)[8]) {
  const int col = 8 * cg, half = r.R / 2;
  const bool turned = col < r.R, pairs = r.interleaved;
  const int64_t p = r.positions[b * r.p_sb + n];
  const bool known = p >= 0 && p < r.rows;
  // adjacent pairs: 4 frequencies from col / 2 on; else 8 from col (mod R/2) on
  const int f = !turned ? 0 : pairs ? col / 2 : col < half ? col : col - half;
  const float* c = r.table + (known ? p * r.R : 0) + f;
  const float* s = c + half;
  const int next = pairs ? 0 : 4;
  const f32x4 c0 = *(const f32x4*)c, c1 = *(const f32x4*)(c + next);
  const f32x4 s0 = *(const f32x4*)s, s1 = *(const f32x4*)(s + next);
  const float flip = r.inverse ? -1.0f : 1.0f, half_sign = col < half ? -flip : flip;
  const float nan = __uint_as_float(0x7fc00000u);   // no angle is known there
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float ce = pairs ? c0[e / 2] : e < 4 ? c0[e] : c1[e - 4];
    const float se = pairs ? s0[e / 2] : e < 4 ? s0[e] : s1[e - 4];
    cs[e] = known ? ce : nan;
    sn[e] = se * (pairs ? (e & 1 ? flip : -flip) : half_sign);
  }
}

// This lane's 8 columns rotated. Every lane of the wave takes part (the half layout's pair lies in
// another lane of the row); columns behind R keep their values.
template <typename T>
__device__ __forceinline__ void rotate8(const Rotary& r, int cg, const float (&cs)[8],
                                        const float (&sn)[8], const u32x4 raw, float (&f)[8]) {
#pragma clang fp contract(off)
  float x[8], y[8];
  unpack8<T>(raw, x);
  if (r.interleaved) {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = x[e ^ 1];
  } else {
    const int lane = threadIdx.x & 63, step = r.R / 16;   // lanes of half of the rotated columns
    const int other = cg < step ? lane + step : cg < 2 * step ? lane - step : lane;
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = (u32)__shfl((int)raw[i], other, 64);
    unpack8<T>(o, y);
  }
  const bool turned = 8 * cg < r.R;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float a = x[e] * cs[e], b = y[e] * sn[e];
    f[e] = turned ? a + b : x[e];
  }
}

template <typename T>
__device__ __forceinline__ u32x4 pack8(const float (&f)[8]) {
  T h[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] = (T)f[e];
  u32x4 w;
  __builtin_memcpy(&w, h, 16);
  return w;
}

// grid: units of one token and HPT heads, CG lanes each. The angles are loaded once for the unit's
// heads; heads of a unit lie HG = ceil(H / HPT) apart, so that adjacent units are adjacent rows. Without
// it every row's fp32 angles are twice its own bytes, from L2.
template <typename T, int D, int HPT>
__global__ __launch_bounds__(THREADS) void rotary_kernel(const T* X, T* O, Rotary r,
                                                         u32 units, u32 H, u32 HG, u32 N,
                                                         int heads_inner, int64_t x_sb, int64_t x_sh,
                                                         int64_t x_sr, int64_t o_sb, int64_t o_sh,
                                                         int64_t o_sr) {
  constexpr int CG = D / 8;
  const u32 t = blockIdx.x * THREADS + threadIdx.x;
  const int cg = t % CG;
  const bool live = t / CG < units;
  const Unit u = unit_of(live ? t / CG : units - 1, N, HG, heads_inner);
  const T* x = X + u.b * x_sb + u.n * x_sr + 8 * cg;
  u32x4 raw[HPT];
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const u32 h = u.h + i * HG;
    raw[i] = *(const u32x4*)(x + (int64_t)(h < H ? h : u.h) * x_sh);
  }
  float cs[8], sn[8];
  rotary_angles(r, u.b, u.n, cg, cs, sn);
  T* o = O + u.b * o_sb + u.n * o_sr + 8 * cg;
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    float f[8];
    rotate8<T>(r, cg, cs, sn, raw[i], f);
    const u32 h = u.h + i * HG;
    if (live && h < H) *(u32x4*)(o + (int64_t)h * o_sh) = pack8<T>(f);
  }
}

// ---------------------------------------------------------------------------------------------
// Quantized rows. The scheme's row scale s = max(RN(amax / M), 1e-12), M = 127 or 448, and codes
// RN(x / s), as the prologue's (one reciprocal per row, div_by). A row that holds a NaN or an
// infinity has no scale: it is held as zero codes under a NaN scale, so that codes are never NaN and
// a masked key of such a row cannot reach the tokens that do not see it.
// ---------------------------------------------------------------------------------------------
template <int CG>
__device__ __forceinline__ u32 row_umax(u32 m) {
  m = umax(m, dpp_u32<0xB1>(m));
  m = umax(m, dpp_u32<0x4E>(m));
  m = umax(m, dpp_u32<0x141>(m));
  if (CG == 16) m = umax(m, dpp_u32<0x140>(m));
  return m;
}

template <bool INT8, int CG>
__device__ __forceinline__ float quantize8(const float (&f)[8], u32x2& codes) {
  u32 top = 0;   // |x| ordered as its bits: infinities and NaNs come out on top
#pragma unroll
  for (int e = 0; e < 8; ++e) top = umax(top, __float_as_uint(f[e]) & 0x7fffffffu);
  top = row_umax<CG>(top);
  if (top >= 0x7f800000u) {
    codes = (u32x2){0u, 0u};
    return __uint_as_float(0x7fc00000u);
  }
  const float m = INT8 ? I8_MAX : P_SCALE;
  const float s = fmaxf(div_by(__uint_as_float(top), m, INT8 ? RCP_I8_MAX : RCP_P_SCALE), SCALE_FLOOR);
  const float y = __fdiv_rn(1.0f, s);
  float q[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) q[e] = div_by(f[e], s, y);
  // |q| is at most an ulp over M, which both conversions round to M
  if (INT8)
    codes = (u32x2){i8x4(q[0], q[1], q[2], q[3]), i8x4(q[4], q[5], q[6], q[7])};
  else
    codes = (u32x2){fp8x4(q[0], q[1], q[2], q[3]), fp8x4(q[4], q[5], q[6], q[7])};
  return s;
}

// grid: one unit per row of K and V, which share the place that they go to: one look at the table for
// both, and twice the loads in flight.
template <typename T, bool KINT8, int D>
__global__ __launch_bounds__(THREADS) void cache_write_kernel(
    const T* __restrict__ K, const T* __restrict__ V, u8* __restrict__ K8, float* __restrict__ SK,
    u8* __restrict__ V8, float* __restrict__ SV, const int* __restrict__ table, int64_t t_sb,
    int64_t max_pages, int64_t num_pages, const int* __restrict__ start, const int* __restrict__ lens,
    Rotary r, u32 units, u32 H, u32 N, int heads_inner, int64_t k_sb, int64_t k_sh, int64_t k_sr,
    int64_t v_sb, int64_t v_sh, int64_t v_sr) {
  constexpr int CG = D / 8;
  const u32 t = blockIdx.x * THREADS + threadIdx.x;
  const int cg = t % CG;
  const bool live = t / CG < units;
  const Unit u = unit_of(live ? t / CG : units - 1, N, H, heads_inner);
  const u32x4 kw = *(const u32x4*)(K + u.b * k_sb + u.h * k_sh + u.n * k_sr + 8 * cg);
  const u32x4 vw = *(const u32x4*)(V + u.b * v_sb + u.h * v_sh + u.n * v_sr + 8 * cg);
  const bool given = live && (lens == nullptr || (int64_t)u.n < lens[u.b]);
  const int64_t row = given ? pool_row(table + u.b * t_sb, max_pages, num_pages, H, u.h,
                                       (int64_t)start[u.b] + u.n)
                            : -1;
  float f[8];
  if (r.table != nullptr) {
    float cs[8], sn[8];
    rotary_angles(r, u.b, u.n, cg, cs, sn);
    rotate8<T>(r, cg, cs, sn, kw, f);
  } else {
    unpack8<T>(kw, f);
  }
  u32x2 kc, vc;
  const float sk = quantize8<KINT8, CG>(f, kc);
  unpack8<T>(vw, f);
  const float sv = quantize8<false, CG>(f, vc);
  if (row < 0) return;
  *(u32x2*)(K8 + row * D + 8 * cg) = kc;
  *(u32x2*)(V8 + row * D + 8 * cg) = vc;
  if (cg == 0) {
    SK[row] = sk;
    SV[row] = sv;
  }
}

template <bool INT8>
__device__ __forceinline__ void codes8(const u32x2 w, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (INT8) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[4 * i + e] = (float)((int)(w[i] << (24 - 8 * e)) >> 24);
    } else {
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false);
      const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
      f[4 * i] = lo[0], f[4 * i + 1] = lo[1], f[4 * i + 2] = hi[0], f[4 * i + 3] = hi[1];
    }
  }
}

// grid: one unit per row of K and V, as in writing. Each value is code * scale, rounded once to T.
template <typename T, bool KINT8, int D>
__global__ __launch_bounds__(THREADS) void cache_read_kernel(
    const u8* __restrict__ K8, const float* __restrict__ SK, const u8* __restrict__ V8,
    const float* __restrict__ SV, const int* __restrict__ table, int64_t t_sb, int64_t max_pages,
    int64_t num_pages, const int* __restrict__ start, const int* __restrict__ lens,
    T* __restrict__ K, T* __restrict__ V, u32 units, u32 H, u32 N, int heads_inner, int64_t k_sb,
    int64_t k_sh, int64_t k_sr, int64_t v_sb, int64_t v_sh, int64_t v_sr) {
  constexpr int CG = D / 8;
  const u32 t = blockIdx.x * THREADS + threadIdx.x;
  const int cg = t % CG;
  if (t / CG >= units) return;
  const Unit u = unit_of(t / CG, N, H, heads_inner);
  const int64_t p = (int64_t)(start ? start[u.b] : 0) + u.n;
  const int64_t row = (int64_t)u.n < lens[u.b]
                          ? pool_row(table + u.b * t_sb, max_pages, num_pages, H, u.h, p)
                          : -1;
  float k[8] = {}, v[8] = {};
  if (row >= 0) {
    const u32x2 kc = *(const u32x2*)(K8 + row * D + 8 * cg), vc = *(const u32x2*)(V8 + row * D + 8 * cg);
    const float sk = SK[row], sv = SV[row];
    codes8<KINT8>(kc, k);
    codes8<false>(vc, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) k[e] *= sk, v[e] *= sv;
  }
  *(u32x4*)(K + u.b * k_sb + u.h * k_sh + u.n * k_sr + 8 * cg) = pack8<T>(k);
  *(u32x4*)(V + u.b * v_sb + u.h * v_sh + u.n * v_sr + 8 * cg) = pack8<T>(v);
}

u32 blocks_for(int64_t units, int64_t D) {
  return (u32)((units * (D / 8) + THREADS - 1) / THREADS);
}

Rotary rotary_of(const RotaryArgs& a) {
  Rotary r;
  r.table = a.table;
  r.rows = a.rows;
  r.positions = a.positions;
  r.p_sb = a.p_sb;
  r.R = (int)a.R;
  r.interleaved = a.interleaved;
  r.inverse = a.inverse;
  return r;
}

// One head a thread while the rows do not fill the card (32768 rows of 128 are 2048 blocks), else four:
// 16384 rows 5.5 us by one, 6.8 by four; 32768 rows 7.3 and 6.7; 2.3 million 266 and 207 (two: 221, eight:
// 219).
template <typename T, int D>
hipError_t rotary_d(const RotaryArgs& a, hipStream_t st) {
  constexpr int HPT = 4;
  const int inner = a.x_sh < a.x_sr;
  const Rotary r = rotary_of(a);
  const int64_t rows = a.B * a.N * a.H;
  if (rows < (int64_t)1 << 15) {
    rotary_kernel<T, D, 1><<<blocks_for(rows, D), THREADS, 0, st>>>(
        (const T*)a.x, (T*)a.o, r, (u32)rows, (u32)a.H, (u32)a.H, (u32)a.N, inner, a.x_sb, a.x_sh,
        a.x_sr, a.o_sb, a.o_sh, a.o_sr);
  } else {
    const int64_t HG = (a.H + HPT - 1) / HPT, units = a.B * a.N * HG;
    rotary_kernel<T, D, HPT><<<blocks_for(units, D), THREADS, 0, st>>>(
        (const T*)a.x, (T*)a.o, r, (u32)units, (u32)a.H, (u32)HG, (u32)a.N, inner, a.x_sb, a.x_sh,
        a.x_sr, a.o_sb, a.o_sh, a.o_sr);
  }
  return hipGetLastError();
}

template <typename T, bool KINT8, int D>
hipError_t write_d(const CacheRowsArgs& a, hipStream_t st) {
  const int64_t units = a.B * a.N * a.H;
  cache_write_kernel<T, KINT8, D><<<blocks_for(units, D), THREADS, 0, st>>>(
      (const T*)a.k, (const T*)a.v, (u8*)a.pool.k8, a.pool.sk, (u8*)a.pool.v8, a.pool.sv, a.pool.table,
      a.pool.t_sb, a.pool.max_pages, a.pool.num_pages, a.start, a.lens, rotary_of(a.rotary), (u32)units,
      (u32)a.H, (u32)a.N, a.k_sh < a.k_sr, a.k_sb, a.k_sh, a.k_sr, a.v_sb, a.v_sh, a.v_sr);
  return hipGetLastError();
}

template <typename T, bool KINT8, int D>
hipError_t read_d(const CacheRowsArgs& a, hipStream_t st) {
  const int64_t units = a.B * a.N * a.H;
  cache_read_kernel<T, KINT8, D><<<blocks_for(units, D), THREADS, 0, st>>>(
      (const u8*)a.pool.k8, a.pool.sk, (const u8*)a.pool.v8, a.pool.sv, a.pool.table, a.pool.t_sb,
      a.pool.max_pages, a.pool.num_pages, a.start, a.lens, (T*)a.k, (T*)a.v, (u32)units, (u32)a.H,
      (u32)a.N, a.k_sh < a.k_sr, a.k_sb, a.k_sh, a.k_sr, a.v_sb, a.v_sh, a.v_sr);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_rotary(const RotaryArgs& a, hipStream_t st) {
  if (a.dtype == 0) return a.D == 128 ? rotary_d<f16, 128>(a, st) : rotary_d<f16, 64>(a, st);
  return a.D == 128 ? rotary_d<bf16, 128>(a, st) : rotary_d<bf16, 64>(a, st);
}

hipError_t launch_cache_write(const CacheRowsArgs& a, hipStream_t st) {
  if (a.dtype == 1) return a.D == 128 ? write_d<bf16, false, 128>(a, st) : write_d<bf16, false, 64>(a, st);
  if (a.pool.k_int8) return a.D == 128 ? write_d<f16, true, 128>(a, st) : write_d<f16, true, 64>(a, st);
  return a.D == 128 ? write_d<f16, false, 128>(a, st) : write_d<f16, false, 64>(a, st);
}

hipError_t launch_cache_read(const CacheRowsArgs& a, hipStream_t st) {
  if (a.dtype == 1) return a.D == 128 ? read_d<bf16, false, 128>(a, st) : read_d<bf16, false, 64>(a, st);
  if (a.pool.k_int8) return a.D == 128 ? read_d<f16, true, 128>(a, st) : read_d<f16, true, 64>(a, st);
  return a.D == 128 ? read_d<f16, false, 128>(a, st) : read_d<f16, false, 64>(a, st);
}

}  // namespace sage
