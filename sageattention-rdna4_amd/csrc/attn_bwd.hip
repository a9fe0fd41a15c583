// Attention's backward pass (gfx950): the gradients of Q, K and V from that of the output, with the
// probabilities recomputed from the kept logsumexp.
//
// For a query row i, its keys j, c = sm_scale log2 e and d_i = dout_i . out_i - dlse_i:
//     P_ij = 2^(c q_i.k_j - lse_i log2 e),      dV_j = sum_i P_ij dout_i,
//     dS_ij = P_ij (dout_i.v_j - d_i),          dQ_i = sm_scale sum_j dS_ij k_j,
//                                               dK_j = sm_scale sum_i dS_ij q_i.
// A row whose logsumexp is -infinity saw nothing: its P are zeros.
//
// Three launches at most. `rows` works out each row's -lse log2 e and -d. `main` holds blocks of two
// kinds: one owns keys and goes over the queries that see them (S, dP, dV, dK), the other owns queries
// and goes over their keys (S, dP, dQ). Seven products, where one kind of block that adds its dQ
// to memory would take five: but added atomically, in an order that changes from call to call, and
// with 4 bytes read and written per pair of query and key in fp32. Where there are too few blocks for
// the card each one's loop is cut into parts, whose fp32 sums `join` adds in order. So results are the
// same from call to call.
//
// Layout. A wave owns 32 T columns (keys, or queries) of 16-bit operands in registers and multiplies
// them with 32 rows of the other side at a time by 32x32x16 MFMAs. The result has a column per lane,
// its rows in the lane's registers: converted to 16 bits it is, lane for lane, the operand of the second
// product when that takes its inner index in the order {16t + 4g + 0..3, 16t + 8 + 4g + 0..3} (g the
// lane's half). So P and dS never leave their lanes. The other operand is read from the same
// LDS tile, transposed (ds_read_b64_tr_b16: 16 lanes exchange a 4 x 16 block).
#include "attn_common.h"
#include "sage_launch.h"

namespace sage {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Vec;
template <>
struct Vec<f16> {
  typedef f16x8 x8;
  typedef f16x4 x4;
};
template <>
struct Vec<bf16> {
  typedef bf16x8 x8;
  typedef bf16x4 x4;
};

__device__ __forceinline__ f32x16 mfma16(const f16x8 a, const f16x8 b, const f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma16(const bf16x8 a, const bf16x8 b, const f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

typedef __fp16 fp16x4 __attribute__((ext_vector_type(4)));   // the builtin's name for four halves
typedef __attribute__((address_space(3))) fp16x4 lds_f16x4;
typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;
__device__ __forceinline__ f16x4 read_tr(const f16* p) {
  return __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_f16x4*)p));
}
__device__ __forceinline__ bf16x4 read_tr(const bf16* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)p);
}

constexpr int BT = 64;                 // rows of the other side in an LDS tile
constexpr float NEG_INF = -__builtin_inff();
// fp16 operands: P is held times 2^12, so that it is a normal number from 2^-26 up and may pass 1 by a
// factor of 15 (a logsumexp of quantized scores is off by some hundredths), dS times a power of two
// that brings its bound into [2^13, 2^14).
template <typename T>
constexpr float P_SHIFT = std::is_same_v<T, f16> ? 12.0f : 0.0f;

// The 16-byte chunk of a tile's row r that lies at position c ^ swz(r). A row read takes 16 rows'
// (or 8 rows' two) chunks in a pass, a transposed read 4 rows' 64 bytes: both touch each bank once.
template <int D>
__device__ __forceinline__ int swz(int r) {
  return D == 128 ? ((r & 3) << 2) | (((r >> 2) & 1) << 1) | ((r >> 3) & 1)
                  : (((r >> 1) & 1) << 2) | (((r >> 2) & 1) << 1) | ((r >> 3) & 1);
}

struct Rows {                          // a (B, H, N, D) view
  const void* p;
  int64_t sb, sh, sr;
};
struct Out {
  void* p;
  int64_t sb, sh, sr;
};
struct Args {
  Rows q, k, v, o, dout;
  Out dq, dk, dv;
  const float* lse;
  const float* dlse;
  int H, H_kv, G, N, N_kv, NP;         // NP: N rounded up to tiles
  int planes_q, planes_kv, nb_q, nb_kv; // planes; tiles of 64 rows in each
  int k_tiles, q_tiles, k_split, q_split, k_blocks;
  float sm_scale, c;
  // workspace
  float* nl;        // (planes_q, NP): P_SHIFT - lse log2 e
  float* nd;        // (planes_q, NP): -d
  float* max_do;    // fp16: (planes_q, nb_q): a tile's largest |dout|^2, |d|, and (planes_kv, nb_kv) |v|^2
  float* max_d;
  float* max_v;
  float* part_k;    // (k_split, planes_kv, k_tiles KB, D) sums of dK, of dV, where k_split > 1
  float* part_v;
  float* part_q;    // (q_split, planes_q, q_tiles QB, D)
};

template <typename T>
__device__ __forceinline__ const T* plane(const Rows& x, int b, int h) {
  return (const T*)x.p + (int64_t)b * x.sb + (int64_t)h * x.sh;
}

// ------------------------------------------------------------------------------------- rows
// 64 rows of a plane per block, D / 8 lanes to a row.
template <typename T, int D>
__global__ void __launch_bounds__(256) rows_kernel(const Args a) {
  constexpr int CG = D / 8, R = 64 / CG, IT = 16 / R;
  constexpr bool F16 = std::is_same_v<T, f16>;
  __shared__ float best[8];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int cg = lane % CG, rg = lane / CG;
  const int blocks_q = a.planes_q * a.nb_q;
  const int blk = blockIdx.x;
  const bool of_v = blk >= blocks_q;
  const int at = of_v ? blk - blocks_q : blk;
  const int nb = of_v ? a.nb_kv : a.nb_q, n_rows = of_v ? a.N_kv : a.N;
  const int p = at / nb, r0 = (at - p * nb) * 64 + 16 * w;
  const int heads = of_v ? a.H_kv : a.H;
  const int b = p / heads, h = p - b * heads;
  float top0 = 0.0f, top1 = 0.0f;
  u32x4 x[IT], y[IT];
  const Rows& first = of_v ? a.v : a.dout;
  const T* px = plane<T>(first, b, h) + 8 * cg;
  const T* py = plane<T>(a.o, of_v ? 0 : b, of_v ? 0 : h) + 8 * cg;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int r = min(r0 + i * R + rg, n_rows - 1);
    x[i] = *(const u32x4*)(px + (int64_t)r * first.sr);
    y[i] = x[i];
    if (!of_v) y[i] = *(const u32x4*)(py + (int64_t)r * a.o.sr);
  }
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int r = r0 + i * R + rg;
    float fx[8], fy[8], dot = 0.0f, sq = 0.0f;
    unpack8<T>(x[i], fx);
    unpack8<T>(y[i], fy);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      dot = __builtin_fmaf(fx[e], fy[e], dot);
      if (F16) sq = __builtin_fmaf(fx[e], fx[e], sq);
    }
#pragma unroll
    for (int m = 1; m < CG; m <<= 1) {
      dot += __shfl_xor(dot, m, 64);
      if (F16) sq += __shfl_xor(sq, m, 64);
    }
    if (!of_v) {
      float nl = NEG_INF, nd = 0.0f;
      if (r < n_rows) {
        const int64_t row = (int64_t)p * a.N + r;
        const float l = a.lse[row];
        nl = l == NEG_INF ? NEG_INF : __builtin_fmaf(-LOG2E_F, l, P_SHIFT<T>);
        nd = (a.dlse ? a.dlse[row] : 0.0f) - dot;
      }
      if (cg == 0) {
        a.nl[(int64_t)p * a.NP + r] = nl;
        a.nd[(int64_t)p * a.NP + r] = nd;
      }
      top1 = fmaxf(top1, fabsf(nd));
    }
    if (r < n_rows) top0 = fmaxf(top0, sq);
  }
  if (F16) {
#pragma unroll
    for (int m = CG; m < 64; m <<= 1) {
      top0 = fmaxf(top0, __shfl_xor(top0, m, 64));
      top1 = fmaxf(top1, __shfl_xor(top1, m, 64));
    }
    if (lane == 0) {
      best[w] = top0;
      best[4 + w] = top1;
    }
    __syncthreads();
    if (tid == 0) {
      top0 = fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3]));
      top1 = fmaxf(fmaxf(best[4], best[5]), fmaxf(best[6], best[7]));
      if (of_v) {
        a.max_v[at] = top0;
      } else {
        a.max_do[at] = top0;
        a.max_d[at] = top1;
      }
    }
  }
}

// ------------------------------------------------------------------------------------- main
// The largest of n values, by a block of 256 threads; NaNs are passed over.
__device__ __forceinline__ float block_max(const float* p, int n, float* lds) {
  float m = 0.0f;
  for (int i = threadIdx.x; i < n; i += 256) m = fmaxf(m, p[i]);
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) m = fmaxf(m, __shfl_xor(m, s, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = m;
  __syncthreads();
  return fmaxf(fmaxf(lds[0], lds[1]), fmaxf(lds[2], lds[3]));
}

// The power of two that brings `bound` into [2^13, 2^14) (an infinite or vanishing one: as far as
// exponents of 100 go).
__device__ __forceinline__ float scale_for(float bound) {
  int e = 0;
  if (bound > 0.0f) {
    (void)frexpf(fminf(bound, 1e30f), &e);
    e = 14 - e;
  }
  return ldexpf(1.0f, min(max(e, -100), 100));
}

// LDS of a block: two tiles of each of two tensors, and of the rows' two constants.
template <int D>
constexpr int LDS_BYTES = 4 * BT * D * 2 + 2 * 2 * BT * 4;

// One tile of BT rows of x from row r0 on into LDS, a quarter by each wave; rows from `n` on are row
// n - 1 again (what they would add is multiplied by P = 0).
template <typename T, int D>
__device__ __forceinline__ void stage(const T* x, int64_t sr, int r0, int n, uint32_t lds, int w,
                                      int lane) {
  constexpr int CPR = D / 8, RPI = 64 / CPR, IT = 16 / RPI;
  const T* base = x + (int64_t)r0 * sr;
  const int last = n - 1 - r0;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int r = 16 * w + RPI * i + lane / CPR, c = (lane % CPR) ^ swz<D>(r);
    dma16(base, (uint32_t)(min(r, last) * (int)(2 * sr) + 16 * c),
          lds + (16 * w + RPI * i) * D * 2);
  }
}

// Offsets, in elements, of a lane's operands within a tile.
template <int D>
struct Offsets {
  int row[D / 16];       // rows lane % 32: chunk 2s + g
  int tr[D / 32][2];     // transposed: 4 rows from 4g (+ 8) on, columns 32 dt .. + 31
  __device__ __forceinline__ Offsets(int lane) {
    const int r = lane & 31, g = lane >> 5, l16 = lane & 15, j = (lane >> 4) & 1;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) row[s] = r * D + 8 * ((2 * s + g) ^ swz<D>(r));
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int hi = 0; hi < 2; ++hi) {
        const int rr = 4 * g + (l16 >> 2) + 8 * hi;
        tr[dt][hi] = rr * D + 8 * ((4 * dt + 2 * j + ((l16 & 3) >> 1)) ^ swz<D>(rr)) + 4 * (l16 & 1);
      }
  }
};

// The transposed operand of 16 rows (from `tile` on) and columns 32 dt .. + 31.
template <typename T, int D>
__device__ __forceinline__ typename Vec<T>::x8 transposed(const T* tile, const Offsets<D>& of, int dt) {
  const auto lo = read_tr(tile + of.tr[dt][0]), hi = read_tr(tile + of.tr[dt][1]);
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// A wave's 32 KT columns of x (rows of memory from r0 on; from n on row n - 1 again) as operands.
template <typename T, int D, int KT>
__device__ __forceinline__ void load_columns(const T* x, int64_t sr, int r0, int n, int lane,
                                             typename Vec<T>::x8 (&f)[KT][D / 16]) {
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    const T* p = x + (int64_t)min(r0 + 32 * kt + (lane & 31), n - 1) * sr + 8 * (lane >> 5);
#pragma unroll
    for (int s = 0; s < D / 16; ++s) f[kt][s] = *(const typename Vec<T>::x8*)(p + 16 * s);
  }
}

// A wave's sums, columns of D values each, times f, into rows from r0 on of a 16-bit view or of fp32
// parts.
template <typename T, int D, int KT>
__device__ __forceinline__ void store_columns(const f32x16 (&acc)[KT][D / 32], const float (&f)[KT],
                                              const Out& o, int b, int h, float* part, int r0, int n,
                                              int lane) {
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) keep_live(acc[kt][dt]);
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    const int r = r0 + 32 * kt + (lane & 31);
    if (r >= n) continue;
    const int col = 4 * (lane >> 5);
    if (part) {
      float* p = part + (int64_t)r * D + col;
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f32x4 x;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = acc[kt][dt][4 * i + e] * f[kt];
          *(f32x4*)(p + 32 * dt + 8 * i) = x;
        }
    } else {
      T* p = (T*)o.p + (int64_t)b * o.sb + (int64_t)h * o.sh + (int64_t)r * o.sr + col;
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          typename Vec<T>::x4 x;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = (T)(acc[kt][dt][4 * i + e] * f[kt]);
          *(typename Vec<T>::x4*)(p + 32 * dt + 8 * i) = x;
        }
    }
  }
}

template <int N>
__device__ __forceinline__ void clear(f32x16 (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) x[i][r] = 0.0f;
}

// A block that owns 128 KT keys of a K/V head.
template <typename T, int D, int KT, bool CAUSAL>
__device__ __forceinline__ void keys_block(const Args& a, u8* smem, int block) {
  constexpr int KB = 128 * KT, TILE = BT * D;
  constexpr bool F16 = std::is_same_v<T, f16>;
  typedef typename Vec<T>::x8 x8;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 5;
  const int pl = block % a.planes_kv, ts = block / a.planes_kv;
  const int tile = ts / a.k_split, sp = ts - tile * a.k_split;
  const int b = pl / a.H_kv, hk = pl - b * a.H_kv;
  const int k0 = tile * KB, kw = k0 + 32 * KT * w;
  // iterations: tiles of queries, head after head of the group
  const int first = CAUSAL ? k0 / BT : 0, per = a.nb_q - first;
  const int n = per * a.G;
  const int it0 = (int)((int64_t)n * sp / a.k_split), it1 = (int)((int64_t)n * (sp + 1) / a.k_split);

  float scale = 1.0f;
  if (F16) {
    const int hq = b * a.H + hk * a.G;
    const float mo = block_max(a.max_do + (int64_t)hq * a.nb_q, a.G * a.nb_q, (float*)smem);
    const float md = block_max(a.max_d + (int64_t)hq * a.nb_q, a.G * a.nb_q, (float*)smem);
    const float mv = block_max(a.max_v + (int64_t)pl * a.nb_kv, a.nb_kv, (float*)smem);
    scale = scale_for(sqrtf(mo) * sqrtf(mv) + md);
    __syncthreads();
  }
  const float fs = scale * __builtin_ldexpf(1.0f, -(int)P_SHIFT<T>);

  T* lds = (T*)smem;
  float* lds_rows = (float*)(lds + 4 * TILE);
  const uint32_t lds0 = lds_addr(smem);
  int gi = it0 / per, ti = first + it0 - gi * per;   // of the next tile to be requested
  auto request = [&](int buf) {
    const int h = hk * a.G + gi, q0 = ti * BT;
    stage<T, D>(plane<T>(a.q, b, h), a.q.sr, q0, a.N, lds0 + buf * TILE * 2, w, lane);
    stage<T, D>(plane<T>(a.dout, b, h), a.dout.sr, q0, a.N, lds0 + (2 + buf) * TILE * 2, w, lane);
    const int64_t row = (int64_t)(b * a.H + h) * a.NP + q0;
    if (w < 2)
      dma4((w ? a.nd : a.nl) + row, 4 * lane, lds0 + 8 * TILE + (2 * buf + w) * BT * 4);
    if (++ti == a.nb_q) {
      ti = first;
      ++gi;
    }
  };

  const Offsets<D> of(lane);
  x8 kf[KT][D / 16], vf[KT][D / 16];
  load_columns<T, D, KT>(plane<T>(a.k, b, hk), a.k.sr, kw, a.N_kv, lane, kf);
  load_columns<T, D, KT>(plane<T>(a.v, b, hk), a.v.sr, kw, a.N_kv, lane, vf);
  f32x16 dk[KT][D / 32], dv[KT][D / 32];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    clear(dk[kt]);
    clear(dv[kt]);
  }
  int tc = ti;                                       // the tile at hand
  if (it0 < it1) request(0);
  int buf = 0;
  for (int it = it0; it < it1; ++it) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const int q0 = tc * BT;
    tc = ti;
    if (it + 1 < it1) request(buf ^ 1);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int qu = q0 + 32 * u;
      if (CAUSAL && qu + 31 < kw) continue;
      const T* tq = lds + buf * TILE + 32 * u * D;
      const T* to = tq + 2 * TILE;
      const float* rows = lds_rows + 2 * buf * BT + 32 * u + 4 * g;
      f32x16 nl, nd;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 x = *(const f32x4*)(rows + 8 * i), y = *(const f32x4*)(rows + BT + 8 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          nl[4 * i + e] = x[e];
          nd[4 * i + e] = y[e];
        }
      }
      f32x16 s[KT], dp[KT];
      clear(s);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) dp[kt] = nd;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const x8 x = *(const x8*)(tq + of.row[i]);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) s[kt] = mfma16(x, kf[kt][i], s[kt]);
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const x8 x = *(const x8*)(to + of.row[i]);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) dp[kt] = mfma16(x, vf[kt][i], dp[kt]);
      }
      x8 pf[KT][2], df[KT][2];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        const int key = kw + 32 * kt + (lane & 31);
        const bool diagonal = CAUSAL && qu < kw + 32 * kt + 31;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][r], a.c, nl[r]));
          if (diagonal && qu + 8 * (r / 4) + 4 * g + r % 4 < key) p = 0.0f;
          pf[kt][r / 8][r % 8] = (T)p;
          if (F16) p *= fs;
          df[kt][r / 8][r % 8] = (T)(p * dp[kt][r]);
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) {
          const x8 x = transposed<T, D>(to + 16 * t * D, of, dt);
          const x8 y = transposed<T, D>(tq + 16 * t * D, of, dt);
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) {
            dv[kt][dt] = mfma16(x, pf[kt][t], dv[kt][dt]);
            dk[kt][dt] = mfma16(y, df[kt][t], dk[kt][dt]);
          }
        }
    }
    buf ^= 1;
  }
  float fk[KT], fv[KT];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    fk[kt] = a.sm_scale / scale;
    fv[kt] = __builtin_ldexpf(1.0f, -(int)P_SHIFT<T>);
  }
  const int64_t part = ((int64_t)sp * a.planes_kv + pl) * a.k_tiles * KB * D;
  store_columns<T, D, KT>(dk, fk, a.dk, b, hk, a.k_split > 1 ? a.part_k + part : nullptr, kw, a.N_kv, lane);
  store_columns<T, D, KT>(dv, fv, a.dv, b, hk, a.k_split > 1 ? a.part_v + part : nullptr, kw, a.N_kv, lane);
}

// A block that owns 128 QT queries of a head.
template <typename T, int D, int QT, bool CAUSAL>
__device__ __forceinline__ void queries_block(const Args& a, u8* smem, int block) {
  constexpr int QB = 128 * QT, TILE = BT * D;
  constexpr bool F16 = std::is_same_v<T, f16>;
  typedef typename Vec<T>::x8 x8;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 5;
  const int pl = block % a.planes_q, ts = block / a.planes_q;
  // the longest tiles, the last of a causal plane, begin first
  const int tile = a.q_tiles - 1 - ts / a.q_split, sp = ts % a.q_split;
  const int b = pl / a.H, h = pl - b * a.H, hk = h / a.G;
  const int q0 = tile * QB, qw = q0 + 32 * QT * w;
  const int n = CAUSAL ? min((q0 + QB + BT - 1) / BT, a.nb_kv) : a.nb_kv;
  const int it0 = (int)((int64_t)n * sp / a.q_split), it1 = (int)((int64_t)n * (sp + 1) / a.q_split);

  float mv = 0.0f;
  if (F16) {
    mv = sqrtf(block_max(a.max_v + (int64_t)(b * a.H_kv + hk) * a.nb_kv, a.nb_kv, (float*)smem));
    __syncthreads();
  }
  T* lds = (T*)smem;
  const uint32_t lds0 = lds_addr(smem);
  const T* pk = plane<T>(a.k, b, hk);
  const T* pv = plane<T>(a.v, b, hk);
  auto request = [&](int it, int buf) {
    stage<T, D>(pk, a.k.sr, it * BT, a.N_kv, lds0 + buf * TILE * 2, w, lane);
    stage<T, D>(pv, a.v.sr, it * BT, a.N_kv, lds0 + (2 + buf) * TILE * 2, w, lane);
  };

  const Offsets<D> of(lane);
  x8 qf[QT][D / 16], of_do[QT][D / 16];
  load_columns<T, D, QT>(plane<T>(a.q, b, h), a.q.sr, qw, a.N, lane, qf);
  load_columns<T, D, QT>(plane<T>(a.dout, b, h), a.dout.sr, qw, a.N, lane, of_do);
  float nl[QT], nd[QT], fs[QT], fq[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int64_t row = (int64_t)pl * a.NP + min(qw + 32 * qt + (lane & 31), a.NP - 1);
    nl[qt] = a.nl[row];
    nd[qt] = a.nd[row];
    float scale = 1.0f;
    if (F16) {
      float sq = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = (float)of_do[qt][i][e];
          sq = __builtin_fmaf(x, x, sq);
        }
      sq += __shfl_xor(sq, 32, 64);
      scale = scale_for(sqrtf(sq) * mv + fabsf(nd[qt]));
    }
    fs[qt] = scale * __builtin_ldexpf(1.0f, -(int)P_SHIFT<T>);
    fq[qt] = a.sm_scale / scale;
  }
  f32x16 dq[QT][D / 32];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) clear(dq[qt]);
  if (it0 < it1) request(it0, 0);
  int buf = 0;
  for (int it = it0; it < it1; ++it) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const int k0 = it * BT;
    if (it + 1 < it1) request(it + 1, buf ^ 1);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int ku = k0 + 32 * u;
      if (ku >= a.N_kv || (CAUSAL && ku > qw + 32 * QT - 1)) continue;
      const T* tk = lds + buf * TILE + 32 * u * D;
      const T* tv = tk + 2 * TILE;
      f32x16 s[QT], dp[QT];
      clear(s);
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
#pragma unroll
        for (int r = 0; r < 16; ++r) dp[qt][r] = nd[qt];
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const x8 x = *(const x8*)(tk + of.row[i]);
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) s[qt] = mfma16(x, qf[qt][i], s[qt]);
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const x8 x = *(const x8*)(tv + of.row[i]);
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) dp[qt] = mfma16(x, of_do[qt][i], dp[qt]);
      }
      x8 df[QT][2];
      const bool ragged = ku + 32 > a.N_kv;
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        const int query = qw + 32 * qt + (lane & 31);
        const bool diagonal = CAUSAL && ku + 31 > qw + 32 * qt;
        const int end = CAUSAL ? min(query + 1, a.N_kv) : a.N_kv;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[qt][r], a.c, nl[qt]));
          if ((ragged || diagonal) && ku + 8 * (r / 4) + 4 * g + r % 4 >= end) p = 0.0f;
          if (F16) p *= fs[qt];
          df[qt][r / 8][r % 8] = (T)(p * dp[qt][r]);
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) {
          const x8 x = transposed<T, D>(tk + 16 * t * D, of, dt);
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) dq[qt][dt] = mfma16(x, df[qt][t], dq[qt][dt]);
        }
    }
    buf ^= 1;
  }
  const int64_t part = ((int64_t)sp * a.planes_q + pl) * a.q_tiles * QB * D;
  store_columns<T, D, QT>(dq, fq, a.dq, b, h, a.q_split > 1 ? a.part_q + part : nullptr, qw, a.N, lane);
}


template <typename T, int D, int KT, bool CAUSAL>
__global__ void __launch_bounds__(256, 3 - KT) main_kernel(const Args a) {
  __shared__ __align__(16) u8 smem[LDS_BYTES<D>];
  if ((int)blockIdx.x < a.k_blocks)
    keys_block<T, D, KT, CAUSAL>(a, smem, blockIdx.x);
  else
    queries_block<T, D, KT, CAUSAL>(a, smem, blockIdx.x - a.k_blocks);
}

// ------------------------------------------------------------------------------------- join
// The parts' sums added in order, eight values a thread: dK and dV where K's loops are cut, then dQ.
struct JoinArgs {
  const float* part[3];
  Out out[3];
  int heads[3], planes[3], rows[3], padded[3], split[3];
  int64_t begin[4];                    // threads ahead of each tensor's
};
template <typename T, int D>
__global__ void __launch_bounds__(256) join_kernel(const JoinArgs a) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= a.begin[3]) return;
  const int x = id >= a.begin[2] ? 2 : id >= a.begin[1] ? 1 : 0;
  const int64_t row = (id - a.begin[x]) / (D / 8);
  const int col = (int)((id - a.begin[x]) % (D / 8)) * 8;
  const int pl = (int)(row / a.rows[x]), r = (int)(row % a.rows[x]);
  const int64_t step = (int64_t)a.planes[x] * a.padded[x] * D;
  const float* p = a.part[x] + ((int64_t)pl * a.padded[x] + r) * D + col;
  f32x4 lo = *(const f32x4*)p, hi = *(const f32x4*)(p + 4);
  for (int s = 1; s < a.split[x]; ++s) {
    p += step;
    lo += *(const f32x4*)p;
    hi += *(const f32x4*)(p + 4);
  }
  typename Vec<T>::x8 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    y[e] = (T)lo[e];
    y[4 + e] = (T)hi[e];
  }
  const int b = pl / a.heads[x], h = pl % a.heads[x];
  *(typename Vec<T>::x8*)((T*)a.out[x].p + (int64_t)b * a.out[x].sb + (int64_t)h * a.out[x].sh +
                          (int64_t)r * a.out[x].sr + col) = y;
}

template <typename T, int D, int KT>
void launch_main(const Args& a, bool causal, int blocks, hipStream_t s) {
  if (causal)
    hipLaunchKernelGGL((main_kernel<T, D, KT, true>), dim3(blocks), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((main_kernel<T, D, KT, false>), dim3(blocks), dim3(256), 0, s, a);
}

template <typename T, int D>
hipError_t launch(const AttnBwdArgs& x, const AttnBwdPlan& p, const Args& a, hipStream_t s) {
  const int rows = a.planes_q * a.nb_q + (x.dtype == 0 ? a.planes_kv * a.nb_kv : 0);
  hipLaunchKernelGGL((rows_kernel<T, D>), dim3(rows), dim3(256), 0, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  launch_main<T, D, 1>(a, x.causal, (int)(p.k_blocks + p.q_blocks), s);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  JoinArgs j = {};
  j.part[0] = a.part_k;
  j.part[1] = a.part_v;
  j.part[2] = a.part_q;
  j.out[0] = a.dk;
  j.out[1] = a.dv;
  j.out[2] = a.dq;
  int64_t at = 0;
  for (int i = 0; i < 3; ++i) {
    const bool q = i == 2;
    j.heads[i] = q ? a.H : a.H_kv;
    j.planes[i] = q ? a.planes_q : a.planes_kv;
    j.rows[i] = q ? a.N : a.N_kv;
    j.padded[i] = (int)(q ? p.q_tiles * p.q_rows : p.k_tiles * p.k_rows);
    j.split[i] = (int)(q ? p.q_split : p.k_split);
    j.begin[i] = at;
    if (j.split[i] > 1) at += (int64_t)j.planes[i] * j.rows[i] * (D / 8);
  }
  j.begin[3] = at;
  if (at == 0) return hipSuccess;
  hipLaunchKernelGGL((join_kernel<T, D>), dim3((unsigned)((at + 255) / 256)), dim3(256), 0, s, j);
  return hipGetLastError();
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The workspace's parts, each from a multiple of 256 bytes on.
struct Offsets64 {
  int64_t nl, nd, max_do, max_d, max_v, part_k, part_v, part_q, end;
};
Offsets64 offsets(const AttnBwdPlan& p, int dtype, int64_t planes_q, int64_t planes_kv, int64_t D) {
  Offsets64 o;
  int64_t at = 0;
  auto take = [&](int64_t floats) {
    const int64_t was = at;
    at += (floats * 4 + 255) / 256 * 256;
    return was;
  };
  const bool f16 = dtype == 0;
  o.nl = take(planes_q * p.nb_q * BT);
  o.nd = take(planes_q * p.nb_q * BT);
  o.max_do = take(f16 ? planes_q * p.nb_q : 0);
  o.max_d = take(f16 ? planes_q * p.nb_q : 0);
  o.max_v = take(f16 ? planes_kv * p.nb_kv : 0);
  const int64_t k = p.k_split > 1 ? p.k_split * planes_kv * p.k_tiles * p.k_rows * D : 0;
  o.part_k = take(k);
  o.part_v = take(k);
  o.part_q = take(p.q_split > 1 ? p.q_split * planes_q * p.q_tiles * p.q_rows * D : 0);
  o.end = at;
  return o;
}

}  // namespace

AttnBwdPlan attn_bwd_plan(int64_t B, int64_t H, int64_t H_kv, int64_t N, int64_t N_kv, int64_t D,
                          bool causal) {
  AttnBwdPlan p;
  p.nb_q = ceil_div(N, BT);
  p.nb_kv = ceil_div(N_kv, BT);
  p.k_rows = p.q_rows = 128;
  p.k_tiles = ceil_div(N_kv, p.k_rows);
  p.q_tiles = ceil_div(N, p.q_rows);
  // As many parts as bring each block's steps (four products over a tile for keys, three for queries)
  // down to its share of what the card runs at once, of 4 tiles or more.
  const int64_t steps_k = p.nb_q * (H / H_kv), steps_q = p.nb_kv;
  const int64_t work = B * H_kv * p.k_tiles * steps_k * 4 + B * H * p.q_tiles * steps_q * 3;
  const int64_t share = ceil_div(work, causal ? 1024 : 512);
  auto parts = [&](int64_t steps, int64_t cost) {
    int64_t n = steps * cost / (share < 1 ? 1 : share);
    if (n > steps / 4) n = steps / 4;
    return n < 1 ? 1 : n > 64 ? 64 : n;
  };
  p.k_split = parts(steps_k, 4);
  p.q_split = parts(steps_q, 3);
  p.k_blocks = B * H_kv * p.k_tiles * p.k_split;
  p.q_blocks = B * H * p.q_tiles * p.q_split;
  return p;
}

int64_t attn_bwd_workspace_bytes(const AttnBwdPlan& p, int dtype, int64_t planes_q, int64_t planes_kv,
                                 int64_t D) {
  return offsets(p, dtype, planes_q, planes_kv, D).end;
}

hipError_t launch_attn_bwd(const AttnBwdArgs& x, hipStream_t s) {
  const AttnBwdPlan p = attn_bwd_plan(x.B, x.H, x.H_kv, x.N, x.N_kv, x.D, x.causal != 0);
  Args a;
  auto rows = [](const View& v) { return Rows{v.p, v.sb, v.sh, v.sr}; };
  auto out = [](const View& v) { return Out{const_cast<void*>(v.p), v.sb, v.sh, v.sr}; };
  a.q = rows(x.q);
  a.k = rows(x.k);
  a.v = rows(x.v);
  a.o = rows(x.o);
  a.dout = rows(x.dout);
  a.dq = out(x.dq);
  a.dk = out(x.dk);
  a.dv = out(x.dv);
  a.lse = x.lse;
  a.dlse = x.dlse;
  a.H = (int)x.H;
  a.H_kv = (int)x.H_kv;
  a.G = (int)(x.H / x.H_kv);
  a.N = (int)x.N;
  a.N_kv = (int)x.N_kv;
  a.nb_q = (int)p.nb_q;
  a.nb_kv = (int)p.nb_kv;
  a.NP = (int)p.nb_q * BT;
  a.planes_q = (int)(x.B * x.H);
  a.planes_kv = (int)(x.B * x.H_kv);
  a.k_tiles = (int)p.k_tiles;
  a.q_tiles = (int)p.q_tiles;
  a.k_split = (int)p.k_split;
  a.q_split = (int)p.q_split;
  a.k_blocks = (int)p.k_blocks;
  a.sm_scale = x.sm_scale;
  a.c = x.sm_scale * LOG2E_F;
  const Offsets64 o = offsets(p, x.dtype, a.planes_q, a.planes_kv, x.D);
  u8* ws = (u8*)x.workspace;
  a.nl = (float*)(ws + o.nl);
  a.nd = (float*)(ws + o.nd);
  a.max_do = (float*)(ws + o.max_do);
  a.max_d = (float*)(ws + o.max_d);
  a.max_v = (float*)(ws + o.max_v);
  a.part_k = (float*)(ws + o.part_k);
  a.part_v = (float*)(ws + o.part_v);
  a.part_q = (float*)(ws + o.part_q);
  if (x.dtype == 0)
    return x.D == 64 ? launch<f16, 64>(x, p, a, s) : launch<f16, 128>(x, p, a, s);
  return x.D == 64 ? launch<bf16, 64>(x, p, a, s) : launch<bf16, 128>(x, p, a, s);
}

}  // namespace sage
