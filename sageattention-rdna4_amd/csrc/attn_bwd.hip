// Attention's backward pass (gfx950): the gradients of Q, K and V from that of the output, with the
// probabilities recomputed from the kept logsumexp.
//
// For a query row i, its keys j, c = sm_scale log2 e and d_i = dout_i . out_i - dlse_i:
//     P_ij = 2^(c q_i.k_j - lse_i log2 e),      dV_j = sum_i P_ij dout_i,
//     dS_ij = P_ij (dout_i.v_j - d_i),          dQ_i = sm_scale sum_j dS_ij k_j,
//                                               dK_j = sm_scale sum_i dS_ij q_i.
// A row whose logsumexp is -infinity saw nothing: its P are zeros.
//
// A call without output and logsumexp (that of a forward pass by 8-bit scores, whose logsumexp is not that of
// the scores formed here) works out both anew: `stats` goes over a query's keys once with a running maximum, for
//     lse_i = log sum_j exp(sm_scale q_i.k_j),      d_i = sum_j P_ij dout_i.v_j - dlse_i,
// so that a row's P sum to 1 and its dS to dlse_i, however far the scores spread and whatever K's mean.
//
// Four launches at most, one in small calls. `rows` works out what S and dP of each row begin with,
// -lse / sm_scale and -d (a product's first summand, so that neither costs an operation). `main` holds blocks
// of two kinds: one owns keys and goes over the queries that see them (S, dP, dV, dK), the other owns queries
// and goes over their keys (S, dP, dQ). Seven products, where one kind of block that adds its dQ
// to memory would take five: but added atomically, in an order that changes from call to call, and
// with 4 bytes read and written per pair of query and key in fp32. Where there are too few blocks for
// the card the longest loops are cut into parts, whose fp32 sums `join` adds in order (bwd_cut.h). So results
// are the same from call to call.
//
// What bounds it. 32 heads on 8 of 16384 causal rows, bf16, head_dim 128: 6.5 to 6.7 ms by the card, the seven
// products at 1160 to 1200 TFLOP/s, where a large library product reaches 1227: the power cap, at a clock
// of 1.7 GHz with the matrix units busy for 66 % of the cycles. 20 heads of 4096 rows of 64 values, fp16, 313 to
// 342 us: the same clock, matrix units 51 %, vector instructions (six to a score) 54 %. `stats` takes 2.56 ms and 142 us
// of these: six vector instructions a score on two products, matrix units 45 and 27 %.
//
// Layout. A wave owns 32 columns (keys, or queries) of 16-bit operands in registers and multiplies
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

constexpr int BT = ATTN_BWD_ROWS;      // rows of the other side in an LDS tile
// Halves of a tile in the loop's code.
template <int D>
constexpr int U = D == 64 ? 2 : 1;
constexpr float NEG_INF = -__builtin_inff();
// fp16 operands: P is held times 2^12, so that it is a normal number from 2^-26 up, dS times a power of two
// that brings its bound (for P of 1 and less) into [2^13, 2^14).
template <typename T>
constexpr float P_SHIFT = std::is_same_v<T, f16> ? 12.0f : 0.0f;
// P passes 1 where a given logsumexp lies under its scores, by some units if it is that of quantized ones (spread
// 100, int8: P of 54). fp16's ends at 2^1.99, so that neither P nor dS passes 65504; a NaN stays one. (One operation a
// score, 313 us for 302 with 20 heads of 4096 rows of 64 values. The mode bit for saturating conversions costs
// nothing, but makes a NaN a number; a tile's largest exponent, and a branch where it is over, 321 us.)
constexpr float P_MOST = 1.99f;

// The 16-byte chunk of a tile's row r that lies at position c ^ swz(r). A row read takes 16 rows'
// (or 8 rows' two) chunks in a pass, a transposed read 4 rows' 64 bytes: both touch each bank once.
template <int D>
__device__ __forceinline__ int swz(int r) {
  return D == 128 ? ((r & 3) << 2) | (((r >> 2) & 1) << 1) | ((r >> 3) & 1)
                  : (((r >> 1) & 1) << 2) | (((r >> 2) & 1) << 1) | ((r >> 3) & 1);
}

// The lane's number, formed where it stands: what follows from it is not kept in registers over the
// main loop, which needs them all.
__device__ __forceinline__ int lane_anew() {
  int x;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(x));
  return x;
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
  AttnBwdCut keys, queries;
  int alone;                            // AttnBwdPlan::alone
  int columns;                          // of a tile
  float sm_scale, c;
  // workspace
  float* nl;        // (planes_q, NP): (P_SHIFT - lse log2 e) / c
  float* nd;        // (planes_q, NP): -d
  float* max_do;    // fp16: (planes_q, nb_q): a tile's largest |dout|^2, |d|, and (planes_kv, nb_kv) |v|^2
  float* max_d;
  float* max_v;
  float* stats;     // without lse: (3, queries.blocks, 128): a part's largest score, sum of weights, of weights times dP
  float* part_k;    // (keys.cut_blocks, columns, D): sums of dK, of dV, by blocks that hold a part of their tile
  float* part_v;
  float* part_q;    // (queries.cut_blocks, columns, D)
};

template <typename T>
__device__ __forceinline__ const T* plane(const Rows& x, int b, int h) {
  return (const T*)x.p + (int64_t)b * x.sb + (int64_t)h * x.sh;
}

// What a row's S begins with: (P_SHIFT - lse log2 e) / c, nothing seen for a logsumexp of -infinity.
template <typename T>
__device__ __forceinline__ float row_start(float lse, float c) {
  return lse == NEG_INF ? NEG_INF : __builtin_fmaf(-LOG2E_F, lse, P_SHIFT<T>) / c;
}

// A row's largest score m, and over its keys the sums l of the weights exp2(c (score - m)) and t of weights times dP;
// nothing seen yet.
struct Stats {
  float m = -3e38f, l = 0.0f, t = 0.0f;
  __device__ __forceinline__ void add(const Stats& x, float c) {
    const float top = fmaxf(m, x.m);
    const float f = __builtin_amdgcn_exp2f((m - top) * c), g = __builtin_amdgcn_exp2f((x.m - top) * c);
    l = l * f + x.l * g;
    t = t * f + x.t * g;
    m = top;
  }
};

// ------------------------------------------------------------------------------------- rows
// 64 rows of a plane per block, D / 8 lanes to a row. ANEW: the constants come from what `stats` left.
template <typename T, int D, bool ANEW>
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
    if (!ANEW && !of_v) y[i] = *(const u32x4*)(py + (int64_t)r * a.o.sr);
  }
  // ANEW: where the parts of the block's rows lie (all in one tile)
  const float* stats = a.stats;
  int parts = 0;
  if (ANEW && !of_v) {
    const int tile = (at - p * nb) * 64 / a.columns;
    const int block = attn_bwd_first_part(a.queries, a.queries.tiles - 1 - tile, a.planes_q, parts) + p;
    stats += (int64_t)block * 128 - tile * a.columns;
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
      if (ANEW) {
        // each of the row's lanes takes some parts (and, of blocks of two pairs of waves, both pairs' sums)
        const int64_t all = (int64_t)a.queries.blocks * 128, step = (int64_t)a.planes_q * 128;
        const int pairs = 128 / a.columns;
        Stats sum;
        for (int k = cg; k < parts * pairs; k += CG) {
          const float* f = stats + k / pairs * step + k % pairs * a.columns + min(r, n_rows - 1);
          Stats x;
          x.m = f[0];
          x.l = f[all];
          x.t = f[2 * all];
          sum.add(x, a.c);
        }
#pragma unroll
        for (int m = 1; m < CG; m <<= 1) {
          Stats x;
          x.m = __shfl_xor(sum.m, m, 64);
          x.l = __shfl_xor(sum.l, m, 64);
          x.t = __shfl_xor(sum.t, m, 64);
          sum.add(x, a.c);
        }
        nl = (P_SHIFT<T> - log2f(sum.l)) / a.c - sum.m;
        dot = sum.t / sum.l;
      }
      if (r < n_rows) {
        const int64_t row = (int64_t)p * a.N + r;
        if (!ANEW) nl = row_start<T>(a.lse[row], a.c);
        nd = (a.dlse ? a.dlse[row] : 0.0f) - dot;
      } else {
        nl = NEG_INF;
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
// Each of the threads' values' largest over a block of 256, through K * 4 floats of LDS; NaNs are passed over.
template <int K>
__device__ __forceinline__ void block_max(float* lds, float (&m)[K]) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) m[k] = fmaxf(m[k], __shfl_xor(m[k], s, 64));
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int k = 0; k < K; ++k) lds[4 * k + (threadIdx.x >> 6)] = m[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k)
    m[k] = fmaxf(fmaxf(lds[4 * k], lds[4 * k + 1]), fmaxf(lds[4 * k + 2], lds[4 * k + 3]));
}
// The largest of n values, as far as this thread has seen them.
__device__ __forceinline__ float largest(const float* p, int n) {
  float m = 0.0f;
  for (int i = threadIdx.x; i < n; i += 256) m = fmaxf(m, p[i]);
  return m;
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

// LDS of a block: two tiles of each of two tensors, and of the rows' two constants (CW = 2: of all tiles',
// where the block works them out).
template <int D, int CW>
constexpr int LDS_BYTES = 4 * BT * D * 2 + 2 * 2 * BT * 4 + (CW == 2 ? ATTN_BWD_ALONE * 2 * BT * 4 : 0);

// A tile of BT rows of a plane on its way into LDS, a quarter by each wave, 1 KB a request: 64 lanes of
// 16 bytes, RPI rows.
template <typename T, int D>
struct Staging {
  static constexpr int CPR = D / 8, RPI = 64 / CPR, IT = 16 / RPI;
  int lane, w;
  __device__ __forceinline__ Staging(int lane, int w) : lane(lane), w(w) {}
  // The tile from `x` on, of which `left` rows or more are the plane's, to LDS address `lds`. Rows behind the
  // last one are that one again: what they would add is multiplied by P = 0.
  __device__ __forceinline__ void operator()(const T* x, int64_t sr, int left, uint32_t lds) const {
    const int l = D == 128 ? lane_anew() : lane;
    const int step = (int)(2 * sr), own = l / CPR;
    const int chunk = 16 * ((l % CPR) ^ swz<D>(own));
    lds = __builtin_amdgcn_readfirstlane(lds + 16 * w * D * 2);
    // (At head_dim 128 the branch costs more than the clamps: 7.20 ms for 6.94, 32 heads of 16384.)
    if (D == 64 && left >= BT) {
      const T* base = x + 16 * w * sr;
      const int at = own * step;
#pragma unroll
      for (int i = 0; i < IT; ++i)
        dma16(base + RPI * i * sr, (uint32_t)(at + (chunk ^ 16 * swz<D>(RPI * i))), lds + RPI * i * D * 2);
    } else {
#pragma unroll
      for (int i = 0; i < IT; ++i)
        dma16(x, (uint32_t)(min(16 * w + RPI * i + own, left - 1) * step + (chunk ^ 16 * swz<D>(RPI * i))),
              lds + RPI * i * D * 2);
    }
  }
};

// Where a lane's operands lie in a tile, in bytes; the chunk's number is part of the address by
// exclusive or alone.
template <int D>
struct Offsets {
  int row, lo, hi;
  __device__ __forceinline__ Offsets(int lane) {
    const int r = lane & 31, g = lane >> 5, l16 = lane & 15, j = (lane >> 4) & 1;
    row = r * D * 2 + 16 * (g ^ swz<D>(r));
    const int r4 = 4 * g + (l16 >> 2), c = 2 * j + ((l16 & 3) >> 1);
    lo = r4 * D * 2 + 16 * (c ^ swz<D>(r4)) + 8 * (l16 & 1);
    hi = (r4 + 8) * D * 2 + 16 * (c ^ swz<D>(r4 + 8)) + 8 * (l16 & 1);
  }
  // In the 32 rows at `at`, a multiple of a row. At head_dim 128 the addresses of a chunk are worked
  // out for its read, at 64 each has a register and `at` stands in the instruction.
  __device__ __forceinline__ Offsets rows(int& at) const {
    Offsets x = *this;
    if (D == 128) {
      asm volatile("" : "+s"(at));
      x.row += at;
      x.lo += at;
      x.hi += at;
      at = 0;
    }
    return x;
  }
};
// Rows lane % 32 of 32, columns 16 s + 8 g .. + 7; `at`: the place of the rows.
template <typename T>
__device__ __forceinline__ typename Vec<T>::x8 row_operand(const u8* smem, int off, int at, int s) {
  return *(const typename Vec<T>::x8*)(smem + (off ^ (32 * s)) + at);
}
// The transposed operand of 16 rows and columns 32 dt .. + 31.
template <typename T>
__device__ __forceinline__ typename Vec<T>::x8 transposed(const u8* smem, int lo, int hi, int at, int dt) {
  const auto a = read_tr((const T*)(smem + (lo ^ (64 * dt)) + at)),
             b = read_tr((const T*)(smem + (hi ^ (64 * dt)) + at));
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// A wave's 32 columns of x (rows of memory from r0 on; from n on row n - 1 again) as operands.
template <typename T, int D>
__device__ __forceinline__ void load_columns(const T* x, int64_t sr, int r0, int n, int lane,
                                             typename Vec<T>::x8 (&f)[D / 16]) {
  const T* p = x + (int64_t)min(r0 + (lane & 31), n - 1) * sr + 8 * (lane >> 5);
#pragma unroll
  for (int s = 0; s < D / 16; ++s) f[s] = *(const typename Vec<T>::x8*)(p + 16 * s);
}

// A wave's sums, 32 columns of D values each, times f, into rows of a 16-bit view from r0 + 32 w on (up to
// n), or of the block's fp32 part.
template <typename T, int D>
__device__ __forceinline__ void store_columns(const f32x16 (&acc)[D / 32], float f, const Out& o, int b,
                                              int h, float* part, int r0, int w, int n) {
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) keep_live(acc[dt]);
  mfma_result_fence32();
  const int lane = lane_anew(), own = 32 * w + (lane & 31), r = r0 + own, col = 4 * (lane >> 5);
  if (r >= n) return;
  if (part) {
    float* p = part + own * D + col;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f32x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = acc[dt][4 * i + e] * f;
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
        for (int e = 0; e < 4; ++e) x[e] = (T)(acc[dt][4 * i + e] * f);
        *(typename Vec<T>::x4*)(p + 32 * dt + 8 * i) = x;
      }
  }
}

// Between the phases of a step: what the compiler moves across costs it registers, at head_dim 64 (a
// 4096-token image at 20 heads: 356 us with, 372 without) and where no branch for masks parts the
// phases (spills). Not for causal calls at head_dim 128: 4 sequences of 2048, 32 heads, 551 us with, 544
// without.
template <int D, bool CAUSAL>
__device__ __forceinline__ void fence() {
  if (D == 64 || !CAUSAL) __builtin_amdgcn_sched_barrier(0);
}

// 2^x; fp16: 2^most at most.
template <typename T>
__device__ __forceinline__ float weight(float x, float most) {
  return __builtin_amdgcn_exp2f(std::is_same_v<T, f16> ? __builtin_elementwise_minimum(x, most) : x);
}

__device__ __forceinline__ void clear(f32x16& x) {
#pragma unroll
  for (int r = 0; r < 16; ++r) x[r] = 0.0f;
}

// The requests of the tile at hand have landed, in all waves, and everyone is done with the other one.
__device__ __forceinline__ void next_tile() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// A constant of each of a result's rows, 8 (r / 4) + 4 g + r % 4; `rows`: from 4 g on.
__device__ __forceinline__ f32x16 row_constants(const float* rows) {
  f32x16 x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x4 y = *(const f32x4*)(rows + 8 * i);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[4 * i + e] = y[e];
  }
  return x;
}

// Blocks of two pairs of waves (CW = 2): the second pair's sums, over the second halves of the steps' rows, are
// added to the first's, by way of the tiles' LDS. True for the waves that hold them.
template <int D, typename... X>
__device__ __forceinline__ bool merge_pairs(u8* smem, int w, X&... x) {
  float* at = (float*)smem + (w & 1) * (sizeof...(X) * 32 * D) + 4 * lane_anew();
  (
      [&](auto& acc) {
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) keep_live(acc[dt]);
      }(x),
      ...);
  mfma_result_fence32();
  __syncthreads();
  auto each = [&](auto&& f) {
    float* p = at;
    auto of = [&](auto& acc) {
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i, p += 256) f(acc[dt], i, (f32x4*)p);
    };
    (of(x), ...);
  };
  if (w >= 2)
    each([](const f32x16& v, int i, f32x4* p) {
      *p = (f32x4){v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
    });
  __syncthreads();
  if (w < 2)
    each([](f32x16& v, int i, const f32x4* p) {
      const f32x4 y = *p;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * i + e] += y[e];
    });
  return w < 2;
}

// A wave works out the constants of a tile's 64 rows (from `g` and `o` on, `left` of them or more): what S and
// dP begin with, to `to` and to + BT. top: the largest |dout|^2 and |d| so far.
template <typename T, int D>
__device__ __forceinline__ void tile_rows(const T* g, int64_t g_sr, const T* o, int64_t o_sr, const float* lse,
                                          const float* dlse, int left, float c, float* to, int lane,
                                          float (&top)[2]) {
  constexpr int CG = D / 8, R = 64 / CG, IT = 8;      // 64 or 32 rows at a time
  const int cg = lane % CG, rg = lane / CG;
#pragma unroll 1
  for (int r0 = rg; r0 < 64; r0 += IT * R) {
    u32x4 x[IT], y[IT];
    float l[IT], dl[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int r = min(r0 + i * R, left - 1);
      x[i] = *(const u32x4*)(g + (int64_t)r * g_sr + 8 * cg);
      y[i] = *(const u32x4*)(o + (int64_t)r * o_sr + 8 * cg);
      l[i] = lse[r];
      dl[i] = dlse ? dlse[r] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      float fx[8], fy[8], dot = 0.0f, sq = 0.0f;
      unpack8<T>(x[i], fx);
      unpack8<T>(y[i], fy);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        dot = __builtin_fmaf(fx[e], fy[e], dot);
        sq = __builtin_fmaf(fx[e], fx[e], sq);
      }
#pragma unroll
      for (int m = 1; m < CG; m <<= 1) {
        dot += __shfl_xor(dot, m, 64);
        if (std::is_same_v<T, f16>) sq += __shfl_xor(sq, m, 64);
      }
      const int r = r0 + i * R;
      const bool live = r < left;
      const float nd = live ? dl[i] - dot : 0.0f;
      top[0] = fmaxf(top[0], sq);
      top[1] = fmaxf(top[1], fabsf(nd));
      if (cg == 0) {
        to[r] = live ? row_start<T>(l[i], c) : NEG_INF;
        to[BT + r] = nd;
      }
    }
  }
}

// The largest |x|^2 of n rows, as far as this thread has seen them.
template <typename T, int D>
__device__ __forceinline__ float largest_row(const T* x, int64_t sr, int n) {
  constexpr int CG = D / 8;
  const int cg = threadIdx.x % CG;
  float m = 0.0f;
  for (int r = threadIdx.x / CG; r < (n + 256 / CG - 1) / (256 / CG) * (256 / CG); r += 256 / CG) {
    float f[8], sq = 0.0f;
    unpack8<T>(*(const u32x4*)(x + (int64_t)min(r, n - 1) * sr + 8 * cg), f);
#pragma unroll
    for (int e = 0; e < 8; ++e) sq = __builtin_fmaf(f[e], f[e], sq);
#pragma unroll
    for (int s = 1; s < CG; s <<= 1) sq += __shfl_xor(sq, s, 64);
    m = fmaxf(m, sq);
  }
  return m;
}

// |x|^2 of a lane's column, and x . y of two.
template <typename T, int D>
__device__ __forceinline__ float column_dot(const typename Vec<T>::x8 (&x)[D / 16],
                                            const typename Vec<T>::x8 (&y)[D / 16]) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) s = __builtin_fmaf((float)x[i][e], (float)y[i][e], s);
  return s + __shfl_xor(s, 32, 64);
}

// A block that owns 32 CW keys of a K/V head.
template <typename T, int D, bool CAUSAL, int CW>
__device__ __forceinline__ void keys_block(const Args& a, u8* smem, int block) {
  constexpr int TILE = BT * D * 2, BC = 32 * CW;
  constexpr bool F16 = std::is_same_v<T, f16>;
  typedef typename Vec<T>::x8 x8;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 5;
  const AttnBwdPlace at = attn_bwd_place(a.keys, block, a.planes_kv);
  const int pl = at.plane, b = pl / a.H_kv, hk = pl - b * a.H_kv;
  const int k0 = at.u * BC, kw = k0 + 32 * (w % CW);
  // tiles of queries, head after head of the group
  const int first = CAUSAL ? k0 / BT : 0, per = a.nb_q - first;
  const int n = per * a.G;
  const int it0 = at.first(n), it1 = at.end(n);

  // LDS: two tiles of Q, two of dout, and of the rows' two constants
  const float* lds_rows = (const float*)(smem + 4 * TILE);
  const uint32_t lds0 = lds_addr(smem);
  const Staging<T, D> stage(lane, w);
  // the next tile to be requested, ti of its head, and where it lies
  int ti = it0 / per;
  const int h0 = hk * a.G + ti;
  ti = first + it0 - ti * per;
  const T* pq = plane<T>(a.q, b, h0) + (int64_t)ti * BT * a.q.sr;
  const T* po = plane<T>(a.dout, b, h0) + (int64_t)ti * BT * a.dout.sr;
  const bool alone = CW == 2 && a.alone;
  float* own_rows = (float*)(smem + 4 * TILE) + 4 * BT;   // alone: constants of all the block's tiles
  const float* pr = alone ? nullptr : (w & 1 ? a.nd : a.nl) + (int64_t)(b * a.H + h0) * a.NP + ti * BT;
  const int64_t head_q = a.q.sh - (int64_t)per * BT * a.q.sr;
  const int64_t head_o = a.dout.sh - (int64_t)per * BT * a.dout.sr;
  auto request = [&](int buf) {
    const int left = a.N - ti * BT;
    stage(pq, a.q.sr, left, lds0 + buf * TILE);
    stage(po, a.dout.sr, left, lds0 + (2 + buf) * TILE);
    if (w < 2 && !alone) dma4(pr, 4 * lane_anew(), lds0 + 4 * TILE + (2 * buf + w) * BT * 4);
    pq += BT * a.q.sr;
    po += BT * a.dout.sr;
    if (!alone) pr += BT;
    if (++ti == a.nb_q) {                            // on to the group's next head
      ti = first;
      pq += head_q;
      po += head_o;
      if (!alone) pr += first * BT;
    }
  };

  int tc = ti;                                       // the tile at hand
  if (it0 < it1) request(0);
  const Offsets<D> offsets(lane);
  x8 kf[D / 16], vf[D / 16];
  load_columns<T, D>(plane<T>(a.k, b, hk), a.k.sr, kw, a.N_kv, lane, kf);
  load_columns<T, D>(plane<T>(a.v, b, hk), a.v.sr, kw, a.N_kv, lane, vf);
  // the largest |dout|^2, |d| and |v|^2
  float scale = 1.0f, m[3] = {0.0f, 0.0f, 0.0f};
  if (alone) {
    float top[2] = {0.0f, 0.0f};
    for (int i = w; i < it1 - it0; i += 4) {
      const int gi = (it0 + i) / per, t = first + it0 + i - gi * per, h = hk * a.G + gi;
      const int64_t row = (int64_t)(b * a.H + h) * a.N + t * BT;
      tile_rows<T, D>(plane<T>(a.dout, b, h) + (int64_t)t * BT * a.dout.sr, a.dout.sr,
                      plane<T>(a.o, b, h) + (int64_t)t * BT * a.o.sr, a.o.sr, a.lse + row,
                      a.dlse ? a.dlse + row : nullptr, a.N - t * BT, a.c, own_rows + 2 * BT * i, lane, top);
    }
    m[0] = top[0];
    m[1] = top[1];
    if (F16) m[2] = column_dot<T, D>(vf, vf);
  } else if (F16) {
    const int64_t hq = (int64_t)(b * a.H + hk * a.G) * a.nb_q;
    m[0] = largest(a.max_do + hq, a.G * a.nb_q);
    m[1] = largest(a.max_d + hq, a.G * a.nb_q);
    m[2] = largest(a.max_v + (int64_t)pl * a.nb_kv, a.nb_kv);
  }
  if (F16) {
    block_max<3>((float*)(smem + 4 * TILE) + 2 * BT, m);   // by way of the second tile's constants
    scale = scale_for(sqrtf(m[0]) * sqrtf(m[2]) + m[1]);
  }
  const float fs = scale * __builtin_ldexpf(1.0f, -(int)P_SHIFT<T>);
  f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) {
    clear(dk[dt]);
    clear(dv[dt]);
  }
  // 32 queries from qu on, which lie at `at`
  auto step = [&](int qu, int at, const float* rows) {
    const Offsets<D> of = offsets.rows(at);
    const int at_do = at + 2 * TILE;
    f32x16 s = row_constants(rows), dp;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) s = mfma16(row_operand<T>(smem, of.row, at, i), kf[i], s);
    if (CAUSAL && qu < kw + 31) {
      const int l = lane_anew(), ahead = kw + (l & 31) - qu - 4 * (l >> 5);
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (8 * (r / 4) + r % 4 < ahead) s[r] = NEG_INF;
    }
    fence<D, CAUSAL>();
    dp = row_constants(rows + BT);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      dp = mfma16(row_operand<T>(smem, of.row, at_do, i), vf[i], dp);
      // P, between dP's products: the matrix unit and the others work at once
#pragma unroll
      for (int r = 256 / D * i; r < 256 / D * (i + 1); ++r) s[r] = weight<T>(s[r] * a.c, P_SHIFT<T> + P_MOST);
    }
    fence<D, CAUSAL>();
    x8 pf[2], df[2];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float p = s[r];
      pf[r / 8][r % 8] = (T)p;
      if (F16) p *= fs;
      df[r / 8][r % 8] = (T)(p * dp[r]);
    }
    fence<D, CAUSAL>();
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) {
        dv[dt] = mfma16(transposed<T>(smem, of.lo, of.hi, at_do + 32 * t * D, dt), pf[t], dv[dt]);
        dk[dt] = mfma16(transposed<T>(smem, of.lo, of.hi, at + 32 * t * D, dt), df[t], dk[dt]);
      }
  };
  // what was loaded so far is here: in the loop the compiler has nothing of its own to wait for
  __builtin_amdgcn_s_waitcnt(0);
  auto tile_of = [&](int it, int buf) {
    next_tile();
    const int q0 = tc * BT;
    tc = ti;
    if (it + 1 < it1) request(buf ^ 1);
    const float* rows = (alone ? own_rows + 2 * BT * (it - it0) : lds_rows + 2 * buf * BT) + 4 * g;
#pragma unroll U<D>
    for (int x = 0; x < CW / 2; ++x) {
      const int u = CW == 4 ? x : w >> 1;
      if (!CAUSAL || q0 + 32 * u + 31 >= kw) step(q0 + 32 * u, (buf * BT + 32 * u) * D * 2, rows + 32 * u);
    }
  };
  if (D == 64) {
    for (int it = it0; it < it1; it += 2) {
      tile_of(it, 0);
      if (it + 1 < it1) tile_of(it + 1, 1);
    }
  } else {
    for (int it = it0; it < it1; ++it) tile_of(it, (it - it0) & 1);
  }
  if (CW == 2 && !merge_pairs<D>(smem, w, dk, dv)) return;
  const bool whole = at.parts == 1;
  const int64_t part = (int64_t)block * BC * D;
  store_columns<T, D>(dk, a.sm_scale / scale, a.dk, b, hk, whole ? nullptr : a.part_k + part, k0, w, a.N_kv);
  store_columns<T, D>(dv, __builtin_ldexpf(1.0f, -(int)P_SHIFT<T>), a.dv, b, hk,
                      whole ? nullptr : a.part_v + part, k0, w, a.N_kv);
}

// A block that owns 32 CW queries of a head.
template <typename T, int D, bool CAUSAL, int CW>
__device__ __forceinline__ void queries_block(const Args& a, u8* smem, int block) {
  constexpr int TILE = BT * D * 2, BC = 32 * CW;
  constexpr bool F16 = std::is_same_v<T, f16>;
  typedef typename Vec<T>::x8 x8;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const AttnBwdPlace at = attn_bwd_place(a.queries, block, a.planes_q);
  const int pl = at.plane, b = pl / a.H, h = pl - b * a.H, hk = h / a.G;
  // the last tile of a causal plane is its longest
  const int q0 = (a.queries.tiles - 1 - at.u) * BC, qw = q0 + 32 * (w % CW);
  const int n = CAUSAL ? min((q0 + BC) / BT, a.nb_kv) : a.nb_kv;
  const int it0 = at.first(n), it1 = at.end(n);

  // LDS: two tiles of K, two of V
  const uint32_t lds0 = lds_addr(smem);
  const T* pk = plane<T>(a.k, b, hk) + (int64_t)it0 * BT * a.k.sr;
  const T* pv = plane<T>(a.v, b, hk) + (int64_t)it0 * BT * a.v.sr;
  const Staging<T, D> stage(lane, w);
  auto request = [&](int it, int buf) {
    const int left = a.N_kv - it * BT;
    stage(pk, a.k.sr, left, lds0 + buf * TILE);
    stage(pv, a.v.sr, left, lds0 + (2 + buf) * TILE);
    pk += BT * a.k.sr;
    pv += BT * a.v.sr;
  };

  if (it0 < it1) request(it0, 0);
  const Offsets<D> offsets(lane);
  x8 qf[D / 16], gf[D / 16];
  load_columns<T, D>(plane<T>(a.q, b, h), a.q.sr, qw, a.N, lane, qf);
  load_columns<T, D>(plane<T>(a.dout, b, h), a.dout.sr, qw, a.N, lane, gf);
  float nl1, nd1, scale = 1.0f, most = 0.0f;           // most: the largest exponent
  if (CW == 2 && a.alone) {
    x8 of[D / 16];
    load_columns<T, D>(plane<T>(a.o, b, h), a.o.sr, qw, a.N, lane, of);
    const int64_t row = (int64_t)pl * a.N + min(qw + (lane & 31), a.N - 1);
    nl1 = row_start<T>(a.lse[row], a.c);
    nd1 = (a.dlse ? a.dlse[row] : 0.0f) - column_dot<T, D>(gf, of);
  } else {
    const int64_t row = (int64_t)pl * a.NP + min(qw + (lane & 31), a.NP - 1);
    nl1 = a.nl[row];
    nd1 = a.nd[row];
  }
  if (F16) {
    const int plane_kv = b * a.H_kv + hk;
    float mv[1] = {CW == 2 && a.alone ? largest_row<T, D>(plane<T>(a.v, b, hk), a.v.sr, a.N_kv)
                                      : largest(a.max_v + (int64_t)plane_kv * a.nb_kv, a.nb_kv)};
    block_max<1>((float*)(smem + 4 * TILE), mv);
    scale = scale_for(sqrtf(column_dot<T, D>(gf, gf)) * sqrtf(mv[0]) + fabsf(nd1));
    // P meets dS alone here: its power of two is part of the exponent
    const float shift = log2f(scale);
    nl1 += (shift - P_SHIFT<T>) / a.c;
    most = shift + P_MOST;
  }
  f32x16 dq[D / 32];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) clear(dq[dt]);
  // what S and dP begin with: a register for each row, all alike
  f32x16 nl, nd;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    nl[r] = nl1;
    nd[r] = nd1;
  }
  // 32 keys from ku on, which lie at `at`
  auto step = [&](int ku, int at) {
    const Offsets<D> of = offsets.rows(at);
    f32x16 s = nl, dp = nd;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) s = mfma16(row_operand<T>(smem, of.row, at, i), qf[i], s);
    if (ku + 31 >= (CAUSAL ? qw + 1 : a.N_kv)) {
      const int l = lane_anew(), query = qw + (l & 31);
      const int left = (CAUSAL ? min(query + 1, a.N_kv) : a.N_kv) - ku - 4 * (l >> 5);
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (8 * (r / 4) + r % 4 >= left) s[r] = NEG_INF;
    }
    fence<D, CAUSAL>();
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      dp = mfma16(row_operand<T>(smem, of.row, at + 2 * TILE, i), gf[i], dp);
#pragma unroll
      for (int r = 256 / D * i; r < 256 / D * (i + 1); ++r) s[r] = weight<T>(s[r] * a.c, most);
    }
    fence<D, CAUSAL>();
    x8 df[2];
#pragma unroll
    for (int r = 0; r < 16; ++r) df[r / 8][r % 8] = (T)(s[r] * dp[r]);
    fence<D, CAUSAL>();
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
        dq[dt] = mfma16(transposed<T>(smem, of.lo, of.hi, at + 32 * t * D, dt), df[t], dq[dt]);
  };
  __builtin_amdgcn_s_waitcnt(0);                     // as in keys_block
  const int end = CAUSAL ? min(qw + 32, a.N_kv) : a.N_kv;
  auto tile_of = [&](int it, int buf) {
    next_tile();
    if (it + 1 < it1) request(it + 1, buf ^ 1);
#pragma unroll U<D>
    for (int x = 0; x < CW / 2; ++x) {
      const int u = CW == 4 ? x : w >> 1;
      if (it * BT + 32 * u < end) step(it * BT + 32 * u, (buf * BT + 32 * u) * D * 2);
    }
  };
  if (D == 64) {
    for (int it = it0; it < it1; it += 2) {
      tile_of(it, 0);
      if (it + 1 < it1) tile_of(it + 1, 1);
    }
  } else {
    for (int it = it0; it < it1; ++it) tile_of(it, (it - it0) & 1);
  }
  if (CW == 2 && !merge_pairs<D>(smem, w, dq)) return;
  store_columns<T, D>(dq, a.sm_scale / scale, a.dq, b, h,
                      at.parts == 1 ? nullptr : a.part_q + (int64_t)block * BC * D, q0, w, a.N);
}

// ------------------------------------------------------------------------------------- stats
// The queries' blocks of the main launch, cut in the same way: S and dP alone, and their sums. Each half of a
// wave has every other four keys of its 32 queries, each pair of waves (CW = 2) half of a step's.
template <typename T, int D, bool CAUSAL, int CW>
__global__ void __launch_bounds__(256, D == 64 ? 4 : 2) stats_kernel(const Args a) {
  constexpr int TILE = BT * D * 2, BC = 32 * CW;
  typedef typename Vec<T>::x8 x8;
  __shared__ __align__(1024) u8 smem[4 * TILE];        // two tiles of K, two of V
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const AttnBwdPlace at = attn_bwd_place(a.queries, blockIdx.x, a.planes_q);
  const int pl = at.plane, b = pl / a.H, h = pl - b * a.H, hk = h / a.G;
  const int q0 = (a.queries.tiles - 1 - at.u) * BC, qw = q0 + 32 * (w % CW);
  const int n = CAUSAL ? min((q0 + BC) / BT, a.nb_kv) : a.nb_kv;
  const int it0 = at.first(n), it1 = at.end(n);
  const uint32_t lds0 = lds_addr(smem);
  const T* pk = plane<T>(a.k, b, hk) + (int64_t)it0 * BT * a.k.sr;
  const T* pv = plane<T>(a.v, b, hk) + (int64_t)it0 * BT * a.v.sr;
  const Staging<T, D> stage(lane, w);
  auto request = [&](int it, int buf) {
    const int left = a.N_kv - it * BT;
    stage(pk, a.k.sr, left, lds0 + buf * TILE);
    stage(pv, a.v.sr, left, lds0 + (2 + buf) * TILE);
    pk += BT * a.k.sr;
    pv += BT * a.v.sr;
  };
  if (it0 < it1) request(it0, 0);
  const Offsets<D> offsets(lane);
  x8 qf[D / 16], gf[D / 16];
  load_columns<T, D>(plane<T>(a.q, b, h), a.q.sr, qw, a.N, lane, qf);
  load_columns<T, D>(plane<T>(a.dout, b, h), a.dout.sr, qw, a.N, lane, gf);
  Stats sum;
  // 32 keys from ku on, which lie at `at`
  auto step = [&](int ku, int at) {
    const Offsets<D> of = offsets.rows(at);
    f32x16 s, dp;
    clear(s);
    clear(dp);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) s = mfma16(row_operand<T>(smem, of.row, at, i), qf[i], s);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) dp = mfma16(row_operand<T>(smem, of.row, at + 2 * TILE, i), gf[i], dp);
    if (ku + 31 >= (CAUSAL ? qw + 1 : a.N_kv)) {
      const int l = lane_anew(), query = qw + (l & 31);
      const int left = (CAUSAL ? min(query + 1, a.N_kv) : a.N_kv) - ku - 4 * (l >> 5);
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (8 * (r / 4) + r % 4 >= left) s[r] = NEG_INF;
    }
    float top = sum.m;
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, s[r]);
    const float f = __builtin_amdgcn_exp2f((sum.m - top) * a.c);
    sum.m = top;
    float l = 0.0f, t = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float p = __builtin_amdgcn_exp2f((s[r] - top) * a.c);
      l += p;
      t = __builtin_fmaf(p, dp[r], t);
    }
    sum.l = __builtin_fmaf(sum.l, f, l);
    sum.t = __builtin_fmaf(sum.t, f, t);
  };
  __builtin_amdgcn_s_waitcnt(0);                       // as in keys_block
  const int end = CAUSAL ? min(qw + 32, a.N_kv) : a.N_kv;
  for (int it = it0; it < it1; ++it) {
    const int buf = (it - it0) & 1;
    next_tile();
    if (it + 1 < it1) request(it + 1, buf ^ 1);
#pragma unroll 1
    for (int x = 0; x < CW / 2; ++x) {
      const int u = CW == 4 ? x : w >> 1;
      if (it * BT + 32 * u < end) step(it * BT + 32 * u, (buf * BT + 32 * u) * D * 2);
    }
  }
  Stats x;
  x.m = __shfl_xor(sum.m, 32, 64);
  x.l = __shfl_xor(sum.l, 32, 64);
  x.t = __shfl_xor(sum.t, 32, 64);
  sum.add(x, a.c);
  if (lane < 32) {
    const int64_t all = (int64_t)a.queries.blocks * 128;
    float* to = a.stats + (int64_t)blockIdx.x * 128 + 32 * w + lane;
    to[0] = sum.m;
    to[all] = sum.l;
    to[2 * all] = sum.t;
  }
}

template <typename T, int D, bool CAUSAL, int CW>
__global__ void __launch_bounds__(256, D == 64 ? 3 : 2) main_kernel(const Args a) {
  __shared__ __align__(1024) u8 smem[LDS_BYTES<D, CW>];
  if ((int)blockIdx.x < a.keys.blocks)
    keys_block<T, D, CAUSAL, CW>(a, smem, blockIdx.x);
  else
    queries_block<T, D, CAUSAL, CW>(a, smem, blockIdx.x - a.keys.blocks);
}

// ------------------------------------------------------------------------------------- join
// The parts of a tile added in order: dK and dV (of = 0, 1) of the keys' cut tiles, then dQ of the queries',
// 256 chunks of 8 values a block.
struct JoinArgs {
  AttnBwdCut cut[2];
  const float* part[3];
  Out out[3];
  int heads[2], planes[2], rows[2], blocks_k;
};
template <typename T, int D, int BC>
__global__ void __launch_bounds__(256) join_kernel(const JoinArgs a) {
  constexpr int SUB = BC * D / 8 / 256;                     // blocks to a tile
  int id = blockIdx.x;
  const bool q = id >= 2 * a.blocks_k;
  if (q) id -= 2 * a.blocks_k;
  const int of = q ? 2 : id >= a.blocks_k;
  if (of == 1) id -= a.blocks_k;
  const AttnBwdCut& c = a.cut[q];
  const int sub = id % SUB, planes = a.planes[q], pl = id / SUB % planes, u = id / SUB / planes;
  int p;
  const int first = attn_bwd_first_part(c, u, planes, p) + pl;       // its block, the other parts' `planes` apart
  const int at = sub * 256 + threadIdx.x, row = at / (D / 8), col = at % (D / 8) * 8;
  const int r = (q ? c.tiles - 1 - u : u) * BC + row;
  if (r >= a.rows[q]) return;
  const float* x = a.part[of] + ((int64_t)first * BC + row) * D + col;
  const int64_t step = (int64_t)planes * BC * D;
  f32x4 s0 = *(const f32x4*)x, s1 = *(const f32x4*)(x + 4);
#pragma unroll 4
  for (int k = 1; k < p; ++k) {
    s0 += *(const f32x4*)(x + k * step);
    s1 += *(const f32x4*)(x + k * step + 4);
  }
  typename Vec<T>::x8 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    y[e] = (T)s0[e];
    y[4 + e] = (T)s1[e];
  }
  const int b = pl / a.heads[q], h = pl % a.heads[q];
  *(typename Vec<T>::x8*)((T*)a.out[of].p + (int64_t)b * a.out[of].sb + (int64_t)h * a.out[of].sh +
                          (int64_t)r * a.out[of].sr + col) = y;
}

template <typename T, int D, int CW>
void launch_main(const Args& a, bool causal, hipStream_t s) {
  const dim3 grid(a.keys.blocks + a.queries.blocks);
  if (causal)
    hipLaunchKernelGGL((main_kernel<T, D, true, CW>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((main_kernel<T, D, false, CW>), grid, dim3(256), 0, s, a);
}
template <typename T, int D, int BC>
hipError_t launch_join(const Args& a, hipStream_t s) {
  constexpr int SUB = BC * D / 8 / 256;
  JoinArgs j = {};
  j.cut[0] = a.keys;
  j.cut[1] = a.queries;
  j.part[0] = a.part_k;
  j.part[1] = a.part_v;
  j.part[2] = a.part_q;
  j.out[0] = a.dk;
  j.out[1] = a.dv;
  j.out[2] = a.dq;
  j.heads[0] = a.H_kv;
  j.heads[1] = a.H;
  j.planes[0] = a.planes_kv;
  j.planes[1] = a.planes_q;
  j.rows[0] = a.N_kv;
  j.rows[1] = a.N;
  j.blocks_k = a.keys.cut * a.planes_kv * SUB;
  const int blocks = 2 * j.blocks_k + a.queries.cut * a.planes_q * SUB;
  if (blocks == 0) return hipSuccess;
  hipLaunchKernelGGL((join_kernel<T, D, BC>), dim3(blocks), dim3(256), 0, s, j);
  return hipGetLastError();
}

template <typename T, int D, int CW>
void launch_stats(const Args& a, bool causal, hipStream_t s) {
  if (causal)
    hipLaunchKernelGGL((stats_kernel<T, D, true, CW>), dim3(a.queries.blocks), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((stats_kernel<T, D, false, CW>), dim3(a.queries.blocks), dim3(256), 0, s, a);
}

template <typename T, int D>
hipError_t launch(const AttnBwdArgs& x, const AttnBwdPlan& p, const Args& a, hipStream_t s) {
  hipError_t e = hipSuccess;
  const int rows = a.planes_q * a.nb_q + (x.dtype == 0 ? a.planes_kv * a.nb_kv : 0);
  if (!x.lse) {
    if (p.columns == 128)
      launch_stats<T, D, 4>(a, x.causal, s);
    else
      launch_stats<T, D, 2>(a, x.causal, s);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    hipLaunchKernelGGL((rows_kernel<T, D, true>), dim3(rows), dim3(256), 0, s, a);
  } else if (!p.alone) {
    hipLaunchKernelGGL((rows_kernel<T, D, false>), dim3(rows), dim3(256), 0, s, a);
  }
  if ((e = hipGetLastError()) != hipSuccess) return e;
  if (p.columns == 128)
    launch_main<T, D, 4>(a, x.causal, s);
  else
    launch_main<T, D, 2>(a, x.causal, s);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  return p.columns == 128 ? launch_join<T, D, 128>(a, s) : launch_join<T, D, 64>(a, s);
}

// The workspace's parts, each from a multiple of 256 bytes on.
struct Offsets64 {
  int64_t nl, nd, max_do, max_d, max_v, stats, part_k, part_v, part_q, end;
};
Offsets64 offsets(const AttnBwdPlan& p, int dtype, bool anew, int64_t planes_q, int64_t planes_kv, int64_t D) {
  Offsets64 o;
  int64_t at = 0;
  auto take = [&](int64_t floats) {
    const int64_t was = at;
    at += (floats * 4 + 255) / 256 * 256;
    return was;
  };
  const bool f16 = dtype == 0 && !p.alone;
  o.nl = take(p.alone ? 0 : planes_q * p.nb_q * BT);
  o.nd = take(p.alone ? 0 : planes_q * p.nb_q * BT);
  o.max_do = take(f16 ? planes_q * p.nb_q : 0);
  o.max_d = take(f16 ? planes_q * p.nb_q : 0);
  o.max_v = take(f16 ? planes_kv * p.nb_kv : 0);
  o.stats = take(anew ? 3 * (int64_t)p.queries.blocks * 128 : 0);
  o.part_k = take((int64_t)p.keys.cut_blocks * p.columns * D);
  o.part_v = take((int64_t)p.keys.cut_blocks * p.columns * D);
  o.part_q = take((int64_t)p.queries.cut_blocks * p.columns * D);
  o.end = at;
  return o;
}

}  // namespace

int64_t attn_bwd_workspace_bytes(int dtype, bool causal, bool anew, int64_t B, int64_t H, int64_t H_kv, int64_t N,
                                 int64_t N_kv, int64_t D) {
  return offsets(attn_bwd_plan(B, H, H_kv, N, N_kv, D, causal, anew), dtype, anew, B * H, B * H_kv, D).end;
}

hipError_t launch_attn_bwd(const AttnBwdArgs& x, hipStream_t s) {
  const AttnBwdPlan p = attn_bwd_plan(x.B, x.H, x.H_kv, x.N, x.N_kv, x.D, x.causal != 0, !x.lse);
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
  a.keys = p.keys;
  a.queries = p.queries;
  a.alone = p.alone;
  a.columns = (int)p.columns;
  a.sm_scale = x.sm_scale;
  a.c = x.sm_scale * LOG2E_F;
  const Offsets64 o = offsets(p, x.dtype, !x.lse, a.planes_q, a.planes_kv, x.D);
  u8* ws = (u8*)x.workspace;
  a.nl = (float*)(ws + o.nl);
  a.nd = (float*)(ws + o.nd);
  a.max_do = (float*)(ws + o.max_do);
  a.max_d = (float*)(ws + o.max_d);
  a.max_v = (float*)(ws + o.max_v);
  a.stats = (float*)(ws + o.stats);
  a.part_k = (float*)(ws + o.part_k);
  a.part_v = (float*)(ws + o.part_v);
  a.part_q = (float*)(ws + o.part_q);
  if (x.dtype == 0)
    return x.D == 64 ? launch<f16, 64>(x, p, a, s) : launch<f16, 128>(x, p, a, s);
  return x.D == 64 ? launch<bf16, 64>(x, p, a, s) : launch<bf16, 128>(x, p, a, s);
}

}  // namespace sage
