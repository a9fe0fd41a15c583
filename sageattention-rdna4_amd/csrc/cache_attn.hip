// Attention of a sequence's newest tokens over its quantized K/V cache (gfx950): one token per
// sequence (decoding), a few in a row, or a tree of drafted ones.
//
// For a row (new token i, head h) and the cached tokens j that it sees, with q of 16 bits and k_j =
// K8_j SK_j, v_j = V8_j SV_j as the cache holds them:
//     t_j = (q . K8_j) SK_j sm_scale log2 e,   o = sum_j 2^t_j v_j / sum_j 2^t_j.
// The codes are exact in fp16 and in bf16, so q . K8_j is a 16-bit MFMA with fp32 sums and no rounding
// of its own. The weight that meets V8 includes V's scale: with u_j = t_j + log2 SV_j and the running
// row maximum m of u,
//     w_j = 2^(u_j - m + 14),   o = (sum_j w_j V8_j) / (sum_j w_j / SV_j):
// w is at most 2^14 whatever the scales, so it is rounded to fp16 (half a step of 2^-11, a quarter of
// what a bf16 weight would lose) without overflow, and 28 binades below a row's largest weight are
// still normal numbers. Sums, maxima and outputs are fp32 until the one rounding of the output.
//
// Layout. A wave holds 16 R rows of one K/V head (row r: token r / G, head r % G of the group) and
// takes 64 keys, a page, at a time: S^T = K Q^T by 16x16x32 MFMAs (keys down, rows across), whose
// results are, lane for lane, the B operand of O^T = V^T W^T when the keys are taken in the order
// 4g .. 4g+3 of two 16-key tiles (g the lane's group of 16). Weights never leave their lanes. A row of
// V is read 16 lanes wide and its bytes converted one by one into the operand whose element is the key.
// What depends on a key alone (ks, lv, 1/SV) is worked out by one lane for each key.
//
// Two kernels share that step:
//   stream: up to 32 rows of a K/V head (decoding, small trees). HBM-bound: each wave has pages of its
//           own, straight from memory to registers, and a block's waves are merged through LDS.
//   shared: more rows. MFMA- and VALU-bound: a block's four waves have rows of their own and share
//           each page, of which every wave converts a quarter to 16 bits in LDS.
// Either cuts a sequence's pages into S interleaved parts, which a second launch joins in order.
#include "sage_device.h"
#include "sage_launch.h"

namespace sage {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr float W_SHIFT = 14.0f;    // weights are at most 2^14
constexpr float SV_LEAST = 0x1p-100f;
constexpr float NEG_INF = -__builtin_inff();
constexpr float LN2_F = 0.6931471805599453f;

template <typename T>
struct Frag;
template <>
struct Frag<f16> {
  typedef f16x8 type;
};
template <>
struct Frag<bf16> {
  typedef bf16x8 type;
};

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// 8 codes as 8 values of the query's type (exact).
template <typename T, bool KINT8>
__device__ __forceinline__ typename Frag<T>::type k_frag(u32 lo, u32 hi) {
  typename Frag<T>::type f;
  if constexpr (KINT8) {
    // bytes + 128 behind the exponent of 1024 are 1152 + code
    u32 w[4];
    const u32 in[2] = {lo ^ 0x80808080u, hi ^ 0x80808080u};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w[2 * i] = __builtin_amdgcn_perm(0x64646464u, in[i], 0x04010400u);
      w[2 * i + 1] = __builtin_amdgcn_perm(0x64646464u, in[i], 0x04030402u);
    }
    __builtin_memcpy(&f, w, 16);
    f -= (f16)1152.0f;
  } else {
    const u32 in[2] = {lo, hi};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if constexpr (std::is_same_v<T, f16>) {
          const f16x2 x = j ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(in[i], 1.0f, true)
                            : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(in[i], 1.0f, false);
          f[4 * i + 2 * j] = x[0], f[4 * i + 2 * j + 1] = x[1];
        } else {
          const bf16x2 x = j ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(in[i], 1.0f, true)
                             : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(in[i], 1.0f, false);
          f[4 * i + 2 * j] = x[0], f[4 * i + 2 * j + 1] = x[1];
        }
      }
  }
  return f;
}

// Byte E of four keys' words, and of four more, as 8 fp16 values (exact).
template <int E>
__device__ __forceinline__ f16x8 v_frag(const u32 (&a)[4], const u32 (&b)[4]) {
  f16x8 f;
  static_for<0, 4>([&](auto ic) {
    constexpr int i = 2 * (decltype(ic)::value % 2);
    const u32* w = decltype(ic)::value < 2 ? a : b;
    f16x2 x = {};
    x = __builtin_amdgcn_cvt_scalef32_f16_fp8(x, (int)w[i], 1.0f, E, false);
    x = __builtin_amdgcn_cvt_scalef32_f16_fp8(x, (int)w[i + 1], 1.0f, E, true);
    f[2 * decltype(ic)::value] = x[0];
    f[2 * decltype(ic)::value + 1] = x[1];
  });
  return f;
}

__device__ __forceinline__ float max_groups(float x) {
  x = fmaxf(x, __shfl_xor(x, 16, 64));
  return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float sum_groups(float x) {
  x += __shfl_xor(x, 16, 64);
  return x + __shfl_xor(x, 32, 64);
}

struct Shape {
  // pool
  const u8* k8;
  const float* sk;
  const u8* v8;
  const float* sv;
  const int* table;
  int64_t t_sb;
  int max_pages, num_pages;
  // queries
  const void* q;
  int64_t q_sb, q_sh, q_sr;
  const int* kv_lens;
  const int* q_lens;
  const u8* mask;
  int64_t m_sb, m_sr;
  void* o;
  int64_t o_sb, o_sh, o_sr;
  float* lse;
  float* part_o;    // (tiles, S, rows of a block, D)
  float* part_ml;   // (tiles, S, rows of a block, 2)
  int H, H_kv, G, T, S, RB, units;
  float c;          // sm_scale log2 e
};

struct Lens {
  int keys;     // cached tokens that the table has pages for
  int kv;       // cached tokens, as given
  int tokens;   // new tokens
};
__device__ __forceinline__ Lens lens_of(const Shape& p, int b) {
  Lens n;
  n.kv = p.kv_lens[b];
  n.kv = n.kv < 0 ? 0 : n.kv;
  const int64_t held = (int64_t)p.max_pages * NPAD;
  n.keys = (int64_t)n.kv < held ? n.kv : (int)held;
  n.tokens = p.q_lens ? p.q_lens[b] : p.T;
  n.tokens = n.tokens < 0 ? 0 : n.tokens > p.T ? p.T : n.tokens;
  return n;
}

// Block -> (plane, part, row block): the row blocks of one part of a plane's pages run on one XCD (blocks
// go round the 8 XCDs), whose L2 then holds the pages that they all read.
struct Place {
  int plane, b, hk, split, rb;
  int64_t part;   // number of (plane, split, row block)
  bool live;
};
__device__ __forceinline__ Place place_of(const Shape& p) {
  Place w;
  const u32 id = blockIdx.x, oct = id / (8u * (u32)p.RB), in = id - oct * 8u * (u32)p.RB;
  w.rb = (int)(in / 8u);
  const u32 unit = oct * 8u + in % 8u;
  w.live = unit < (u32)p.units;
  w.plane = (int)(unit / (u32)p.S);
  w.split = (int)(unit - (u32)w.plane * (u32)p.S);
  w.b = w.plane / p.H_kv;
  w.hk = w.plane - w.b * p.H_kv;
  w.part = (int64_t)unit * p.RB + w.rb;
  return w;
}

// A wave's rows and running sums.
template <typename T, int D, int R>
struct Rows {
  typename Frag<T>::type q[R][D / 32];
  int token[R];
  f32x4 acc[R][D / 16];
  float m[R], l[R];

  // lane l15 holds row l15 of each 16, columns 64c + 16g + 8s in k-step 2c + s
  __device__ __forceinline__ void load(const Shape& p, int b, int hk, int row0, int l15, int g) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = row0 + 16 * r + l15;
      token[r] = row / p.G;
      const int h = hk * p.G + row - token[r] * p.G;
      const bool live = token[r] < p.T;
      const T* src = (const T*)p.q + b * p.q_sb + (live ? h * p.q_sh + token[r] * p.q_sr : 0) + 16 * g;
#pragma unroll
      for (int t = 0; t < D / 32; ++t) {
        u32x4 w = *(const u32x4*)(src + 64 * (t >> 1) + 8 * (t & 1));
        if (!live) w = (u32x4){0, 0, 0, 0};
        __builtin_memcpy(&q[r][t], &w, 16);
      }
      m[r] = NEG_INF, l[r] = 0.0f;
#pragma unroll
      for (int e = 0; e < D / 16; ++e) acc[r][e] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    }
  }
};

// What the softmax needs of each key, by one lane a key, into 3 x 64 floats: SK sm_scale log2 e, log2 SV
// and 1 / SV. A scale of 0 (a token never written) weighs as its key says and adds zeros; one of NaN (a
// row that is not finite) makes the weights of the rows that see it NaN, and 1/SV 0, so that the
// others' weights of 0 leave their sums alone. So do keys behind the sequence's end.
__device__ __forceinline__ void key_consts(float* dst, int key, float sk, float sv, float c, bool held) {
  const float v = sv < SV_LEAST ? SV_LEAST : sv;
  dst[key] = sk * c;
  dst[64 + key] = __builtin_amdgcn_logf(v);
  dst[128 + key] = held ? fmaxf(__builtin_amdgcn_rcpf(v), 0.0f) : 0.0f;
}

// Scores to weights: u = t + log2 SV, where the page holds new tokens or ends the sequence only for the
// keys that each row sees; then the running maximum and sum, and the weights as the PV MFMA takes them.
template <typename T, int D, int R>
__device__ __forceinline__ void softmax_step(const Shape& p, const Lens& n, int b, int key0,
                                             const float* consts, int g, Rows<T, D, R>& w,
                                             f32x4 (&s)[R][4], f16x8 (&wf)[R][2]) {
  const int prefix = n.kv - n.tokens;    // tokens that every new token sees
#pragma unroll
  for (int kt = 0; kt < 4; ++kt) {
    const f32x4 ks = *(const f32x4*)(consts + 16 * kt + 4 * g);
    const f32x4 lv = *(const f32x4*)(consts + 64 + 16 * kt + 4 * g);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[r][kt][i] = __builtin_fmaf(s[r][kt][i], ks[i], lv[i]);
  }
  if (key0 + NPAD > prefix || key0 + NPAD > n.keys) {
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = key0 + 16 * kt + 4 * g + i, draft = key - prefix;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          bool seen = key < n.keys;
          if (seen && draft >= 0) {
            if (p.mask)
              seen = w.token[r] < n.tokens && p.mask[b * p.m_sb + w.token[r] * p.m_sr + draft] != 0;
            else
              seen = draft <= w.token[r];
          }
          s[r][kt][i] = seen ? s[r][kt][i] : NEG_INF;
        }
      }
  }
  float top[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    top[r] = NEG_INF;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) top[r] = fmaxf(top[r], s[r][kt][i]);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) top[r] = max_groups(top[r]);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (__builtin_amdgcn_ballot_w64(top[r] > w.m[r])) {
      const float now = fmaxf(top[r], w.m[r]);
      // a row that has seen nothing keeps sums of zero
      const float alpha = __builtin_amdgcn_exp2f(w.m[r] - (now == NEG_INF ? 0.0f : now));
      w.m[r] = now;
      w.l[r] *= alpha;
#pragma unroll
      for (int e = 0; e < D / 16; ++e) w.acc[r][e] *= alpha;
    }
    const float shift = (w.m[r] == NEG_INF ? 0.0f : w.m[r]) - W_SHIFT;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      const f32x4 rsv = *(const f32x4*)(consts + 128 + 16 * kt + 4 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = __builtin_amdgcn_exp2f(s[r][kt][i] - shift);
        w.l[r] = __builtin_fmaf(x, rsv[i], w.l[r]);
        wf[r][kt >> 1][4 * (kt & 1) + i] = (f16)x;
      }
    }
  }
}

// N columns of an output row.
template <typename T, int N>
__device__ __forceinline__ void store_row(T* o, const float (&f)[N], float inv, bool some) {
  T out[N];
#pragma unroll
  for (int e = 0; e < N; ++e) out[e] = (T)(some ? f[e] * inv : 0.0f);
  if constexpr (N == 8) {
    u32x4 w;
    __builtin_memcpy(&w, out, 16);
    *(u32x4*)o = w;
  } else if constexpr (N == 4) {
    u32x2 w;
    __builtin_memcpy(&w, out, 8);
    *(u32x2*)o = w;
  } else {
    u32 w;
    __builtin_memcpy(&w, out, 4);
    *(u32*)o = w;
  }
}

__device__ __forceinline__ float lse_of(float top, float sum) {
  return (top - W_SHIFT + __log2f(sum)) * LN2_F;
}

// A row's N columns from col on: to the output where the call has one part, else to the workspace
// (at row `at` of the parts), where nothing is read that a part with a sum of 0 did not write.
template <typename T, int D, int N>
__device__ __forceinline__ void finish_row(const Shape& p, const Lens& n, int b, int hk, int row,
                                           int64_t at, int col, const float (&f)[N], float top,
                                           float sum) {
  const int tok = row / p.G, h = hk * p.G + row - tok * p.G;
  if (tok >= p.T) return;
  if (p.S > 1) {
    if (col == 0) *(float2*)(p.part_ml + 2 * at) = make_float2(top, sum);
    if (sum != 0.0f) {
#pragma unroll
      for (int e = 0; e < N; e += 4)
        *(f32x4*)(p.part_o + at * D + col + e) = (f32x4){f[e], f[e + 1], f[e + 2], f[e + 3]};
    }
    return;
  }
  const bool some = tok < n.tokens && sum != 0.0f;
  store_row<T, N>((T*)p.o + b * p.o_sb + h * p.o_sh + tok * p.o_sr + col, f, some ? 1.0f / sum : 0.0f,
                  some);
  if (p.lse && col == 0)
    p.lse[((int64_t)b * p.H + h) * p.T + tok] = some ? lse_of(top, sum) : NEG_INF;
}

// grid: one block per part of a plane (row blocks: 1). Wave w of part s takes pages s W + w, then every
// (S W)-th: which these are does not wait for the sequence's length.
template <typename T, bool KINT8, int D, int R, int W>
__global__ __launch_bounds__(64 * W, 2) void cache_attn_stream_kernel(Shape p) {
  typedef typename Frag<T>::type frag;
  constexpr int KC = D / 64, KT = D / 32, VE = D / 16, VW = VE / 4, LD = D + 4;
  __shared__ __attribute__((aligned(16))) float lds_o[W][16][LD];
  __shared__ float lds_ml[W][16][2];
  __shared__ __attribute__((aligned(16))) float lds_c[W][192];

  const int lane = threadIdx.x & 63, l15 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Place at = place_of(p);
  if (!at.live) return;
  const int b = at.b, hk = at.hk;
  const Lens n = lens_of(p, b);
  Rows<T, D, R> w;
  w.load(p, b, hk, 0, l15, g);

  const int pages = n.tokens > 0 ? (n.keys + NPAD - 1) / NPAD : 0;
  const int* table = p.table + b * p.t_sb;
  for (int pg = at.split * W + wave; pg < pages; pg += p.S * W) {
    const int id = __builtin_amdgcn_readfirstlane(table[pg]);
    if (id < 0 || id >= p.num_pages) continue;   // no page: nothing to see
    const int64_t base = ((int64_t)id * p.H_kv + hk) * NPAD;
    const u8* kp = p.k8 + base * D + (int64_t)l15 * D + 16 * g;
    const u8* vp = p.v8 + base * D + (int64_t)(4 * g) * D + l15 * VE;
    const float sk = p.sk[base + lane], sv = p.sv[base + lane];
    u32x4 kw[4][KC];
    u32 vw[4][VW][4];   // [key tile][word of the row's 4 VW bytes][key 4g + j]
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int c = 0; c < KC; ++c) kw[kt][c] = *(const u32x4*)(kp + 16 * kt * D + 64 * c);
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u8* src = vp + (16 * kt + j) * D;
        if constexpr (VW == 2) {
          const u32x2 x = *(const u32x2*)src;
          vw[kt][0][j] = x[0], vw[kt][1][j] = x[1];
        } else {
          vw[kt][0][j] = *(const u32*)src;
        }
      }
    const int key0 = pg * NPAD;
    key_consts(lds_c[wave], lane, sk, sv, p.c, key0 + lane < n.keys);

    f32x4 s[R][4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
      for (int r = 0; r < R; ++r) s[r][kt] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        const frag kf = k_frag<T, KINT8>(kw[kt][t >> 1][2 * (t & 1)], kw[kt][t >> 1][2 * (t & 1) + 1]);
#pragma unroll
        for (int r = 0; r < R; ++r) s[r][kt] = mfma(kf, w.q[r][t], s[r][kt]);
      }
    }
    if (key0 + NPAD > n.keys) {   // whatever lies behind the end: no NaN may meet a weight of zero
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (key0 + 16 * kt + 4 * g + j >= n.keys) {
#pragma unroll
            for (int x = 0; x < VW; ++x) vw[kt][x][j] = 0;
          }
    }
    f16x8 wf[R][2];
    softmax_step<T, D, R>(p, n, b, key0, lds_c[wave], g, w, s, wf);

    // O^T += V^T W^T: tile e's row x is column VE x + e
    static_for<0, 2>([&](auto uc) {
      constexpr int u = decltype(uc)::value;
      static_for<0, VE>([&](auto ec) {
        constexpr int e = decltype(ec)::value;
        const f16x8 vf = v_frag<e % 4>(vw[2 * u][e / 4], vw[2 * u + 1][e / 4]);
#pragma unroll
        for (int r = 0; r < R; ++r) w.acc[r][e] = mfma(vf, wf[r][u], w.acc[r][e]);
      });
    });
  }

  // the waves' results merged, 16 rows at a time; each thread has N columns of a row
  constexpr int TPR = 4 * W, N = D / TPR;   // threads of a row
  const int tid = threadIdx.x, orow = tid / TPR, ocol = (tid % TPR) * N;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float total = sum_groups(w.l[r]);
    if (r) __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < VE; e += 4)
        *(f32x4*)&lds_o[wave][l15][VE * (4 * g + i) + e] =
            (f32x4){w.acc[r][e][i], w.acc[r][e + 1][i], w.acc[r][e + 2][i], w.acc[r][e + 3][i]};
    if (g == 0) lds_ml[wave][l15][0] = w.m[r], lds_ml[wave][l15][1] = total;
    __syncthreads();
    float top = NEG_INF;
#pragma unroll
    for (int x = 0; x < W; ++x) top = fmaxf(top, lds_ml[x][orow][0]);
    const float use = top == NEG_INF ? 0.0f : top;
    float sum = 0.0f, f[N] = {};
#pragma unroll
    for (int x = 0; x < W; ++x) {
      const float a = __builtin_amdgcn_exp2f(lds_ml[x][orow][0] - use);
      sum += lds_ml[x][orow][1] * a;
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] += lds_o[x][orow][ocol + e] * a;
    }
    finish_row<T, D, N>(p, n, b, hk, 16 * r + orow, at.part * (16 * R) + 16 * r + orow, ocol, f, top, sum);
  }
}

// grid: row blocks of 64 R rows x parts of a plane. Part s takes pages s, s + S, ... The page in work
// lies in LDS as the MFMAs' operands (K: key tile x k-step, V: half x column tile; 1 KB each, one
// 16-byte piece a lane), the next one's bytes in registers: wave w converts key tile w of K and four
// operands of V.
template <typename T, bool KINT8, int D, int R>
__global__ __launch_bounds__(256, 2) void cache_attn_shared_kernel(Shape p) {
  typedef typename Frag<T>::type frag;
  constexpr int KC = D / 64, KT = D / 32, VE = D / 16, NV = 2 * VE / 4, ROWS = 64 * R;
  __shared__ __attribute__((aligned(16))) u32x4 lds_k[2][4][KT][64];
  __shared__ __attribute__((aligned(16))) u32x4 lds_v[2][2][VE][64];
  __shared__ __attribute__((aligned(16))) float lds_c[2][192];

  const int lane = threadIdx.x & 63, l15 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Place at = place_of(p);
  if (!at.live) return;
  const int b = at.b, hk = at.hk;
  const Lens n = lens_of(p, b);
  const int row0 = at.rb * ROWS + 16 * R * wave;
  Rows<T, D, R> w;
  w.load(p, b, hk, row0, l15, g);

  const int pages = at.rb * ROWS < n.tokens * p.G ? (n.keys + NPAD - 1) / NPAD : 0;
  const int* table = p.table + b * p.t_sb;
  // operands u = wave / 2, e = first .. first + NV - 1 of V: bytes of word `word` of a row's VE
  const int vu = wave >> 1, vfirst = (wave & 1) * NV;
  u32x4 kw[KC];
  u32 vw[2][4];
  float sk = 0.0f, sv = 0.0f;
  bool there = false;
  auto fetch = [&](int pg) {
    const int id = pg < pages ? __builtin_amdgcn_readfirstlane(table[pg]) : -1;
    there = id >= 0 && id < p.num_pages;
    if (!there) return;
    const int64_t base = ((int64_t)id * p.H_kv + hk) * NPAD;
    const u8* kp = p.k8 + (base + 16 * wave + l15) * D + 16 * g;
#pragma unroll
    for (int c = 0; c < KC; ++c) kw[c] = *(const u32x4*)(kp + 64 * c);
    const u8* vp = p.v8 + (base + 32 * vu + 4 * g) * D + l15 * VE + (VE == 8 ? vfirst : 0);
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int j = 0; j < 4; ++j) vw[x][j] = *(const u32*)(vp + (16 * x + j) * D);
    if (wave == 0) sk = p.sk[base + lane], sv = p.sv[base + lane];
  };
  auto convert = [&](int pg, int buf) {
    if (!there) return;
    const int key0 = pg * NPAD;
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      const frag f = k_frag<T, KINT8>(kw[t >> 1][2 * (t & 1)], kw[t >> 1][2 * (t & 1) + 1]);
      __builtin_memcpy(&lds_k[buf][wave][t][lane], &f, 16);
    }
    if (key0 + NPAD > n.keys) {   // whatever lies behind the end: no NaN may meet a weight of zero
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (key0 + 32 * vu + 16 * x + 4 * g + j >= n.keys) vw[x][j] = 0;
    }
    static_for<0, 4>([&](auto ec) {
      constexpr int e = decltype(ec)::value;
      if constexpr (NV == 4) {
        const f16x8 f = v_frag<e>(vw[0], vw[1]);
        __builtin_memcpy(&lds_v[buf][vu][vfirst + e][lane], &f, 16);
      } else if (e / NV == (wave & 1)) {
        const f16x8 f = v_frag<e>(vw[0], vw[1]);
        __builtin_memcpy(&lds_v[buf][vu][e][lane], &f, 16);
      }
    });
    if (wave == 0) key_consts(lds_c[buf], lane, sk, sv, p.c, key0 + lane < n.keys);
  };

  int pg = at.split, buf = 0;
  fetch(pg);
  convert(pg, 0);
  bool work = there;   // whether the page in LDS is one
  __syncthreads();
  for (; pg < pages; pg += p.S) {
    fetch(pg + p.S);
    if (work) {
      f32x4 s[R][4];
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
        for (int r = 0; r < R; ++r) s[r][kt] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          frag kf;
          __builtin_memcpy(&kf, &lds_k[buf][kt][t][lane], 16);
#pragma unroll
          for (int r = 0; r < R; ++r) s[r][kt] = mfma(kf, w.q[r][t], s[r][kt]);
        }
      }
      f16x8 wf[R][2];
      softmax_step<T, D, R>(p, n, b, pg * NPAD, lds_c[buf], g, w, s, wf);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          f16x8 vf;
          __builtin_memcpy(&vf, &lds_v[buf][u][e][lane], 16);
#pragma unroll
          for (int r = 0; r < R; ++r) w.acc[r][e] = mfma(vf, wf[r][u], w.acc[r][e]);
        }
    }
    convert(pg + p.S, buf ^ 1);   // the other buffer: its readers passed the last barrier
    work = there;
    buf ^= 1;
    __syncthreads();
  }

#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float sum = sum_groups(w.l[r]);
    const int row = row0 + 16 * r + l15;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) f[e] = w.acc[r][e][i];
      finish_row<T, D, VE>(p, n, b, hk, row, at.part * ROWS + row - at.rb * ROWS, VE * (4 * g + i), f,
                           w.m[r], sum);
    }
  }
}

// The parts joined, in their order: a wave per output row, D/64 columns a lane; lane s first has the
// part s's maximum and sum (S is at most 64).
template <typename T, int D>
__global__ __launch_bounds__(256) void cache_attn_join_kernel(Shape p, int rows_per_block, u32 rows) {
  constexpr int N = D / 64;
  const int lane = threadIdx.x & 63;
  const u32 at = __builtin_amdgcn_readfirstlane(blockIdx.x * 4u + (threadIdx.x >> 6));
  if (at >= rows) return;
  // rows in the order (b, K/V head, row of the plane)
  const u32 M = (u32)p.T * (u32)p.G;
  const u32 plane = at / M, row = at - plane * M;
  const int b = (int)(plane / (u32)p.H_kv), hk = (int)(plane - (u32)b * (u32)p.H_kv);
  const int tok = (int)(row / (u32)p.G), h = hk * p.G + (int)row - tok * p.G;
  const Lens n = lens_of(p, b);
  const u32 rb = row / (u32)rows_per_block, in = row - rb * (u32)rows_per_block;
  const int64_t first = ((int64_t)plane * p.S * p.RB + rb) * rows_per_block + in;
  const int64_t step = (int64_t)p.RB * rows_per_block;
  float2 ml = make_float2(NEG_INF, 0.0f);
  if (lane < p.S) ml = *(const float2*)(p.part_ml + 2 * (first + lane * step));
  float top = ml.x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  const float a = __builtin_amdgcn_exp2f(ml.x - (top == NEG_INF ? 0.0f : top));
  const bool full = ml.y != 0.0f;
  float sum = full ? ml.y * a : 0.0f;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
  const uint64_t parts = __builtin_amdgcn_ballot_w64(full);
  float f[N] = {};
  const float* src = p.part_o + first * D + lane * N;
  for (int s0 = 0; s0 < p.S; s0 += 8) {   // eight parts requested together
    float x[8][N];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int s = s0 + i < p.S ? s0 + i : p.S - 1;
#pragma unroll
      for (int e = 0; e < N; ++e) x[i][e] = src[s * step * D + e];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int s = s0 + i;
      if (s >= p.S || !((parts >> s) & 1)) continue;
      const float as = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(a), s));
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] += x[i][e] * as;
    }
  }
  const bool some = tok < n.tokens && sum != 0.0f;
  const float inv = some ? 1.0f / sum : 0.0f;
  T* o = (T*)p.o + b * p.o_sb + h * p.o_sh + tok * p.o_sr + lane * N;
  if constexpr (N == 2)
    store_row<T, 2>(o, f, inv, some);
  else
    *o = (T)(some ? f[0] * inv : 0.0f);
  if (p.lse && lane == 0)
    p.lse[((int64_t)b * p.H + h) * p.T + tok] = some ? lse_of(top, sum) : NEG_INF;
}

template <typename T, bool KINT8, int D>
hipError_t run(const CacheAttnArgs& a, hipStream_t st) {
  const CacheAttnPlan plan = cache_attn_plan(a.B, a.H, a.H_kv, a.T, a.pool.max_pages);
  Shape p;
  p.k8 = (const u8*)a.pool.k8;
  p.sk = a.pool.sk;
  p.v8 = (const u8*)a.pool.v8;
  p.sv = a.pool.sv;
  p.table = a.pool.table;
  p.t_sb = a.pool.t_sb;
  p.max_pages = (int)a.pool.max_pages;
  p.num_pages = (int)a.pool.num_pages;
  p.q = a.q;
  p.q_sb = a.q_sb;
  p.q_sh = a.q_sh;
  p.q_sr = a.q_sr;
  p.kv_lens = a.kv_lens;
  p.q_lens = a.q_lens;
  p.mask = (const u8*)a.mask;
  p.m_sb = a.m_sb;
  p.m_sr = a.m_sr;
  p.o = a.o;
  p.o_sb = a.o_sb;
  p.o_sh = a.o_sh;
  p.o_sr = a.o_sr;
  p.lse = a.lse;
  p.H = (int)a.H;
  p.H_kv = (int)a.H_kv;
  p.G = (int)(a.H / a.H_kv);
  p.T = (int)a.T;
  p.S = (int)plan.splits;
  p.RB = (int)plan.row_blocks;
  p.units = (int)plan.units;
  p.c = a.sm_scale * LOG2E_F;
  p.part_o = (float*)a.workspace;
  p.part_ml = p.part_o + plan.units * plan.row_blocks * plan.rows * D;
  const u32 blocks = (u32)plan.blocks;
  if (plan.rows == 16)
    cache_attn_stream_kernel<T, KINT8, D, 1, 4><<<blocks, 256, 0, st>>>(p);
  else if (plan.rows == 32)
    cache_attn_stream_kernel<T, KINT8, D, 2, 4><<<blocks, 256, 0, st>>>(p);
  else if (plan.rows == 64)
    cache_attn_shared_kernel<T, KINT8, D, 1><<<blocks, 256, 0, st>>>(p);
  else
    cache_attn_shared_kernel<T, KINT8, D, 2><<<blocks, 256, 0, st>>>(p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || plan.splits == 1) return e;
  const int64_t rows = a.B * a.H * a.T;
  cache_attn_join_kernel<T, D><<<(u32)((rows + 3) / 4), 256, 0, st>>>(p, (int)plan.rows, (u32)rows);
  return hipGetLastError();
}

template <int D>
hipError_t run_d(const CacheAttnArgs& a, hipStream_t st) {
  if (a.dtype == 1) return run<bf16, false, D>(a, st);
  return a.pool.k_int8 ? run<f16, true, D>(a, st) : run<f16, false, D>(a, st);
}

}  // namespace

CacheAttnPlan cache_attn_plan(int64_t B, int64_t H, int64_t H_kv, int64_t T, int64_t max_pages) {
  CacheAttnPlan p;
  const int64_t M = T * (H / H_kv), planes = B * H_kv;
  p.rows = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
  p.row_blocks = (M + p.rows - 1) / p.rows;
  const int64_t tiles = planes * p.row_blocks;
  const bool stream = p.rows <= 32;
  // stream: four blocks' worth of work for each compute unit, so that sequences of different lengths
  // even out, and a page at least for each wave; shared: two
  int64_t s = ((stream ? 1024 : 512) + tiles - 1) / tiles;
  const int64_t most = stream ? (max_pages + 3) / 4 : max_pages;
  if (s > most) s = most;
  if (s > 64) s = 64;
  p.splits = s < 1 ? 1 : s;
  p.units = planes * p.splits;
  p.blocks = (p.units + 7) / 8 * 8 * p.row_blocks;
  return p;
}

size_t cache_attn_workspace_bytes(const CacheAttnPlan& p, int64_t D) {
  return p.splits > 1 ? (size_t)(p.units * p.row_blocks * p.rows * (D + 2)) * sizeof(float) : 0;
}

hipError_t launch_cache_attn(const CacheAttnArgs& a, hipStream_t st) {
  return a.D == 128 ? run_d<128>(a, st) : run_d<64>(a, st);
}

}  // namespace sage
