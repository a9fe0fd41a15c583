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
// Layout. A wave holds 16 R rows of one K/V head (row r: token r / G, head r % G of the group), and
// takes a page of 64 keys at a time straight from memory to registers: S^T = K Q^T by 16x16x32 MFMAs
// (keys down, rows across), whose results are, lane for lane, the B operand of O^T = V^T W^T when
// the keys are taken in the order 4g .. 4g+3 of two 16-key tiles (g the lane's group of 16). Weights
// never leave their lanes. A row of V is read 16 lanes wide and its bytes converted one by one into
// the operand whose element is the key.
#include "sage_device.h"
#include "sage_launch.h"

namespace sage {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int WAVES = 4;            // of a block
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
  int H, H_kv, G, T, S, RB;
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

// grid: block = (tile * S + split), tile = (b * H_kv + K/V head) * RB + row block of 16 R rows. The
// block's waves take its pages in turn and are merged through LDS.
template <typename T, bool KINT8, int D, int R>
__global__ __launch_bounds__(64 * WAVES) void cache_attn_kernel(Shape p) {
  typedef typename Frag<T>::type frag;
  constexpr int KC = D / 64, KT = D / 32, VE = D / 16, VW = VE / 4, ROWS = 16 * R, LD = D + 4;
  __shared__ __attribute__((aligned(16))) float lds_o[WAVES][16][LD];
  __shared__ float lds_ml[WAVES][16][2];

  const int lane = threadIdx.x & 63, l15 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const u32 tile = blockIdx.x / (u32)p.S, split = blockIdx.x - tile * (u32)p.S;
  const u32 plane = tile / (u32)p.RB;
  const int rb = (int)(tile - plane * (u32)p.RB);
  const int b = (int)(plane / (u32)p.H_kv), hk = (int)(plane - (u32)b * (u32)p.H_kv);
  const Lens n = lens_of(p, b);
  const int prefix = n.kv - n.tokens;    // tokens that every new token sees
  const int row0 = rb * ROWS;

  // rows of Q: lane l15 holds row l15 of each 16, columns 64c + 16g + 8s in k-step 2c + s
  frag qf[R][KT];
  int token[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = row0 + 16 * r + l15;
    token[r] = row / p.G;
    const int h = hk * p.G + row - token[r] * p.G;
    const bool live = token[r] < p.T;
    const T* q = (const T*)p.q + b * p.q_sb + (live ? h * p.q_sh + token[r] * p.q_sr : 0) + 16 * g;
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      u32x4 w = *(const u32x4*)(q + 64 * (t >> 1) + 8 * (t & 1));
      if (!live) w = (u32x4){0, 0, 0, 0};
      __builtin_memcpy(&qf[r][t], &w, 16);
    }
  }

  f32x4 acc[R][VE];
  float m[R], l[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = NEG_INF, l[r] = 0.0f;
#pragma unroll
    for (int e = 0; e < VE; ++e) acc[r][e] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  }

  const int pages = row0 < n.tokens * p.G ? (n.keys + NPAD - 1) / NPAD : 0;
  const int per = (pages + p.S - 1) / p.S;
  const int first = (int)split * per, last = first + per < pages ? first + per : pages;
  const int* table = p.table + b * p.t_sb;

  for (int pg = first + wave; pg < last; pg += WAVES) {
    const int id = __builtin_amdgcn_readfirstlane(table[pg]);
    if (id < 0 || id >= p.num_pages) continue;   // no page: nothing to see
    const int64_t base = ((int64_t)id * p.H_kv + hk) * NPAD;
    const u8* kp = p.k8 + base * D + (int64_t)l15 * D + 16 * g;
    const u8* vp = p.v8 + base * D + (int64_t)(4 * g) * D + l15 * VE;
    u32x4 kw[4][KC];
    u32 vw[4][VW][4];   // [key tile][word of the row's 4 VW bytes][key 4g + j]
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int c = 0; c < KC; ++c) kw[kt][c] = *(const u32x4*)(kp + 16 * kt * D + 64 * c);
    f32x4 sk[4], sv[4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      sk[kt] = *(const f32x4*)(p.sk + base + 16 * kt + 4 * g);
      sv[kt] = *(const f32x4*)(p.sv + base + 16 * kt + 4 * g);
    }
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u8* at = vp + (16 * kt + j) * D;
        if constexpr (VW == 2) {
          const u32x2 w = *(const u32x2*)at;
          vw[kt][0][j] = w[0], vw[kt][1][j] = w[1];
        } else {
          vw[kt][0][j] = *(const u32*)at;
        }
      }

    // S^T, then u = t + log2 SV
    f32x4 s[R][4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
      for (int r = 0; r < R; ++r) s[r][kt] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        const frag kf = k_frag<T, KINT8>(kw[kt][t >> 1][2 * (t & 1)], kw[kt][t >> 1][2 * (t & 1) + 1]);
#pragma unroll
        for (int r = 0; r < R; ++r) s[r][kt] = mfma(kf, qf[r][t], s[r][kt]);
      }
    }
    f32x4 rsv[4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // a scale of 0 (a token never written) weighs as its key says and adds zeros; one of NaN (a row
        // that is not finite) makes the weights of the rows that see it NaN, and 1/SV 0, so that the
        // others' weights of 0 leave their sums alone
        const float v = sv[kt][i] < SV_LEAST ? SV_LEAST : sv[kt][i];
        const float lv = __builtin_amdgcn_logf(v), ks = sk[kt][i] * p.c;
        rsv[kt][i] = fmaxf(__builtin_amdgcn_rcpf(v), 0.0f);
#pragma unroll
        for (int r = 0; r < R; ++r) s[r][kt][i] = __builtin_fmaf(s[r][kt][i], ks, lv);
      }

    const int key0 = pg * NPAD;
    if (key0 + NPAD > prefix || key0 + NPAD > n.keys) {
      // the page holds new tokens or ends the sequence: each row sees what its mask leaves it
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = key0 + 16 * kt + 4 * g + i, draft = key - prefix;
          const bool held = key < n.keys;
          if (!held) {   // whatever lies behind the sequence's end: no NaN may meet a zero weight
            rsv[kt][i] = 0.0f;
#pragma unroll
            for (int w = 0; w < VW; ++w) vw[kt][w][i] = 0;
          }
#pragma unroll
          for (int r = 0; r < R; ++r) {
            bool seen = held;
            if (held && draft >= 0) {
              if (p.mask)
                seen = token[r] < n.tokens && p.mask[b * p.m_sb + token[r] * p.m_sr + draft] != 0;
              else
                seen = draft <= token[r];
            }
            s[r][kt][i] = seen ? s[r][kt][i] : NEG_INF;
          }
        }
    }

    f16x8 wf[R][2];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = NEG_INF;
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, s[r][kt][i]);
      top = max_groups(top);
      if (__builtin_amdgcn_ballot_w64(top > m[r])) {
        const float now = fmaxf(top, m[r]);
        // a row that has seen nothing keeps sums of zero
        const float alpha = __builtin_amdgcn_exp2f(m[r] - (now == NEG_INF ? 0.0f : now));
        m[r] = now;
        l[r] *= alpha;
#pragma unroll
        for (int e = 0; e < VE; ++e) acc[r][e] *= alpha;
      }
      const float shift = (m[r] == NEG_INF ? 0.0f : m[r]) - W_SHIFT;
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float w = __builtin_amdgcn_exp2f(s[r][kt][i] - shift);
          l[r] = __builtin_fmaf(w, rsv[kt][i], l[r]);
          wf[r][kt >> 1][4 * (kt & 1) + i] = (f16)w;
        }
    }

    // O^T += V^T W^T: tile e's row x is column VE x + e
    static_for<0, 2>([&](auto uc) {
      constexpr int u = decltype(uc)::value;
      static_for<0, VE>([&](auto ec) {
        constexpr int e = decltype(ec)::value;
        const f16x8 vf = v_frag<e % 4>(vw[2 * u][e / 4], vw[2 * u + 1][e / 4]);
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r][e] = mfma(vf, wf[r][u], acc[r][e]);
      });
    });
  }

  // the waves' results merged, 16 rows at a time; thread tid: row tid / 16, columns VE (tid % 16)
  const int tid = threadIdx.x, orow = tid >> 4, ocol = (tid & 15) * VE;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float total = sum_groups(l[r]);
    if (r) __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < VE; e += 4)
        *(f32x4*)&lds_o[wave][l15][VE * (4 * g + i) + e] =
            (f32x4){acc[r][e][i], acc[r][e + 1][i], acc[r][e + 2][i], acc[r][e + 3][i]};
    if (g == 0) lds_ml[wave][l15][0] = m[r], lds_ml[wave][l15][1] = total;
    __syncthreads();
    float top = NEG_INF;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, lds_ml[w][orow][0]);
    const float use = top == NEG_INF ? 0.0f : top;
    float sum = 0.0f, f[8] = {};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float a = __builtin_amdgcn_exp2f(lds_ml[w][orow][0] - use);
      sum += lds_ml[w][orow][1] * a;
#pragma unroll
      for (int e = 0; e < VE; ++e) f[e] += lds_o[w][orow][ocol + e] * a;
    }
    const int row = row0 + 16 * r + orow, tok = row / p.G, h = hk * p.G + row - tok * p.G;
    if (p.S > 1) {
      const int64_t at = (int64_t)blockIdx.x * ROWS + 16 * r + orow;
      if (ocol == 0) *(float2*)(p.part_ml + 2 * at) = make_float2(top, sum);
      if (sum != 0.0f) {
#pragma unroll
        for (int e = 0; e < VE; e += 4)
          *(f32x4*)(p.part_o + at * D + ocol + e) = (f32x4){f[e], f[e + 1], f[e + 2], f[e + 3]};
      }
    } else if (tok < p.T) {
      const bool some = tok < n.tokens && sum != 0.0f;
      const float inv = some ? 1.0f / sum : 0.0f;
      T* o = (T*)p.o + b * p.o_sb + h * p.o_sh + tok * p.o_sr + ocol;
      T out[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) out[e] = (T)(some ? f[e] * inv : 0.0f);
      if constexpr (VE == 8) {
        u32x4 w;
        __builtin_memcpy(&w, out, 16);
        *(u32x4*)o = w;
      } else {
        u32x2 w;
        __builtin_memcpy(&w, out, 8);
        *(u32x2*)o = w;
      }
      if (p.lse && ocol == 0)
        p.lse[((int64_t)b * p.H + h) * p.T + tok] =
            some ? (top - W_SHIFT + __log2f(sum)) * LN2_F : NEG_INF;
    }
  }
}

// The splits' results joined, in the order of the splits: D/4 lanes per output row.
template <typename T, int D>
__global__ __launch_bounds__(256) void cache_attn_join_kernel(Shape p, int rows_per_block, u32 rows) {
  constexpr int LPR = D / 4;
  const u32 t = blockIdx.x * 256u + threadIdx.x;
  const u32 at = t / LPR;
  const int c = (int)(t % LPR) * 4;
  if (at >= rows) return;
  // rows in the order (b, K/V head, row of the plane)
  const u32 M = (u32)p.T * (u32)p.G;
  const u32 plane = at / M, row = at - plane * M;
  const int b = (int)(plane / (u32)p.H_kv), hk = (int)(plane - (u32)b * (u32)p.H_kv);
  const int tok = (int)(row / (u32)p.G), h = hk * p.G + (int)row - tok * p.G;
  const Lens n = lens_of(p, b);
  const u32 rb = row / (u32)rows_per_block;
  const int64_t first = (((int64_t)plane * p.RB + rb) * p.S) * rows_per_block +
                        (row - rb * (u32)rows_per_block);
  float top = NEG_INF, sum = 0.0f;
  f32x4 f = {0.0f, 0.0f, 0.0f, 0.0f};
  if (tok < n.tokens) {
    for (int s = 0; s < p.S; ++s) {
      const float2 ml = *(const float2*)(p.part_ml + 2 * (first + (int64_t)s * rows_per_block));
      top = fmaxf(top, ml.x);
    }
    const float use = top == NEG_INF ? 0.0f : top;
    for (int s = 0; s < p.S; ++s) {
      const int64_t i = first + (int64_t)s * rows_per_block;
      const float2 ml = *(const float2*)(p.part_ml + 2 * i);
      if (ml.y == 0.0f) continue;
      const float a = __builtin_amdgcn_exp2f(ml.x - use);
      sum += ml.y * a;
      f += *(const f32x4*)(p.part_o + i * D + c) * a;
    }
  }
  const bool some = sum != 0.0f;
  const float inv = some ? 1.0f / sum : 0.0f;
  T out[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = (T)(some ? f[e] * inv : 0.0f);
  u32x2 w;
  __builtin_memcpy(&w, out, 8);
  *(u32x2*)((T*)p.o + b * p.o_sb + h * p.o_sh + tok * p.o_sr + c) = w;
  if (p.lse && c == 0)
    p.lse[((int64_t)b * p.H + h) * p.T + tok] = some ? (top - W_SHIFT + __log2f(sum)) * LN2_F : NEG_INF;
}

template <typename T, bool KINT8, int D, int R>
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
  p.c = a.sm_scale * LOG2E_F;
  const int64_t blocks = plan.blocks;
  p.part_o = (float*)a.workspace;
  p.part_ml = p.part_o + blocks * plan.rows * D;
  cache_attn_kernel<T, KINT8, D, R><<<(u32)blocks, 64 * WAVES, 0, st>>>(p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || plan.splits == 1) return e;
  const int64_t rows = a.B * a.H * a.T;
  cache_attn_join_kernel<T, D><<<(u32)((rows * (D / 4) + 255) / 256), 256, 0, st>>>(
      p, (int)plan.rows, (u32)rows);
  return hipGetLastError();
}

template <int D>
hipError_t run_d(const CacheAttnArgs& a, hipStream_t st) {
  if (a.dtype == 1) return run<bf16, false, D, 1>(a, st);
  return a.pool.k_int8 ? run<f16, true, D, 1>(a, st) : run<f16, false, D, 1>(a, st);
}

}  // namespace

CacheAttnPlan cache_attn_plan(int64_t B, int64_t H, int64_t H_kv, int64_t T, int64_t max_pages) {
  CacheAttnPlan p;
  p.rows = 16;
  p.row_blocks = (T * (H / H_kv) + p.rows - 1) / p.rows;
  const int64_t tiles = B * H_kv * p.row_blocks;
  // two blocks per compute unit, and four pages at least for each block
  int64_t s = (512 + tiles - 1) / tiles;
  const int64_t most = (max_pages + WAVES - 1) / WAVES;
  if (s > most) s = most;
  p.splits = s < 1 ? 1 : s;
  p.blocks = tiles * p.splits;
  return p;
}

size_t cache_attn_workspace_bytes(const CacheAttnPlan& p, int64_t D) {
  return p.splits > 1 ? (size_t)(p.blocks * p.rows * (D + 2)) * sizeof(float) : 0;
}

hipError_t launch_cache_attn(const CacheAttnArgs& a, hipStream_t st) {
  return a.D == 128 ? run_d<128>(a, st) : run_d<64>(a, st);
}

}  // namespace sage
