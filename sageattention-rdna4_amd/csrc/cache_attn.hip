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
// w is at most 2^14 whatever the scales, so it is rounded to fp16 (by 2^-11 of it at most, an eighth of what
// a bf16 weight would lose) without overflow, and 28 binades below a row's largest weight are still
// normal numbers. Sums, maxima and outputs are fp32 until the one rounding of the output.
//
// Layout. A wave holds 16 R rows of one K/V head (row r: token r / G, head r % G of the group) and
// takes 64 keys, a page, at a time: S^T = K Q^T by 16x16x32 MFMAs (keys down, rows across), whose
// results are, lane for lane, the B operand of O^T = V^T W^T when the keys are taken in the order
// 4g .. 4g+3 of two 16-key tiles (g the lane's group of 16). Weights never leave their lanes. A row of
// V is read 16 lanes wide and its bytes converted, pairs of keys at a time, into the operand whose element
// is the key.
// What depends on a key alone (ks, lv, 1/SV) is worked out by one lane for each key.
//
// Two kernels share that step:
//   stream: up to 32 rows of a K/V head (decoding, small trees). HBM-bound: each wave has pages of its
//           own, straight from memory to registers, and a block's waves are merged through LDS.
//   shared: more rows. MFMA- and VALU-bound: a block's four waves have rows of their own and share
//           each page, of which every wave converts a quarter to 16 bits in LDS.
// Their blocks either take a plane each (a sequence's K/V head; a second block, and so on, for more rows
// than one holds), or, spread, equal runs of the pages of all planes in a row, whatever the sequences'
// lengths: about as many blocks as the card runs at once. A run may end one plane, hold others whole and
// begin another; the planes that lie in several runs are joined by a second launch, in order.
#include "sage_device.h"
#include "sage_launch.h"

namespace sage {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr float W_SHIFT = 14.0f;    // weights are at most 2^14
// What a value scale of less counts as (0: a token never written; the scheme's own are 1e-12 or more). Its
// key's share of a row's sum is at most 2^(14 + 64), so that the 2^30 tokens that a table may have pages
// for add up to no more than 2^108.
constexpr float SV_LEAST = 0x1p-64f;
// A float's exponential ends at 2^-126, and in a bf16 cache value scales may lie 2^183 apart: a row of zeros
// (1e-12) that scores as a row of bf16's largest values does has a weight that low, but half of the sum. So
// from the first scale of a part over this one on (values over 3e13), its sums are added up and scaled by
// square roots, one after the other, which end at 2^-252; all sums of bf16 are merged so. Up to it, what
// falls under 2^-126 is 2^(-126 + 36 + 64) = 2^-26 of the largest share of the sum or less. (fp16 values have
// scales of 2^7.2 at most.) A branch in the loop that scales sums took 5 to 12 % longer than a loop of its
// own does, which costs other bf16 calls 0 to 1 %: 64 sequences of up to 8192 tokens, M = 4, 109.8 us and
// 109.6 without.
constexpr float SV_FAR = 0x1p36f;
template <typename T>
constexpr bool MAY_BE_FAR = std::is_same_v<T, bf16>;
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

// Bytes of eight keys' words (keys 4g .. 4g+3 of two key tiles, x in a and b) as the operands of four
// column tiles, byte e being tile e's: 16-bit halves of two keys' words interleaved by bytes convert
// pairwise, 24 operations for 32 values. (Converted byte by byte, with the half-words that the
// convert keeps set to zero first: 48.)
__device__ __forceinline__ void v_frags(const u32x4 a, const u32x4 b, f16x8 (&f)[4]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {   // bytes 2h and 2h + 1
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32 k0 = i < 2 ? a[2 * i] : b[2 * i - 4], k1 = i < 2 ? a[2 * i + 1] : b[2 * i - 3];
      const u32 w = __builtin_amdgcn_perm(k1, k0, h ? 0x07030602u : 0x05010400u);
      const f16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
      const f16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
      f[2 * h][2 * i] = lo[0], f[2 * h][2 * i + 1] = lo[1];
      f[2 * h + 1][2 * i] = hi[0], f[2 * h + 1][2 * i + 1] = hi[1];
    }
  }
}

__device__ __forceinline__ float max_groups(float x) {
  x = fmaxf(x, __shfl_xor(x, 16, 64));
  return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float sum_groups(float x) {
  x += __shfl_xor(x, 16, 64);
  return x + __shfl_xor(x, 32, 64);
}

// 2^d, d at most 0, for accumulators (a) and for sums: in bf16 as two square roots, down to d = -252.
template <typename T>
struct Down {
  float root, a;
  __device__ __forceinline__ explicit Down(float d) {
    root = __builtin_amdgcn_exp2f(MAY_BE_FAR<T> ? 0.5f * d : d);
    a = MAY_BE_FAR<T> ? root * root : root;
  }
  __device__ __forceinline__ float sum(float y) const { return MAY_BE_FAR<T> ? y * root * root : y * a; }
};

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
  float* part_o;    // (runs, RB, 2, rows, D): a run's last part of a plane begun before it, and its
  float* part_ml;   // part of the plane that goes on behind it; (runs, RB, 2, rows, 2)
  uint2* starts;    // (planes): where its pages begin in the row of all planes, and the runs' length
  int B, H, H_kv, G, T, RB;
  int rows;         // of a row block
  int units;        // planes, or runs
  int least;        // length of a run at least; 0: a block for each plane
  int ahead;        // cost of beginning a plane, in pages
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

__device__ __forceinline__ int pages_of(const Shape& p, int b) {
  const Lens n = lens_of(p, b);
  return n.tokens > 0 ? (n.keys + NPAD - 1) / NPAD : 0;
}

// Inclusive sum over the wave's lanes.
__device__ __forceinline__ u32 scan_lanes(u32 x, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u32 y = (u32)__shfl_up((int)x, o, 64);
    if (lane >= o) x += y;
  }
  return x;
}
__device__ __forceinline__ u32 lane_of(u32 x, int lane) {
  return (u32)__builtin_amdgcn_readlane((int)x, lane);
}

// All planes in a row: each is as long as its pages and, ahead of them, what it costs to begin a plane,
// in pages (so that the runs that hold many short planes do not end last). Every wave works it out by
// itself, 64 sequences at a time; the entry point bounds the sum by 2^31.
struct Runs {
  u32 mine, upto;   // length of sequence `lane`'s planes, and of those up to its own, one of each head
  u32 total, per;   // of the row, and of a run
};
__device__ __forceinline__ u32 length_of(const Shape& p, int b) {
  const u32 pages = b < p.B ? (u32)pages_of(p, b) : 0u;
  return pages ? pages + (u32)p.ahead : 0u;
}
__device__ __forceinline__ Runs runs_of(const Shape& p, int lane) {
  Runs r;
  r.mine = length_of(p, lane);
  r.upto = scan_lanes(r.mine, lane);
  u32 length = lane_of(r.upto, 63);
  for (int b0 = 64; b0 < p.B; b0 += 64)
    length += lane_of(scan_lanes(length_of(p, b0 + lane), lane), 63);
  r.total = length * (u32)p.H_kv;
  const u32 even = (r.total + (u32)p.units - 1) / (u32)p.units;
  r.per = even < (u32)p.least ? (u32)p.least : even;
  return r;
}
// The sequence at y of the row with one plane of each, its planes' length and that of those before it.
struct Seq {
  int b;
  u32 length, before;
};
__device__ __forceinline__ Seq find_seq(const Shape& p, const Runs& r, int lane, u32 y) {
  u32 mine = r.mine, upto = r.upto, base = 0;
  for (int b0 = 0;;) {
    const uint64_t hit = __builtin_amdgcn_ballot_w64(base + upto > y);
    if (hit || b0 + 64 >= p.B) {   // y lies below the sum: there is one
      const int at = hit ? __builtin_ctzll(hit) : 0;
      const u32 n = lane_of(mine, at);
      return {b0 + at, n, base + lane_of(upto, at) - n};
    }
    base += lane_of(upto, 63);
    b0 += 64;
    mine = length_of(p, b0 + lane);
    upto = scan_lanes(mine, lane);
  }
}

// Block -> (plane or run, row block): the row blocks of one unit run on one XCD (blocks go round the 8
// XCDs), whose L2 then holds the pages that they all read. The last rows, which see most, begin first.
struct Place {
  u32 unit;
  int rb;
};
__device__ __forceinline__ Place place_of(const Shape& p) {
  const u32 id = blockIdx.x, oct = id / (8u * (u32)p.RB), in = id - oct * 8u * (u32)p.RB;
  return {oct * 8u + in % 8u, p.RB - 1 - (int)(in / 8u)};
}

// A block's part of a plane: pages first .. last - 1, the whole of it or not.
struct Part {
  int b, hk, first, last;
  bool whole;
  int64_t row;   // of the parts in the workspace
};
// Calls f(Part) for each part of the block's unit.
template <typename F>
__device__ __forceinline__ void for_parts(const Shape& p, const Place& at, int lane, F&& f) {
  if (at.unit >= (u32)p.units) return;
  u32 left, per = 0;          // of the run; its length
  int b, hk, pages, at0 = 0;   // plane, its pages, and the page (from -ahead on) where the run is
  u32 x = 0;                   // place of the plane's page 0 in the row
  if (!p.least) {
    b = (int)(at.unit / (u32)p.H_kv);
    hk = (int)(at.unit - (u32)b * (u32)p.H_kv);
    pages = pages_of(p, b);
    left = (u32)pages;
  } else {
    const Runs r = runs_of(p, lane);
    per = r.per;
    const u32 begin = at.unit * per;   // below 2^31 + the length of a run
    if (begin >= r.total) return;
    left = r.total - begin < per ? r.total - begin : per;
    const Seq q = find_seq(p, r, lane, begin / (u32)p.H_kv);
    const u32 in = begin - q.before * (u32)p.H_kv;
    b = q.b;
    hk = (int)(in / q.length);
    pages = (int)q.length - p.ahead;
    at0 = (int)(in - (u32)hk * q.length) - p.ahead;
    x = begin - (u32)at0;
  }
  for (;;) {
    const u32 rest = (u32)(pages - at0);   // of the plane
    const int first = at0 < 0 ? 0 : at0, last = rest < left ? pages : at0 + (int)left;
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    if (last > first || !p.least) {
      if (p.least && first == 0 && at.rb == 0 && tid == 0)
        p.starts[b * p.H_kv + hk] = make_uint2(x, per);   // for the join
      f(Part{b, hk, first, last, first == 0 && last == pages,
             (((int64_t)at.unit * p.RB + at.rb) * 2 + (first == 0)) * p.rows});
    }
    if (rest >= left) return;
    left -= rest;
    x += (u32)pages + (u32)p.ahead;
    at0 = -p.ahead;
    if (++hk == p.H_kv) {
      hk = 0;
      do {   // one with pages follows: the run ends below the row's length
        if (++b >= p.B) return;
        pages = pages_of(p, b);
      } while (pages == 0);
    }
  }
}

// Time for the last products to be written before anything else may read them (a copy on the way out of
// a loop, say): the 16 cycles that such an MFMA takes, where the compiler's table has 8 wait states.
__device__ __forceinline__ void results_done() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 15" : : : "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// N operands from LDS, each used once, three more requested ahead of the one in use. The memory clobber
// keeps each request where it stands: left to itself the compiler reads every operand into the same
// registers, right before its use, and waits for LDS N times in a row.
template <int N, typename Read, typename Use>
__device__ __forceinline__ void run_operands(Read&& read, Use&& use) {
  u32x4 x[4];
#pragma unroll
  for (int j = 0; j < 3; ++j) x[j] = read(j);
  static_for<0, N>([&](auto jc) {
    constexpr int j = decltype(jc)::value;
    if constexpr (j + 3 < N) x[(j + 3) & 3] = read(j + 3);
    asm volatile("" : "+v"(x[j & 3]) : : "memory");
    use(jc, x[j & 3]);
  });
}

// A wave's rows and running sums.
template <typename T, int D, int R>
struct Rows {
  typename Frag<T>::type q[R][D / 32];
  int row0, step;   // lane l15 holds row row0 + step r + l15 of the plane in tile r
  f32x4 acc[R][D / 16];
  float m[R], l[R];

  // columns 64c + 16g + 8s of its row in k-step 2c + s
  __device__ __forceinline__ void load(const Shape& p, int b, int hk, int first, int step_) {
    row0 = first, step = step_;
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));   // addresses are worked out here, not held from part to part
    const int l15 = lane & 15, g = lane >> 4;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = row0 + step * r + l15, token = row / p.G, h = hk * p.G + row - token * p.G;
      const bool live = token < p.T;
      const T* src = (const T*)p.q + b * p.q_sb + (live ? h * p.q_sh + token * p.q_sr : 0) + 16 * g;
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
// others' weights of 0 leave their sums alone. Keys that are not held weigh nothing: with a score of 0,
// which is neither infinite nor NaN, their u is -infinity.
__device__ __forceinline__ void key_consts(float* dst, int key, float sk, float sv, float c, bool held) {
  const float v = sv < SV_LEAST ? SV_LEAST : sv;
  dst[key] = held ? sk * c : 0.0f;
  dst[64 + key] = held ? __builtin_amdgcn_logf(v) : NEG_INF;
  dst[128 + key] = held ? fmaxf(__builtin_amdgcn_rcpf(v), 0.0f) : 0.0f;
}

// Which keys of a page this lane's row sees, of those whose scores it holds: bit 16 (kt & 1) + i of half
// kt / 2 for key 16 kt + 4g + i. token: the row's new token.
struct Seen {
  u32 half[2];
};
__device__ __forceinline__ Seen seen_causal(const Lens& n, int key0, int held, int token, int g) {
  const int upto = n.kv - n.tokens + token + 1 - key0, count = upto < held ? upto : held;
  const uint64_t seen = count >= 64 ? ~0ull : count <= 0 ? 0ull : (1ull << count) - 1;
  return {{(u32)seen >> (4 * g), (u32)(seen >> 32) >> (4 * g)}};
}
// Under a mask, key tile kt's four keys are bytes of the row's from column d = key - prefix on, read as one
// word of any alignment at the nearest place s that lies in the row (rows of fewer than four bytes: byte by
// byte). 2 sequences of 90 tokens, 51 of them drafted, M = 408: 13.3 us; with 16 bytes and ballots for each
// row tile, a row at a time, 15.3; without a mask 12.4.
__device__ __forceinline__ int draft_of(const Lens& n, int key0, int kt, int g) {
  return key0 + 16 * kt + 4 * g - (n.kv - n.tokens);
}
__device__ __forceinline__ int mask_place(const Shape& p, int d) {
  const int most = p.T < 4 ? 0 : p.T - 4;
  return d < 0 ? 0 : d < most ? d : most;
}
__device__ __forceinline__ u32x4 mask_words(const Shape& p, const Lens& n, int b, int key0, int token,
                                            int g) {
  // n.tokens is 1 or more here
  const u8* row = p.mask + b * p.m_sb + (token < n.tokens ? token : n.tokens - 1) * p.m_sr;
  u32x4 w;
  if (p.T >= 4) {
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      u32 x;
      __builtin_memcpy(&x, row + mask_place(p, draft_of(n, key0, kt, g)), 4);
      w[kt] = x;
    }
  } else {
    const u32 x = row[0] | (u32)row[p.T > 1 ? 1 : 0] << 8 | (u32)row[p.T > 2 ? 2 : 0] << 16;
    w = (u32x4){x, x, x, x};
  }
  return w;
}
__device__ __forceinline__ Seen seen_masked(const Shape& p, const Lens& n, const u32x4 w, int key0,
                                            int held, int g) {
  Seen out;
#pragma unroll
  for (int kt = 0; kt < 4; ++kt) {
    const int d = draft_of(n, key0, kt, g), s = mask_place(p, d), left = held - 16 * kt - 4 * g;
    u32 x = (((w[kt] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w[kt]) >> 7 & 0x01010101u;   // bytes that are not 0
    x = (x | x >> 7 | x >> 14 | x >> 21) & 15u;
    // key i is byte d + i - s; every new token sees those before d = 0; none those from `held` on
    const int before = d < 0 ? (d < -4 ? 4 : -d) : 0, skip = d > s ? (d - s > 4 ? 4 : d - s) : 0;
    x = (((x >> skip) + 1) << before) - 1;
    x &= (1u << (left < 0 ? 0 : left > 4 ? 4 : left)) - 1;
    out.half[kt >> 1] = kt & 1 ? out.half[kt >> 1] | x << 16 : x;
  }
  return out;
}

// Scores to weights: u = t + log2 SV, where the page holds new tokens or ends the sequence only for the
// keys that each row sees; then the running maximum and sum, and the weights as the PV MFMA takes them.
// For the first NR of the wave's row tiles. FAR: one of the part's value scales is over SV_FAR.
template <int NR, bool FAR, typename T, int D, int R>
__device__ __forceinline__ void softmax_step(const Shape& p, const Lens& n, int b, int key0, int held,
                                             const float* consts, int g, Rows<T, D, R>& w,
                                             f32x4 (&s)[R][4], f16x8 (&wf)[R][2]) {
  const int prefix = n.kv - n.tokens;
  f32x4 ks[4], lv[4], rsv[4];
#pragma unroll
  for (int kt = 0; kt < 4; ++kt) {
    ks[kt] = *(const f32x4*)(consts + 16 * kt + 4 * g);
    lv[kt] = *(const f32x4*)(consts + 64 + 16 * kt + 4 * g);
  }
#pragma unroll
  for (int kt = 0; kt < 4; ++kt) rsv[kt] = *(const f32x4*)(consts + 128 + 16 * kt + 4 * g);
  asm volatile("" : : : "memory");   // all requested here
#pragma unroll
  for (int kt = 0; kt < 4; ++kt)
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[r][kt][i] = __builtin_fmaf(s[r][kt][i], ks[kt][i], lv[kt][i]);
  if (key0 + NPAD > prefix || held < NPAD) {
    int tid = threadIdx.x, G = p.G;
    asm volatile("" : "+v"(tid), "+s"(G));   // what follows is worked out here, not held over the loop
    const int at = tid >> 4 & 3;
    Seen seen[NR];
    if (p.mask) {
      u32x4 words[NR];
#pragma unroll
      for (int r = 0; r < NR; ++r)
        words[r] = mask_words(p, n, b, key0, (w.row0 + w.step * r + (tid & 15)) / G, at);
#pragma unroll
      for (int r = 0; r < NR; ++r) seen[r] = seen_masked(p, n, words[r], key0, held, at);
    } else {
#pragma unroll
      for (int r = 0; r < NR; ++r)
        seen[r] = seen_causal(n, key0, held, (w.row0 + w.step * r + (tid & 15)) / G, at);
    }
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s[r][kt][i] = (seen[r].half[kt >> 1] >> (16 * (kt & 1) + i)) & 1 ? s[r][kt][i] : NEG_INF;
  }
  float top[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    top[r] = NEG_INF;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) top[r] = fmaxf(top[r], s[r][kt][i]);
  }
#pragma unroll
  for (int r = 0; r < NR; ++r) top[r] = max_groups(top[r]);
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    if (__builtin_amdgcn_ballot_w64(top[r] > w.m[r])) {
      const float now = fmaxf(top[r], w.m[r]);
      // a row that has seen nothing keeps sums of zero
      const std::conditional_t<FAR, Down<T>, Down<f16>> alpha(w.m[r] - (now == NEG_INF ? 0.0f : now));
      w.m[r] = now;
      w.l[r] = alpha.sum(w.l[r]);
#pragma unroll
      for (int e = 0; e < D / 16; ++e) w.acc[r][e] *= alpha.a;
    }
    const float shift = (w.m[r] == NEG_INF ? 0.0f : w.m[r]) - W_SHIFT;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = __builtin_amdgcn_exp2f(s[r][kt][i] - shift);
        if constexpr (FAR) {
          const float root = __builtin_amdgcn_exp2f(0.5f * (s[r][kt][i] - shift));
          w.l[r] = __builtin_fmaf(root * rsv[kt][i], root, w.l[r]);
        } else {
          w.l[r] = __builtin_fmaf(x, rsv[kt][i], w.l[r]);
        }
        wf[r][kt >> 1][4 * (kt & 1) + i] = (f16)x;
      }
    }
  }
}

// N columns of an output row. A mean of fp16 values is no larger than fp16's largest, 65504, but with weights
// rounded up by 2^-11 it may come out as up to 65536, an infinity: such ones are 65504. (bf16 would need 2^-9.)
template <typename T, int N>
__device__ __forceinline__ void store_row(T* o, const float (&f)[N], float inv, bool some) {
  T out[N];
#pragma unroll
  for (int e = 0; e < N; ++e) {
    float x = some ? f[e] * inv : 0.0f;
    if constexpr (std::is_same_v<T, f16>)
      x = fabsf(x) < 65568.0f ? fminf(fmaxf(x, -65504.0f), 65504.0f) : x;
    out[e] = (T)x;
  }
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

// A row's N columns from col on: to the output where the part is the whole plane, else to the workspace
// (at row `at` of the parts), where nothing is read that a part with a sum of 0 did not write.
template <typename T, int D, int N>
__device__ __forceinline__ void finish_row(const Shape& p, const Lens& n, const Part& part, int row,
                                           int64_t at, int col, const float (&f)[N], float top,
                                           float sum) {
  const int tok = row / p.G, h = part.hk * p.G + row - tok * p.G;
  if (tok >= p.T) return;
  if (!part.whole) {
    if (col == 0) *(float2*)(p.part_ml + 2 * at) = make_float2(top, sum);
    if (sum != 0.0f) {
      if constexpr (N % 4 == 0) {
#pragma unroll
        for (int e = 0; e < N; e += 4)
          *(f32x4*)(p.part_o + at * D + col + e) = (f32x4){f[e], f[e + 1], f[e + 2], f[e + 3]};
      } else {
        *(float2*)(p.part_o + at * D + col) = make_float2(f[0], f[1]);
      }
    }
    return;
  }
  const bool some = tok < n.tokens && sum != 0.0f;
  store_row<T, N>((T*)p.o + part.b * p.o_sb + h * p.o_sh + tok * p.o_sr + col, f,
                  some ? 1.0f / sum : 0.0f, some);
  if (p.lse && col == 0)
    p.lse[((int64_t)part.b * p.H + h) * p.T + tok] = some ? lse_of(top, sum) : NEG_INF;
}

// Up to 16 R rows of a plane. Wave w of a part takes its pages first + w, then every W-th. The next
// page's K is requested when the scores are done with this one's, its V when the products are: a wave has
// 17 KB in flight at head_dim 128, a CU 8 waves. Bound by HBM where there are enough pages: 64 sequences
// of up to 8192 tokens, 8 K/V heads, M = 4: 103 us, 5.4 TB/s; 4 of 131072, M = 6: 191 us, 5.8 TB/s (a
// large copy: 4.9, read and written). A call of a few pages is a chain of latencies (lengths, page number,
// K and V, the waves' exchange): 517 tokens 10 us.
template <typename T, bool KINT8, int D, int R, int W>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu((R == 2 && D == 128) ? 1 : 2, (R == 2 && D == 128) ? 1 : 2))) void cache_attn_stream_kernel(Shape p) {
  typedef typename Frag<T>::type frag;
  constexpr int KC = D / 64, KT = D / 32, VE = D / 16, VW = VE / 4, LD = D + 4;
  __shared__ __attribute__((aligned(16))) float lds_o[W][16][LD];
  __shared__ float lds_ml[W][16][2];
  __shared__ __attribute__((aligned(16))) float lds_c[W][192];

  const int lane = threadIdx.x & 63, l15 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  for_parts(p, place_of(p), lane, [&](const Part& part) {
    const int b = part.b;
    const Lens n = lens_of(p, b);
    Rows<T, D, R> w;
    w.load(p, b, part.hk, 0, 16);

    // The page in work and what is known of the next one: its place, and the keys that it holds (0 where
    // there is no page; 64 or more: all). Its number is requested a page before that, ahead of all bytes.
    // Loads stand in no branch, where the compiler would wait for them at its end: a wave without a next
    // page asks for one line of its last one again.
    u32x4 kw[4][KC];
    u32x4 vw[4][VW];   // [key tile][word of the row's 4 VW bytes][key 4g + j]
    float sk, sv;
    const int* numbers = p.table + b * p.t_sb;
    int pg = part.first + wave;
    const int end = part.last;
    int number = numbers[pg < p.max_pages ? pg : 0], held = 0;
    int64_t base = 0;
    bool more = false;
    auto look_ahead = [&](int page) {   // at page's number, and request the next one's
      const int cur = __builtin_amdgcn_readfirstlane(number);
      const bool there = cur >= 0 && cur < p.num_pages;
      more = page < end;
      number = numbers[page + W < end ? page + W : 0];
      held = there && more ? n.keys - page * NPAD : 0;
      base = more ? ((int64_t)(there ? cur : 0) * p.H_kv + part.hk) * NPAD : base;
    };
    auto load_k = [&]() {
      const u8* kp = p.k8 + base * D;
      u32 at = more ? (u32)(l15 * D + 16 * g) : 0u;
      asm volatile("" : "+v"(at));
      sk = (p.sk + base)[(u32)lane];
      sv = (p.sv + base)[(u32)lane];
      asm volatile("" : : : "memory");   // ahead of the rows, so that the look at them waits for no row
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int c = 0; c < KC; ++c) kw[kt][c] = *(const u32x4*)(kp + (at + 16 * kt * D + 64 * c));
    };
    auto load_v = [&]() {
      const u8* vp = p.v8 + base * D;
      u32 at = more ? (u32)(4 * g * D + l15 * VE) : 0u;
      asm volatile("" : "+v"(at));
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u8* src = vp + (at + (16 * kt + j) * D);
          if constexpr (VW == 2) {
            const u32x2 x = *(const u32x2*)src;
            vw[kt][0][j] = x[0], vw[kt][1][j] = x[1];
          } else {
            vw[kt][0][j] = *(const u32*)src;
          }
        }
    };
    auto pages = [&](auto fc) {   // up to the first one with a scale over SV_FAR, or from there on
      constexpr bool FAR = decltype(fc)::value;
      for (; pg < end; pg += W) {
        const int key0 = pg * NPAD, now = held;
        if constexpr (MAY_BE_FAR<T> && !FAR)
          if (__builtin_amdgcn_ballot_w64(lane < now && sv > SV_FAR)) return;
        key_consts(lds_c[wave], lane, sk, sv, p.c, lane < now);
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
        look_ahead(pg + W);
        load_k();
        if (now < NPAD) {   // whatever lies behind the end, or on no page: no NaN may meet a weight of zero
          const int left = now - 4 * g;
#pragma unroll
          for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int x = 0; x < VW; ++x) vw[kt][x][j] = 16 * kt + j < left ? vw[kt][x][j] : 0u;
        }
        f16x8 wf[R][2];
        softmax_step<R, FAR>(p, n, b, key0, now, lds_c[wave], g, w, s, wf);

        // O^T += V^T W^T: tile e's row x is column VE x + e
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int x = 0; x < VW; ++x) {
            f16x8 vf[4];
            v_frags(vw[2 * u][x], vw[2 * u + 1][x], vf);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int r = 0; r < R; ++r) w.acc[r][4 * x + e] = mfma(vf[e], wf[r][u], w.acc[r][4 * x + e]);
          }
        load_v();
        results_done();
      }
    };
    if (pg < end) {
      look_ahead(pg);
      load_k();
      load_v();
      pages(std::false_type{});
      if constexpr (MAY_BE_FAR<T>) pages(std::true_type{});
    }

    // the waves' results merged, 16 rows at a time; each thread has N columns of a row
    constexpr int TPR = 4 * W, N = D / TPR;   // threads of a row
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));   // addresses are worked out here, not held over the loop
    const int orow = tid / TPR, ocol = (tid % TPR) * N;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float total = sum_groups(w.l[r]);
      __syncthreads();   // the readers of what was merged before
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
        const Down<T> to(lds_ml[x][orow][0] - use);
        sum += to.sum(lds_ml[x][orow][1]);
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] += lds_o[x][orow][ocol + e] * to.a;
      }
      finish_row<T, D, N>(p, n, part, 16 * r + orow, part.row + 16 * r + orow, ocol, f, top, sum);
    }
  });
}

// Row blocks of up to 64 R rows of a plane, the row tiles of 16 dealt to the four waves in turn. The page
// in work lies in LDS as the MFMAs' operands (K: key tile x k-step, V: half x column tile; 1 KB each,
// one 16-byte piece a lane), the next one's bytes in registers: wave w converts key tile w of K and
// half w / 2 of V, four column tiles of it at D = 128 and two at 64. One barrier a page: the page after
// it goes to the other half of the buffers, whose readers passed the barrier before. Two blocks share a
// CU, whose matrix cores and vector units each serve one while the other waits.
// 8 sequences of 32768 tokens, 4 K/V heads, M = 512: 345 to 369 us by the card, 0.80 to 0.75 PFLOP/s (a large
// matrix product: 1.21). Of a page's time for a SIMD's two waves, 128 MFMAs are 2048 cycles and 680 vector
// operations, 64 of them exponentials, about 3500; the two overlap little (matrix cores busy for 32 % of
// the cycles, vector units for 52 %). More rows to a block would share the conversion, a
// third of those operations, further, but: 8 waves in two groups, one at its products while the other is
// at its softmax, took 404 us or more, three row tiles a wave (one block a CU) 1095 for want of registers
// and of a second block, the conversion spread among the second products 2 % more.
template <typename T, bool KINT8, int D, int R>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void cache_attn_shared_kernel(Shape p) {
  typedef typename Frag<T>::type frag;
  constexpr int KC = D / 64, KT = D / 32, VE = D / 16;
  __shared__ __attribute__((aligned(16))) u32x4 lds_k[2][4][KT][64];
  __shared__ __attribute__((aligned(16))) u32x4 lds_v[2][2][VE][64];
  __shared__ __attribute__((aligned(16))) float lds_c[2][192];

  const int lane = threadIdx.x & 63, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Place at = place_of(p);

  for_parts(p, at, lane, [&](const Part& part) {
    const int b = part.b;
    const Lens n = lens_of(p, b);
    const int block0 = at.rb * p.rows, row0 = block0 + 16 * wave;
    // rows of the block that are there, and the wave's tiles of them
    const int rows = n.tokens * p.G - block0 < p.rows ? n.tokens * p.G - block0 : p.rows;
    const int tiles = rows > 16 * wave ? (rows - 16 * wave + 63) / 64 : 0;
    Rows<T, D, R> w;
    w.load(p, b, part.hk, row0, 64);

    // in causal order, the pages behind its last row's token are none of the block's (4096 tokens by
    // themselves, 32 heads on 8: 479 us, 817 with them)
    const int upto = n.kv - n.tokens + (block0 + rows - 1) / p.G;   // that token
    const int seen = p.mask ? part.last : upto < 0 ? 0 : upto / NPAD + 1;
    const int last = rows <= 0 ? part.first : part.last < seen ? part.last : seen;
    // this wave's share of the next page, and the keys' scales, by lane
    u32x4 kw[KC];
    u32 vw[8];
    float sk, sv;
    int held;   // keys of that page, 0 where there is none (and 64 or more: all)
    bool far = false;
    // page numbers are requested a page before they are used, ahead of that page's bytes
    const int* numbers = p.table + b * p.t_sb;
    int number = 0;
    // Requests page pg's share (the last page's again behind it), without a branch: nothing but the
    // conversion waits for these loads. Offsets that hang on the lane or the wave are worked out here and
    // in convert, not held over the loop, where registers are short.
    auto fetch = [&](int pg) {
      const int cur = __builtin_amdgcn_readfirstlane(number);
      const bool there = cur >= 0 && cur < p.num_pages;
      number = numbers[pg + 1 < last ? pg + 1 : last - 1];
      held = there ? n.keys - pg * NPAD : 0;
      const int64_t base = ((int64_t)(there ? cur : 0) * p.H_kv + part.hk) * NPAD;
      int ln = lane, me = wave;
      asm volatile("" : "+v"(ln), "+s"(me));
      const u8* kp = p.k8 + base * D;
      const u8* vp = p.v8 + base * D;
      u32 ko = (u32)((16 * me + (ln & 15)) * D + (ln >> 4) * 16);
      u32 vo = (u32)((32 * (me >> 1) + (ln >> 4) * 4) * D + (ln & 15) * VE + (VE == 8 ? 4 * (me & 1) : 0));
      asm volatile("" : "+v"(ko), "+v"(vo));
#pragma unroll
      for (int c = 0; c < KC; ++c) kw[c] = *(const u32x4*)(kp + (ko + 64 * c));
#pragma unroll
      for (int i = 0; i < 8; ++i) vw[i] = *(const u32*)(vp + (vo + (16 * (i >> 2) + (i & 3)) * D));
      sk = (p.sk + base)[(u32)ln];
      sv = (p.sv + base)[(u32)ln];
    };
    // The requested page to LDS. What lies behind the sequence's end, or on no page, is zeros under the
    // constants of a key that weighs nothing: no NaN may meet a weight of zero.
    auto convert = [&](int pg) {
      const int buf = pg & 1;
      int ln = lane, me = wave;
      asm volatile("" : "+v"(ln), "+s"(me));
      if (held < NPAD) {
        const int left = held - 32 * (me >> 1) - (ln >> 4) * 4;
#pragma unroll
        for (int i = 0; i < 8; ++i) vw[i] = 16 * (i >> 2) + (i & 3) < left ? vw[i] : 0u;
#pragma unroll
        for (int c = 0; c < KC; ++c)
          if (16 * me + (ln & 15) >= held) kw[c] = (u32x4){0, 0, 0, 0};
      }
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        const frag f = k_frag<T, KINT8>(kw[t >> 1][2 * (t & 1)], kw[t >> 1][2 * (t & 1) + 1]);
        __builtin_memcpy(&lds_k[buf][me][t][ln], &f, 16);
      }
      f16x8 vf[4];
      v_frags((u32x4){vw[0], vw[1], vw[2], vw[3]}, (u32x4){vw[4], vw[5], vw[6], vw[7]}, vf);
      if constexpr (VE == 8) {
#pragma unroll
        for (int e = 0; e < 4; ++e) __builtin_memcpy(&lds_v[buf][me >> 1][4 * (me & 1) + e][ln], &vf[e], 16);
      } else {   // both waves of a half have all four tiles, and write two each
        const bool odd = me & 1;
        const f16x8 v0 = odd ? vf[2] : vf[0], v1 = odd ? vf[3] : vf[1];
        __builtin_memcpy(&lds_v[buf][me >> 1][2 * (me & 1)][ln], &v0, 16);
        __builtin_memcpy(&lds_v[buf][me >> 1][2 * (me & 1) + 1][ln], &v1, 16);
      }
      if (me == 0) key_consts(lds_c[buf], ln, sk, sv, p.c, ln < held);
      if constexpr (MAY_BE_FAR<T>) far |= __builtin_amdgcn_ballot_w64(ln < held && sv > SV_FAR) != 0;
    };
    f32x4 s[R][4];
    f16x8 wf[R][2];
    auto scores = [&](auto nr, int pg) {
      constexpr int NR = decltype(nr)::value;
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) s[r][kt] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
      // two key tiles at a time, so that no MFMA waits for the one before it
      auto tile = [](int i) { return i / (2 * KT) * 2 + (i & 1); };
      auto step = [](int i) { return i % (2 * KT) / 2; };
      const auto* k = lds_k[pg & 1];
      run_operands<4 * KT>([&](int i) { return k[tile(i)][step(i)][lane]; },
                           [&](auto i, const u32x4& x) {
                             constexpr int I = decltype(i)::value;
                             frag kf;
                             __builtin_memcpy(&kf, &x, 16);
#pragma unroll
                             for (int r = 0; r < NR; ++r)
                               s[r][tile(I)] = mfma(kf, w.q[r][step(I)], s[r][tile(I)]);
                           });
    };
    auto values = [&](auto nr, int pg) {
      constexpr int NR = decltype(nr)::value;
      const auto* v = lds_v[pg & 1];
      run_operands<2 * VE>([&](int i) { return v[i / VE][i % VE][lane]; },
                           [&](auto i, const u32x4& x) {
                             constexpr int I = decltype(i)::value;
                             f16x8 vf;
                             __builtin_memcpy(&vf, &x, 16);
#pragma unroll
                             for (int r = 0; r < NR; ++r)
                               w.acc[r][I % VE] = mfma(vf, wf[r][I / VE], w.acc[r][I % VE]);
                           });
    };
    int pg = part.first;
    // pages for the wave's first NR row tiles: up to the first one with a scale over SV_FAR, which all
    // waves have read, or from there on
    auto pages = [&](auto nr, auto fc) {
      constexpr int NR = decltype(nr)::value;
      constexpr bool FAR = decltype(fc)::value;
      for (; pg < last; ++pg) {
        if constexpr (MAY_BE_FAR<T> && !FAR)
          if (far) return;
        const int now = held;
        fetch(pg + 1);
        if constexpr (NR > 0) {
          scores(nr, pg);
          softmax_step<NR, FAR>(p, n, b, pg * NPAD, now, lds_c[pg & 1], g, w, s, wf);
          values(nr, pg);
        }
        if (pg + 1 < last) convert(pg + 1);
        __syncthreads();
      }
    };

    if (part.first < last) {
      number = numbers[part.first];
      fetch(part.first);
      convert(part.first);   // the readers of the part before have passed its last barrier
      __syncthreads();
      // (two tiles a wave are taken for five or more, so that a wave without any is rare there)
      auto all = [&](auto nr) {
        pages(nr, std::false_type{});
        if constexpr (MAY_BE_FAR<T>) pages(nr, std::true_type{});
      };
      if (tiles == R)
        all(std::integral_constant<int, R>{});
      else
        all(std::integral_constant<int, R - 1>{});
    }

    int ln = threadIdx.x & 63;
    asm volatile("" : "+v"(ln));   // addresses are worked out here, not held over the loop
    const int in0 = 16 * wave + (ln & 15), col0 = VE * 4 * (ln >> 4);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float sum = sum_groups(w.l[r]);
      const int in = 64 * r + in0;   // row of the block
      if (in < p.rows) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float f[VE];
#pragma unroll
          for (int e = 0; e < VE; ++e) f[e] = w.acc[r][e][i];
          finish_row<T, D, VE>(p, n, part, block0 + in, part.row + in, col0 + VE * i, f, w.m[r], sum);
        }
      }
    }
  });
}

// Planes in several runs joined, part after part, and the rows of those that have no pages cleared. grid:
// (row tile, plane), D/4 lanes to a row and SL slices of its parts; 8 parts are requested at a time.
template <typename T, int D, int SL>
__global__ __launch_bounds__(256) void cache_attn_join_kernel(Shape p, u32 row_tiles) {
  constexpr int LPR = D / 4, ROWS = 256 / (LPR * SL);
  __shared__ __attribute__((aligned(16))) f32x4 lds_f[SL > 1 ? 256 : 1];
  __shared__ float2 lds_ml[SL > 1 ? 256 : 1];
  const int tid = threadIdx.x, col = tid % LPR * 4, slice = tid / LPR % SL;
  const u32 plane = blockIdx.x / row_tiles, rt = blockIdx.x - plane * row_tiles;
  const int b = (int)(plane / (u32)p.H_kv), hk = (int)(plane - (u32)b * (u32)p.H_kv);
  const int row = (int)rt * ROWS + tid / (LPR * SL);
  const u32 pages = (u32)pages_of(p, b);
  u32 run0 = 0;
  int parts = 0;
  if (pages) {
    const uint2 at = p.starts[plane];
    run0 = at.x / at.y;
    parts = (int)((at.x + pages - 1) / at.y - run0) + 1;
    if (parts == 1) return;   // its one run has written the plane
  }
  const int tok = row / p.G, h = hk * p.G + row - tok * p.G;
  const bool live = tok < p.T;
  const int rb = row / p.rows, in = row - rb * p.rows;
  // part i's row: of the first run its last part, of the others their first
  auto row_of = [&](int i) {
    return (((int64_t)(run0 + (u32)i) * p.RB + rb) * 2 + (i == 0)) * p.rows + in;
  };
  float top = NEG_INF, sum = 0.0f;
  f32x4 f = {0.0f, 0.0f, 0.0f, 0.0f};
  if (live) {
    for (int i0 = slice; i0 < parts; i0 += 8 * SL) {
      float2 ml[8];
      f32x4 y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = i0 + j * SL;
        const int64_t at = row_of(i < parts ? i : i0);
        ml[j] = *(const float2*)(p.part_ml + 2 * at);
        y[j] = *(const f32x4*)(p.part_o + at * D + col);
        if (i >= parts) ml[j] = make_float2(NEG_INF, 0.0f);
      }
      float now = top;
#pragma unroll
      for (int j = 0; j < 8; ++j) now = fmaxf(now, ml[j].x);
      const float use = now == NEG_INF ? 0.0f : now;
      const Down<T> old(top - use);
      top = now;
      sum = old.sum(sum);
      f *= old.a;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const Down<T> to(ml[j].x - use);
        const bool full = ml[j].y != 0.0f;   // else nothing was written there
        sum += full ? to.sum(ml[j].y) : 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] += full ? y[j][e] * to.a : 0.0f;
      }
    }
  }
  if constexpr (SL > 1) {
    lds_f[tid] = f;
    lds_ml[tid] = make_float2(top, sum);
    __syncthreads();
    if (slice != 0) return;
#pragma unroll
    for (int x = 1; x < SL; ++x) top = fmaxf(top, lds_ml[tid + x * LPR].x);
    const float use = top == NEG_INF ? 0.0f : top;
    sum = 0.0f;
    f = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int x = 0; x < SL; ++x) {
      const float2 ml = lds_ml[tid + x * LPR];
      const Down<T> to(ml.x - use);
      sum += to.sum(ml.y);
      f += lds_f[tid + x * LPR] * to.a;
    }
  }
  if (!live) return;
  const bool some = tok < lens_of(p, b).tokens && sum != 0.0f;
  const float out[4] = {f[0], f[1], f[2], f[3]};
  store_row<T, 4>((T*)p.o + b * p.o_sb + h * p.o_sh + tok * p.o_sr + col, out, some ? 1.0f / sum : 0.0f,
                  some);
  if (p.lse && col == 0)
    p.lse[((int64_t)b * p.H + h) * p.T + tok] = some ? lse_of(top, sum) : NEG_INF;
}

template <typename T, bool KINT8, int D>
hipError_t run(const CacheAttnArgs& a, hipStream_t st) {
  const CacheAttnPlan plan = cache_attn_plan(a.B, a.H, a.H_kv, a.T, a.pool.max_pages, D);
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
  p.B = (int)a.B;
  p.H = (int)a.H;
  p.H_kv = (int)a.H_kv;
  p.G = (int)(a.H / a.H_kv);
  p.T = (int)a.T;
  p.RB = (int)plan.row_blocks;
  p.rows = (int)plan.rows;
  p.units = (int)plan.units;
  p.least = (int)plan.least;
  p.ahead = plan.ahead;
  p.c = a.sm_scale * LOG2E_F;
  p.part_o = (float*)a.workspace;
  p.part_ml = p.part_o + plan.part_rows * D;
  p.starts = (uint2*)(p.part_ml + plan.part_rows * 2);
  const u32 blocks = (u32)plan.blocks;
  switch (plan.kernel) {
    case CACHE_ATTN_STREAM16:
      cache_attn_stream_kernel<T, KINT8, D, 1, 4><<<blocks, 256, 0, st>>>(p);
      break;
    case CACHE_ATTN_STREAM16_WIDE:
      cache_attn_stream_kernel<T, KINT8, D, 1, 8><<<blocks, 512, 0, st>>>(p);
      break;
    case CACHE_ATTN_STREAM32:
      cache_attn_stream_kernel<T, KINT8, D, 2, 4><<<blocks, 256, 0, st>>>(p);
      break;
    case CACHE_ATTN_SHARED64:
      cache_attn_shared_kernel<T, KINT8, D, 1><<<blocks, 256, 0, st>>>(p);
      break;
    default:
      cache_attn_shared_kernel<T, KINT8, D, 2><<<blocks, 256, 0, st>>>(p);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !plan.least) return e;
  const u32 M = (u32)(a.T * (a.H / a.H_kv)), planes = (u32)(a.B * a.H_kv);
  if (plan.wide_join) {
    constexpr u32 ROWS = 256 / (D / 4 * 8);
    const u32 tiles = (M + ROWS - 1) / ROWS;
    cache_attn_join_kernel<T, D, 8><<<planes * tiles, 256, 0, st>>>(p, tiles);
  } else {
    constexpr u32 ROWS = 256 / (D / 4);
    const u32 tiles = (M + ROWS - 1) / ROWS;
    cache_attn_join_kernel<T, D, 1><<<planes * tiles, 256, 0, st>>>(p, tiles);
  }
  return hipGetLastError();
}

template <int D>
hipError_t run_d(const CacheAttnArgs& a, hipStream_t st) {
  if (a.dtype == 1) return run<bf16, false, D>(a, st);
  return a.pool.k_int8 ? run<f16, true, D>(a, st) : run<f16, false, D>(a, st);
}

}  // namespace

// Which kernel: by the rows M that read one K/V head. Up to 32 rows leave the matrix cores idle enough
// for every wave to convert its own pages (stream); more share the conversion. Measured, 8 sequences of
// 8192 tokens, 8 K/V heads, us: M = 32 stream 37, shared 48; M = 64 shared 55.
//
// Which cut (for the whole card, 256 CUs in 8 XCDs; on a part of it calls are served, but not filled so): as
// many runs as blocks are resident at once (512 threads' registers of a CU hold two blocks
// of 4 waves, but one of the 32-row kernel at head_dim 128), so that all runs begin and end together.
// 8 x 3000 tokens, M = 4: 512 runs 20 us, 1024 runs 26; 8 x 8192, M = 32: 256 runs 37, 1024 runs 61. The
// row blocks of a run share an XCD, so the runs are as many as each of the 8 XCDs holds whole: three row
// blocks (M = 384) in 168 runs 176 us, in 171 (two XCDs with blocks left for a second turn) 237. From 65 row
// blocks on (M over 8192: a prompt's part of over 2048 tokens, 4 heads to a K/V head) none holds a run whole,
// and there are as few runs as make about 512 blocks, or one: less than 8 leave XCDs without work (4096
// tokens: 4 runs of 128 row blocks on 4 of the 8), as do fewer than 8 planes of a block each. Runs
// shorter than a page for each wave (or two pages, shared) cost more in their beginnings than they save.
// A run's beginning of a plane counts as `ahead` pages: the more, the less else a CU has to do meanwhile.
// M = 32 at head_dim 128 (one block a CU), 64 ragged sequences of up to 8192 tokens: 4 pages 180 us, 8
// 146, 12 126, 16 130; head_dim 64: 4 pages 86, 8 64, 16 65. M = 4, up to 4096 tokens, head_dim 64: 4
// pages 35, 8 33, 16 35; head_dim 128: 2 pages 64, 4 53, 8 54, 16 57. Shared, M = 128, 16 of up to 4096: 4
// pages 56, 8 58, 16 61. No more than a run is long: no run can begin a plane for another (49 planes of 19
// ragged pages, M = 30, 4 pages 14.9, 12 pages 16.7).
//
// A block for each plane saves the second launch and the parts' way through memory, but waits for the
// longest: taken for tables of up to so many pages as either takes as long (us, one launch / spread), the
// more the better the planes fill the card. 8 K/V heads, M = 4, 12 pages, 1 sequence 11.4 / 11.6, 8
// sequences 11.7 / 11.9; 16 pages 13.1 / 11.7 and 13.4 / 14.4; 32 ragged sequences, 16 pages 14.9 / 18.9,
// 32 pages 21.6 / 24.1, 64 pages 33.6 / 33.7. M = 32, 8 sequences, 16 pages 17.9 / 18.5, 24 pages 22.1 /
// 19.3. M = 128, 8 sequences, 8 pages 24.9 / 29.3, 16 pages 40.6 / 33.5; 32 ragged, 16 pages 43.6 / 49.0, 32
// pages 74 / 62; 64 ragged, 32 pages 92 / 100. Planes that fill the card four times always take it.
CacheAttnPlan cache_attn_plan(int64_t B, int64_t H, int64_t H_kv, int64_t T, int64_t max_pages,
                              int64_t D) {
  CacheAttnPlan p;
  const int64_t M = T * (H / H_kv), planes = B * H_kv, tiles = (M + 15) / 16;
  p.kernel = M <= 16 ? CACHE_ATTN_STREAM16 : M <= 32 ? CACHE_ATTN_STREAM32
             : M <= 64 ? CACHE_ATTN_SHARED64 : CACHE_ATTN_SHARED128;
  const bool stream = M <= 32;
  const int64_t most = M <= 16 ? 1 : M <= 32 ? 2 : M <= 64 ? 4 : 8;   // tiles of a row block
  p.row_blocks = (tiles + most - 1) / most;
  p.rows = 16 * ((tiles + p.row_blocks - 1) / p.row_blocks);
  p.planes = planes;
  const int64_t blocks = planes * p.row_blocks;
  int64_t one_launch;   // pages
  if (stream)
    one_launch = blocks >= 256 ? 32 : blocks >= 32 ? 16 : (M <= 16 ? 12 : 8) * (128 / D);
  else
    one_launch = blocks >= 512 ? 32 : blocks >= 256 ? 16 : blocks >= 64 ? 10 : 4;
  p.ahead = CACHE_ATTN_LEAST_AHEAD;
  if (max_pages <= one_launch || blocks >= 2048) {
    p.units = planes;
    p.least = 0;
    p.part_rows = 0;
    p.wide_join = false;
    // fewer planes than CUs: twice the waves for each
    if (M <= 16 && blocks <= 256) p.kernel = CACHE_ATTN_STREAM16_WIDE;
  } else {
    p.least = stream ? 4 : 2;
    const int64_t resident = p.kernel == CACHE_ATTN_STREAM32 && D == 128 ? 256 : 512;
    int64_t runs = resident / 8 / p.row_blocks * 8;
    if (runs < 8) runs = resident / p.row_blocks > 1 ? resident / p.row_blocks : 1;
    const int64_t longest = (planes * (max_pages + CACHE_ATTN_LEAST_AHEAD) + p.least - 1) / p.least;
    if (runs > longest) runs = longest;
    if (runs > 128 * planes) runs = 128 * planes;   // parts of a plane that the join reads
    p.units = runs;
    const int64_t most_ahead = !stream ? 4 : D == 64 ? 8 : M <= 16 ? 4 : CACHE_ATTN_MOST_AHEAD;
    const int64_t length = planes * max_pages / runs;   // of a run, at most
    p.ahead = (int)(length < CACHE_ATTN_LEAST_AHEAD ? CACHE_ATTN_LEAST_AHEAD
                    : length < most_ahead ? length : most_ahead);
    p.part_rows = runs * p.row_blocks * 2 * p.rows;
    p.wide_join = runs > 16 * planes;
  }
  p.blocks = (p.units + 7) / 8 * 8 * p.row_blocks;
  return p;
}

size_t cache_attn_workspace_bytes(const CacheAttnPlan& p, int64_t D) {
  return p.least ? (size_t)(p.part_rows * (D + 2) + 2 * p.planes) * sizeof(float) : 0;
}

hipError_t launch_cache_attn(const CacheAttnArgs& a, hipStream_t st) {
  return a.D == 128 ? run_d<128>(a, st) : run_d<64>(a, st);
}

}  // namespace sage
