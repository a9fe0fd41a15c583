// Host-side launchers shared between the kernel translation units and the C ABI (capi.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace sage {

// Geometry of the two-launch prologue for BH planes of N rows, padded to N_pad (a multiple of 64,
// at least ceil(N/64)*64). The workspace is sized for head_dim 128, which covers 64.
//   stats pass: C1 blocks per plane (1-D grid of C1*BH), each owning R1 consecutive rows; R1 and
//               C1 follow from Nc = ceil(N/64)*64, and the plane's last block also covers the
//               rows up to N_pad, so extra padding never changes the workspace;
//   quant pass: C2 blocks per plane (1-D grid of C2*BH), each owning R2 rows of N_pad.
// Each grid is one round of resident blocks on MI355X (prologue.hip), so C1 stays small and the
// quant blocks' reduction of the C1 mean partials (128 fp64 each) stays short.
struct PrologueGeom {
  int64_t R1, C1, R2, C2;
};
// cus: the device's compute units; the grids are sized for min(cus, 256) (the workspace bound,
// prologue_workspace_bytes, is the 256-CU geometry's, which has the most mean partials).
PrologueGeom prologue_geom(int64_t BH, int64_t N, int64_t N_pad, int64_t step = 128,
                           int64_t cus = 256);
// bytes of workspace for BH planes of N rows (any N_pad)
size_t prologue_workspace_bytes(int64_t BH, int64_t N);

struct PrologueArgs {
  int dtype, k_int8, smooth_k, smooth_v, fold;
  const void* k;
  int64_t k_sb, k_sh, k_sr;
  const void* v;
  int64_t v_sb, v_sh, v_sr;
  int64_t B, H, N, N_pad;
  int64_t D;       // head_dim: 64 or 128
  void* k8;
  float* sk;
  void* v8t;
  float* sv;
  float* mean;
  float* vmean;    // required with smooth_v: V's sequence mean (B*H, 128) fp32
  float* s;
  float* kconst;   // optional: the main loop's per-key constants (B*H, N_pad/64, 2, 64) fp32
  void* workspace;
  int64_t cus;     // compute units of the launch device (<= 0: 256)
};
hipError_t launch_prologue(const PrologueArgs& a, hipStream_t stream);
// The smooth_k mean alone: K's fp64 column partials (stats pass, K only), then MEAN, with the
// same summation order and rounding as the prologue's MEAN output.
hipError_t launch_kseq_mean(const PrologueArgs& a, hipStream_t stream);

struct AttnArgs {
  int dtype, qk_int8, causal;
  const void* q;
  int64_t q_sb, q_sh, q_sr;
  const void* k8;
  const float* kconst;      // per-key constants in the prologue's KCONST layout, or NULL and:
  const float* sk;          //   SK (B*H_kv, N_kv_pad) and
  const float* svp;         //   SV' (B*H_kv, N_kv_pad), the reference's arrays
  const void* v8t;
  const float* s;
  void* o;
  int64_t o_sb, o_sh, o_sr;
  int64_t B, H, N;          // query side: B*H planes of N rows
  int64_t D;                // head_dim: 64 or 128 (the 256-query kernel serves 128 only)
  int64_t H_kv, N_kv, N_kv_pad;   // key/value side: B*H_kv planes of N_kv rows (H % H_kv == 0)
  float sm_scale;
  float* lse;              // optional (B*H, N) fp32 row logsumexp
  const float* kmean;      // optional (B*H_kv, 128) fp32 smooth_k mean, for the logsumexp correction
  const float* vmean;      // optional (B*H_kv, 128) fp32 smooth_v mean, added to the output
  int64_t cus = 0;         // compute units of the launch device (<= 0: 256)
};
hipError_t launch_attn_fwd(const AttnArgs& a, hipStream_t stream);
// the two-group ping-pong form of the same main loop (256 queries per block of 8 waves)
hipError_t launch_attn_fwd_pp(const AttnArgs& a, hipStream_t stream);
// the software-pipelined form (128 queries per block of 4 waves, three or four blocks per CU)
hipError_t launch_attn_fwd_pl(const AttnArgs& a, hipStream_t stream);
// the same kernel in its key-split form (non-causal, head_dim 64; 64 queries per block, the even
// and the odd key blocks run by two wave pairs that exchange their block maxima, merged in LDS)
hipError_t launch_attn_fwd_split(const AttnArgs& a, hipStream_t stream);

struct QuantQArgs {
  int dtype, qk_int8;
  const void* q;
  int64_t q_sb, q_sh, q_sr;
  int64_t B, H, N;
  int64_t D;       // head_dim: 64 or 128
  float sm_scale;
  void* q8;
  float* sq;
  float* cq;
};
hipError_t launch_quant_q(const QuantQArgs& a, hipStream_t stream);

hipError_t launch_layout_probe(const void* a, const void* bt, int32_t* c, const void* e,
                               const void* ft, float* d, hipStream_t stream);
// MFMA throughput probe: blocks x 256 threads, each wave `iters` rounds of 4 independent MFMAs.
hipError_t launch_mfma_peak(bool int8, int64_t blocks, int64_t iters, int64_t* clocks,
                            hipStream_t stream);

// Rotary positions: a pair (a, b) of the first R columns becomes (a c - b s, b c + a s). `table` holds
// R/2 cosines and R/2 sines per position; null where a cache write rotates nothing.
struct RotaryArgs {
  int dtype;
  const void* x;
  int64_t x_sb, x_sh, x_sr;
  void* o;
  int64_t o_sb, o_sh, o_sr;
  const float* table;
  int64_t rows, R;
  const int32_t* positions;   // (B, N), rows p_sb apart
  int64_t p_sb;
  int64_t B, H, N, D;
  int interleaved, inverse;
};
hipError_t launch_rotary(const RotaryArgs& a, hipStream_t stream);

// A cache's pool of pages of 64 tokens, (num_pages, H_kv, 64, D) codes and (num_pages, H_kv, 64)
// scales, and the page numbers of B sequences.
struct CachePool {
  int k_int8;
  void* k8;
  float* sk;
  void* v8;
  float* sv;
  int64_t num_pages;
  const int32_t* table;       // (B, max_pages), rows t_sb apart
  int64_t t_sb, max_pages;
};
// Rows written to (k, v are read) or read from (k, v are written) positions start[b] + n of sequence
// b, n < lens[b]. start null: 0 (reading only); lens null: all N (writing only).
struct CacheRowsArgs {
  int dtype;
  void* k;
  int64_t k_sb, k_sh, k_sr;
  void* v;
  int64_t v_sb, v_sh, v_sr;
  int64_t B, H, N, D;
  CachePool pool;
  const int32_t* start;
  const int32_t* lens;
  RotaryArgs rotary;          // of K, when writing: table, rows, R, positions, p_sb, interleaved
};
hipError_t launch_cache_write(const CacheRowsArgs& a, hipStream_t stream);
hipError_t launch_cache_read(const CacheRowsArgs& a, hipStream_t stream);

struct CacheAttnArgs {
  int dtype;
  const void* q;
  int64_t q_sb, q_sh, q_sr;
  void* o;
  int64_t o_sb, o_sh, o_sr;
  int64_t B, H, T, H_kv, D;
  CachePool pool;
  const int32_t* kv_lens;
  const int32_t* q_lens;      // null: T each
  const void* mask;           // (B or 1, T, T) bytes; null: causal among the new tokens
  int64_t m_sb, m_sr;
  float sm_scale;
  float* lse;                 // optional (B, H, T)
  void* workspace;
};
// How a call is cut up: row blocks of `rows` of a K/V head's T * H / H_kv rows, and `units` planes (least
// = 0) or equal runs of all planes' pages, of `least` pages or more, whose parts (part_rows rows of D
// + 2 floats) a second launch joins. Sizes alone decide it, so a captured call and its workspace agree.
enum CacheAttnKernel {
  CACHE_ATTN_STREAM16,        // up to 16 rows, 4 waves
  CACHE_ATTN_STREAM16_WIDE,   // 8 waves
  CACHE_ATTN_STREAM32,        // up to 32 rows
  CACHE_ATTN_SHARED64,        // row blocks of up to 64
  CACHE_ATTN_SHARED128,       // and 128 rows
};
// What beginning a plane costs a run, in pages of its own (CacheAttnPlan::ahead).
constexpr int CACHE_ATTN_LEAST_AHEAD = 4, CACHE_ATTN_MOST_AHEAD = 12;
struct CacheAttnPlan {
  CacheAttnKernel kernel;
  int64_t rows, row_blocks, planes, units, least, part_rows, blocks;
  int ahead;
  bool wide_join;
};
CacheAttnPlan cache_attn_plan(int64_t B, int64_t H, int64_t H_kv, int64_t T, int64_t max_pages,
                              int64_t D);
size_t cache_attn_workspace_bytes(const CacheAttnPlan& p, int64_t D);
hipError_t launch_cache_attn(const CacheAttnArgs& a, hipStream_t stream);

}  // namespace sage
