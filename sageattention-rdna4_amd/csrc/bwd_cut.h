// How a backward call is cut into blocks (host and device; no HIP dependency, so that a host program can
// check that every step of every tile is taken once).
//
// A tile is 128 columns (keys, or queries) of a plane, 64 in small calls; its block goes over the other side
// in steps of 64 rows.
// Where tiles are few, or some far longer than a resident block's share, they are cut into parts of
// so many steps, each a block of its own, and a further launch adds the parts' sums in order.
#pragma once
#include <stdint.h>

#if defined(__HIPCC__)
#define SAGE_HD __host__ __device__ __forceinline__
#else
#define SAGE_HD inline
#endif

namespace sage {

constexpr int ATTN_BWD_ROWS = 64, ATTN_BWD_SEGMENTS = 32, ATTN_BWD_ALONE = 6;

// One kind of block's tiles, the longest first. Those of `parts` parts come first, end[0] of them, then
// those of one part less, up to tile end[1], and so on; from tile `cut` on they are whole. Blocks are numbered
// tile by tile, part by part, plane by plane: cut_blocks of them hold parts.
struct AttnBwdCut {
  int tiles, parts, cut, cut_blocks, blocks;
  int end[ATTN_BWD_SEGMENTS];
};
struct AttnBwdPlan {
  int64_t columns;            // of a tile
  bool alone;                 // no launch ahead: blocks work out their rows' constants by themselves
  int64_t nb_q, nb_kv;        // steps in a plane of queries, of keys
  AttnBwdCut keys, queries;
};

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Tiles u = 0 .. of min(top, base - drop u) steps each in `planes` planes, no part of more than `most`.
inline AttnBwdCut cut_tiles(int64_t tiles, int64_t base, int64_t drop, int64_t top, int64_t most,
                            int64_t planes) {
  const int64_t longest = base < top ? base : top;
  int64_t parts = ceil_div(longest, most);
  if (drop && parts > ATTN_BWD_SEGMENTS) {
    most = ceil_div(longest, ATTN_BWD_SEGMENTS);
    parts = ceil_div(longest, most);
  }
  AttnBwdCut c = {};
  int64_t lo = 0, blocks = 0;
  int i = 0;
  for (int64_t p = parts;; --p, ++i) {
    int64_t hi = tiles;                       // the end of the tiles of more than (p - 1) most steps
    const int64_t over = (p - 1) * most;
    if (p > 1 && drop) hi = over >= longest ? 0 : ceil_div(base - over, drop);
    hi = hi > tiles ? tiles : hi < lo ? lo : hi;
    c.end[i] = (int)hi;
    blocks += (hi - lo) * p * planes;
    if (p > 1) {
      c.cut = (int)hi;
      c.cut_blocks = (int)blocks;
    }
    lo = hi;
    if (p == 1 || hi == tiles) break;
  }
  c.tiles = (int)tiles;
  c.parts = (int)parts;
  c.blocks = (int)blocks;
  return c;
}

// anew: the call works out its logsumexp by itself, in launches ahead.
inline AttnBwdPlan attn_bwd_plan(int64_t B, int64_t H, int64_t H_kv, int64_t N, int64_t N_kv, int64_t D,
                                 bool causal, bool anew = false) {
  AttnBwdPlan p;
  p.nb_q = ceil_div(N, ATTN_BWD_ROWS);
  p.nb_kv = ceil_div(N_kv, ATTN_BWD_ROWS);
  const int64_t G = H / H_kv, k_planes = B * H_kv, q_planes = B * H;
  // Blocks of four waves own 128 columns, 32 a wave. Where there is less than one for each compute unit and
  // their loops are short, they own 64: two pairs of waves, each of which takes half of a step's rows, so
  // that a step takes half as long. (Long loops are better cut, below.) 128 and 64 columns (us): 8 heads of 257
  // causal rows 28 and 23, of 1024 42 and 36, 12 of 900 48 and 38, 10 of 1024 rows of 64 values 39 and 29; 4
  // of 2048, in parts, 59 and 64.
  const int64_t k_long = G * p.nb_q, q_long = p.nb_kv;
  const bool few = k_planes * ceil_div(N_kv, 128) + q_planes * ceil_div(N, 128) <= 256;
  p.columns = few && k_long <= 24 && q_long <= 24 ? 64 : 128;
  // With loops this short a block also works out its rows' constants, a tile a wave, which takes about as long
  // as a launch ahead but spares the host one (8 heads, in a graph, so and with a launch: 128 rows of 64
  // values 8.6 and 9.7 us, 257 12.8 and 11.8, 512 15.5 and 13.8, 128 rows of 128 values 14.6 and 13.7, 257
  // 22.5 and 17.4; a call takes the host 13.0 and 16.4 us).
  const int64_t steps = ATTN_BWD_ALONE * 64 / D;
  p.alone = !anew && p.columns == 64 && k_long <= steps && q_long <= steps;
  const int64_t wide = p.columns / ATTN_BWD_ROWS, k_tiles = ceil_div(N_kv, p.columns), q_tiles = ceil_div(N, p.columns);
  // The steps of the longest tiles, and of all of them, at two products' time for keys and one and a half
  // for queries, twice that for 128 columns; `share` is each resident block's part of it all.
  const int64_t k_all = k_planes * (causal ? G * (p.nb_q * k_tiles - wide * k_tiles * (k_tiles - 1) / 2) : k_long * k_tiles);
  const int64_t q_all = q_planes * (causal ? wide * q_tiles * (q_tiles + 1) / 2 : q_long * q_tiles);
  const int64_t resident = (D == 64 ? 3 : 2) * 256;
  const int64_t k_cost = 4 * wide, q_cost = 3 * wide;
  const int64_t share = (k_cost * k_all + q_cost * q_all) / resident;
  // A part may take a little more than that: parts are written in fp32 and read again, and tiles that are all
  // alike fit the card in one go with a fifth more. A tile is cut only where that saves more than the
  // joining launch costs (for each kind by itself, also where the other one's parts need that launch anyway); no part is
  // under 4 steps. Measured, all tiles in as many parts as the longest one
  // and so: 2 x 8 heads on 2 of 6449 causal rows of 64 values 358 and 292 us, one head of 16384 rows 550 and
  // 408, 6 heads on 1 of 1541 rows 101 and 93, 4096 causal rows, 32 heads on 8, 472 and 479.
  const int64_t may = share + share / (causal ? 20 : 5);
  auto most = [&](int64_t longest, int64_t cost) {
    if (longest * cost <= may + 56) return longest;
    const int64_t steps = ceil_div(may, cost);
    return steps < 4 ? (int64_t)4 : steps;
  };
  const int64_t most_k = most(k_long, k_cost), most_q = most(q_long, q_cost);
  p.keys = cut_tiles(k_tiles, k_long, causal ? wide * G : 0, k_long, most_k, k_planes);
  p.queries = causal ? cut_tiles(q_tiles, wide * q_tiles, wide, q_long, most_q, q_planes)
                     : cut_tiles(q_tiles, q_long, 0, q_long, most_q, q_planes);
  return p;
}

// A block's place in a cut: its tile, its plane, and which of its tile's parts it holds.
struct AttnBwdPlace {
  int u, plane, part, parts;
  // the part's share of n steps
  SAGE_HD int first(int n) const {
    const int left = n % parts;
    return n / parts * part + (part < left ? part : left);
  }
  SAGE_HD int end(int n) const { return first(n) + n / parts + (part < n % parts ? 1 : 0); }
};
SAGE_HD AttnBwdPlace attn_bwd_place(const AttnBwdCut& c, int block, int planes) {
  int lo = 0, p = c.parts;
  for (int i = 0; p > 1; ++i, --p) {
    const int hi = c.end[i], here = (hi - lo) * p * planes;
    if (block < here) break;
    block -= here;
    lo = hi;
  }
  const int x = block / planes, t = x / p;
  return {lo + t, block - x * planes, x - t * p, p};
}
// The block that holds the first part of tile u in plane 0 (those of the other planes follow it, the next
// part's are `planes` further on), and the tile's parts.
SAGE_HD int attn_bwd_first_part(const AttnBwdCut& c, int u, int planes, int& parts) {
  int lo = 0, p = c.parts, first = 0;
  for (int i = 0; u >= c.end[i]; ++i, --p) {
    first += (c.end[i] - lo) * p * planes;
    lo = c.end[i];
  }
  parts = p;
  return first + (u - lo) * p * planes;
}

}  // namespace sage
