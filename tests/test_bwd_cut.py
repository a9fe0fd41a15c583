"""The backward pass's cut into blocks (`csrc/bwd_cut.h`), compiled for the host: every step of every tile
is taken once, by a block of its own place, and the joining launch finds a tile's parts where they are."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = os.path.join(ROOT, "sageattention-rdna4_amd", "csrc", "bwd_cut.h")

_MAIN = r"""
#include "%s"
#include <cstdio>
#include <vector>
using namespace sage;
static int bad(const char* what, long a, long b, long c) {
  std::printf("%%s %%ld %%ld %%ld\n", what, a, b, c);
  return 1;
}
// steps(u): of tile u, the longest first
template <typename F>
int check(const AttnBwdCut& c, int planes, F steps) {
  std::vector<int> taken((size_t)c.tiles * planes, 0), next((size_t)c.tiles * planes, 0);
  int before = 1 << 30;
  for (int u = 0; u < c.tiles; ++u) {
    if (steps(u) > before) return bad("order", u, steps(u), before);
    before = steps(u);
  }
  for (int b = 0; b < c.blocks; ++b) {
    const AttnBwdPlace at = attn_bwd_place(c, b, planes);
    if (at.u < 0 || at.u >= c.tiles || at.plane < 0 || at.plane >= planes) return bad("place", b, at.u, at.plane);
    const size_t i = (size_t)at.u * planes + at.plane;
    if (at.part != next[i]++) return bad("part", b, at.u, at.part);
    const int n = steps(at.u);
    if (at.first(n) != taken[i]) return bad("first", b, at.first(n), taken[i]);
    if (at.parts > 1 && at.end(n) <= at.first(n)) return bad("empty", b, at.first(n), at.end(n));
    taken[i] = at.end(n);
    if ((at.parts > 1) != (b < c.cut_blocks) || (at.parts > 1) != (at.u < c.cut)) return bad("cut", b, at.u, at.parts);
    if (at.parts > 1) {
      int parts = 0;
      const int first = attn_bwd_first_part(c, at.u, planes, parts);
      if (parts != at.parts || first + at.plane + at.part * planes != b) return bad("join", b, first, parts);
    }
  }
  for (int u = 0; u < c.tiles; ++u)
    for (int p = 0; p < planes; ++p)
      if (taken[(size_t)u * planes + p] != steps(u)) return bad("steps", u, p, taken[(size_t)u * planes + p]);
  return 0;
}
int main() {
  long plans = 0, cut = 0, narrow = 0;
  const int lengths[] = {1, 2, 63, 64, 65, 128, 129, 257, 500, 777, 1024, 1541, 1777, 2048, 4097, 6449, 11000, 16384, 47520};
  for (int B : {1, 2, 3, 9}) for (int H_kv : {1, 2, 8, 10}) for (int G : {1, 3, 4, 6, 32}) for (int D : {64, 128})
    for (int N : lengths) for (int N_kv : lengths) for (int causal = 0; causal < 2; ++causal) {
      if (causal && N != N_kv) continue;
      if ((long)B * H_kv * G * N > 2000000) continue;
      const AttnBwdPlan p = attn_bwd_plan(B, (long)H_kv * G, H_kv, N, N_kv, D, causal);
      const int nb = (int)p.nb_q, nk = (int)p.nb_kv, tq = p.queries.tiles, c = (int)p.columns, wide = c / 64;
      if (c != 64 && c != 128) return bad("columns", c, 0, 0);
      if (p.keys.tiles != (N_kv + c - 1) / c || tq != (N + c - 1) / c) return bad("tiles", N, N_kv, tq);
      if (check(p.keys, B * H_kv, [&](int u) { return G * (nb - (causal ? wide * u : 0)); })) return 1;
      if (check(p.queries, B * H_kv * G, [&](int u) {
            const int end = wide * (tq - u);
            return causal ? (end < nk ? end : nk) : nk;
          })) return 1;
      ++plans;
      cut += p.keys.cut > 0;
      narrow += wide == 1;
    }
  std::printf("plans %%ld %%ld %%ld\n", plans, cut, narrow);
  return 0;
}
"""


def _run(tmp_path, header):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    src, exe = tmp_path / "cut.cpp", tmp_path / "cut"
    src.write_text(_MAIN % header)
    subprocess.run(["g++", "-O2", "-std=c++17", "-o", str(exe), str(src)], check=True)
    return subprocess.run([str(exe)], capture_output=True, text=True)


def test_every_step_once(tmp_path):
    res = _run(tmp_path, SRC)
    assert res.returncode == 0, res.stdout
    plans, cut, narrow = (int(x) for x in res.stdout.split()[1:])
    assert plans > 10000 and cut > 2000 and 500 < narrow < plans - 500


def test_a_lost_step_is_found(tmp_path):
    text = open(SRC).read()
    old = "return n / parts * part + (part < left ? part : left);"
    assert old in text
    planted = tmp_path / "bwd_cut.h"
    planted.write_text(text.replace(old, "return n / parts * part;"))
    assert _run(tmp_path, planted).returncode == 1
