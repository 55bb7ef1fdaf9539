"""CPU check of the tiles that the window attention's kernels visit (csrc/window_geometry.h).

A probe built with g++ from the kernels' own header walks the tiles of each pass as they do, for many lengths, windows,
first tokens and tables, and checks that

* every distance that a pass looks up in the bias table lies in the table (the select behind the lookup would discard a
  wrong value, but not the address);
* every visible pair is visited, once: by the query passes, and by the key pass's band or its first tokens' chunks.
"""

import os
import subprocess
import tempfile

from conftest import PKG_ROOT

GEOMETRY = os.path.join(PKG_ROOT, "csrc", "window_geometry.h")

PROBE = r"""
#include <stdio.h>
#include <string.h>
#include <vector>
#include "GEOMETRY"
using namespace dfl;

struct Args { int M, N, window, n_sink, causal; };
static unsigned rng = 12345u;
static int rnd(int n) { rng = rng * 1664525u + 1013904223u; return (int)((rng >> 8) % (unsigned)n); }
static int fails = 0;
static long looked = 0;

static void lookup(const char* pass, const Args& a, const RelSpec& r, int t0, int j0) {
  const int lo = rel_lut_base(r) + t0 - (j0 + 31), hi = rel_lut_base(r) + t0 + 31 - j0;
  ++looked;
  if (lo >= 0 && hi < rel_lut_size(r)) return;
  if (++fails < 20)
    printf("%s reads [%d, %d] of %d: M %d N %d window %d n_sink %d causal %d dist %d t0 %d j0 %d\n", pass, lo, hi,
           rel_lut_size(r), a.M, a.N, a.window, a.n_sink, a.causal, r.dist(), t0, j0);
}

static void walk(const Args& a, const RelSpec& r) {
  const WinVis vis(a);
  const int shift = a.N - a.M, G = 64;
  std::vector<unsigned char> seen((size_t)a.M * a.N), keyed((size_t)a.M * a.N);
  for (int BK = 32; BK <= 64; BK += 32) {  // query passes: the forward skips whole tiles, the backward halves
    for (int backward = 0; backward < 2; ++backward) {
      memset(seen.data(), 0, seen.size());
      for (int i128 = 0; i128 < a.M; i128 += 128) {
        const KeyTiles kt(a, i128 + shift, win_min(a.M, i128 + 128) - 1 + shift, BK);
        for (int wave = 0; wave < 4; ++wave)
          for (int it = 0; it < kt.total; ++it) {
            const int j0 = kt.tile(it) * BK, t0 = i128 + 32 * wave + shift;
            if (!backward && vis.none(t0, j0, BK)) continue;
            const bool one = !backward && rel_far(r, t0, j0, BK) >= 0;
            for (int js = j0; js < j0 + BK; js += 32) {
              if (vis.none(t0, js)) continue;
              if (!one && rel_far(r, t0, js) < 0) lookup(backward ? "backward" : "forward", a, r, t0, js);
              for (int t = t0; t < t0 + 32 && t < a.N; ++t)
                for (int j = js; j < js + 32 && j < a.N; ++j) seen[(size_t)(t - shift) * a.N + j] += vis.sees(t, j);
            }
          }
      }
      for (int i = 0; i < a.M; ++i)
        for (int j = 0; j < a.N; ++j)
          if (seen[(size_t)i * a.N + j] != (vis.sees(i + shift, j) ? 1 : 0) && ++fails < 20)
            printf("query pass: pair %d %d\n", i, j);
    }
  }
  for (int k0 = 0; k0 < a.N; k0 += G) {  // the key pass's band
    const int k1 = win_min(a.N, k0 + G) - 1, ilo = win_max(0, k0 - vis.off - shift);
    const int ihi = win_min(a.M, k1 - vis.off + (int)vis.range - shift);
    for (int i0 = ilo; i0 < ihi; i0 += 32)
      for (int j0 = k0; j0 < k0 + G; j0 += 32) {
        const int t0 = i0 + shift;
        if (vis.none_near(t0, j0)) continue;
        if (rel_far(r, t0, j0) < 0) lookup("band", a, r, t0, j0);
        for (int i = i0; i < i0 + 32 && i < ihi; ++i)
          for (int j = j0; j < j0 + 32 && j < a.N; ++j) keyed[(size_t)i * a.N + j] += vis.near(i + shift, j);
      }
  }
  const int ns = win_min(a.n_sink, a.N), first = a.causal ? win_max(0, win_min(a.window, a.N) - shift) : 0;
  if (a.N > a.window)
    for (int i0 = first; i0 < a.M; i0 += 32)  // its first tokens
      for (int j0 = 0; j0 < ns; j0 += 32) {
        const int t0 = i0 + shift;
        if (!vis.some_first(t0, j0)) continue;
        if (rel_far(r, t0, j0) < 0) lookup("first tokens", a, r, t0, j0);
        for (int i = i0; i < i0 + 32 && i < a.M; ++i)
          for (int j = j0; j < j0 + 32 && j < ns; ++j)
            keyed[(size_t)i * a.N + j] += !vis.near(i + shift, j) & vis.first(i + shift, j);
      }
  for (int i = 0; i < a.M; ++i)
    for (int j = 0; j < a.N; ++j)
      if (keyed[(size_t)i * a.N + j] != (vis.sees(i + shift, j) ? 1 : 0) && ++fails < 20)
        printf("key pass: pair %d %d of M %d N %d window %d n_sink %d causal %d\n", i, j, a.M, a.N, a.window, a.n_sink, a.causal);
}

int main() {
  const int windows[] = {1, 2, 7, 31, 32, 33, 64, 100, 250, 1000}, sinks[] = {0, 1, 4, 31, 33, 64, 100, 128};
  const int dists[] = {1, 2, 31, 48, 63, 64, 65, 130, 500, 2048};
  for (int k = 0; k < 3000; ++k) {
    Args a;
    a.N = 1 + rnd(k % 3 ? 330 : 70);
    a.M = rnd(2) ? a.N : 1 + rnd(a.N);
    if (k % 7 == 0) a.M = win_max(1, a.N - rnd(66));
    a.window = windows[rnd(10)];
    a.n_sink = sinks[rnd(8)];
    a.causal = rnd(2);
    RelSpec r;
    r.n = 1;
    r.both = !a.causal;
    r.edge[0] = dists[rnd(10)];
    walk(a, r);
  }
  printf("lookups %ld fails %d\n", looked, fails);
  return fails != 0;
}
"""


def test_lookups_stay_in_the_table_and_pairs_are_visited_once():
    with tempfile.TemporaryDirectory() as td:
        src, exe = os.path.join(td, "geometry.cpp"), os.path.join(td, "geometry")
        open(src, "w").write(PROBE.replace("GEOMETRY", GEOMETRY))
        subprocess.run(["g++", "-std=c++17", "-O2", "-o", exe, src], check=True)
        out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout[-3000:]
    assert int(out.stdout.split()[1]) > 10000
