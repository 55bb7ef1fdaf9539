"""Launches of more threads than a grid's x dimension may have (csrc/launch_slices.h): a probe built with g++ from the header
checks that the slices are the workgroups, each once, that none has 2^32 threads, and that the first failure ends them."""

import os
import subprocess

from conftest import PKG_ROOT

PROBE = r"""
#include <cstdio>
#include "launch_slices.h"
using namespace dfl;

int main() {
  long long slices = 0;
  const int sizes[] = {64, 128, 256, 512, 768, 1024};
  for (int threads : sizes) {
    const long long most = launch_most(threads);
    if (most * threads >= (1ll << 32) || (most + 1) * threads < (1ll << 32)) return 1;
    const long long counts[] = {0, 1, 255, most - 1, most, most + 1, 2 * most, 2 * most + 7, (1ll << 31) - 1};
    for (long long blocks : counts) {
      long long at = 0;
      bool fine = true;
      const int e = launch_slices(blocks, threads, [&](long long first, long long count) {
        fine = fine && first == at && count > 0 && count * threads < (1ll << 32);
        at = first + count;
        ++slices;
        return 0;
      });
      if (e || !fine || at != blocks) return 2;
      int calls = 0;
      const int failed = launch_slices(blocks, threads, [&](long long, long long) { return ++calls == 2 ? 7 : 0; });
      if (failed != (blocks > most ? 7 : 0) || calls > 2) return 3;
    }
  }
  std::printf("slices %lld\n", slices);
}
"""


def test_slices_are_the_workgroups(tmp_path):
    src, exe = tmp_path / "probe.cpp", tmp_path / "probe"
    src.write_text(PROBE)
    subprocess.run(["g++", "-std=c++17", "-O2", "-I", os.path.join(PKG_ROOT, "csrc"), "-o", exe, src], check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0, (out.returncode, out.stdout)
    assert int(out.stdout.split()[1]) > 50
