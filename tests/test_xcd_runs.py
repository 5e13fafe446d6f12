"""Every run of a step is some workgroup's, whatever the number of CUs: the launch and the
kernels' arithmetic (csrc/xcd_runs.h), compiled for the host."""

import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pipeswift_amd", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <vector>
#include "xcd_runs.h"
using namespace psk_detail;
// runs that no workgroup of a launch of `grid` takes, or that two take
static int wrong(int64_t grid, int64_t runs) {
  std::vector<int> taken(runs, 0);
  for (int64_t w = 0; w < grid; ++w) {
    const int64_t j = run_of_xcd(runs, w & 7, w >> 3);
    if (j < runs) ++taken[j];
  }
  int n = 0;
  for (int t : taken) n += t != 1;
  return n;
}
int main() {
  for (int64_t slots = 0; slots <= 600; ++slots) {
    const int64_t grid = xcd_rounds(slots);
    if (grid % 8 || grid < 8 || (slots >= 8 && grid > slots)) return std::printf("grid %d of %d\n", int(grid), int(slots)), 1;
    for (int64_t runs = 1; runs <= grid; ++runs)
      if (wrong(grid, runs)) return std::printf("%d runs of %d\n", int(runs), int(grid)), 1;
  }
  if (wrong(76, 76) != 3) return std::printf("76 workgroups are no whole rounds: three runs are lost\n"), 1;
  return 0;
}
"""


def test_every_run_is_taken_once(tmp_path):
    cxx = shutil.which("g++") or shutil.which("clang++")
    if cxx is None:
        pytest.skip("no host compiler")
    (tmp_path / "runs.cpp").write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-O2", "-I", CSRC, str(tmp_path / "runs.cpp"), "-o", str(tmp_path / "runs")], check=True)
    done = subprocess.run([str(tmp_path / "runs")], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout


def test_launches_of_runs_are_whole_rounds():
    """No launch that deals runs out by XCD takes its count from elsewhere."""
    for name in ("tree_attention.hip", "attention_weights.hip"):
        with open(os.path.join(CSRC, name)) as f:
            text = f.read()
        counts = [line for line in text.splitlines() if "max_runs =" in line]
        assert counts and all("xcd_rounds(" in c or "s.max_runs)" in c or "= 1;" in c for c in counts), counts
