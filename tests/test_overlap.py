"""csrc/eg_overlap.h against enumeration: random small matrices of any strides, whether one overlaps itself and whether two
share a byte.  Where the header does not look (columns apart, of different strides) it may only say "apart"."""
from __future__ import annotations

import subprocess

from tests.conftest import ROOT

PROGRAM = r"""
#include "eg_overlap.h"
#include <stdio.h>
#include <random>
#include <set>
using eg::Extent;
static std::mt19937 gen(1);
static int rnd(int a, int b) { return a + (int)(gen() % (unsigned)(b - a + 1)); }
struct Made { Extent extent; std::set<int64_t> bytes; bool self; };
static Made make() {
  const int item = rnd(0, 1) ? 2 : 4, rows = rnd(1, 6), cols = rnd(1, 6), at = 1000 + 2 * rnd(-40, 40);
  int s0 = rnd(0, 9), s1 = rnd(0, 1) ? 1 : rnd(0, 9);
  if (rnd(0, 2) == 0) std::swap(s0, s1);
  if (rnd(0, 9) == 0) s0 = -s0;
  Made m{Extent((void*)(intptr_t)at, rows, cols, s0, s1, item), {}, false};
  for (int i = 0; i < rows; ++i)
    for (int j = 0; j < cols; ++j)
      for (int b = 0; b < item; ++b)
        if (!m.bytes.insert(at + (i * s0 + j * s1) * item + b).second) m.self = true;
  return m;
}
int main() {
  int shared = 0, exact = 0;
  for (int k = 0; k < 200000; ++k) {
    const Made a = make(), b = make();
    bool want = false;
    for (int64_t x : a.bytes) want = want || b.bytes.count(x);
    const bool got = overlap(a.extent, b.extent);
    const bool looks = (a.extent.rows_whole() && b.extent.rows_whole()) ||
                       (a.extent.step[0] == b.extent.step[0] && a.extent.step[1] == b.extent.step[1]);
    if (overlaps_itself(a.extent) != a.self || (got && !want) || (looks && got != want) || got != overlap(b.extent, a.extent))
      return fprintf(stderr, "pair %d: self %d, shared %d, said %d\n", k, a.self, want, got), 1;
    shared += want;
    exact += looks;
  }
  return shared > 20000 && exact > 20000 ? 0 : 2;
}
"""


def test_against_enumeration(tmp_path):
    source, program = tmp_path / "overlap.cpp", tmp_path / "overlap"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", str(ROOT / "engraft-ngram_amd" / "csrc"), str(source), "-o", str(program)],
                   check=True, timeout=120)
    done = subprocess.run([str(program)], capture_output=True, text=True, timeout=100)
    assert done.returncode == 0, done.stderr
