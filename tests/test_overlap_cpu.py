"""Which tensors of rows share memory (csrc/overlap.h), compiled by itself and compared with sets of bytes."""
import subprocess

from theano_b200 import build

PROGRAM = r"""
#include <stdio.h>
#include <stdlib.h>
#include <random>
#include <set>
#include <vector>
#include "overlap.h"
using namespace b200;
struct Rows { long long base, seq, row, sequences, length, width; };
static std::vector<int> bytes(const Rows& r, int es) {
  std::vector<int> seen(6000, 0);
  for (long long s = 0; s < r.sequences; ++s)
    for (long long t = 0; t < r.length; ++t)
      for (long long k = 0; k < r.width * es; ++k) ++seen[r.base + (s * r.seq + t * r.row) * es + k];
  return seen;
}
int main() {
  std::mt19937 g(1);
  auto pick = [&](int lo, int hi) { return lo + static_cast<int>(g() % (hi - lo + 1)); };
  int met = 0, in_itself = 0, same = 0;
  for (int n = 0; n < 200000; ++n) {
    const int es = pick(0, 1) ? 2 : 4;
    Rows r[2];
    for (int k = 0; k < 2; ++k) {
      r[k].sequences = pick(0, 4); r[k].length = pick(0, 6); r[k].width = pick(1, 6);
      r[k].row = pick(0, 20); r[k].seq = pick(0, 60);
      r[k].base = pick(0, 200) * es;
    }
    if (pick(0, 2)) { r[1].row = r[0].row; r[1].seq = r[0].seq; }
    if (pick(0, 3) == 0) { r[1].sequences = r[0].sequences; r[1].length = r[0].length; }
    if (pick(0, 9) == 0) r[1] = r[0];
    static char memory[8192];
    Region a[2];
    std::vector<int> b[2];
    for (int k = 0; k < 2; ++k) {
      b200conv_rows rows = {r[k].row, r[k].seq, 0, 0};
      a[k] = region("", memory + r[k].base, rows, r[k].sequences, r[k].length, r[k].width, es);
      b[k] = bytes(r[k], es);
      bool twice = false;
      for (int v : b[k]) twice |= v > 1;
      if (folded(a[k]) != twice) { printf("folded %d\n", n); return 1; }
      in_itself += twice;
    }
    bool want = false;
    for (size_t i = 0; i < b[0].size(); ++i) want |= b[0][i] && b[1][i];
    if (overlap(a[0], a[1]) != want || overlap(a[1], a[0]) != want) { printf("overlap %d: %d\n", n, want); return 1; }
    if (same_place(a[0], a[1])) { ++same; if (!a[0].empty() && !want) return 2; }
    met += want;
  }
  Region none = region("", nullptr, 100), flat = region("", reinterpret_cast<void*>(4096), 100), next = region("", reinterpret_cast<void*>(4196), 8);
  if (overlap(none, flat) || overlap(flat, next) || !overlap(flat, region("", reinterpret_cast<void*>(4195), 8))) return 3;
  // far apart in one address space, tensors of many rows
  b200conv_rows halves = {1 << 14, 1LL << 40, 0, 0};
  Region x = region("", reinterpret_cast<void*>(1LL << 20), halves, 4, 1 << 26, 1 << 13, 2), y = region("", reinterpret_cast<void*>((1LL << 20) + (1 << 14)), halves, 4, 1 << 26, 1 << 13, 2);
  if (overlap(x, y) || folded(x)) return 4;
  puts(met > 20000 && in_itself > 20000 && same > 5000 ? "ok" : "too few cases");
}
"""


def test_against_sets_of_bytes(tmp_path):
    src, exe = tmp_path / "overlap.cpp", tmp_path / "overlap"
    src.write_text(PROGRAM)
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-I", build.CSRC, str(src), "-o", str(exe)])
    p = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and p.stdout.strip() == "ok", (p.returncode, p.stdout)
