"""The index arithmetic of the norm's row kernels, enumerated on the host: no
thread reads outside of the weight, also where the last CTA has more rows than
the tensor, and every element of every row is covered once."""

import os
import subprocess

from tests.conftest import ROOT

PROGRAM = r"""
#include <cstdio>
#include <vector>
#include "norm_index.cuh"
using namespace i8moe;

template <int kVec, int kPer, bool kShift>
int check(int k, int64_t rows) {
  const RowBlock b = row_block<kVec, kPer, kShift>(k);
  if (b.x > 1024) return 0;
  const int64_t ctas = (rows + b.y - 1) / b.y;
  std::vector<int> seen(rows * k, 0);
  for (int64_t c = 0; c < ctas; ++c)
    for (int y = 0; y < b.y; ++y)
      for (int tid = 0; tid < b.x; ++tid) {
        const int64_t r = c * b.y + y;
        const RowPart part = row_part<kVec, kShift>(r, rows, k, tid);
        for (int p = 0; p < kPer; ++p) {
          const int i = p * b.x * kVec + part.first;
          if (i >= part.k) continue;  // the kernels' only test
          if (r >= rows) return std::printf("row %lld of %lld has a column, k %d\n", (long long)r, (long long)rows, k);
          for (int e = 0; e < kVec; ++e) {
            const int at = nearest_element(i + e, part.k);
            if (at < 0 || at >= k) return std::printf("reads element %d of %d\n", at, k);
            if (i + e >= 0 && i + e < k) ++seen[r * k + i + e];
          }
        }
      }
  for (int n : seen)
    if (n != 1) return std::printf("an element is covered %d times, k %d\n", n, k);
  return 0;
}

int main() {
  for (int k = 1; k < 300; ++k)
    for (int64_t rows : {1, 2, 3, 5, 7, 8, 31, 83, 129}) {
      int bad = check<1, 8, false>(k, rows);
      if (k % 8 == 0) bad += check<8, 1, false>(k, rows) + check<8, 2, false>(k, rows);
      if (k % 4 == 0) bad += check<4, 1, false>(k, rows) + check<4, 2, false>(k, rows);
      if (k >= 8) bad += check<8, 1, true>(k, rows) + check<8, 2, true>(k, rows);
      if (k >= 4) bad += check<4, 1, true>(k, rows) + check<4, 2, true>(k, rows);
      if (bad) return 1;
    }
  for (int k : {1001, 2047, 4095, 4097, 8191})
    if (check<8, 1, true>(k, 9) + check<4, 2, true>(k, 9)) return 1;
  return 0;
}
"""


def test_no_thread_reads_outside_of_the_weight(tmp_path):
    src, exe = tmp_path / "index.cpp", tmp_path / "index"
    src.write_text(PROGRAM)
    cxx = os.environ.get("CXX", "g++")
    include = ROOT / "int8blockwisegemm_b200" / "csrc"
    res = subprocess.run([cxx, "-O2", "-std=c++17", "-xc++", f"-I{include}", str(src), "-o", str(exe)],
                         capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0, res.stdout
