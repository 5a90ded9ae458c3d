"""Which items of a join its workgroups take (csrc/kv_walk.hpp), on the CPU: those of each row of each sequence once, those of
other rows never, whatever lies between the sequences and however many there are."""
import os
import shutil
import subprocess

import pytest

import example_matmul_metal4_amd as mtk

PROGRAM = r"""
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>
#include "kv_walk.hpp"

// A batch as the kernels see it: 64 sequences at a time.
struct View {
  const std::vector<int> &start;
  int T, b0 = 0, steps = 0;
  int B() const { return (int)start.size() - 1; }
  kv_seq seq(int b) const { return kv_sequence(start[b], start[b + 1], 0, T, 1, 4); }
  int windows() const { return (B() + 63) / 64; }
  int hit(int t) const {
    for (int i = 0; i < 64 && b0 + i < B(); ++i)
      if (seq(b0 + i).first <= t && t < seq(b0 + i).first + seq(b0 + i).rows) return i;
    return -1;
  }
  int later(int t) const {
    int x = INT32_MAX;
    for (int i = 0; i < 64 && b0 + i < B(); ++i)
      if (seq(b0 + i).rows > 0 && seq(b0 + i).first > t) x = std::min(x, seq(b0 + i).first);
    return x;
  }
  void step() {
    b0 = b0 + 64 < B() ? b0 + 64 : 0;
    ++steps;
  }
  kv_rows rows_of(int l) const { return kv_rows{seq(b0 + l).first, seq(b0 + l).rows}; }
};

int main() {
  std::mt19937 rng(5);
  auto log = [&](int lo, int hi) { return (int)(lo * std::pow((double)hi / lo, std::uniform_real_distribution<>(0, 1)(rng))); };
  for (int n = 0; n < 4000; ++n) {
    const int B = log(1, 400), T = log(1, 3000), per_row = log(1, 9), S_q = rng() % 2 ? T : log(1, T + 1), grid = log(1, 1200);
    std::vector<int> start(B + 1);
    for (int &x : start) x = (int)(rng() % (T + 1));
    std::sort(start.begin(), start.end());
    if (n % 4 == 1) std::fill(start.begin(), start.begin() + B / 2 + 1, start[B / 2]);  // rows in front, sequences of none
    if (n % 4 == 2) std::fill(start.begin() + (B + 1) / 2, start.end(), start[(B + 1) / 2]);  // rows behind the last
    if (n % 8 == 3 && B > 1) {  // starts that do not ascend, no row claimed twice: the front half's behind the others'
      std::rotate(start.begin(), start.begin() + B / 2, start.end());
    }
    std::vector<int> want(T, 0), got(T * per_row, 0);
    for (int b = 0; b < B; ++b) {
      const kv_seq s = kv_sequence(start[b], start[b + 1], 0, T, 1, 4);
      for (int i = 0; i < std::min(s.rows, S_q); ++i) ++want[s.first + i];
    }
    int most = 0;
    for (int w = 0; w < grid; ++w) {
      View v{start, T};
      int open_at = -1;
      kv_walk(v, T, per_row, S_q, w, grid, [&](int l) { return open_at = v.b0 + l, true; }, [&](int it) {
        const kv_seq s = v.seq(open_at);
        if (it % grid != w || it / per_row < s.first || it / per_row >= s.first + s.rows) printf("item %d\n", it), exit(1);
        ++got[it];
      });
      most = std::max(most, v.steps);
    }
    for (int it = 0; it < T * per_row; ++it)
      if (got[it] != want[it / per_row])
        return printf("B %d T %d per row %d S_q %d grid %d: item %d (row %d) %d times, not %d\n", B, T, per_row, S_q, grid, it, it / per_row,
                      got[it], want[it / per_row]), 1;
    // the windows are walked once, and once more for the rows in front and behind
    if (n % 8 != 3 && most > 3 * ((B + 63) / 64)) return printf("B %d: %d steps\n", B, most), 1;
  }
  return 0;
}
"""


def test_every_row_of_a_sequence_is_joined_once(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    src, exe = tmp_path / "walk.cpp", tmp_path / "walk"
    src.write_text(PROGRAM)
    r = subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                        f"-I{os.path.join(mtk.PKG, 'csrc')}", str(src), "-o", str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.stdout + r.stderr)[-3000:]
