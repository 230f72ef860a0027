"""CPU tests of how the serving kernels share out their work (csrc/serve_sched.h): a
host program built from the header checks, over seeded random batches, that the classes
of row blocks hold every block once, longest first, and that the parts of requests hold
every tile once and fit the workspace that is planned for them."""
import os
import shutil
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "custom_ops_amd", "csrc")

PROGRAM = r"""
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>
#include <vector>
#include "serve_sched.h"
using namespace mi355fa;
#define REQUIRE(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); exit(1); } } while (0)

int main() {
  std::mt19937 g(7);
  auto pick = [&](int lo, int hi) { return lo + (int)(g() % (unsigned)(hi - lo + 1)); };
  for (int round = 0; round < 3000; ++round) {
    RowSpans s{pick(0, 1), pick(0, 2) ? kNoWindow : pick(1, 3000), pick(5, 8)};
    const int n = pick(1, 20);
    std::vector<int> rows(n), keys(n);
    int64_t total = 0;
    for (int i = 0; i < n; ++i) {
      rows[i] = pick(0, 3) ? pick(0, 2000) : pick(0, 40);
      keys[i] = pick(0, 2) ? rows[i] : pick(0, 4000);
      total += rows[i];
    }
    int most = 0, blocks = 0;
    for (int i = 0; i < n; ++i) {
      const int c = block_count(s, rows[i]);
      blocks += c;
      for (int b = 0; b < c; ++b) {
        const int x = block_span(s, rows[i], keys[i], b);
        REQUIRE(x >= 0 && x <= std::max(keys[i], 0));
        if (b) REQUIRE(x >= block_span(s, rows[i], keys[i], b - 1));
        most = std::max(most, x);
      }
    }
    REQUIRE(blocks <= (total >> s.shift) + n);   // the grid holds two more segments
    for (int levels : {1, 4}) {
      std::set<std::pair<int, int>> seen;
      for (int level = 0; level < levels; ++level) {
        const int lo = class_floor(most, level, levels), hi = class_ceil(most, level);
        for (int i = 0; i < n; ++i) {
          const int b0 = first_over(s, rows[i], keys[i], lo), b1 = first_over(s, rows[i], keys[i], hi);
          REQUIRE(b0 <= b1);
          for (int b = b0; b < b1; ++b) {
            const int x = block_span(s, rows[i], keys[i], b);
            REQUIRE(x > lo && x <= hi);
            REQUIRE(seen.insert({i, b}).second);
          }
        }
      }
      REQUIRE((int)seen.size() == blocks);
    }
  }
  for (int round = 0; round < 2000; ++round) {   // every rank has a block of its own
    const int ranks = pick(1, 300), fold = pick(0, 200);
    std::set<int> seen;
    for (int r = 0; r < ranks; ++r) {
      const int b = folded(r, fold, ranks);
      REQUIRE(b >= 0 && b < ranks && seen.insert(b).second);
      REQUIRE((b < fold) == (r < fold) && (b < 2 * fold) == (r < 2 * fold));
    }
  }
  // the largest sizes
  {
    RowSpans s{1, kNoWindow, 5};
    const int big = 1 << 30;
    REQUIRE(block_count(s, big) == big >> 5);
    REQUIRE(block_span(s, big, big, (big >> 5) - 1) == big);
    REQUIRE(first_over(s, big, big, INT_MAX) == big >> 5);
    REQUIRE(first_over(s, big, 0, -1) == 0);
    RowSpans w{0, kNoWindow - 1, 8};
    REQUIRE(block_span(w, big, big, 0) == big);
  }
  for (int round = 0; round < 3000; ++round) {
    const int b = pick(1, 200), groups = pick(1, 40), target = pick(1, 2000), least = pick(1, 40);
    const int window = pick(0, 1) ? kNoWindow : pick(1, 5000);
    const int64_t cap = pick(0, 1) ? 1 << 20 : pick(0, 9000);
    std::vector<KeySpan> k(b);
    int64_t sum = 0;
    for (auto& x : k) {
      const int len = pick(0, 4) ? pick(-3, 20000) : pick(0, 2000000);
      x = key_span(len, cap, window);
      REQUIRE(x.len >= 0 && x.len <= cap && x.first >= 0 && x.first <= x.len && x.tiles >= 0);
      REQUIRE(x.tile0 * kDecTile <= x.first && (x.tile0 + x.tiles) * kDecTile >= x.len);
      sum += weighed(x.tiles);
    }
    REQUIRE(sum < INT_MAX);
    const int per = part_size((int)sum, groups, target, least);
    int64_t parts = 0;
    for (auto& x : k) {
      const int n = part_count(x.tiles, per);
      REQUIRE(n >= 1);
      parts += (int64_t)n * groups;
      int at = 0;
      for (int p = 0; p < n; ++p) {
        REQUIRE(part_start(x.tiles, n, p) == at);
        at = part_start(x.tiles, n, p + 1);
        REQUIRE(at >= part_start(x.tiles, n, p) && at <= x.tiles);
      }
      REQUIRE(at == x.tiles);
    }
    REQUIRE(parts <= (int64_t)target + (int64_t)b * groups);   // the workgroups and slots that are planned
  }
  // the longest span that a table may have
  const KeySpan x = key_span(INT_MAX, (int64_t)1 << 30, kNoWindow);
  REQUIRE(x.len == 1 << 30 && x.tiles == 1 << 25);
  printf("ok\n");
}
"""


def test_schedules(tmp_path):
    src, exe = tmp_path / "sched.cpp", tmp_path / "sched"
    src.write_text(PROGRAM)
    cxx = os.environ.get("CXX") or shutil.which("g++")
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout == "ok\n", out.stdout + out.stderr[-2000:]
