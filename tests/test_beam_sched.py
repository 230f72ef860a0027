"""CPU tests of how the kernels for several continuations of a prompt share out their work
(csrc/beam_sched.h): a host program built from the header checks, over seeded random
batches, that every seen key is read once, by the group or by its request, and that the
parts hold every tile once and fit the grid."""
import os
import shutil
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "custom_ops_amd", "csrc")

PROGRAM = r"""
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>
#include "beam_sched.h"
using namespace mi355fa;
#define REQUIRE(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); exit(1); } } while (0)

int main() {
  std::mt19937 g(7);
  auto pick = [&](int lo, int hi) { return lo + (int)(g() % (unsigned)(hi - lo + 1)); };
  for (int round = 0; round < 4000; ++round) {
    const int n = pick(1, 9), prefix = pick(0, 3) ? pick(0, 700) : pick(0, 40);
    const int window = pick(0, 2) ? kNoWindow : pick(1, 900);
    std::vector<int> len(n);
    int least = INT_MAX, most = 0;
    for (int& x : len) {
      x = pick(0, 5) ? prefix + pick(0, 300) : pick(0, 400);
      if (x > 0) least = std::min(least, x), most = std::max(most, x);
    }
    const TileSpan s = most ? shared_tiles(prefix, least, most, window, n) : TileSpan{0, 0};
    REQUIRE(s.t0 >= 0 && s.t0 <= s.t1 && s.t1 * kDecTile <= prefix);
    for (int x : len) {
      const OwnTiles o = own_tiles(x, window, s);
      REQUIRE(o.count >= 0 && (x > 0 || o.count == 0));
      std::vector<int> read(x + 1, 0);
      for (int i = 0; i < o.count; ++i)
        for (int e = 0; e < kDecTile; ++e) {
          const int key = own_tile(o, i) * kDecTile + e;
          REQUIRE(key >= 0);
          if (key >= o.lo && key < o.len) ++read[key];
        }
      if (x > 0)
        for (int t = s.t0 * kDecTile; t < s.t1 * kDecTile; ++t) {
          REQUIRE(t < x && t >= x - window);   // a shared tile hides nothing
          ++read[t];
        }
      for (int key = 0; key < x; ++key) REQUIRE(read[key] == (key >= x - window ? 1 : 0));
    }
  }
  REQUIRE(own_tiles(1 << 30, kNoWindow, TileSpan{0, 0}).count == 1 << 25);
  for (int round = 0; round < 4000; ++round) {
    const int items = pick(1, 60), groups = pick(0, items), target = pick(128, 1024), ways = 1 << pick(0, 2), weight = own_weight(128 / ways);
    std::vector<int> tiles(items), units(items);
    int64_t sum = 0, of_groups = 0, own = 0, units_g = 0, units_r = 0;
    for (int i = 0; i < items; ++i) {
      tiles[i] = pick(0, 3) ? pick(0, 3000) : pick(0, 3) ? 0 : 1 << pick(0, 25);
      units[i] = pick(1, 64);
      sum += (int64_t)tiles[i] * units[i] * (i < groups ? 4 / ways : weight);
      (i < groups ? units_g : units_r) += units[i];
    }
    const int steps = share_steps(sum, target), per = share_size(steps, ways), wave_per = wave_share_size(steps, weight);
    REQUIRE(steps >= 1 && per >= 4 && per >= steps * ways && wave_per >= 1 && wave_per * weight >= steps);
    int last = -1, unit = 0;   // of requests: the last part's row
    for (int i = 0; i < items; ++i) {
      if (i < groups) {
        const int n = share_count(tiles[i], per);
        of_groups += (int64_t)n * units[i];
        REQUIRE((n == 0) == (tiles[i] == 0));
        for (int p = 0; p < n; ++p) {
          const int a = share_start(tiles[i], n, p), b = share_start(tiles[i], n, p + 1);
          REQUIRE(a < b && b - a <= per);
        }
        if (n) REQUIRE(share_start(tiles[i], n, 0) == 0 && share_start(tiles[i], n, n) == tiles[i]);
        continue;
      }
      const WaveTile at = wave_tile(own, wave_per);
      REQUIRE(at.wave == own / wave_per && at.before == own % wave_per);
      for (int u = 0; u < units[i]; ++u, ++unit) {
        if (tiles[i] == 0) continue;
        const uint32_t from = (uint32_t)at.before + (uint32_t)u * (uint32_t)tiles[i];
        const int first = at.wave + (int)(from / wave_per) + unit, end = at.wave + (int)((from + (uint32_t)tiles[i] - 1) / wave_per) + unit;
        REQUIRE(first > last && end >= first);   // a part's row is its own
        last = end;
      }
      own += (int64_t)tiles[i] * units[i];
    }
    const int64_t waves = (own + wave_per - 1) / wave_per;
    REQUIRE(of_groups + (waves + 3) / 4 <= target + units_g + 1);
    REQUIRE(of_groups <= target + units_g && last < waves + units_r && waves <= 4 * ((int64_t)target + 1));   // rows of partial sums
  }
  for (int round = 0; round < 4000; ++round) {   // a unit's parts: each once, eight at a time next to those of the other blocks
    const int n = pick(1, 40), heads = pick(1, 9), blocks = pick(1, 9), all = heads * n;
    std::vector<int> seen(all * blocks, 0);
    for (int x = 0; x < all * blocks; ++x) {
      const UnitPart u = unit_part(x, n, heads, blocks);
      REQUIRE(u.hk >= 0 && u.hk < heads && u.block >= 0 && u.block < blocks && u.part >= 0 && u.part < n);
      REQUIRE(!seen[(u.hk * blocks + u.block) * n + u.part]++);
      const int item = u.hk * n + u.part;
      if (item < all / 8 * 8) REQUIRE(x % 8 == item % 8 && x / (8 * blocks) == item / 8);
    }
  }
  printf("ok\n");
  return 0;
}
"""


def test_schedules(tmp_path):
    src, exe = tmp_path / "sched.cpp", tmp_path / "sched"
    src.write_text(PROGRAM)
    cxx = os.environ.get("CXX") or shutil.which("g++") or "g++"
    res = subprocess.run([cxx, "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{CSRC}", str(src), "-o", str(exe)],
                         capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-2000:]
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=110)
    assert res.returncode == 0 and "ok" in res.stdout, (res.stdout, res.stderr)
