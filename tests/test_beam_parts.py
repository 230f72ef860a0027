"""CPU tests of how a selection splits its rows (csrc/beam_sched.h): every token lies in one
part and one step of it, for every vocabulary that a call may have, and no bound passes 32 bits."""
import os
import shutil
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "custom_ops_amd", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <random>
#include "beam_sched.h"
using namespace mi355fa;
#define REQUIRE(x) do { if (!(x)) { printf("line %d: %s (rows %lld beams %d vocab %d k %d)\n", __LINE__, #x, (long long)rows, beams, vocab, k); exit(1); } } while (0)

void look(int64_t rows, int beams, int vocab, int k, int vectors, int cus) {
  const SelectSplit s = select_split(rows, beams, vocab, k, vectors, cus);
  REQUIRE(s.parts >= 1 && s.per >= 1 && (int64_t)beams * s.parts * k <= kSelCandidates);
  const int step = kSelThreads * 8 * (s.wide ? vectors : 1);
  REQUIRE(s.per % step == 0);
  int next = 0;
  for (int p = 0; p < s.parts; ++p) {
    const SelectSpan x = select_span(p, s.per, vocab);
    REQUIRE(x.begin == next && x.begin < x.end && x.end <= vocab && x.end - x.begin <= s.per);
    next = x.end;
    // the steps, as the kernel takes them: whole ones, and the last one to the part's end
    int at = x.begin;
    int64_t steps = 1;
    if (x.end - x.begin > 64 * step) steps += (x.end - x.begin) / step - 8, at += (x.end - x.begin) / step * step - 8 * step;
    for (;; at += step, ++steps) {
      const int left = x.end - at;
      REQUIRE(left > 0);
      if (left <= step) break;
    }
    REQUIRE(steps == (x.end - x.begin + (int64_t)step - 1) / step);
  }
  REQUIRE(next == vocab);
}

int main() {
  std::mt19937 g(11);
  auto pick = [&](int lo, int hi) { return lo + (int)(g() % ((unsigned)hi - (unsigned)lo + 1u)); };
  const int most = INT_MAX;
  for (int vectors : {2, 4})
    for (int k : {1, 4, 32, 33, 64})
      for (int64_t rows : {1, 2, 129, 512, 513, 1025, 100000})
        for (int vocab : {1, 2047, 2048, 2049, 8192, 8193, (1 << 30) - 1, 1 << 30, (1 << 30) + 1, most - (1 << 21), most - 8192, most - 1, most})
          look(rows, 1, vocab, k, vectors, 256);
  for (int i = 0; i < 20000; ++i) {
    const int beams = pick(0, 1) ? 1 : pick(1, 256), limit = most / beams;
    const int vocab = pick(0, 2) ? pick(1, limit) : limit - pick(0, limit < 20000 ? limit - 1 : 20000);
    look((int64_t)beams * pick(1, 2000), beams, vocab, pick(1, 64), pick(0, 1) ? 2 : 4, pick(0, 3) ? 256 : pick(1, 304));
  }
  printf("ok\n");
  return 0;
}
"""


def test_parts_of_rows(tmp_path):
    src, exe = tmp_path / "parts.cpp", tmp_path / "parts"
    src.write_text(PROGRAM)
    cxx = os.environ.get("CXX") or shutil.which("g++") or "g++"
    res = subprocess.run([cxx, "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{CSRC}", str(src), "-o", str(exe)],
                         capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-2000:]
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=110)
    assert res.returncode == 0 and "ok" in res.stdout, (res.stdout, res.stderr)
