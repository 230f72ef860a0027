"""CPU test of the attention plan's place in LDS (csrc/beam_sched.h): what lies behind it is
stored and read 16 bytes at a time."""
import os
import shutil
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "custom_ops_amd", "csrc")

PROGRAM = r"""
#include <cstdio>
#include "beam_sched.h"
using namespace mi355fa;
int main() {
  printf("%d %d\n", kShMax, kShWords);
  return 0;
}
"""


def test_plan_takes_whole_vectors(tmp_path):
    src, exe = tmp_path / "lds.cpp", tmp_path / "lds"
    src.write_text(PROGRAM)
    cxx = os.environ.get("CXX") or shutil.which("g++") or "g++"
    res = subprocess.run([cxx, "-std=c++17", f"-I{CSRC}", str(src), "-o", str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-2000:]
    most, words = map(int, subprocess.run([str(exe)], capture_output=True, text=True, timeout=60).stdout.split())
    assert words * 4 % 16 == 0
    assert words >= 64 + 8 * most + 1   # eight arrays, one of them with an element more, behind 64 words
    assert words * 4 <= 40 * 1024
