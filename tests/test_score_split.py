"""How token scores deal rows to workgroups (score_split.hpp), built for the CPU: what the kernel relies on holds for every
number of rows, vocabulary and type."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r"""
#include <cstdio>
#include <initializer_list>
#include "score_split.hpp"
using namespace pcp;
static int check(int64_t rows, int64_t vocab, int bytes) {
  const ScoreSplit s = score_split(rows, vocab, bytes);
  const int64_t nv = vocab * bytes / 16, batch = kScoreBlock * kScoreU;
  const char* wrong = nullptr;
  if (s.group < 1) wrong = "a group holds no batch";                                       // the kernel divides by it
  else if ((s.per + batch - 1) / batch > int64_t(s.group) * kScoreGroups) wrong = "more groups than a lane keeps";
  else if (s.parts < 1 || s.parts > kScoreParts) wrong = "parts that one wave cannot merge";
  else if (s.parts > 1 && (rows >= kScoreTickets || s.per < batch)) wrong = "a row in parts without a ticket";
  else if (s.parts * s.per < nv || (s.parts > 1 && (s.parts - 1) * s.per >= nv)) wrong = "parts that do not cover the row";
  else if (s.per % kScoreBlock != 0) wrong = "a part that ends within a step";
  if (wrong) printf("%s: %lld rows of %lld, %d bytes each: %lld parts of %lld, groups of %d\n", wrong, (long long)rows,
                    (long long)vocab, bytes, (long long)s.parts, (long long)s.per, s.group);
  return wrong != nullptr;
}
int main() {
  int bad = 0;
  long n = 0;
  for (int bytes : {2, 4})
    for (int64_t rows : {1, 2, 3, 5, 16, 37, 64, 100, 127, 128, 200, 254, 255, 256, 257, 4096, 2147483647}) {
      for (int64_t v = 1; v <= 70000 && bad < 5; v += v < 300 ? 1 : 61, ++n) bad += check(rows, v, bytes);
      for (int64_t v = 70000; v < (1 << 24) && bad < 5; v += v / 97 + 1, ++n) bad += check(rows, v, bytes);
      bad += check(rows, 1 << 24, bytes);
    }
  printf("%ld\n", n);
  return bad != 0;
}
"""


def test_split_of_rows(tmp_path):
    src, exe = tmp_path / "split.cpp", tmp_path / "split"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(ROOT, "pcp_amd", "csrc"), str(src), "-o", str(exe)],
                   check=True)
    got = subprocess.run([str(exe)], capture_output=True, text=True)
    assert got.returncode == 0, got.stdout
    assert int(got.stdout.split()[-1]) > 40000
