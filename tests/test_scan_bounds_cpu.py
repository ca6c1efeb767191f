"""The sequence bounds of the selective scan on the host: the kernels' own functions, walked as the kernels walk blocks and segments.

Every state that is read or written has to be one of the batch's, whatever is in the array of bounds, and for an array as the interface asks for it
each sequence starts and ends exactly once in either direction."""
import os
import random
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "palimpsa_amd", "csrc")

WALK = r"""
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <vector>
using std::max; using std::min;
#include "scan_seqs.h"
using namespace pal;
struct Args { const int32_t* cu; int seqs, T; };
constexpr int kTok = 8;
static std::vector<int> starts, ends, dstarts, dends, hands, dhands;
static int bad = 0;
static void touch(std::vector<int>& v, int n) {          // state n is read or written
  if (n < 0 || n >= (int)v.size()) ++bad; else ++v[n];
}
static void hand_over(std::vector<int>& v, int n, int end) { for (; n < end; ++n) touch(v, n); }
static void forward(const Args& a, int t0, int t1) {
  ScanSeq cur = seq_at(a, 0, t0);
  if (t0 == 0) hand_over(hands, 0, cur.n);
  for (int tb = t0; tb < t1; tb += kTok) {
    const int nt = min(kTok, t1 - tb);
    for (int lo = 0, hi; lo < nt; lo = hi) {
      if (tb + lo == cur.s) touch(starts, cur.n);
      hi = max(lo + 1, min(nt, cur.e - tb));
      if (tb + hi == cur.e) {
        touch(ends, cur.n);
        const ScanSeq next = next_seq(a, cur);
        hand_over(hands, cur.n + 1, next.n);
        cur = next;
      }
    }
  }
}
static void states_of_block(const Args& a, int tb, int nt) {     // the backward's walk forward through a block
  ScanSeq fw = seq_at(a, 0, tb);
  for (int lo = 0, hi; lo < nt; lo = hi) {
    std::vector<int> any(a.seqs);
    if (tb + lo == fw.s) touch(any, fw.n);
    hi = max(lo + 1, min(nt, fw.e - tb));
    if (hi < nt) fw = next_seq(a, fw);
  }
}
static void backward(const Args& a, int t0, int t1) {
  ScanSeq cur = seq_at(a, 0, t1 - 1);
  if (t1 == a.T) hand_over(dhands, cur.n + 1, a.seqs);
  for (int tb = t0 + (t1 - 1 - t0) / kTok * kTok; tb >= t0; tb -= kTok) {
    const int nt = min(kTok, t1 - tb);
    states_of_block(a, tb, nt);
    for (int hi = nt, lo; hi > 0; hi = lo) {
      lo = min(hi - 1, max(0, cur.s - tb));
      if (tb + hi == cur.e) touch(dends, cur.n);
      if (tb + lo == cur.s) {
        touch(dstarts, cur.n);
        const ScanSeq prev = prev_seq(a, cur);
        hand_over(dhands, prev.n + 1, cur.n);
        cur = prev;
      }
    }
  }
}
// reads: T, tokens of a segment, sequences, bounds ..; prints: accesses out of range, then the six counts of every sequence
int main() {
  int T, seg, seqs;
  while (scanf("%d %d %d", &T, &seg, &seqs) == 3) {
    std::vector<int32_t> cu(seqs + 1);
    for (auto& c : cu) if (scanf("%d", &c) != 1) return 1;
    const Args a{cu.data(), seqs, T};
    for (auto* v : {&starts, &ends, &dstarts, &dends, &hands, &dhands}) v->assign(seqs, 0);
    bad = 0;
    for (int t0 = 0; t0 < T; t0 += seg) { forward(a, t0, min(T, t0 + seg)); backward(a, t0, min(T, t0 + seg)); }
    printf("%d", bad);
    for (auto* v : {&starts, &ends, &hands, &dstarts, &dends, &dhands}) for (int x : *v) printf(" %d", x);
    printf("\n");
  }
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    cxx = os.environ.get("CXX") or shutil.which("g++") or shutil.which("c++")
    if not cxx:
        pytest.skip("no C++ compiler")
    d = tmp_path_factory.mktemp("walk")
    (d / "walk.cpp").write_text(WALK)
    subprocess.run([cxx, "-std=c++17", "-O1", "-ftrapv", "-D__device__=", "-D__forceinline__=inline",
                    f"-I{CSRC}", str(d / "walk.cpp"), "-o", str(d / "walk")], check=True)

    def run(cases):
        text = "\n".join(" ".join(map(str, (T, seg, len(cu) - 1, *cu))) for T, seg, cu in cases)
        out = subprocess.run([str(d / "walk")], input=text, capture_output=True, text=True, timeout=60, check=True).stdout
        return [[int(x) for x in line.split()] for line in out.splitlines()]

    return run


def test_bounds_that_are_not_as_they_should_be(walk):
    low, high = -(1 << 31), (1 << 31) - 1
    arrays = [[0, 10, 20], [0, 0, 0], [5, 20, 30], [7, 7, 7], [0, 10, 50], [0, 40, 30], [30, 20, 10, 0], [30, 30, 30], [-4, 10, 30], [0, -3, 30],
              [low, high], [high, low], [low, low, low], [high, high, high], [0, high, 30], [0, low, 30], [29, 30, 31, 32], [0, 31], [31, 31], [0, 15, 14, 30]]
    rng = random.Random(1)
    arrays += [[rng.randint(-5, 40) for _ in range(rng.randint(2, 9))] for _ in range(300)]
    cases = [(30, seg, cu) for cu in arrays for seg in (8, 16, 32)]
    for case, line in zip(cases, walk(cases)):
        assert line[0] == 0, case


def test_every_sequence_starts_and_ends_once(walk):
    rng, cases = random.Random(2), []
    for _ in range(200):
        T = rng.randint(1, 90)
        inner = sorted(rng.choice([0, T, 8, rng.randint(0, T)]) if T >= 8 else rng.randint(0, T) for _ in range(rng.randint(0, 7)))
        cases += [(T, seg, [0, *inner, T]) for seg in (8, 32, 96)]
    for (T, seg, cu), line in zip(cases, walk(cases)):
        n = len(cu) - 1
        have = [int(b > a) for a, b in zip(cu, cu[1:])]
        starts, ends, hands, dstarts, dends, dhands = (line[1 + i * n:1 + (i + 1) * n] for i in range(6))
        assert line[0] == 0 and starts == ends == dstarts == dends == have, (T, seg, cu)
        assert hands == dhands == [1 - h for h in have], (T, seg, cu)
