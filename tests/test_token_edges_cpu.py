"""The edges of sequences as the convolution and the selective scan find them
(csrc/ltc_tokens.h), run on the host: for boundaries of any order and range every token has
a sequence that holds it or none, and every state that an edge names is one that is there;
for boundaries in order, the edges are those of the definition."""

from __future__ import annotations

import os
import shutil
import subprocess

import pytest

import ltc_cuda

CSRC = os.path.join(os.path.dirname(os.path.abspath(ltc_cuda.__file__)), "csrc")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")

pytestmark = pytest.mark.skipif(
    shutil.which("g++") is None or not os.path.isfile(os.path.join(ROCM, "include", "hip", "hip_runtime.h")),
    reason="needs g++ and the HIP headers")

# g++ takes the device functions for ordinary ones.
SOURCE = r"""
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <vector>
using std::max;
using std::min;
#include "ltc_tokens.h"
using namespace ltc;

constexpr int L = 4;  // tokens of a batch

#define CHECK(c) do { if (!(c)) { std::printf("line %d: %s\n", __LINE__, #c); for (int v : cu) std::printf(" %d", v); \
  std::printf(" | N %d first %d len %d back %d\n", N, c0, len, back); return 1; } } while (0)

// A walk over the chunk of `len` tokens from c0, forward or back.
int walk(const std::vector<int>& cu, int N, int c0, int len, bool back) {
  const int S = (int)cu.size() - 1, c1 = min(c0 + len, N);
  const bool sorted = std::is_sorted(cu.begin(), cu.end()) && cu[0] >= 0 && cu.back() <= N;
  Seq q{-1, 0, 0, 0};
  const int last = c0 + (c1 - 1 - c0) / L * L;
  for (int t = back ? last : c0; back ? t >= c0 : t < c1; t += back ? -L : L) {
    EdgesOf<L> ed;
    ed.find(cu.data(), S, N, N, t, c1, q);
    for (int i = 0; i < L; ++i) {
      const bool start = ed.start >> i & 1, end = ed.end >> i & 1, valid = ed.valid >> i & 1;
      CHECK(!(start || end || valid) || t + i < c1);
      CHECK(valid || (!start && !end));
      int s = -1;
      if (start || end)
        at_edge(cu.data(), S, N, N, t + i, [&](int found) {
          s = found;
          if (s < 0) s = -2;
        });
      CHECK(s >= -1 && s < S);
      if (!sorted || t + i >= c1) continue;
      int want = -1;
      for (int k = 0; k < S; ++k)
        if (cu[k] <= t + i && t + i < cu[k + 1]) want = k;
      CHECK(valid == (want >= 0));
      CHECK(start == (want >= 0 && cu[want] == t + i));
      CHECK(end == (want >= 0 && cu[want + 1] == t + i + 1));
      CHECK(!(start || end) || s == want);
    }
    for (unsigned rest = ed.valid, seg; rest != 0; rest &= ~seg) {
      seg = ed.last(rest);
      CHECK(seg != 0 && (seg & ~rest) == 0 && seg > (rest & ~seg));
    }
  }
  return 0;
}

int check(const std::vector<int>& cu, int N) {
  const int S = (int)cu.size() - 1, c0 = 0, len = 0;
  const bool back = false;
  for (int t = 0; t < N; ++t) {
    const Seq q = seq_of(cu.data(), S, N, N, t, 0, 0);
    CHECK(q.s >= -1 && q.s < S && 0 <= q.lo && q.lo <= t && t < q.hi && q.hi <= N);
  }
  for (int s = 0; s < S; ++s) {
    int lo, hi;
    span_of(cu.data(), N, N, s, lo, hi);
    CHECK(0 <= lo && lo <= hi && hi <= N);
  }
  for (int size : {2 * L, N})
    for (int from = 0; from < N; from += size)
      for (int b = 0; b < 2; ++b)
        if (walk(cu, N, from, size, b)) return 1;
  return 0;
}

int main() {
  const int values[] = {-3, 0, 1, 3, 4, 5, 7, 8, 9, 12, 13, 20, 2147483647, -2147483647 - 1};
  constexpr int V = sizeof(values) / sizeof(values[0]);
  for (int N : {1, 5, 13})
    for (int S = 0; S <= 4; ++S) {
      std::vector<int> at(S + 1, 0), cu(S + 1);
      for (;;) {
        for (int i = 0; i <= S; ++i) cu[i] = values[at[i]];
        if (check(cu, N)) return 1;
        int i = 0;
        while (i <= S && ++at[i] == V) at[i++] = 0;
        if (i > S) break;
      }
    }
  std::puts("done");
  return 0;
}
"""


def test_edges_of_any_boundaries(tmp_path):
    src, exe = tmp_path / "edges.cpp", tmp_path / "edges"
    src.write_text(SOURCE)
    made = subprocess.run(["g++", "-O2", "-std=c++17", "-w", "-D__HIP_PLATFORM_AMD__=1", f"-I{ROCM}/include",
                           f"-I{CSRC}", str(src), "-o", str(exe)], capture_output=True, text=True)
    assert made.returncode == 0, made.stderr[-3000:]
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=100)
    assert run.returncode == 0 and run.stdout.strip() == "done", run.stdout[-2000:]
