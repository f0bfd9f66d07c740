"""The rounds in which the sampling kernels walk a row (ako_amd/csrc/row_rounds.h), compiled with g++ from the
header itself: every row that is kept in LDS is read back from inside its array, and every element of a row is
met once, whatever is left behind the last whole packet and the last whole group of rounds."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "ako_amd" / "csrc"

DRIVER = r"""
#include <cstdio>
#include <vector>
#include "row_rounds.h"

constexpr int kThreads = 1024;
long rows = 0, outside = 0, missed = 0, planted = 0;

template <int E, bool AGAIN>
void walk(int vocab, bool every) {
  const int whole = vocab / E, rest = vocab % E, n = ako::rounds_of(whole, rest, kThreads);
  std::vector<int> met(every ? vocab : 0);
  int loaded[4] = {-1, -1, -1, -1}, used = 0;
  ako::in_groups<4, AGAIN>(n, [&](int u, int k) {
    loaded[u] = k;
    outside += k >= n || k * kThreads + kThreads - 1 >= ako::held_places(kThreads);
  }, [&](int u, int k) {
    missed += loaded[u] != k || k != used++;
    if (!every) return;
    const bool behind = rest > 0 && k == n - 1;
    for (int t = 0; t < kThreads; ++t) {
      const int i = ako::index_in_round<E>(whole, rest, kThreads, k, t);
      if (behind ? t < rest : k * kThreads + t < whole)
        for (int e = 0; e < (behind ? 1 : E); ++e) {
          if (i + e < 0 || i + e >= vocab) ++missed;
          else ++met[i + e];
        }
    }
  });
  missed += used != n;
  for (int m : met) missed += m != 1;
  // The check has teeth: groups that are always whole read behind the array.
  for (int k0 = 0; k0 < n; k0 += 4) planted += (k0 + 3) * kThreads + kThreads - 1 >= ako::held_places(kThreads);
  ++rows;
}

int main() {
  for (int v = 1; v <= ako::kHeldBytes / 4; ++v) {
    walk<4, false>(v, v % 61 == 0 || v > 12280);
    walk<4, true>(v, false);
  }
  for (int v = 1; v <= ako::kHeldBytes / 2; ++v) {
    walk<8, false>(v, v % 61 == 0 || (v > 24570 && v < 24610) || v > 32760);
    walk<8, true>(v, false);
  }
  std::printf("rows=%ld outside=%ld missed=%ld planted=%ld\n", rows, outside, missed, planted);
  return outside || missed || !planted;
}
"""


def test_rounds_stay_inside_and_meet_everything(tmp_path) -> None:
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ is not available")
    src = tmp_path / "rounds.cpp"
    src.write_text(DRIVER)
    exe = tmp_path / "rounds"
    subprocess.run([gxx, "-O2", "-std=c++17", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout + out.stderr
    assert "rows=98304 outside=0 missed=0" in out.stdout
