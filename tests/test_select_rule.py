"""How many token rows a launch of the block choice takes (ako_amd/csrc/select_rule.h), compiled with g++ from the
header itself: for every number of key heads, tile and head size the work-items of a full slice stay below 2^32, and a
slice is whole tiles."""

from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "ako_amd" / "csrc"

DRIVER = r"""
#include <cstdio>
#include "select_rule.h"

int main() {
  long checks = 0, bad = 0, planted = 0;
  for (int64_t heads = 1; heads <= 0x7fffffff / 65536; ++heads)
    for (int dim = 16; dim <= 256; dim += 16)
      for (int64_t tile = 1; tile <= 16; tile *= 2) {
        const int threads = ako::tile_threads(dim, tile == 1);
        const int64_t rows = ako::tile_slice(dim, tile, heads);
        bad += rows < tile || rows % tile || rows / tile * heads * threads >= int64_t(1) << 32;
        // Twice the workgroups that 256 work-items each allow are too many.
        planted += 2 * ako::slice_groups(256) / heads * heads * threads >= int64_t(1) << 32;
        ++checks;
      }
  bad += 256 * ako::slice_groups(256) >= int64_t(1) << 32;
  std::printf("checks=%ld bad=%ld planted=%ld\n", checks, bad, planted);
  return bad || !planted;
}
"""


def test_a_slice_stays_below_the_bound(tmp_path) -> None:
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ is not available")
    src = tmp_path / "slice.cpp"
    src.write_text(DRIVER)
    exe = tmp_path / "slice"
    subprocess.run([gxx, "-O2", "-std=c++17", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout + out.stderr
    assert "bad=0" in out.stdout


def test_the_launches_go_by_it() -> None:
    """Every launch of the choice takes its threads and its slice from the rule."""
    text = (CSRC / "paged_select.hip").read_text()
    tiles = re.findall(r"AKO_LAUNCH\(\(select_tile<[^>]*, (\w+), (?:true|false)>\), grid, dim3\((\w+) \* kWave\)", text)
    assert len(tiles) == 4 and {w for pair in tiles for w in pair} == {"kOneWaves", "kTileWaves"} and all(a == b for a, b in tiles)
    assert "tile_slice(a.c.head_dim, d.tile, a.c.kv_heads)" in text and "constexpr int64_t kSlice = slice_groups(256);" in text
