"""The 4-bit weight's layout without a GPU: every load that the tile kernel forms stays inside the weight."""

from __future__ import annotations

import pathlib
import shutil
import subprocess

import pytest

from lastkv_amd import _lib

CSRC = pathlib.Path(__file__).resolve().parents[1] / "lastkv_amd" / "csrc"

# The loads of one workgroup, as mx4_tile_kernel forms them from the layout's functions: kbn row tiles from nt0 on, all
# column tiles and units (the last ones are asked for again), 16 bytes of 64 lanes of codes, 4 bytes of scales.
HARNESS = r"""
#include <stdio.h>
#include <stdlib.h>
#include <initializer_list>
#include "mx_layout.h"
using namespace lkv;
int main(int argc, char** argv) {
  for (int a = 1; a + 1 < argc; a += 2) {
    const int n = atoi(argv[a]), k = atoi(argv[a + 1]);
    const int units = mx4_units(k), stride = mx4_tile_stride(units), ntiles = (n + 15) / 16, columns = (k + 127) / 128;
    const long long bytes = static_cast<long long>(ntiles) * stride;
    for (const int kbn : {8, 16}) {
      for (int nt0 = 0; nt0 < ntiles; nt0 += kbn) {
        if (nt0 > 0 && nt0 + 2 * kbn < ntiles) continue;  // (the first and the last two workgroups)
        const int tiles = kbn < ntiles - nt0 ? kbn : ntiles - nt0;
        const long long base = static_cast<long long>(nt0) * stride, buffer = static_cast<long long>(tiles) * stride;
        for (int i = 0; i < kbn; ++i) {
          const long long at = mx4_tile_start(i, tiles, stride);
          for (const int kt : {0, columns / 2, columns - 1}) {
            const long long end = at + mx4_codes_at(kt) + 63 * 16 + 16;
            if (at < 0 || end > buffer || base + end > bytes) {
              printf("%d x %d: codes of tile %d + %d, column tile %d end at %lld of %lld\n", n, k, nt0, i, kt, end, buffer);
              return 1;
            }
          }
          const long long end = at + mx4_scales_at(units - 1) + 63 * 4 + 4;
          if (end > buffer || base + end > bytes) {
            printf("%d x %d: scales of tile %d + %d end at %lld of %lld\n", n, k, nt0, i, end, buffer);
            return 1;
          }
        }
      }
    }
  }
  return 0;
}
"""

SHAPES = [(1, 32), (15, 96), (16, 128), (17, 544), (33, 160), (100, 1056), (129, 4096), (255, 14336), (257, 1 << 20), (2060, 96),
          (4095, 4064), (6161, 416), (8001, 640), (28672, 4096), (28700, 32), (128256, 4096), ((1 << 24) - 1, 32)]


def test_tile_loads_stay_inside_the_weight(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("needs a host compiler")
    (tmp_path / "loads.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", f"-I{CSRC}", str(tmp_path / "loads.cpp"), "-o", str(tmp_path / "loads")],
                   check=True)
    run = subprocess.run([str(tmp_path / "loads"), *(str(v) for shape in SHAPES for v in shape)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout


def test_sizes_that_no_weight_has_need_no_bytes():
    size = _lib.load().lkv_mx4_weight_bytes
    assert size(1 << 24, 1 << 20) == (1 << 20) * (((1 << 11) * 17) | 1) * 256
    for n, k in ((0, 32), (16, 0), (-1, 64), ((1 << 24) + 1, 32), (16, (1 << 20) + 32), (16, (1 << 31) - 32), ((1 << 31) - 1, (1 << 31) - 32)):
        assert size(n, k) == 0, (n, k)
