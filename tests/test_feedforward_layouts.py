"""How the products of the value tests are laid out over 148 SMs (host code, compiled and run here), so that the tests
keep covering the layouts that they are meant for: whole tiles with shares behind them, 256 columns wide; shares alone;
tiles of any width; the kernel for few rows.  test_feedforward_layouts_gpu.py runs the shapes of SHARES."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlp_megakernel_b200", "csrc")
SOURCE = """
#include <initializer_list>
#include <cstdio>
#include <cstdlib>
#include "few_rows_plan.cuh"
#include "product_plan.cuh"
using namespace mlpk;
int main(int argc, char** argv) {  // rows cols outputs nk split any few
  for (int i = 1; i + 6 < argc; i += 7) {
    long v[7];
    for (int k = 0; k < 7; ++k) v[k] = std::atol(argv[i + k]);
    const ProductPlan p = product_plan(v[0], v[1], v[2], 256, v[3], 74, v[4], true, v[5]);
    const bool few = v[6] && v[0] <= 2048 && (v[0] <= 64 || few_plan(v[0], v[1], v[3], 128, 148).us <= p.us + 0.5);
    std::printf("%d %d %ld %ld %d\\n", few, p.cols, long(p.full), long(p.tail), p.splits);
  }
}
"""


def blocks(n):
    return -(-n // 64)


def forward(rows, k, n, keep=False):
    return rows, n, 1, blocks(k), int(not keep), 1, 1


def dx(rows, k, n, count=1):
    return rows, k, 1, count * blocks(n), 1, 1, 1


def dw(rows, k, n, count=1, transposed=False):
    return *((n, k) if transposed else (k, n)), count, blocks(rows), 1, 1, 0


# (call, its sizes) -> (whole tiles, shared ones, shares of each): 256 columns wide
SHARES = {
    (forward, (3000, 4104, 1560)): (74, 10, 4), (forward, (1500, 4104, 3144)): (74, 4, 6), (forward, (8000, 2608, 1560)): (222, 2, 7),
    (dx, (3000, 1560, 4104)): (74, 10, 4), (dx, (2000, 2608, 2600, 2)): (74, 14, 4),
    (dw, (3000, 1288, 3144)): (74, 4, 6), (dw, (3000, 3144, 1288, 1, True)): (74, 4, 6), (dw, (3000, 520, 3144, 2)): (74, 4, 6),
}
# Shapes of test_feedforward_gpu.py: shares of 128 columns alone, and the widths of whole tiles.
ALONE = {(forward, (300, 4096, 128)): (2, 11), (forward, (700, 5000, 264)): (9, 5), (forward, (2100, 4096, 136)): (18, 4),
         (dx, (600, 200, 4600)): (6, 6), (dw, (20000, 264, 136)): (4, 15), (dw, (20000, 264, 136, 1, True)): (3, 21)}
WIDTHS = {(forward, (513, 136, 3088, True)): 160, (forward, (600, 200, 4600, True)): 192, (forward, (2500, 72, 1400, True)): 224,
          (forward, (4000, 4096, 520)): 160, (dx, (700, 5000, 264)): 224, (dx, (20000, 264, 136)): 160, (dw, (520, 2000, 1288)): 160,
          (dw, (769, 520, 4656)): 224, (dw, (769, 520, 4656, 1, True)): 192}
FEW = [(forward, (129, 2056, 520)), (forward, (1000, 4096, 1000)), (forward, (512, 4096, 136, True)), (dx, (513, 136, 3088))]


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no g++")
    at = tmp_path_factory.mktemp("layouts")
    (at / "plan.cpp").write_text(SOURCE)
    subprocess.run([cxx, "-O1", "-std=c++17", "-I", CSRC, "-o", str(at / "plan"), str(at / "plan.cpp")], check=True)

    def of(cases):
        said = subprocess.run([str(at / "plan"), *(str(v) for call, sizes in cases for v in call(*sizes))],
                              check=True, capture_output=True, text=True).stdout
        return [tuple(int(v) for v in line.split()) for line in said.splitlines()]

    return of


def test_whole_tiles_and_shares_256_wide(plans):
    for (case, want), got in zip(SHARES.items(), plans(SHARES), strict=True):
        assert got == (0, 256, *want), (case, got)


def test_shares_alone_128_wide(plans):
    for (case, want), got in zip(ALONE.items(), plans(ALONE), strict=True):
        assert got == (0, 128, 0, *want), (case, got)


def test_widths_of_whole_tiles(plans):
    for (case, want), got in zip(WIDTHS.items(), plans(WIDTHS), strict=True):
        assert got[:2] == (0, want) and got[4] == 1, (case, got)


def test_few_rows(plans):
    for case, got in zip(FEW, plans(FEW), strict=True):
        assert got[0] == 1, (case, got)
