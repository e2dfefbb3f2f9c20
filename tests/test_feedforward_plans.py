"""How the feed-forward products are laid out over the SMs (host code, compiled and
run here): every tile and every block of the reduction is taken once, shares lie
apart in the workspace, and what is asked of an SM is there."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlp_megakernel_b200", "csrc")
PRODUCT = """
#include <cstdio>
#include <vector>
#include "product_plan.cuh"
using namespace mlpk;
int main() {
  long bad = 0, seen = 0;
  const int64_t some_rows[] = {1, 8, 255, 256, 257, 1000, 5003, 20011, 65536, 1000000};
  const int some_cols[] = {8, 120, 128, 136, 256, 1000, 2056, 11008, 16384};
  for (int pairs : {1, 2, 37, 66, 74, 80})
    for (int64_t rows : some_rows)
      for (int cols : some_cols)
        for (int nk : {1, 2, 3, 4, 7, 8, 16, 33, 64, 344, 15626})
          for (int outputs : {1, 2})
            for (int mode = 0; mode < 5; ++mode) {
              const int out_cols = mode & 1 ? 128 : 256;
              const bool split = mode == 0 || mode >= 2, narrow = mode < 2 || mode == 4, any = mode == 4;
              const ProductPlan p = product_plan(rows, cols, outputs, out_cols, nk, pairs, split, narrow, any);
              const int each = out_cols * p.cols / 256;
              const int64_t tm = (rows + 255) / 256, tn = (cols + each - 1) / each;
              bool ok = (p.cols == 256 || (p.cols == 128 && narrow) || (any && p.cols > 128 && p.cols < 256 && p.cols % 32 == 0)) && p.full + p.tail == tm * tn * outputs &&
                        p.splits >= 1 && (split || p.splits == 1) && (p.splits > 1 || p.tail == 0) && p.tail < pairs &&
                        (p.splits == 1 || (nk / p.splits >= 4 && p.cols % 128 == 0)) &&
                        p.partials() == (p.splits > 1 ? p.tail * p.splits * 256 * p.cols : 0);
              if (p.tail) ok = ok && p.full % pairs == 0;  // whole turns of whole tiles, then the shares
              // A share's blocks, as the kernel cuts them.
              int64_t covered = 0;
              for (int s = 0; s < p.splits; ++s) {
                const int64_t k0 = int64_t(s) * nk / p.splits, k1 = int64_t(s + 1) * nk / p.splits;
                ok = ok && k0 == covered && k1 > k0;
                covered = k1;
              }
              ok = ok && covered == nk;
              ++seen;
              if (!ok && ++bad < 10)
                std::printf("rows %ld cols %d nk %d outputs %d pairs %d mode %d\\n", long(rows), cols, nk, outputs, pairs, mode);
            }
  // Every tile once.
  for (int tm : {1, 2, 7, 8, 9, 16, 20, 79})
    for (int tn : {1, 3, 8, 43})
      for (int outputs : {1, 2}) {
        std::vector<int> hit(tm * tn * outputs);
        for (int t = 0; t < tm * tn * outputs; ++t) {
          const TileAt at = product_tile(t, tm, tn, outputs, 8);
          if (at.m < 0 || at.m >= tm || at.n < 0 || at.n >= tn || at.output < 0 || at.output >= outputs) { ++bad; continue; }
          ++hit[(at.output * tn + at.n) * tm + at.m];
        }
        for (int h : hit) bad += h != 1;
        ++seen;
      }
  // Every value of a share at its own place, and where the kernel's warps put it.
  for (int cols : {128, 256}) {
    std::vector<int> hit(64 * cols);
    const int chunks = cols / 128;
    for (int rank = 0; rank < 2; ++rank)
      for (int w = 0; w < 16; ++w)
        for (int c = 0; c < chunks; ++c)
          for (int lane = 0; lane < 32; ++lane)
            for (int u = 0; u < 8; ++u) {
              const int quarter = (w + 2) & 3;  // warp w + 2 of the CTA reads this quarter of its TMEM lanes
              const int row = rank * 128 + quarter * 32 + lane, col = w / 4 * 32 + c * 128 + u * 4;
              const int there = ((rank * 16 + w) * chunks + c) * 256 + lane * 8 + (u ^ (lane & 7));
              const int unit = share_unit(row, col, cols);
              if (unit != there || unit < 0 || unit >= 64 * cols) { ++bad; continue; }
              ++hit[unit];
            }
    for (int h : hit) bad += h != 1;
    ++seen;
  }
  std::printf("%ld seen, %ld bad\\n", seen, bad);
  return bad != 0;
}
"""
FEW = """
#include <initializer_list>
#include <cstdio>
#include "few_rows_plan.cuh"
using namespace mlpk;
int main() {
  long bad = 0, seen = 0;
  for (int sms : {2, 16, 74, 132, 148, 160})
    for (int64_t rows = 1; rows <= 3 * kFewMostRows; ++rows)
      for (int cols : {8, 64, 72, 128, 136, 4096, 14336, 65536})
        for (int nk : {1, 2, 3, 4, 5, 7, 8, 16, 31, 32, 64, 224, 1000})
          for (int tile : {64, 128}) {
            const FewPlan p = few_plan(rows, cols, nk, tile, sms);
            // The instruction's N (a multiple of 16), its columns of TMEM (512 for the CTAs of an SM).
            const int at_once = p.each_sm, columns = p.nt <= 32 ? 32 : p.nt <= 64 ? 64 : p.nt <= 128 ? 128 : 256;
            bool ok = (at_once == 1 || at_once == 2) && p.nt >= 16 && p.nt <= 256 && p.nt % 16 == 0 && int64_t(p.nt) * p.row_tiles >= rows &&
                      int64_t(p.nt) * (p.row_tiles - 1) < rows &&
                      columns * at_once <= 512 && p.stages >= 2 && p.stages <= kFewMaxStages &&
                      few_smem(p.nt, p.stages) * at_once <= 227 * 1024 && int64_t(p.tiles) * tile >= cols &&
                      int64_t(p.tiles - 1) * tile < cols;
            // A cluster of the portable size; each of its CTAs has blocks to add.
            ok = ok && p.ranks >= 1 && p.ranks <= kFewMaxRanks && p.ranks <= nk;
            for (int r = 0; r < p.ranks; ++r) ok = ok && int64_t(r + 1) * nk / p.ranks > int64_t(r) * nk / p.ranks;
            // The fp32 tile fits where the ring was.
            const int ring = p.stages * (kFewWBytes + p.nt * 128), tile_bytes = p.nt * 128 * 4;
            ok = ok && few_smem(p.nt, p.stages) >= 1024 + (ring > tile_bytes ? ring : tile_bytes) + 8 * (2 * kFewMaxStages + 1) + 8;
            ++seen;
            if (!ok && ++bad < 10) std::printf("rows %ld cols %d nk %d tile %d sms %d\\n", long(rows), cols, nk, tile, sms);
          }
  std::printf("%ld seen, %ld bad\\n", seen, bad);
  return bad != 0;
}
"""


@pytest.mark.parametrize("source", [PRODUCT, FEW], ids=["product", "few_rows"])
def test_plans(tmp_path, source):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no g++")
    (tmp_path / "plan.cpp").write_text(source)
    exe = tmp_path / "plan"
    subprocess.run([cxx, "-O1", "-std=c++17", "-I", CSRC, "-o", str(exe), str(tmp_path / "plan.cpp")], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout
