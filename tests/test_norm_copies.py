"""Where the RMS norm's kernels copy, load and store: their own index arithmetic
(RowSpan, row_plan and the rest of csrc/norm_kernel.cuh and norm_launch.cuh),
compiled for the host and gone over for shapes and launches of every kind.  The
copies run ahead of the rows they are for, so they must not run past the tensor."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlp_megakernel_b200", "csrc")
SOURCE = r"""
#include <cstdio>
#include <random>
#include <set>
#include <vector>
#include "norm_launch.cuh"
using namespace mlpk;
using namespace mlpk::norm;

long shapes, copies, bad;
void fail(const char* what, int64_t rows, int width, int64_t row, int lane, int i) {
  if (++bad < 20) std::printf("%s: %ld x %d, row %ld, lane %d, vector %d\n", what, long(rows), width, long(row), lane, i);
}

// A block's row group `sub`, thread `lane` of it: every copy of the kernel's loop.
template <class T, int KIND>
void thread(int64_t rows, const RowPlan& p, int width, int64_t block, int64_t blocks, int sub, int lane, int stages) {
  constexpr int VEC = kVecOf<T>;
  const int64_t first = block * p.rows_per_block + sub, step = blocks * p.rows_per_block, total = rows * width;
  const RowSpan<T, 1, KIND> span(rows, width, p.tpr, lane, first);
  const int64_t begin0 = span.begin(first), loops = first < rows ? (rows - 1 - first) / step + 1 : 0;
  for (int64_t n = 0; n <= loops + stages; ++n) {
    if (n == 3 && loops > 6) n = loops - 2;  // the first ones and the last ones
    const int64_t row = first + n * step, begin = begin0 + n * step * width;
    if (begin != span.begin(row)) fail("begin", rows, width, row, lane, 0);
    if (span.exists(begin) != (row < rows)) fail("a row that is not there", rows, width, row, lane, 0);
    if (!span.exists(begin)) continue;
    for (int i = 0; i < p.nv; ++i) {
      if (!span.has(i)) continue;
      const int64_t at = span.at(begin, i);
      const int bytes = span.bytes(begin, i);
      ++copies;
      if (at < 0 || at % VEC || bytes < 1 || bytes > 16 || at * int64_t(sizeof(T)) + bytes > total * int64_t(sizeof(T)))
        fail("a copy outside", rows, width, row, lane, i);
      if (at != row * width + span.col(i)) fail("a copy of other columns", rows, width, row, lane, i);
      for (int e = 0; e < VEC; ++e)
        if (span.owns(i, e) != (span.col(i) + e >= 0 && span.col(i) + e < width)) fail("owns", rows, width, row, lane, i);
    }
  }
}

// Every column of a row belongs to one element of one vector of one thread.
template <class T, int KIND>
void cover(int64_t rows, const RowPlan& p, int width, int64_t first) {
  std::vector<int> seen(width);
  for (int lane = 0; lane < p.tpr; ++lane) {
    const RowSpan<T, 1, KIND> span(rows, width, p.tpr, lane, first);
    for (int i = 0; i < p.nv; ++i)
      for (int e = 0; e < kVecOf<T> && span.has(i); ++e)
        if (span.owns(i, e)) {
          if (span.col(i) + e < 0 || span.col(i) + e >= width) fail("a column outside", rows, width, first, lane, i);
          else ++seen[span.col(i) + e];
        }
  }
  for (int c = 0; c < width; ++c)
    if (seen[c] != 1) {
      fail("a column of none or several", rows, width, first, c, seen[c]);
      break;
    }
}

template <class T, int KIND>
void launch(int64_t rows, int width, const RowPlan& p, int64_t resident, int stages) {
  const int64_t blocks = loop_blocks(rows, p, kVecOf<T>, resident);
  std::set<int64_t> some = {0, 1, blocks / 2, blocks - 1, rows / p.rows_per_block % blocks, (rows - 1) / p.rows_per_block % blocks};
  std::set<int> lanes = {0, 1, 2, p.tpr / 2, p.tpr - 2, p.tpr - 1}, subs = {0, 1, p.rows_per_block - 1};
  for (int64_t b : some)
    for (int sub : subs)
      for (int lane : lanes)
        if (b >= 0 && b < blocks && sub < p.rows_per_block && lane >= 0 && lane < p.tpr)
          thread<T, KIND>(rows, p, width, b, blocks, sub, lane, stages);
  ++shapes;
}

template <class T>
void shape(int64_t rows, int width, int sms) {
  const RowPlan p = row_plan(width, kVecOf<T>);
  if (p.nv * p.tpr * kVecOf<T> < width || p.threads > 1024 || p.tpr * p.rows_per_block != p.threads)
    fail("plan", rows, width, 0, p.tpr, p.nv);
  if (p.full && p.nv * p.tpr * kVecOf<T> != width) fail("full", rows, width, 0, p.tpr, p.nv);
  auto every = [&](int64_t resident, int stages) {
    if (p.ragged) launch<T, kRagged>(rows, width, p, resident, stages);
    else if (p.full) launch<T, kFull>(rows, width, p, resident, stages);
    else launch<T, kPart>(rows, width, p, resident, stages);
  };
  for (int streams = 1; streams <= 2; ++streams)
    for (int per_sm = 1; per_sm <= 2048 / p.threads && per_sm <= 8; per_sm += 3)
      every(int64_t(sms) * per_sm, stages_of(p, streams, 52 * 1024));
  for (int streams = 2; streams <= 4; ++streams)
    every(int64_t(sms) * bwd_per_sm(p), stages_of(p, streams, 200 * 1024 / bwd_per_sm(p)));
  for (int64_t first = 0; first < 8; ++first) {
    if (p.ragged) cover<T, kRagged>(rows, p, width, first);
    else if (p.full) cover<T, kFull>(rows, p, width, first);
    else cover<T, kPart>(rows, p, width, first);
  }
}

int main() {
  std::mt19937_64 rng(5);
  std::uniform_real_distribution<double> u(0, 1);
  const int widths[] = {1, 2, 3, 7, 8, 9, 31, 33, 64, 127, 128, 129, 255, 256, 257, 300, 511, 513, 517, 520, 1000, 1023, 1024,
                        1025, 1032, 1999, 2048, 2049, 4096, 4097, 5120, 8190, 8191, 8192, 8193, 16383, 16384, 16385, 28673,
                        32761, 32767, 32768};
  const int64_t counts[] = {1, 2, 7, 8, 9, 147, 148, 149, 296, 592, 1776, 5003, 70001};
  for (int width : widths)
    for (int64_t rows : counts) {
      shape<__half>(rows, width, 148);
      shape<float>(rows, width, 148);
    }
  for (int n = 0; n < 3000; ++n) {
    const int width = std::min(32768, int(std::exp2(15 * u(rng)) + 0.5));
    const int64_t rows = int64_t(std::exp2(18 * u(rng)) + 0.5);
    const int sms = n % 4 ? 148 : 1 + int(200 * u(rng));
    if (n % 2) shape<__half>(rows, width, sms);
    else shape<float>(rows, width, sms);
  }
  std::printf("%ld launches, %ld copies, %ld bad\n", shapes, copies, bad);
  return bad != 0;
}
"""


def test_copies_stay_inside(tmp_path):
    from mlp_megakernel_b200 import build

    try:
        nvcc = build.nvcc_path()
    except RuntimeError:
        pytest.skip("no nvcc")
    assert shutil.which("g++")
    (tmp_path / "copies.cu").write_text(SOURCE)
    exe = tmp_path / "copies"
    subprocess.run([nvcc, *build.NVCC_FLAGS, "-I", CSRC, "-o", str(exe), str(tmp_path / "copies.cu")], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout
