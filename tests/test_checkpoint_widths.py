"""Very wide rows of the 8-bit checkpoints: the widths that are refused, and the index arithmetic of the kernels up to
there (their own, compiled for the host)."""
import os
import shutil
import subprocess

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mlp_megakernel_b200 as m

ops = torch.ops.mlpk
FP8, F16, F32 = torch.float8_e4m3fn, torch.float16, torch.float32
MOST = 2 ** 31 - 1
CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlp_megakernel_b200", "csrc")
STEPS = r"""
#include <cstdio>
#include "ff_kernel.cuh"
using namespace mlpk;
int main() {
  long bad = 0, seen = 0;
  const int minors[] = {1, 2, 127, 4096, 1 << 24, 1000000007, 0x7fffffff - 5000000, 0x7fffffff - 15, 0x7ffffff0, 0x7fffffff};
  // Grids of the restoring kernel (16 values a thread, 256 threads) and of the other one (teams).
  for (int64_t step : {int64_t(1), int64_t(3), int64_t(148) * 8 * 32, int64_t(148) * 8 * 256 * 16, int64_t(132) * 4 * 256 * 16, int64_t(1) << 33})
    for (int n : minors)
      for (int64_t first : {int64_t(0), int64_t(16), step - 1, step / 2, int64_t(n) - 1}) {
        Steps at(first, step, n);
        for (int64_t k = 0; k < 3000; ++k) {
          const int64_t i = first + k * step;
          ++seen;
          if (at.major != i / n || at.minor != i % n) {
            if (++bad < 10) std::printf("step %ld of %ld, %d: turn %ld at %ld, %d\n", long(step), long(first), n, long(k), long(at.major), at.minor);
            break;
          }
          at.next();
        }
      }
  std::printf("%ld seen, %ld bad\n", seen, bad);
  return bad != 0;
}
"""


def test_steps_over_rows_of_any_width(tmp_path):
    """Where the kernels' next values lie, up to rows within a step of 2^31 columns."""
    from mlp_megakernel_b200 import build

    try:
        nvcc = build.nvcc_path()
    except RuntimeError:
        pytest.skip("no nvcc")
    assert shutil.which("g++")
    (tmp_path / "steps.cu").write_text(STEPS)
    exe = tmp_path / "steps"
    subprocess.run([nvcc, *build.NVCC_FLAGS, "-I", CSRC, "-o", str(exe), str(tmp_path / "steps.cu")], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout


@pytest.mark.parametrize("width", [MOST + 1, 2 ** 32 - 8, 5 * 10 ** 9])
def test_rows_wider_than_an_int_are_refused(width):
    """The C calls take the width as an int: 5e9 columns would be 705,032,704 of them."""
    with FakeTensorMode():
        x, q = torch.empty(1, width, dtype=F16, device="cuda"), torch.empty(1, width, dtype=FP8, device="cuda")
        scale = torch.empty(1, -(-width // 128), dtype=F32, device="cuda")
        for call in (lambda: m.fp8_checkpoint(x), lambda: ops.fp8_checkpoint(x), lambda: m.fp8_restore(q, scale),
                     lambda: ops.fp8_restore(q, scale, F16)):
            with pytest.raises(ValueError, match="columns"):
                call()


def test_the_widest_rows_are_taken():
    with FakeTensorMode():
        q, scale = m.fp8_checkpoint(torch.empty(2, MOST, dtype=F16, device="cuda"))
        assert q.shape == (2, MOST) and scale.shape == (2, 2 ** 24)
        assert m.fp8_restore(q, scale, F16).shape == (2, MOST)
