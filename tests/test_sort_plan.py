"""How a sort by expert is launched, for devices of any size (host code, compiled
and run here).  What each line says of a plan is what the kernels rely on."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlp_megakernel_b200", "csrc")
SOURCE = """
#include <cstdio>
#include "expert_plan.cuh"
using namespace mlpk;
int main() {
  long bad = 0, seen = 0;
  const int64_t some[] = {0, 1, 31, 32, 33, 4095, 4096, 4097, 8192, 32769, 65535, 65536, 65537, 65600, 100000, 131072,
                          262144, 606208, 606209, 1 << 20, 2200001, 1 << 30, 0x7fffffff};
  for (int sms = 1; sms <= 200; ++sms)
    for (int64_t slots : some) {
      const SortPlan p = sort_plan(slots, sms);
      ++seen;
      bool ok = p.blocks >= 1 && p.part >= 32 && p.part % 32 == 0 && p.blocks * kSortWarps * p.part >= slots;
      if (p.cluster)  // a power of two of blocks; all of a warp's slots are in registers
        ok = ok && (p.blocks & (p.blocks - 1)) == 0 && p.blocks <= kSortCluster && p.part <= 32 * kSortGroups &&
             p.workspace(64) == 0;
      else
        ok = ok && p.blocks <= sms && p.workspace(64) == 65 * 4 * static_cast<int64_t>(p.blocks);
      ok = ok && p.cluster == sort_plan(slots, 1).cluster && p.cluster == (slots <= kSortCluster * kSortBlockSlots);
      if (!ok && ++bad < 10) std::printf("%ld slots, %d SMs: blocks %d, part %ld\\n", long(slots), sms, p.blocks, long(p.part));
    }
  std::printf("%ld plans, %ld bad\\n", seen, bad);
  return bad != 0;
}
"""


def test_sort_plan(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no g++")
    (tmp_path / "plan.cpp").write_text(SOURCE)
    exe = tmp_path / "plan"
    subprocess.run([cxx, "-std=c++17", "-I", CSRC, "-o", str(exe), str(tmp_path / "plan.cpp")], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout
