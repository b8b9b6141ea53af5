"""The table of shared-memory limits (csrc/smem_limits.h), with a stand-in for the
CUDA call: more kernels and devices than one process has, from several threads."""
import shutil
import subprocess
from pathlib import Path

import pytest

import int8_kernel_lab_b200 as m

PROGRAM = r"""
#include <atomic>
#include <cstdio>
#include <thread>
#include <vector>
#include "smem_limits.h"

constexpr int kKernels = 700, kDevices = 8;
static std::atomic<int> calls[kDevices][kKernels], limit[kDevices][kKernels], lowered;

int main() {
  i8c::SmemLimits limits;
  static char kernels[kKernels];
  auto run = [&](int seed) {
    for (int pass = 0; pass < 3; ++pass)
      for (int i = 0; i < kDevices * kKernels; ++i) {
        const int at = (i * 131 + seed * 977) % (kDevices * kKernels);
        const int d = at / kKernels, k = at % kKernels;
        const int bytes = 1000 * (1 + (seed + pass) % 3);
        const bool ok = limits.ensure(d, kernels + k, bytes, [&](int b) {
          ++calls[d][k];
          if (limit[d][k].exchange(b) >= b) ++lowered;
          return true;
        });
        if (!ok || limit[d][k] < bytes) ++lowered;
      }
  };
  std::vector<std::thread> threads;
  for (int t = 0; t < 4; ++t) threads.emplace_back(run, t);
  for (auto &t : threads) t.join();
  int most = 0;
  for (auto &row : calls)
    for (auto &c : row) most = c > most ? c.load() : most;
  // A limit that could not be set is tried again.
  bool refused = !limits.ensure(0, &limits, 5, [](int) { return false; });
  bool later = limits.ensure(0, &limits, 5, [](int) { return true; });
  bool kept = limits.ensure(0, &limits, 5, [](int) { return false; });
  std::printf("%d %d %d\n", lowered.load(), most, refused && later && kept);
}
"""


def test_limits_are_set_once_and_never_lowered(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    (tmp_path / "limits.cpp").write_text(PROGRAM)
    csrc = Path(m.__file__).parent / "csrc"
    subprocess.run([cxx, "-std=c++17", "-O1", "-pthread", f"-I{csrc}", "-o", str(tmp_path / "limits"),
                    str(tmp_path / "limits.cpp")], check=True)
    out = subprocess.run([str(tmp_path / "limits")], capture_output=True, text=True, check=True,
                         timeout=60).stdout.split()
    lowered, most, again = map(int, out)
    assert lowered == 0 and 1 <= most <= 3 and again == 1   # three sizes: three calls at most
