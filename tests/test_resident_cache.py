"""The kernels' shared-memory limits under calls from several host threads (host code, no GPU needed).

``resident_ctas`` (csrc/pim_common.cuh) raises a kernel's dynamic shared-memory limit as calls need more.  It is compiled here
against stand-ins of the CUDA calls that it makes, with two threads meeting in the middle of one.
"""

from __future__ import annotations

import os
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
NVCC = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"

PROGRAM = r"""
#include <stdio.h>

#include <atomic>
#include <thread>

#include "pim_common.cuh"

extern std::atomic<int> limit, small_inside;
static void kernel(int) {}

int main() {
  static pim::ResidentCache cache;
  auto call = [&](int smem) {
    cudaError_t e;
    return pim::resident_ctas(kernel, 32, smem, cache, &e) == 1 && e == cudaSuccess;
  };
  bool a = false, b = false;
  std::thread small([&] { a = call(30000); });
  while (!small_inside) std::this_thread::yield();
  std::thread large([&] { b = call(90000); });
  small.join();
  large.join();
  printf("%d %d %d ", a, b, (int)limit);
  const bool c = call(60000);  // a size between the two, later
  printf("%d %d\n", c, (int)limit);
}
"""

# `limit`: what the device would hold a launch to.  A call that sets the smaller size takes long: it waits for the larger
# one to be set, if that comes.  (8: cudaFuncAttributeMaxDynamicSharedMemorySize)
STAND_INS = r"""
#include <atomic>
#include <chrono>
#include <cstddef>
#include <thread>

std::atomic<int> limit{0}, small_inside{0};
static std::atomic<int> large_set{0};
extern "C" int cudaGetDevice(int* d) { *d = 0; return 0; }
extern "C" int cudaFuncSetAttribute(const void*, int what, int value) {
  if (what != 8) return 0;
  if (value == 30000) {
    small_inside = 1;
    for (int i = 0; i < 300 && !large_set; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
  }
  limit = value;
  if (value == 90000) large_set = 1;
  return 0;
}
extern "C" int cudaOccupancyMaxActiveBlocksPerMultiprocessor(int* n, const void*, int, size_t) { *n = 1; return 0; }
extern "C" int cudaOccupancyMaxActiveBlocksPerMultiprocessorWithFlags(int* n, const void*, int, size_t, unsigned) {
  *n = 1;
  return 0;
}
"""


@pytest.mark.skipif(not Path(NVCC).exists(), reason="needs nvcc")
def test_two_threads_leave_the_limit_at_the_larger_size(tmp_path):
    src, fake, exe = tmp_path / "resident.cu", tmp_path / "stand_ins.cpp", tmp_path / "resident"
    src.write_text(PROGRAM)
    fake.write_text(STAND_INS)
    r = subprocess.run([NVCC, "-std=c++17", "-O1", "--expt-relaxed-constexpr", "-gencode", "arch=compute_100a,code=sm_100a",
                        "-cudart", "shared", "-I", str(ROOT / "flagos-pim-compiler_b200" / "csrc"), "-o", str(exe), str(src),
                        str(fake)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    got = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert got.returncode == 0 and got.stdout.split() == ["1", "1", "90000", "1", "90000"], got.stdout + got.stderr
