"""The shared-memory limit of a kernel from two threads (no GPU needed): ``csrc/func_attr.h`` compiled against a runtime whose
cudaFuncSetAttribute only stores the limit."""

import os
import shutil
import subprocess

import pytest

from conftest import ROOT

RUNTIME = r"""
#pragma once
typedef int cudaError_t;
enum { cudaSuccess = 0 };
enum { cudaFuncAttributeMaxDynamicSharedMemorySize = 8 };
cudaError_t cudaFuncSetAttribute(void (*kern)(), int attr, int bytes);
"""

PROGRAM = r"""
#include "func_attr.h"
#include <chrono>
#include <condition_variable>
#include <cstdio>
#include <thread>

static std::atomic<int> limit{0}, started{0};
static std::atomic<bool> large_set{false};
cudaError_t cudaFuncSetAttribute(void (*)(), int, int bytes) {
  if (bytes == 50) {  // the small limit arrives late: after the large one where that can overtake it
    started = 1;
    for (int i = 0; i < 300 && !large_set; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
  }
  limit = bytes;
  if (bytes == 100) large_set = true;
  return cudaSuccess;
}
static void kern() {}

int main() {
  static mdlc::SmemLimit seen;
  std::thread small([] { mdlc::allow_smem(seen, 0, kern, 50); });
  while (!started) std::this_thread::yield();
  std::thread large([] { mdlc::allow_smem(seen, 0, kern, 100); });
  small.join();
  large.join();
  mdlc::allow_smem(seen, 0, kern, 100);  // what every later launch asks for
  const int two = limit;
  mdlc::allow_smem(seen, 0, kern, 20);   // a smaller one changes nothing
  mdlc::allow_smem(seen, 3, kern, 30);   // another device has its own
  std::printf("%d %d %d\n", two, (int)limit, (int)seen.set[0].load());
}
"""


def test_a_smaller_limit_never_replaces_a_larger_one(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    (tmp_path / "cuda_runtime.h").write_text(RUNTIME)
    (tmp_path / "main.cpp").write_text(PROGRAM)
    exe = tmp_path / "limits"
    subprocess.run([cxx, "-std=c++17", "-O1", "-pthread", "-I", str(tmp_path), "-I", os.path.join(ROOT, "mdlc_b200", "csrc"),
                    str(tmp_path / "main.cpp"), "-o", str(exe)], check=True)
    for _ in range(3):
        out = subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=60).stdout.split()
        assert out == ["100", "30", "100"]
