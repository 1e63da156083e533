"""The shared-memory limit of a kernel whose launches differ in size, set by
two threads at once: compiled against a stand-in for the CUDA runtime, which
holds the first call until the second thread is through."""

from __future__ import annotations

import os
import shutil
import subprocess

import pytest

from conftest import ROOT

RUNTIME = r"""
#include <atomic>
#include <chrono>
#include <thread>
#include <cuda_runtime_api.h>

std::atomic<int> limit{48 * 1024}, calls{0}, released{0};

extern "C" {
void** __cudaRegisterFatBinary(void*) { static void* p; return &p; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
char __cudaInitModule(void**) { return 1; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
cudaError_t cudaFuncGetAttributes(cudaFuncAttributes* a, const void*) {
  *a = cudaFuncAttributes{};
  a->sharedSizeBytes = 1024;
  return cudaSuccess;
}
cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int value) {
  if (value + 1024 > 232448) return cudaErrorInvalidValue;
  limit = value;
  if (calls++ == 0)  // the first caller stays here until it is released
    for (int i = 0; i < 5000 && !released; ++i)
      std::this_thread::sleep_for(std::chrono::milliseconds(1));
  return cudaSuccess;
}
}
"""

CALLS = r"""
#include <atomic>
#include <cstdio>
#include <thread>
#include "sg_common.cuh"

extern std::atomic<int> limit, calls, released;

namespace sg {
void set_cuda_error(cudaError_t) {}
int max_dyn_smem() { return 232448; }
int num_sms() { return 148; }
int current_device() { return 0; }
}  // namespace sg

static void kernel(int) {}

int main() {
  static int cache[64];
  int a = -1, b = -1;
  std::thread large([&] { a = sg::ensure_dyn_smem(kernel, 150000, cache); });
  while (!calls) std::this_thread::yield();
  std::thread small([&] { b = sg::ensure_dyn_smem(kernel, 60000, cache); });
  small.join();
  released = 1;
  large.join();
  if (a != SG_OK || b != SG_OK) return 2;
  // a later large call finds the limit set, and far too much is refused
  if (sg::ensure_dyn_smem(kernel, 150000, cache) != SG_OK) return 3;
  if (limit < 150000) {
    std::printf("limit %d after calls with 150000 and 60000\n", limit.load());
    return 1;
  }
  if (sg::ensure_dyn_smem(kernel, 232448, cache) != SG_ERR_UNSUPPORTED)
    return 4;
  if (sg::ensure_dyn_smem(kernel, 231424, cache) != SG_OK || limit < 231424)
    return 5;
  return 0;
}
"""


def test_two_threads_first_calls(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    (tmp_path / "runtime.cpp").write_text(RUNTIME)
    (tmp_path / "calls.cu").write_text(CALLS)
    exe = tmp_path / "limit"
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a",
                    "-std=c++17", "-cudart", "none",
                    "-I" + os.path.join(ROOT, "suffixgpu_b200", "csrc"),
                    str(tmp_path / "calls.cu"), str(tmp_path / "runtime.cpp"),
                    "-o", str(exe), "-lpthread", "-ldl"],
                   check=True, capture_output=True, text=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, (r.returncode, r.stdout)
