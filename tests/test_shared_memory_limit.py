"""The dynamic shared-memory limit of a kernel whose need depends on the shape, raised by two host threads at
once: the code of common.cuh, compiled for the host with the two CUDA calls it makes replaced."""
import os
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")

HARNESS = r"""
#include <cuda_runtime.h>
#include <atomic>
#include <chrono>
#include <cstdio>
#include <thread>
static std::atomic<int> limit{0};  // what the driver would hold
static cudaError_t get_device(int *d) { *d = 3; return cudaSuccess; }
template <typename K>
static cudaError_t set_attribute(K, cudaFuncAttribute, int bytes) {
  limit = bytes;
  if (bytes > 100000) std::this_thread::sleep_for(std::chrono::milliseconds(400));  // a first call loads the kernel
  return cudaSuccess;
}
#define cudaGetDevice get_device
#define cudaFuncSetAttribute set_attribute
#include "common.cuh"
namespace mq {
int fail(int code, const char *, ...) { return code; }
}
static void kernel() {}
int main() {
  static size_t seen[64] = {};
  std::thread large([&] { mq::ensure_smem(kernel, 200000, seen, "large"); });
  std::this_thread::sleep_for(std::chrono::milliseconds(100));
  std::thread small([&] { mq::ensure_smem(kernel, 50000, seen, "small"); });
  large.join(), small.join();
  mq::ensure_smem(kernel, 200000, seen, "again");
  std::printf("%d\n", limit.load());
  return limit >= 200000 ? 0 : 1;
}
"""


def test_two_threads_leave_the_larger_limit(tmp_path):
    if not os.path.exists(NVCC):
        pytest.skip("no nvcc")
    src, exe = tmp_path / "limit.cu", tmp_path / "limit"
    src.write_text(HARNESS)
    subprocess.run([NVCC, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-I", os.path.join(REPO, "include"), "-I",
                    os.path.join(REPO, "mojo-adreno_b200", "csrc"), "--expt-relaxed-constexpr", "-Xcompiler", "-pthread", str(src), "-o",
                    str(exe)], check=True, capture_output=True, text=True)
    ran = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert ran.returncode == 0, ran.stdout + ran.stderr
