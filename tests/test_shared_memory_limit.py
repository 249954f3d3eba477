"""``allow_shared`` (csrc/common.cuh), which raises a kernel's limit of dynamic shared memory, from two host threads at once: built here against a
fake of the runtime's two calls, in which both threads meet inside the setting where they can.  No GPU."""
import os
import shutil
import subprocess

import pytest

from qutai_b200.build import ARCH_FLAGS, CSRC, INCLUDE

SOURCE = r"""
#include <cuda_runtime.h>
#include <atomic>
#include <chrono>
#include <cstdio>
#include <thread>

std::atomic<int> inside{0}, limit{0};
std::atomic<bool> large_set{false}, small_set{false};

template <typename F> void wait_for(F done) {        // half a second at most: a thread that the other may not join goes on alone
    for (int i = 0; i < 500 && !done(); ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
}
cudaError_t fake_device(int* device) { *device = 0; return cudaSuccess; }
// The larger amount is set first and returns last
cudaError_t fake_set(const void*, cudaFuncAttribute, int bytes) {
    ++inside;
    wait_for([] { return inside >= 2; });
    if (bytes < 150000) wait_for([] { return large_set.load(); });
    limit = bytes;
    if (bytes < 150000) { small_set = true; return cudaSuccess; }
    large_set = true;
    wait_for([] { return small_set.load(); });
    std::this_thread::sleep_for(std::chrono::milliseconds(50));
    return cudaSuccess;
}
#define cudaGetDevice fake_device
#define cudaFuncSetAttribute(kernel, which, bytes) fake_set((const void*)(kernel), which, bytes)
#include "common.cuh"

__global__ void some_kernel() {}

int main() {
    std::thread large([] { (void)qmoe::allow_shared<some_kernel>(200000); });
    std::thread small([] { (void)qmoe::allow_shared<some_kernel>(100000); });
    large.join();
    small.join();
    (void)qmoe::allow_shared<some_kernel>(200000);
    std::printf("%d\n", limit.load());
    return 0;
}
"""


def test_two_threads_leave_the_larger_limit(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("needs nvcc")
    source, binary = tmp_path / "limit.cu", tmp_path / "limit"
    source.write_text(SOURCE)
    subprocess.run([nvcc, *ARCH_FLAGS, "-std=c++17", "-I", CSRC, "-I", INCLUDE, "-o", str(binary), str(source)], check=True, capture_output=True, text=True)
    result = subprocess.run([str(binary)], check=True, capture_output=True, text=True, timeout=60)
    assert int(result.stdout) == 200000
