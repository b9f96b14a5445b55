"""The cached shared-memory limit of a kernel (csrc/smem_limit.h) under two host threads, against a fake runtime."""
from __future__ import annotations

import os
import shutil
import subprocess

import pytest

from conftest import PKG

SOURCE = r"""
#include <atomic>
#include <chrono>
#include <stdio.h>
#include <thread>
#include "%s"

static std::atomic<int> limit{0}, sets{0}, large_set{0}, small_set{0};
static const int LARGE = 200000, SMALL = 100000;

static void wait_for(std::atomic<int> &x)
{
    for (int i = 0; i < 500 && !x; i++) std::this_thread::sleep_for(std::chrono::milliseconds(1));
}
extern "C" cudaError_t cudaGetDevice(int *device)
{
    *device = 0;
    return cudaSuccess;
}
// The larger size is set first and its caller goes on last, where the callers can get so far.
extern "C" cudaError_t cudaFuncSetAttribute(const void *, cudaFuncAttribute, int bytes)
{
    sets++;
    if (bytes == LARGE) {
        limit = bytes;
        large_set = 1;
        wait_for(small_set);
    } else {
        wait_for(large_set);
        limit = bytes;
        small_set = 1;
    }
    return cudaSuccess;
}

int main()
{
    static dsv4cu::SmemLimit lim;
    auto call = [](int bytes) { dsv4cu::smem_limit(lim, nullptr, bytes); };
    std::thread a(call, LARGE), b(call, SMALL);
    a.join();
    b.join();
    call(LARGE);
    const int after = sets;
    call(SMALL);
    call(LARGE);
    printf("%%d %%d", limit.load(), sets.load() - after);
    return 0;
}
"""


def test_two_threads_leave_the_larger_limit(tmp_path):
    """Calls of two sizes at once: a launch of the larger size fits afterwards, and nothing is set again."""
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc))), "include")
    if not os.path.exists(os.path.join(include, "cuda_runtime_api.h")):
        pytest.skip("no CUDA headers")
    src, exe = tmp_path / "s.cpp", str(tmp_path / "s")
    src.write_text(SOURCE % os.path.join(PKG, "csrc", "smem_limit.h"))
    subprocess.run(["g++", "-std=c++17", "-pthread", "-I", include, str(src), "-o", exe], check=True)
    for _ in range(5):
        out = subprocess.run([exe], capture_output=True, check=True, timeout=60).stdout.split()
        assert [int(x) for x in out] == [200000, 0]
