// smem_limit.h - the dynamic shared-memory limit of a kernel, host side.
#pragma once

#include <atomic>
#include <mutex>

#include <cuda_runtime_api.h>

namespace dsv4cu {

// One per call site: the largest limit set for its kernel on each device, so a
// call costs no attribute call after the first. Threads with a context each
// come here with different sizes: looking, setting and noting are one step, or
// a smaller size set last would stand below a larger one noted last and every
// later launch of the larger size would fail.
struct SmemLimit {
    std::mutex lock;
    std::atomic<int> set[64];
};
static inline cudaError_t smem_limit(SmemLimit &c, const void *kernel, int bytes)
{
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const bool cache = dev >= 0 && dev < 64;
    if (cache && c.set[dev].load(std::memory_order_acquire) >= bytes) return cudaSuccess;
    std::lock_guard<std::mutex> hold(c.lock);
    if (cache && c.set[dev].load(std::memory_order_relaxed) >= bytes) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && cache) c.set[dev].store(bytes, std::memory_order_release);
    return e;
}

}  // namespace dsv4cu
