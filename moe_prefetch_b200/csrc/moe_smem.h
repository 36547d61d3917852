// moe_smem.h -- the dynamic shared memory limit of a kernel.
#pragma once

#include <cuda_runtime_api.h>

#include <atomic>
#include <mutex>

namespace moe {

// cudaFuncSetAttribute of a kernel's dynamic shared memory, only where a launch on
// this device needs more than any before (the call costs a microsecond).  One
// object per kernel.  Launches may come from several threads: the limit and
// the record of it change together, under the lock, so that it only rises.
class SmemAttr {
    std::atomic<int> set_[64];   // zero-initialised as a static
    std::mutex lock_;

public:
    cudaError_t need(const void *fn, int bytes) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        if (dev < 64 && set_[dev].load(std::memory_order_acquire) >= bytes) return cudaSuccess;
        const std::lock_guard<std::mutex> hold(lock_);
        if (dev < 64 && set_[dev].load(std::memory_order_relaxed) >= bytes) return cudaSuccess;
        e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess && dev < 64) set_[dev].store(bytes, std::memory_order_release);
        return e;
    }
};

}  // namespace moe
