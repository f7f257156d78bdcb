// Host side: the dynamic shared-memory limit of a kernel.
#pragma once
#include <cuda_runtime_api.h>
#include <stddef.h>

#include <atomic>
#include <mutex>

namespace ygg {

// The limit, raised once per device to the largest size asked for so far (the attribute is per device; raising it on every
// launch would cost a driver call per step). One SmemLimits per kernel. The record never says more than the attribute holds,
// whatever sizes several host threads ask for: it is raised, and both written, by one thread at a time.
constexpr int kMaxDevices = 64;
struct SmemLimits { std::atomic<size_t> set[kMaxDevices]; };
inline cudaError_t raise_smem_limit(const void *fn, size_t smem, SmemLimits &lim) {
    static std::mutex raising;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const bool known = dev >= 0 && dev < kMaxDevices;
    if (known && lim.set[dev].load(std::memory_order_acquire) >= smem) return cudaSuccess;
    std::lock_guard<std::mutex> one(raising);
    if (known && lim.set[dev].load(std::memory_order_relaxed) >= smem) return cudaSuccess;
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess && known) lim.set[dev].store(smem, std::memory_order_release);
    return e;
}

}  // namespace ygg
