// What the operators without a model handle share: the element types, the calling thread's device, and the dispatch of
// a type given as a number.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "ygg_b200.h"

namespace ygg {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f(float v, float &o) { o = v; }
__device__ __forceinline__ void from_f(float v, __half &o) { o = __float2half_rn(v); }
__device__ __forceinline__ void from_f(float v, __nv_bfloat16 &o) { o = __float2bfloat16_rn(v); }

struct OnDevice {   // makes `device` the calling thread's for the length of a call
    int prev = -1;
    bool ok;
    explicit OnDevice(int device) {
        ok = cudaGetDevice(&prev) == cudaSuccess && (prev == device || cudaSetDevice(device) == cudaSuccess);
        if (!ok || prev == device) prev = -1;
    }
    ~OnDevice() {
        if (prev >= 0) cudaSetDevice(prev);
    }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;
};

// The SMs of the calling thread's device.
inline int sm_count() {
    static int counts[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    if (!counts[dev] && cudaDeviceGetAttribute(&counts[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return 148;
    return counts[dev];
}

// f of a value of the type that a YGG_DTYPE_ number names.
template <typename F> int by_type(int dtype, F f) {
    switch (dtype) {
        case YGG_DTYPE_FLOAT: f(float()); return YGG_OK;
        case YGG_DTYPE_HALF: f(__half()); return YGG_OK;
        case YGG_DTYPE_BFLOAT: f(__nv_bfloat16()); return YGG_OK;
        default: return YGG_E_UNSUPPORTED;
    }
}

}  // namespace ygg
