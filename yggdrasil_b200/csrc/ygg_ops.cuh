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

// A vector of 16 bytes as floats.
template <typename T> constexpr int kPer = 16 / sizeof(T);
__device__ __forceinline__ void unpack(const uint4 &q, float (&v)[4], float) {
    v[0] = __uint_as_float(q.x), v[1] = __uint_as_float(q.y), v[2] = __uint_as_float(q.z), v[3] = __uint_as_float(q.w);
}
__device__ __forceinline__ void unpack(const uint4 &q, float (&v)[8], __nv_bfloat16) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ void unpack(const uint4 &q, float (&v)[8], __half) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*(const __half2 *)&w[i]);
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
}
// 16 bytes that this launch reads once. volatile: a load in plain asm counts as free of side effects, so that the compiler
// may issue it before the branch that guards its address.
__device__ __forceinline__ uint4 load_stream(const void *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// The same where the launch comes back to some of the bytes soon: they stay in L1.
__device__ __forceinline__ uint4 load_again(const void *p) {
    uint4 v;
    asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// A launch that follows another in its stream may begin before that one ends; it waits here before it reads what the
// other wrote. The other says when it may begin.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

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
