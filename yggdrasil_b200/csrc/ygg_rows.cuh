// What the kernels over rows of logits share: 16-byte pieces of rows that begin anywhere, their largest entries, pairs of
// floats, and 2^x.
#pragma once
#include <math.h>

#include "ygg_ops.cuh"

namespace ygg {

constexpr float kLog2e = 1.4426950408889634f;

// 2^x, results below 2^-126 as 0 (keeping them costs three instructions more, and no sum of a row would show them).
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Integers in the order of the floats: NaN as -inf, -0 as +0.
__device__ __forceinline__ int order(float x) {
    x = isnan(x) ? -INFINITY : x + 0.0f;
    const int b = __float_as_int(x);
    return b >= 0 ? b : b ^ 0x7FFFFFFF;
}
__device__ __forceinline__ float unorder(int k) { return __int_as_float(k >= 0 ? k : k ^ 0x7FFFFFFF); }

// Rows may begin anywhere: a row is read from the 16-byte boundary at or before it, `off` entries early, and place u of
// what is read holds the entry u - off (32 bits: a row has less than 2^31 entries). The places outside the row lie in the same 16 bytes as one of its own entries.
template <typename T> __device__ __forceinline__ uint32_t offset_of(const T *x) { return ((uint32_t)(uintptr_t)x & 15) / sizeof(T); }

template <typename T> constexpr uint32_t kMinusInf = 0;
template <> constexpr uint32_t kMinusInf<float> = 0xFF800000u;
template <> constexpr uint32_t kMinusInf<__half> = 0xFC00u;
template <> constexpr uint32_t kMinusInf<__nv_bfloat16> = 0xFF80u;

// A warp's run of 32 kPer places from u0 on, lane l those from u0 + l kPer on; -inf outside the row's places [off, end).
template <typename T, bool AGAIN = false>
__device__ __forceinline__ uint4 load_run(const T *from, uint32_t u0, uint32_t off, uint32_t end, int lane) {
    constexpr int N = kPer<T>;
    const uint32_t u = u0 + lane * N;
    uint4 q = make_uint4(0, 0, 0, 0);
    if (u < end) q = AGAIN ? load_again(from + u) : load_stream(from + u);
    if (u + N > end || u < off) {
        uint32_t *w = (uint32_t *)&q;
#pragma unroll
        for (int i = 0; i < N; i++)
            if (u + i >= end || u + i < off) {
                if (N == 4) w[i] = kMinusInf<T>;
                else w[i / 2] = (w[i / 2] & (0xFFFFu << (i & 1 ? 0 : 16))) | kMinusInf<T> << (i & 1 ? 16 : 0);
            }
    }
    return q;
}
template <typename T>
__device__ __forceinline__ void load_run(const T *from, uint32_t u0, uint32_t off, uint32_t end, int lane, float (&v)[kPer<T>]) {
    unpack(load_run(from, u0, off, end, lane), v, T());
}

// The largest of a vector, NaN left out. 16-bit types compare in pairs.
__device__ __forceinline__ float largest(const uint4 &q, float) {
    return fmaxf(fmaxf(__uint_as_float(q.x), __uint_as_float(q.y)), fmaxf(__uint_as_float(q.z), __uint_as_float(q.w)));
}
__device__ __forceinline__ float largest(const uint4 &q, __half) {
    const __half2 *h = (const __half2 *)&q;
    const float2 f = __half22float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(f.x, f.y);
}
__device__ __forceinline__ float largest(const uint4 &q, __nv_bfloat16) {
    const __nv_bfloat162 *h = (const __nv_bfloat162 *)&q;
    const float2 f = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(f.x, f.y);
}

// Two floats to an instruction.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float a, float b) {
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 split(Pair v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ Pair add(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Pair mul(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ Pair exp2_approx(Pair v) {
    const float2 f = split(v);
    return pair(exp2_approx(f.x), exp2_approx(f.y));
}

__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *(const uint32_t *)&h;
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *(const uint32_t *)&h;
}
__device__ __forceinline__ uint4 pack(const float (&v)[4], float) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
template <typename T> __device__ __forceinline__ uint4 pack(const float (&v)[8], T t) {
    return make_uint4(pack2(v[0], v[1], t), pack2(v[2], v[3], t), pack2(v[4], v[5], t), pack2(v[6], v[7], t));
}

// The i-th pair of a vector.
__device__ __forceinline__ Pair pair_of(const uint4 &q, int i, float) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    return pair(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
}
__device__ __forceinline__ Pair pair_of(const uint4 &q, int i, __nv_bfloat16) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    return pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
}
__device__ __forceinline__ Pair pair_of(const uint4 &q, int i, __half) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    const float2 f = __half22float2(*(const __half2 *)&w[i]);
    return pair(f.x, f.y);
}

}  // namespace ygg
