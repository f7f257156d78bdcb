// Log-probabilities of given tokens, entropy and top alternatives of rows of logits, and their gradient.
//
// A row x of V logits gives, with m = max x, s = sum_j e^(x_j - m) and p_j = e^(x_j - m) / s,
//   lse = m + log s,   logprob = x_t - lse,   H = -sum_j p_j log p_j = log s - (sum_j e^(x_j - m) (x_j - m)) / s,
// and the `top` largest entries by (value descending, index ascending).
// The gradient of g . logprob + g_H H + g_lse lse + sum_k g_k (x_ak - lse) is
//   dx_j = g [j = t] + sum_k g_k [j = a_k] + p_j (g_lse - g - sum_k g_k) - g_H p_j (log p_j + H).
// Everything is held in 32 bits as y_j = x_j - m and e_j = 2^(y_j log2 e): the difference first, so that a mask of the
// type's lowest value does not overflow in the product.
//
// Edge rules: -inf entries have probability 0 and add nothing; a row of -inf alone is empty (logprob and lse -inf,
// entropy 0, gradient 0); NaN or +inf anywhere makes the row's values NaN, and NaN ranks as -inf among the
// alternatives. A negative token is padding (logprob 0, no gradient), a token >= V gives NaN.
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "ygg_ops.cuh"

namespace {

using namespace ygg;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFloor = -200.0f;   // e^-200 is 0 in 32 bits: y below it only has to stay finite

struct Rows {
    const void *logits;
    int64_t rows, vocab, stride;
    const void *tokens;   // int32 or int64
    int token_bytes, top;
    float *logprob, *entropy, *lse;
    int32_t *top_ids;
    float *top_logprobs;
    float4 *stats;        // m, 1 / s, log s, H: what the gradient needs; or null
};

struct Grad {
    const void *logits;
    int64_t rows, vocab, stride;
    const void *tokens;
    int token_bytes, top;
    const int32_t *top_ids;
    const float4 *stats;
    const float *g_logprob, *g_entropy, *g_lse, *g_top;   // each may be null
    void *grad;
    int64_t grad_stride;
};

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Integers in the order of the floats: NaN as -inf, -0 as +0.
__device__ __forceinline__ int order(float x) {
    x = isnan(x) ? -INFINITY : x + 0.0f;
    const int b = __float_as_int(x);
    return b >= 0 ? b : b ^ 0x7FFFFFFF;
}
__device__ __forceinline__ float unorder(int k) { return __int_as_float(k >= 0 ? k : k ^ 0x7FFFFFFF); }

// Running softmax sums relative to m: s = sum e^y, t = sum e^y y.
struct Sums { float m, s, t; };

__device__ __forceinline__ Sums none() { return {-INFINITY, 0.0f, 0.0f}; }

// The sums relative to a larger m. An m of -inf stands for an empty part; a row that holds +inf becomes NaN.
__device__ __forceinline__ void raise(Sums &a, float m) {
    if (a.m == m) return;
    const float by = a.m == -INFINITY ? 0.0f : a.m - m, f = exp2_approx(by * kLog2e);
    a.t = f * fmaf(a.s, fmaxf(by, kFloor), a.t);
    a.s *= f;
    a.m = m;
}
__device__ __forceinline__ void join(Sums &a, Sums b) {
    const float m = fmaxf(a.m, b.m);
    raise(a, m);
    raise(b, m);
    a.s += b.s;
    a.t += b.t;
}
__device__ __forceinline__ void add(Sums &a, float x) {
    if (x > a.m) raise(a, x);
    const float y = x - (a.m == -INFINITY ? 0.0f : a.m), e = exp2_approx(y * kLog2e);
    a.s += e;
    a.t = fmaf(e, fmaxf(y, kFloor), a.t);
}

__device__ __forceinline__ int64_t token_of(const void *tokens, int bytes, int64_t row) {
    return bytes == 8 ? ((const int64_t *)tokens)[row] : (int64_t)((const int32_t *)tokens)[row];
}

template <typename T> __global__ void __launch_bounds__(256) logprobs_kernel(const Rows p) {
    __shared__ Sums part[8];
    __shared__ unsigned long long best[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T *x = (const T *)p.logits + row * p.stride;
        Sums a = none();
        for (int64_t j = threadIdx.x; j < p.vocab; j += blockDim.x) add(a, to_f(x[j]));
#pragma unroll
        for (int o = 16; o; o >>= 1)
            join(a, Sums{__shfl_xor_sync(~0u, a.m, o), __shfl_xor_sync(~0u, a.s, o), __shfl_xor_sync(~0u, a.t, o)});
        if (lane == 0) part[warp] = a;
        __syncthreads();
        a = part[0];
        for (int w = 1; w < 8; w++) join(a, part[w]);
        const bool empty = a.s == 0.0f;
        const float m = empty ? 0.0f : a.m, ls = empty ? -INFINITY : logf(a.s);
        const float H = empty ? 0.0f : ls - a.t / a.s;
        if (threadIdx.x == 0) {
            const int64_t t = token_of(p.tokens, p.token_bytes, row);
            float lp = 0.0f;
            if (t >= p.vocab) lp = NAN;
            else if (t >= 0) lp = empty ? -INFINITY : (to_f(x[t]) - m) - ls;
            p.logprob[row] = lp;
            p.entropy[row] = H;
            p.lse[row] = m + ls;
            if (p.stats) p.stats[row] = make_float4(m, empty ? 0.0f : 1.0f / a.s, empty ? 0.0f : ls, H);
        }
        // the k-th best is the best key below the last: value above, then the lower index
        unsigned long long last = ~0ull;
        for (int k = 0; k < p.top; k++) {
            unsigned long long mine = 0;
            for (int64_t j = threadIdx.x; j < p.vocab; j += blockDim.x) {
                const unsigned long long key =
                    ((unsigned long long)((unsigned)order(to_f(x[j])) ^ 0x80000000u) << 32) | (unsigned)~(unsigned)j;
                if (key < last && key > mine) mine = key;
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) mine = max(mine, __shfl_xor_sync(~0u, mine, o));
            __syncthreads();
            if (lane == 0) best[warp] = mine;
            __syncthreads();
            for (int w = 0; w < 8; w++) mine = max(mine, best[w]);
            last = mine;
            if (threadIdx.x == 0) {
                const float v = unorder((int)((unsigned)(mine >> 32) ^ 0x80000000u));
                p.top_ids[row * p.top + k] = (int32_t)~(unsigned)mine;
                p.top_logprobs[row * p.top + k] = empty ? -INFINITY : (v - m) - ls;
            }
        }
        __syncthreads();
    }
}

// The gradient of one entry, less the terms of the row's given tokens: p (A + B y).
__device__ __forceinline__ float dense(float x, float m, float inv_s, float A, float B) {
    const float y = x - m;
    return exp2_approx(y * kLog2e) * inv_s * fmaf(B, fmaxf(y, kFloor), A);
}

// A warp per (row, chunk of kChunk entries).
constexpr int kChunk = 1024;
template <typename T> __global__ void __launch_bounds__(256) logprobs_grad_kernel(const Grad p) {
    const int lane = threadIdx.x & 31;
    const int64_t chunks = (p.vocab + kChunk - 1) / kChunk, items = p.rows * chunks;
    for (int64_t it = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); it < items; it += (int64_t)gridDim.x * 8) {
        const int64_t row = it / chunks, j0 = (it - row * chunks) * kChunk, j1 = min(j0 + (int64_t)kChunk, p.vocab);
        const T *x = (const T *)p.logits + row * p.stride;
        T *g = (T *)p.grad + row * p.grad_stride;
        const float4 st = p.stats[row];
        const int64_t t = token_of(p.tokens, p.token_bytes, row);
        const bool given = t >= 0 && t < p.vocab;
        const float gl = p.g_logprob && given ? p.g_logprob[row] : 0.0f, gh = p.g_entropy ? p.g_entropy[row] : 0.0f;
        float c = (p.g_lse ? p.g_lse[row] : 0.0f) - gl;
        if (p.g_top)
            for (int k = 0; k < p.top; k++) c -= p.g_top[row * p.top + k];
        const float A = c - gh * (st.w - st.z), B = -gh;
        for (int64_t j = j0 + lane; j < j1; j += 32) from_f(dense(to_f(x[j]), st.x, st.y, A, B), g[j]);
        __syncwarp();
        // the given token and the alternatives: written again, whole, so that they are rounded once
        const bool live = st.y != 0.0f;
        for (int q = lane; q <= (p.g_top ? p.top : 0); q += 32) {
            const int64_t j = q == 0 ? (given ? t : -1) : p.top_ids[row * p.top + q - 1];
            if (j < j0 || j >= j1 || !live || (q > 0 && given && j == t)) continue;
            float more = q == 0 ? gl : p.g_top[row * p.top + q - 1];
            if (q == 0 && p.g_top)
                for (int k = 0; k < p.top; k++)
                    if (p.top_ids[row * p.top + k] == j) more += p.g_top[row * p.top + k];
            from_f(dense(to_f(x[j]), st.x, st.y, A, B) + more, g[j]);
        }
    }
}

}  // namespace

extern "C" {

int ygg_token_logprobs(int device, int dtype, int64_t rows, int64_t vocab, const void *d_logits, int64_t row_stride,
                       const void *d_tokens, int token_bytes, int top, float *d_logprob, float *d_entropy, float *d_lse,
                       int32_t *d_top_ids, float *d_top_logprobs, float *d_stats, void *stream) {
    if (rows < 0 || vocab < 1 || vocab > INT32_MAX || top < 0 || top > YGG_TOP_MAX || top > vocab ||
        (token_bytes != 4 && token_bytes != 8))
        return YGG_E_ARG;
    if (rows == 0) return YGG_OK;
    if (!d_logits || !d_tokens || !d_logprob || !d_entropy || !d_lse || (top && (!d_top_ids || !d_top_logprobs)) ||
        ((uintptr_t)d_stats & 15))
        return YGG_E_ARG;
    OnDevice on(device);
    if (!on.ok) return YGG_E_DEVICE;
    const Rows p{d_logits, rows, vocab, row_stride, d_tokens, token_bytes, top, d_logprob, d_entropy, d_lse, d_top_ids,
                 d_top_logprobs, (float4 *)d_stats};
    const int grid = (int)std::min<int64_t>(rows, 148 * 8);
    const int rc = by_type(dtype, [&](auto t) {
        logprobs_kernel<decltype(t)><<<grid, 256, 0, (cudaStream_t)stream>>>(p);
    });
    if (rc != YGG_OK) return rc;
    return cudaGetLastError() == cudaSuccess ? YGG_OK : YGG_E_CUDA;
}

int ygg_token_logprobs_backward(int device, int dtype, int64_t rows, int64_t vocab, const void *d_logits,
                                int64_t row_stride, const void *d_tokens, int token_bytes, int top,
                                const int32_t *d_top_ids, const float *d_stats, const float *d_grad_logprob,
                                const float *d_grad_entropy, const float *d_grad_lse, const float *d_grad_top,
                                void *d_grad, int64_t grad_stride, void *stream) {
    if (rows < 0 || vocab < 1 || vocab > INT32_MAX || top < 0 || top > YGG_TOP_MAX || top > vocab ||
        (token_bytes != 4 && token_bytes != 8))
        return YGG_E_ARG;
    if (rows == 0) return YGG_OK;
    if (!d_logits || !d_tokens || !d_stats || ((uintptr_t)d_stats & 15) || !d_grad || (d_grad_top && !d_top_ids))
        return YGG_E_ARG;
    OnDevice on(device);
    if (!on.ok) return YGG_E_DEVICE;
    const Grad p{d_logits, rows, vocab, row_stride, d_tokens, token_bytes, top, d_top_ids, (const float4 *)d_stats,
                 d_grad_logprob, d_grad_entropy, d_grad_lse, d_grad_top, d_grad, grad_stride};
    const int64_t items = rows * ((vocab + kChunk - 1) / kChunk);
    const int grid = (int)std::min<int64_t>((items + 7) / 8, 148 * 16);
    const int rc = by_type(dtype, [&](auto t) {
        logprobs_grad_kernel<decltype(t)><<<grid, 256, 0, (cudaStream_t)stream>>>(p);
    });
    if (rc != YGG_OK) return rc;
    return cudaGetLastError() == cudaSuccess ? YGG_OK : YGG_E_CUDA;
}

}  // extern "C"
