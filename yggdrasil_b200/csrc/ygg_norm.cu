// Layer norm of rows, and its gradient.
//
// A row x of D entries gives mu = sum x / D, r = 1 / sqrt(sum (x - mu)^2 / D + eps), h = (x - mu) r and y = h w + b (w 1 and b
// 0 where they are absent). With the gradient g that arrives at y,
//   dx = r (g w - sum(g w) / D - h sum(g w h) / D),   dw = sum over rows of g h,   db = sum over rows of g.
// All sums are held in 32 bits; the variance is that of the differences, so that a large mean does not cancel it. The sums
// over rows are cut by the number of rows and columns alone and joined in one order: results repeat bit for bit.
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "ygg_ops.cuh"

namespace {

using namespace ygg;

struct Affine {          // a weight or a bias: null for none
    int dtype;
    const void *v;
};
struct Norm {
    const void *x;
    int64_t rows, stride;
    int dim;
    Affine weight, bias;
    float eps;
    void *y;             // rows dim entries apart
    float2 *stats;       // mu, r of each row, or null
};
struct NormGrad {
    const void *x, *g;
    int64_t rows, stride, g_stride;
    int dim;
    Affine weight;
    const float2 *stats;
    void *dx;            // rows dim entries apart, or null
};
struct Columns {
    const void *x, *g;
    int64_t rows, stride, g_stride, each;   // each: rows of a part
    int dim, parts;
    const float2 *stats;
    float *dw, *db;      // [parts][dim], each may be null
};

__device__ __forceinline__ float at(const Affine &a, int i, float none) {
    if (!a.v) return none;
    if (a.dtype == YGG_DTYPE_FLOAT) return ((const float *)a.v)[i];
    if (a.dtype == YGG_DTYPE_HALF) return __half2float(((const __half *)a.v)[i]);
    return __bfloat162float(((const __nv_bfloat16 *)a.v)[i]);
}

// The sum over the block's 256 threads, the same in each.
__device__ __forceinline__ float block_sum(float v, float *part) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; w++) v += part[w];
    return v;
}

template <typename T> __global__ void __launch_bounds__(256) norm_kernel(const Norm p) {
    __shared__ float part[8];
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T *x = (const T *)p.x + row * p.stride;
        float sum = 0.0f, sq = 0.0f;
        for (int j = threadIdx.x; j < p.dim; j += 256) sum += to_f(x[j]);
        const float mu = block_sum(sum, part) / (float)p.dim;
        for (int j = threadIdx.x; j < p.dim; j += 256) {
            const float d = to_f(x[j]) - mu;
            sq = fmaf(d, d, sq);
        }
        const float r = 1.0f / sqrtf(block_sum(sq, part) / (float)p.dim + p.eps);
        T *y = (T *)p.y + row * p.dim;
        for (int j = threadIdx.x; j < p.dim; j += 256) from_f(fmaf((to_f(x[j]) - mu) * r, at(p.weight, j, 1.0f), at(p.bias, j, 0.0f)), y[j]);
        if (p.stats && threadIdx.x == 0) p.stats[row] = make_float2(mu, r);
    }
}

template <typename T> __global__ void __launch_bounds__(256) grad_kernel(const NormGrad p) {
    __shared__ float part[8];
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T *x = (const T *)p.x + row * p.stride, *g = (const T *)p.g + row * p.g_stride;
        const float2 s = p.stats[row];
        float a = 0.0f, c = 0.0f;
        for (int j = threadIdx.x; j < p.dim; j += 256) {
            const float gw = to_f(g[j]) * at(p.weight, j, 1.0f);
            a += gw;
            c = fmaf(gw, (to_f(x[j]) - s.x) * s.y, c);
        }
        a = block_sum(a, part) / (float)p.dim;
        c = block_sum(c, part) / (float)p.dim;
        T *dx = (T *)p.dx + row * p.dim;
        for (int j = threadIdx.x; j < p.dim; j += 256) {
            const float h = (to_f(x[j]) - s.x) * s.y;
            from_f(s.y * (to_f(g[j]) * at(p.weight, j, 1.0f) - a - h * c), dx[j]);
        }
    }
}

template <typename T> __global__ void __launch_bounds__(128) columns_kernel(const Columns p) {
    const int j = blockIdx.x * 128 + threadIdx.x;
    if (j >= p.dim) return;
    const int64_t first = (int64_t)blockIdx.y * p.each, end = min(first + p.each, p.rows);
    float w = 0.0f, b = 0.0f;
    for (int64_t row = first; row < end; row++) {
        const float2 s = p.stats[row];
        const float g = to_f(((const T *)p.g)[row * p.g_stride + j]);
        w = fmaf(g, (to_f(((const T *)p.x)[row * p.stride + j]) - s.x) * s.y, w);
        b += g;
    }
    const int64_t to = (int64_t)blockIdx.y * p.dim + j;
    if (p.dw) p.dw[to] = w;
    if (p.db) p.db[to] = b;
}

template <typename T> __global__ void __launch_bounds__(128) join_kernel(const float *part, int parts, int dim, T *out) {
    const int j = blockIdx.x * 128 + threadIdx.x;
    if (j >= dim) return;
    float v = 0.0f;
    for (int i = 0; i < parts; i++) v += part[(int64_t)i * dim + j];
    from_f(v, out[j]);
}

int parts_of(int64_t rows) { return (int)std::min<int64_t>((rows + 31) / 32, 256); }

unsigned grid_of(int64_t rows) { return (unsigned)std::min<int64_t>(rows, 1 << 20); }

bool type_ok(int t) { return t >= YGG_DTYPE_FLOAT && t <= YGG_DTYPE_BFLOAT; }
size_t size_of(int t) { return t == YGG_DTYPE_FLOAT ? 4 : 2; }

}  // namespace

extern "C" {

int ygg_layer_norm(int device, int dtype, int64_t rows, int64_t dim, const void *d_x, int64_t row_stride, int weight_dtype,
                   const void *d_weight, int bias_dtype, const void *d_bias, float eps, void *d_y, float *d_stats,
                   void *stream) {
    if (rows < 0 || dim < 1) return YGG_E_ARG;
    if (dim > INT32_MAX / 2 || !type_ok(weight_dtype) || !type_ok(bias_dtype)) return YGG_E_UNSUPPORTED;
    if (rows == 0) return YGG_OK;
    if (!d_x || !d_y) return YGG_E_ARG;
    OnDevice on(device);
    if (!on.ok) return YGG_E_DEVICE;
    const Norm p{d_x, rows, row_stride, (int)dim, {weight_dtype, d_weight}, {bias_dtype, d_bias}, eps, d_y, (float2 *)d_stats};
    const int rc = by_type(dtype, [&](auto t) { norm_kernel<decltype(t)><<<grid_of(rows), 256, 0, (cudaStream_t)stream>>>(p); });
    return rc != YGG_OK ? rc : cudaGetLastError() == cudaSuccess ? YGG_OK : YGG_E_CUDA;
}

size_t ygg_layer_norm_workspace(int64_t rows, int64_t dim) {
    if (rows < 0 || dim < 1 || dim > INT32_MAX / 2) return 0;
    return 2 * sizeof(float) * (size_t)parts_of(rows) * (size_t)dim + 16;
}

int ygg_layer_norm_backward(int device, int dtype, int64_t rows, int64_t dim, const void *d_x, int64_t row_stride,
                            int weight_dtype, const void *d_weight, int bias_dtype, const float *d_stats, const void *d_grad,
                            int64_t grad_stride, void *d_dx, void *d_dweight, void *d_dbias, void *d_workspace,
                            size_t workspace_bytes, void *stream) {
    if (rows < 0 || dim < 1) return YGG_E_ARG;
    if (dim > INT32_MAX / 2 || !type_ok(dtype) || !type_ok(weight_dtype) || !type_ok(bias_dtype)) return YGG_E_UNSUPPORTED;
    OnDevice on(device);
    if (!on.ok) return YGG_E_DEVICE;
    const cudaStream_t st = (cudaStream_t)stream;
    if (rows == 0) {
        cudaError_t e = cudaSuccess;
        if (d_dweight) e = cudaMemsetAsync(d_dweight, 0, dim * size_of(weight_dtype), st);
        if (d_dbias && e == cudaSuccess) e = cudaMemsetAsync(d_dbias, 0, dim * size_of(bias_dtype), st);
        return e == cudaSuccess ? YGG_OK : YGG_E_CUDA;
    }
    if (!d_x || !d_stats || !d_grad) return YGG_E_ARG;
    if ((d_dweight || d_dbias) && (!d_workspace || ((uintptr_t)d_workspace & 15) || workspace_bytes < ygg_layer_norm_workspace(rows, dim)))
        return YGG_E_ARG;
    const int parts = parts_of(rows);
    float *dw = (float *)d_workspace, *db = dw + (size_t)parts * dim;
    const NormGrad p{d_x, d_grad, rows, row_stride, grad_stride, (int)dim, {weight_dtype, d_weight}, (const float2 *)d_stats, d_dx};
    const Columns c{d_x, d_grad, rows, row_stride, grad_stride, (rows + parts - 1) / parts, (int)dim, parts,
                    (const float2 *)d_stats, d_dweight ? dw : nullptr, d_dbias ? db : nullptr};
    const unsigned wide = (unsigned)((dim + 127) / 128);
    by_type(dtype, [&](auto t) {
        using T = decltype(t);
        if (d_dx) grad_kernel<T><<<grid_of(rows), 256, 0, st>>>(p);
        if (d_dweight || d_dbias) columns_kernel<T><<<dim3(wide, parts), 128, 0, st>>>(c);
    });
    if (d_dweight)
        by_type(weight_dtype, [&](auto t) { join_kernel<decltype(t)><<<wide, 128, 0, st>>>(dw, parts, (int)dim, (decltype(t) *)d_dweight); });
    if (d_dbias)
        by_type(bias_dtype, [&](auto t) { join_kernel<decltype(t)><<<wide, 128, 0, st>>>(db, parts, (int)dim, (decltype(t) *)d_dbias); });
    return cudaGetLastError() == cudaSuccess ? YGG_OK : YGG_E_CUDA;
}

}  // extern "C"
