// Linear layers in 8-bit integers: rows of activations quantised as they come, weights quantised once.
//
// Row m of x (K values) has the scale s_m = max|x_m| / 127 and the codes c = rint(x 127 / max|x_m|), in [-127, 127];
// a weight row n (one output channel) has codes w and its scale s_n. Then
//   y[m][n] = (sum_k c[m][k] w[n][k]) s_m s_n + b[n],
// (the channel's factor first: a row's scale may be near the end of the type's range, where only a result beyond it may
// overflow), with the sum exact in int32 (K <= 131072 keeps |sum| below 127 127 2^17 < 2^31), one rounding to float, one for each
// factor and the bias, and one to the output's type. Integer sums have no order: results repeat bit for bit.
// A row of zeros (or so small that its scale rounds to 0) has scale 0 and codes 0; a row that holds NaN or infinity has
// scale NaN and codes 0, so that its outputs are NaN.
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "ygg_ops.cuh"

namespace {

using namespace ygg;

struct Quantize {
    const void *x;
    int64_t rows, stride;
    int k, padded;          // the codes of a row are zero from k to padded
    int8_t *codes;
    int64_t code_stride;
    float *scale;
};

struct Linear {
    const int8_t *codes, *weight;
    int64_t code_stride, weight_stride;
    const float *row_scale, *scale, *bias;   // bias: null for none
    int64_t rows, n;
    int k;
    void *out;
    int64_t out_stride;
};

// The two factors of a row from its largest magnitude: 127 / most for the codes, most / 127 for the products. NaN or
// infinity in the row (most is not finite): codes 0, scale NaN.
struct Factors { float inverse, scale; };
__device__ __forceinline__ Factors factors(float most) {
    if (!(most < INFINITY)) return {0.0f, NAN};
    const float scale = __fdiv_rn(most, 127.0f), inverse = __fdiv_rn(127.0f, most);
    if (scale == 0.0f || inverse == INFINITY) return {0.0f, 0.0f};
    return {inverse, scale};
}
__device__ __forceinline__ int code(float x, float inverse) {
    if (inverse == 0.0f) return 0;
    return max(-127, min(127, __float2int_rn(__fmul_rn(x, inverse))));
}
// max that keeps NaN
__device__ __forceinline__ float most_of(float a, float b) { return (a > b || a != a) ? a : b; }

template <typename T> __global__ void __launch_bounds__(256) quantize_kernel(const Quantize p) {
    __shared__ float part[8];
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T *x = (const T *)p.x + row * p.stride;
        float most = 0.0f;
        for (int j = threadIdx.x; j < p.k; j += 256) most = most_of(fabsf(to_f(x[j])), most);
#pragma unroll
        for (int o = 16; o; o >>= 1) most = most_of(__shfl_xor_sync(~0u, most, o), most);
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = most;
        __syncthreads();
        for (int w = 0; w < 8; w++) most = most_of(part[w], most);
        __syncthreads();
        const Factors f = factors(most);
        for (int j = threadIdx.x; j < p.padded; j += 256)
            p.codes[row * p.code_stride + j] = j < p.k ? (int8_t)code(to_f(x[j]), f.inverse) : (int8_t)0;
        if (threadIdx.x == 0) p.scale[row] = f.scale;
    }
}

// 64 rows x 64 channels a block, 4 x 4 a thread, 64 bytes of K at a time through shared memory, dp4a.
constexpr int kTile = 64, kPitch = 64 + 16;

__device__ __forceinline__ uint4 chunk_of(const int8_t *base, int64_t row, int64_t rows, int64_t stride, int at, int k) {
    if (row >= rows || at >= k) return make_uint4(0, 0, 0, 0);
    uint4 v = *(const uint4 *)(base + row * stride + at);   // 16-byte chunks: stride and base are multiples of 16
    if (at + 16 > k) {                                      // bytes past k are not the row's
        uint32_t *w = (uint32_t *)&v;
        for (int i = 0; i < 4; i++) {
            const int left = k - at - 4 * i;
            w[i] = left >= 4 ? w[i] : left <= 0 ? 0u : w[i] & ((1u << (8 * left)) - 1);
        }
    }
    return v;
}

template <typename T> __global__ void __launch_bounds__(256) linear_kernel(const Linear p) {
    __shared__ __align__(16) int8_t a[kTile][kPitch], b[kTile][kPitch];
    const int64_t m0 = (int64_t)blockIdx.y * kTile, n0 = (int64_t)blockIdx.x * kTile;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 16;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < p.k; k0 += 64) {
        *(uint4 *)&a[r][c] = chunk_of(p.codes, m0 + r, p.rows, p.code_stride, k0 + c, p.k);
        *(uint4 *)&b[r][c] = chunk_of(p.weight, n0 + r, p.n, p.weight_stride, k0 + c, p.k);
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < 64; kk += 4) {
            int av[4], bv[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                av[i] = *(const int *)&a[ty + 16 * i][kk];
                bv[i] = *(const int *)&b[tx + 16 * i][kk];
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = __dp4a(av[i], bv[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int64_t m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
            if (m >= p.rows || n >= p.n) continue;
            const float v = __int2float_rn(acc[i][j]) * p.scale[n] * p.row_scale[m];
            from_f(p.bias ? v + p.bias[n] : v, ((T *)p.out)[m * p.out_stride + n]);
        }
}

int padded_of(int64_t k) { return (int)((k + 15) / 16 * 16); }

bool rows_ok(int64_t rows, int64_t k) { return rows >= 0 && rows < ((int64_t)1 << 40) && k >= 1; }

int quantize(int dtype, const Quantize &p, cudaStream_t st) {
    const int grid = (int)std::min<int64_t>(p.rows, 148 * 8);
    return by_type(dtype, [&](auto t) { quantize_kernel<decltype(t)><<<grid, 256, 0, st>>>(p); });
}

int linear(int out_dtype, const Linear &p, cudaStream_t st) {
    const int64_t step = (int64_t)65535 * kTile;   // rows a launch can hold in its grid's second dimension
    for (int64_t m = 0; m < p.rows; m += step) {
        Linear q = p;
        q.rows = std::min(step, p.rows - m);
        q.codes += m * p.code_stride;
        q.row_scale += m;
        q.out = (char *)p.out + m * p.out_stride * (out_dtype == YGG_DTYPE_FLOAT ? 4 : 2);
        const dim3 grid((unsigned)((q.n + kTile - 1) / kTile), (unsigned)((q.rows + kTile - 1) / kTile));
        const int rc = by_type(out_dtype, [&](auto t) { linear_kernel<decltype(t)><<<grid, 256, 0, st>>>(q); });
        if (rc != YGG_OK) return rc;
    }
    return YGG_OK;
}

bool aligned16(const void *p, int64_t stride) { return ((uintptr_t)p & 15) == 0 && stride % 16 == 0; }

}  // namespace

extern "C" {

int ygg_quantize_rows(int device, int dtype, int64_t rows, int64_t k, const void *d_x, int64_t row_stride,
                      int8_t *d_codes, int64_t code_stride, float *d_scale, void *stream) {
    if (!rows_ok(rows, k)) return YGG_E_ARG;
    if (k > YGG_LINEAR_MAX_K) return YGG_E_UNSUPPORTED;
    if (rows == 0) return YGG_OK;
    if (!d_x || !d_codes || !d_scale || !aligned16(d_codes, code_stride) || code_stride < padded_of(k)) return YGG_E_ARG;
    OnDevice on(device);
    if (!on.ok) return YGG_E_DEVICE;
    const int rc = quantize(dtype, {d_x, rows, row_stride, (int)k, padded_of(k), d_codes, code_stride, d_scale},
                            (cudaStream_t)stream);
    return rc != YGG_OK ? rc : cudaGetLastError() == cudaSuccess ? YGG_OK : YGG_E_CUDA;
}

size_t ygg_linear_workspace(int64_t rows, int64_t k) {
    if (!rows_ok(rows, k) || k > YGG_LINEAR_MAX_K) return 0;
    return (size_t)rows * padded_of(k) + (size_t)rows * sizeof(float) + 16;
}

int ygg_linear_quantized(int device, int64_t rows, int64_t k, int64_t n, const int8_t *d_codes, int64_t code_stride,
                         const float *d_row_scale, const int8_t *d_weight, int64_t weight_stride,
                         const float *d_scale, const float *d_bias, int out_dtype, void *d_out, int64_t out_stride,
                         void *stream) {
    if (!rows_ok(rows, k) || n < 1 || n > INT32_MAX) return YGG_E_ARG;
    if (k > YGG_LINEAR_MAX_K) return YGG_E_UNSUPPORTED;
    if (rows == 0) return YGG_OK;
    if (!d_codes || !d_row_scale || !d_weight || !d_scale || !d_out || !aligned16(d_codes, code_stride) ||
        !aligned16(d_weight, weight_stride) || code_stride < k || weight_stride < k)
        return YGG_E_ARG;
    OnDevice on(device);
    if (!on.ok) return YGG_E_DEVICE;
    const int rc = linear(out_dtype, {d_codes, d_weight, code_stride, weight_stride, d_row_scale, d_scale, d_bias, rows,
                                      n, (int)k, d_out, out_stride}, (cudaStream_t)stream);
    return rc != YGG_OK ? rc : cudaGetLastError() == cudaSuccess ? YGG_OK : YGG_E_CUDA;
}

int ygg_linear(int device, int dtype, int64_t rows, int64_t k, int64_t n, const void *d_x, int64_t row_stride,
               const int8_t *d_weight, int64_t weight_stride, const float *d_scale, const float *d_bias, int out_dtype,
               void *d_out, int64_t out_stride, void *d_workspace, size_t workspace_bytes, void *stream) {
    if (!rows_ok(rows, k) || n < 1 || n > INT32_MAX) return YGG_E_ARG;
    if (k > YGG_LINEAR_MAX_K) return YGG_E_UNSUPPORTED;
    if (rows == 0) return YGG_OK;
    if (!d_workspace || ((uintptr_t)d_workspace & 15) || workspace_bytes < ygg_linear_workspace(rows, k)) return YGG_E_ARG;
    const int64_t padded = padded_of(k);
    int8_t *codes = (int8_t *)d_workspace;
    float *scale = (float *)(codes + rows * padded);
    const int rc = ygg_quantize_rows(device, dtype, rows, k, d_x, row_stride, codes, padded, scale, stream);
    if (rc != YGG_OK) return rc;
    return ygg_linear_quantized(device, rows, k, n, codes, padded, scale, d_weight, weight_stride, d_scale, d_bias,
                                out_dtype, d_out, out_stride, stream);
}

}  // extern "C"
