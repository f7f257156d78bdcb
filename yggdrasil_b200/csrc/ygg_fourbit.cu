// Linear layers with 4-bit weights: a code -8..7 for each weight, a scale for each channel and each group of inputs.
//
//   y[m][n] = sum_g s[n][g] sum_{k in g} x[m][k] q[n][k] + b[n],   group g: inputs g group .. g group + group - 1
//
// with x as it is. A code is exact in either 16-bit type, so that a group's sum is a product of x and codes with float sums,
// and the scale is applied once a group, in floats: no weight is rounded.
//
// The layout of a channel's codes (64 bytes for 128 inputs, rows padded with zeros): of 128 inputs, four runs of 32, each of
// four pieces of 8, piece t of run i is the word 4 t + i; inputs 0, 2, 4, 6 of a piece are the four lowest fields of 4 bits,
// 1, 3, 5, 7 the upper four, each as code + 8. So 16 bytes hold the pieces t of the four runs, a run's inputs are spread over
// the four lanes that multiply them together, and two neighbouring inputs come out of one mask side by side.
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "ygg_ops.cuh"

namespace {

using namespace ygg;

struct FourBit {
    const void *x;
    int64_t rows, x_stride, n;
    int k, blocks, group, groups;   // blocks: of 128 inputs
    const uint8_t *codes;           // [n][64 blocks]
    int scale_dtype;
    const void *scale;              // [n][groups]
    const float *bias;              // null for none
    int out_dtype;
    void *out;
    int64_t out_stride;
};

__device__ __forceinline__ float load_as(int dtype, const void *p, int64_t at) {
    if (dtype == YGG_DTYPE_FLOAT) return ((const float *)p)[at];
    if (dtype == YGG_DTYPE_HALF) return __half2float(((const __half *)p)[at]);
    return __bfloat162float(((const __nv_bfloat16 *)p)[at]);
}
__device__ __forceinline__ void store_as(int dtype, void *p, int64_t at, float v) {
    if (dtype == YGG_DTYPE_FLOAT) ((float *)p)[at] = v;
    else if (dtype == YGG_DTYPE_HALF) ((__half *)p)[at] = __float2half_rn(v);
    else ((__nv_bfloat16 *)p)[at] = __float2bfloat16_rn(v);
}

// The first input of a word of a row, and where an input of a piece stands in its word.
__device__ __forceinline__ int first_of(int word) { return (word >> 4) * 128 + (word & 3) * 32 + (word >> 2 & 3) * 8; }
__device__ __forceinline__ int field_of(int e) { return (e >> 1) * 4 + (e & 1) * 16; }

// ------------------------------------------------------------------------------------------------------ weights

struct Codes {
    const void *w;           // what to quantise, or the codes themselves (int8)
    int64_t n, stride;
    int k, blocks, group, groups;
    uint32_t *codes;
    void *scale;
};

// A warp a channel and group; the last groups of a row pad it to whole blocks. T int8_t: codes that are there already.
template <typename T> __global__ void __launch_bounds__(256) codes_kernel(const Codes p) {
    const int per_row = (p.blocks * 128 + p.group - 1) / p.group, lane = threadIdx.x & 31;
    const int64_t id = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (id >= p.n * per_row) return;
    const int64_t ch = id / per_row;
    const int g = (int)(id - ch * per_row), k0 = g * p.group, end = min(k0 + p.group, p.k);
    const T *w = (const T *)p.w + ch * p.stride;
    float scale = 1.0f;
    if constexpr (sizeof(T) > 1) {
        uint32_t most = 0;
        for (int j = k0 + lane; j < end; j += 32) most = max(most, __float_as_uint(to_f(w[j])) & 0x7FFFFFFFu);
        most = __reduce_max_sync(~0u, most);
        const float m = __uint_as_float(most);
        T s;
        from_f(m < INFINITY ? __fdiv_rn(m, 7.0f) : NAN, s);
        if (lane == 0 && g < p.groups) ((T *)p.scale)[ch * p.groups + g] = s;
        scale = to_f(s);
    }
    uint32_t *row = p.codes + ch * p.blocks * 16;
    const int words = min(k0 + p.group, p.blocks * 128) / 8;
    for (int at = k0 / 8 + lane; at < words; at += 32) {   // piece `at` of the row
        const int run = at >> 2, word = (run >> 2) * 16 + (at & 3) * 4 + (run & 3);
        uint32_t v = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int j = at * 8 + e;
            int q = 0;
            if (j < end) {
                if constexpr (sizeof(T) == 1) q = (int)w[j];
                else if (scale > 0.0f) q = min(max(__float2int_rn(__fdiv_rn(to_f(w[j]), scale)), -8), 7);
            }
            v |= ((uint32_t)(q + 8) & 15u) << field_of(e);
        }
        row[word] = v;
    }
}

template <typename T> cudaError_t launch_codes(const Codes &p, cudaStream_t st) {
    const int64_t warps = p.n * ((p.blocks * 128 + p.group - 1) / p.group);
    codes_kernel<T><<<(unsigned)((warps + 7) / 8), 256, 0, st>>>(p);
    return cudaGetLastError();
}

// ----------------------------------------------------------------------------------------------------- products

// A warp a channel and up to 8 rows; a lane takes a word at a time.
template <typename T> __global__ void __launch_bounds__(256) plain_kernel(const FourBit p) {
    const int lane = threadIdx.x & 31;
    const int64_t ch = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (ch >= p.n) return;
    const uint32_t *codes = (const uint32_t *)p.codes + ch * p.blocks * 16;
    for (int64_t m0 = (int64_t)blockIdx.y * 8; m0 < p.rows; m0 += (int64_t)gridDim.y * 8) {
        const int rows = (int)min((int64_t)8, p.rows - m0);
        float acc[8] = {};
        for (int word = lane; word < p.blocks * 16; word += 32) {
            const int k0 = first_of(word);
            if (k0 >= p.k) continue;
            const uint32_t v = codes[word];
            const float s = load_as(p.scale_dtype, p.scale, ch * p.groups + k0 / p.group);
#pragma unroll
            for (int r = 0; r < 8; r++) {
                if (r >= rows) break;
                const T *x = (const T *)p.x + (m0 + r) * p.x_stride;
                float sum = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (k0 + e < p.k) sum = fmaf(to_f(x[k0 + e]), (float)((int)(v >> field_of(e) & 15u) - 8), sum);
                acc[r] = fmaf(s, sum, acc[r]);
            }
        }
#pragma unroll
        for (int r = 0; r < 8; r++) {
            float sum = acc[r];
#pragma unroll
            for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
            if (lane == 0 && r < rows) store_as(p.out_dtype, p.out, (m0 + r) * p.out_stride + ch, sum + (p.bias ? p.bias[ch] : 0.0f));
        }
    }
}

template <typename T> cudaError_t launch_plain(const FourBit &p, cudaStream_t st) {
    plain_kernel<T><<<dim3((unsigned)((p.n + 7) / 8), (unsigned)std::min<int64_t>((p.rows + 7) / 8, 65535)), 256, 0, st>>>(p);
    return cudaGetLastError();
}

bool shape_ok(int64_t n, int64_t k, int64_t group) {
    return n >= 1 && n <= INT32_MAX && k >= 1 && group >= 32 && (group & (group - 1)) == 0;
}
int blocks_of(int64_t k) { return (int)((k + 127) / 128); }
int groups_of(int64_t k, int64_t group) { return (int)((k + group - 1) / group); }

}  // namespace

extern "C" {

int ygg_fourbit_quantize(int device, int dtype, int64_t n, int64_t k, int64_t group, const void *d_weight, int64_t row_stride,
                         uint8_t *d_codes, void *d_scale, void *stream) {
    if (!shape_ok(n, k, group)) return YGG_E_ARG;
    if (k > YGG_LINEAR_MAX_K || group > YGG_LINEAR_MAX_K) return YGG_E_UNSUPPORTED;
    if (!d_weight || !d_codes || !d_scale || ((uintptr_t)d_codes & 15)) return YGG_E_ARG;
    OnDevice on(device);
    if (!on.ok) return YGG_E_DEVICE;
    cudaError_t e = cudaSuccess;
    const int rc = by_type(dtype, [&](auto t) {
        e = launch_codes<decltype(t)>({d_weight, n, row_stride, (int)k, blocks_of(k), (int)group, groups_of(k, group),
                                       (uint32_t *)d_codes, d_scale}, (cudaStream_t)stream);
    });
    return rc != YGG_OK ? rc : e == cudaSuccess ? YGG_OK : YGG_E_CUDA;
}

int ygg_fourbit_pack(int device, int64_t n, int64_t k, const int8_t *d_in, int64_t row_stride, uint8_t *d_codes,
                     void *stream) {
    if (!shape_ok(n, k, 128)) return YGG_E_ARG;
    if (k > YGG_LINEAR_MAX_K) return YGG_E_UNSUPPORTED;
    if (!d_in || !d_codes || ((uintptr_t)d_codes & 15)) return YGG_E_ARG;
    OnDevice on(device);
    if (!on.ok) return YGG_E_DEVICE;
    return launch_codes<int8_t>({d_in, n, row_stride, (int)k, blocks_of(k), 128, blocks_of(k), (uint32_t *)d_codes, nullptr},
                                (cudaStream_t)stream) == cudaSuccess ? YGG_OK : YGG_E_CUDA;
}

int ygg_fourbit_linear(int device, int dtype, int64_t rows, int64_t k, int64_t n, int64_t group, const void *d_x,
                       int64_t row_stride, const uint8_t *d_codes, int scale_dtype, const void *d_scale,
                       const float *d_bias, int out_dtype, void *d_out, int64_t out_stride, void *stream) {
    if (rows < 0 || rows >= ((int64_t)1 << 40) || !shape_ok(n, k, group)) return YGG_E_ARG;
    if (k > YGG_LINEAR_MAX_K || group > YGG_LINEAR_MAX_K || out_dtype < YGG_DTYPE_FLOAT || out_dtype > YGG_DTYPE_BFLOAT ||
        scale_dtype < YGG_DTYPE_FLOAT || scale_dtype > YGG_DTYPE_BFLOAT)
        return YGG_E_UNSUPPORTED;
    if (rows == 0) return YGG_OK;
    if (!d_x || !d_codes || !d_scale || !d_out || ((uintptr_t)d_codes & 15)) return YGG_E_ARG;
    OnDevice on(device);
    if (!on.ok) return YGG_E_DEVICE;
    const FourBit p{d_x, rows, row_stride, n, (int)k, blocks_of(k), (int)group, groups_of(k, group), d_codes, scale_dtype,
                    d_scale, d_bias, out_dtype, d_out, out_stride};
    cudaError_t e = cudaSuccess;
    const int rc = by_type(dtype, [&](auto t) { e = launch_plain<decltype(t)>(p, (cudaStream_t)stream); });
    return rc != YGG_OK ? rc : e == cudaSuccess ? YGG_OK : YGG_E_CUDA;
}

}  // extern "C"
