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
#include "ygg_tensor.cuh"

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

// ---------------------------------------------------------------------------------------------------- tensor cores
//
// D[channel][row] = W C^T on tcgen05 (kind::i8): channels along M (128 lanes of tensor memory a CTA, 256 for a pair),
// rows of x along N. A thread of the epilogue then holds one channel, and the 32 lanes of a warp store 32 channels of a
// row side by side. Both operands are K-major, so TMA brings 128 bytes of K for each row and channel as they lie in
// memory, swizzled; it fills with zeros what is past k, the rows or the channels.
//
// A block is persistent over tiles: one warp issues the copies into a ring of stages, one the products, eight read the
// accumulators (two, so that a tile's epilogue runs under the next one's products). In a pair each CTA holds its own 128
// channels and half of the rows of x; the leader issues the products of both.
//
// Every wait is bounded: one that runs out raises the library's fault word (ygg_linear_status), gives its copies in
// flight time to land and leaves.

constexpr int kMaxStages = 12, kStageK = 128, kRing = 192 * 1024;
constexpr int kEpilogueWarps = 8, kTcThreads = (kEpilogueWarps + 2) * 32;

__device__ int g_fault;   // a bounded wait ran out

struct Tiles {
    int64_t rows, n;
    int k_blocks, tn, stages, channel_blocks, row_blocks, tmem_cols;
    const float *row_scale, *scale, *bias;
    void *out;
    int64_t out_stride;
};

struct TcShared {   // at the end of dynamic shared memory
    uint64_t full[kMaxStages], empty[kMaxStages], done[2], drained[2];
    float row_scale[kEpilogueWarps][256];   // each warp its own: no barrier among them
    uint32_t tmem;
};

constexpr int kBand = 8;   // channel blocks that share the rows of x while they are in L2

__device__ __forceinline__ void tile_at(const Tiles &p, int t, int &cb, int &rb) {
    const int band = kBand * p.row_blocks, first = t / band * kBand, left = min(kBand, p.channel_blocks - first);
    t %= band;
    cb = first + t % left;
    rb = t / left;
}

template <int CTAS, typename T>
__global__ void __launch_bounds__(kTcThreads, 1)
    tc_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, const Tiles p) {
    extern __shared__ __align__(1024) uint8_t ring[];
    TcShared &sh = *(TcShared *)(ring + kRing);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = CTAS == 2 ? cluster_rank() : 0;
    const int tiles = p.channel_blocks * p.row_blocks, first = blockIdx.x / CTAS, step = gridDim.x / CTAS;
    const int x_rows = p.tn / CTAS, stage_bytes = 128 * kStageK + x_rows * kStageK;
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; s++) {
            mbar_init(smem_addr(&sh.full[s]), 1);
            mbar_init(smem_addr(&sh.empty[s]), 1);
        }
        for (int s = 0; s < 2; s++) {
            mbar_init(smem_addr(&sh.done[s]), 1);
            mbar_init(smem_addr(&sh.drained[s]), CTAS * kEpilogueWarps);
        }
        fence_mbar_init();
    }
    if (warp == kEpilogueWarps) tmem_alloc<CTAS>(smem_addr(&sh.tmem), p.tmem_cols);
    tmem_fence_before();
    __syncthreads();
    if (CTAS == 2) cluster_sync();
    tmem_fence_after();
    const uint32_t tmem = *(volatile uint32_t *)&sh.tmem;
    bool ok = true;

    if (warp == kEpilogueWarps) {          // copies
        if (lane == 0) {
            int s = 0;
            uint32_t phase = 1;
            for (int t = first; t < tiles && ok; t += step) {
                int cb, rb;
                tile_at(p, t, cb, rb);
                const int ch = (cb * CTAS + rank) * 128, row = rb * p.tn + rank * x_rows;
                for (int kb = 0; kb < p.k_blocks; kb++) {
                    if (!(ok = mbar_wait_bounded(smem_addr(&sh.empty[s]), phase))) break;
                    uint32_t bar = smem_addr(&sh.full[s]);
                    if (rank == 0) mbar_expect_tx(bar, CTAS * stage_bytes);
                    if (CTAS == 2) bar = at_rank(bar, 0);
                    const uint32_t a = smem_addr(ring + s * stage_bytes);
                    tma_load<CTAS>(a, &wmap, kb * kStageK, ch, bar);
                    tma_load<CTAS>(a + 128 * kStageK, &xmap, kb * kStageK, row, bar);
                    if (++s == p.stages) s = 0, phase ^= 1;
                }
            }
        }
    } else if (warp == kEpilogueWarps + 1) {   // products
        if (lane == 0 && rank == 0) {
            const uint32_t shape = product_s8(128 * CTAS, p.tn);
            int s = 0, it = 0;
            uint32_t phase = 0;
            for (int t = first; t < tiles && ok; t += step, it++) {
                const int acc = it & 1;
                if (!(ok = mbar_wait_bounded(smem_addr(&sh.drained[acc]), ((it >> 1) & 1) ^ 1))) break;
                tmem_fence_after();
                const uint32_t d = tmem + acc * (p.tmem_cols / 2);
                for (int kb = 0; kb < p.k_blocks; kb++) {
                    if (!(ok = mbar_wait_bounded(smem_addr(&sh.full[s]), phase))) break;
                    tmem_fence_after();
                    const uint32_t at = smem_addr(ring + s * stage_bytes);
                    const uint64_t a = operand_128b(at), b = operand_128b(at + 128 * kStageK);
#pragma unroll
                    for (int j = 0; j < kStageK / 32; j++) mma_s8<CTAS>(d, a + 2 * j, b + 2 * j, shape, kb > 0 || j > 0);
                    mma_commit<CTAS>(smem_addr(&sh.empty[s]));
                    if (++s == p.stages) s = 0, phase ^= 1;
                }
                if (ok) mma_commit<CTAS>(smem_addr(&sh.done[acc]));
            }
        }
    } else {                               // epilogue
        const int quad = warp & 3, half = warp >> 2;
        float *rs = sh.row_scale[warp];
        int it = 0;
        for (int t = first; t < tiles; t += step, it++) {
            int cb, rb;
            tile_at(p, t, cb, rb);
            const int acc = it & 1;
            const int64_t row0 = (int64_t)rb * p.tn, ch = (int64_t)(cb * CTAS + rank) * 128 + quad * 32 + lane;
            const int rows = (int)min((int64_t)p.tn, p.rows - row0);
            __syncwarp();
            for (int c = lane; c < rows; c += 32) rs[c] = p.row_scale[row0 + c];
            const bool live = ch < p.n;
            const float sn = live ? p.scale[ch] : 0.0f, bn = live && p.bias ? p.bias[ch] : 0.0f;
            if (!(ok = __all_sync(~0u, mbar_wait_bounded(smem_addr(&sh.done[acc]), (it >> 1) & 1)))) break;
            tmem_fence_after();
            const uint32_t d = tmem + acc * (p.tmem_cols / 2) + ((uint32_t)(quad * 32) << 16);
            T *out = (T *)p.out + row0 * p.out_stride + ch;
            for (int c = half * 16; c < p.tn; c += 32) {
                uint32_t v[16];
                __syncwarp();
                tmem_load16(d + c, v);
                tmem_loaded();
                if (live) {
#pragma unroll
                    for (int j = 0; j < 16; j++)
                        if (c + j < rows) {
                            const float y = __int2float_rn((int)v[j]) * sn * rs[c + j];
                            from_f(p.bias ? y + bn : y, out[(int64_t)(c + j) * p.out_stride]);
                        }
                }
            }
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) {
                const uint32_t bar = smem_addr(&sh.drained[acc]);
                if (CTAS == 2) mbar_arrive_cluster(at_rank(bar, 0));
                else mbar_arrive(bar);
            }
        }
    }
    if (!ok) {
        *(volatile int *)&g_fault = 1;
        const long long t0 = clock64();
        while (clock64() - t0 < 50000000LL) {}
    }
    __syncwarp();
    tmem_fence_before();
    __syncthreads();
    if (CTAS == 2) cluster_sync();
    if (warp == kEpilogueWarps) tmem_free<CTAS>(tmem, p.tmem_cols);
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            f = nullptr;
        return (EncodeTiled)f;
    }();
    return fn;
}

// Rows of k bytes, `stride` apart, in tiles of 128 bytes by `box` rows.
bool map_rows(CUtensorMap *map, const int8_t *base, int64_t rows, int64_t stride, int k, int box) {
    const EncodeTiled encode = encode_tiled();
    if (!encode) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride};
    const cuuint32_t tile[2] = {kStageK, (cuuint32_t)box}, steps[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void *)base, dims, strides, tile, steps,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int CTAS, typename T> int launch_tc(const Linear &q, int tn, cudaStream_t st) {
    static SmemLimits limits;
    const size_t smem = kRing + sizeof(TcShared);
    Tiles p{q.rows, q.n, (q.k + kStageK - 1) / kStageK, tn, 0, (int)((q.n + 128 * CTAS - 1) / (128 * CTAS)),
            (int)((q.rows + tn - 1) / tn), 32, q.row_scale, q.scale, q.bias, q.out, q.out_stride};
    p.stages = std::min(kMaxStages, kRing / ((128 + tn / CTAS) * kStageK));
    while (p.tmem_cols < 2 * tn) p.tmem_cols *= 2;
    CUtensorMap wmap, xmap;
    if (!map_rows(&wmap, q.weight, q.n, q.weight_stride, q.k, 128) ||
        !map_rows(&xmap, q.codes, q.rows, q.code_stride, q.k, tn / CTAS) ||
        raise_smem_limit((const void *)tc_kernel<CTAS, T>, smem, limits) != cudaSuccess)
        return YGG_E_CUDA;
    const int64_t tiles = (int64_t)p.channel_blocks * p.row_blocks;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)std::min<int64_t>(tiles, sm_count() / CTAS) * CTAS);
    cfg.blockDim = dim3(kTcThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CTAS;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, tc_kernel<CTAS, T>, wmap, xmap, p) == cudaSuccess ? YGG_OK : YGG_E_CUDA;
}

int padded_of(int64_t k) { return (int)((k + 15) / 16 * 16); }

bool rows_ok(int64_t rows, int64_t k) { return rows >= 0 && rows < ((int64_t)1 << 40) && k >= 1; }

int quantize(int dtype, const Quantize &p, cudaStream_t st) {
    const int grid = (int)std::min<int64_t>(p.rows, 148 * 8);
    return by_type(dtype, [&](auto t) { quantize_kernel<decltype(t)><<<grid, 256, 0, st>>>(p); });
}

int linear(int out_dtype, const Linear &p, cudaStream_t st) {
    const int64_t step = (int64_t)1 << 24;   // rows a launch counts its tiles over
    for (int64_t m = 0; m < p.rows; m += step) {
        Linear q = p;
        q.rows = std::min(step, p.rows - m);
        q.codes += m * p.code_stride;
        q.row_scale += m;
        q.out = (char *)p.out + m * p.out_stride * (out_dtype == YGG_DTYPE_FLOAT ? 4 : 2);
        int done = YGG_OK;
        const int rc = by_type(out_dtype, [&](auto t) {
            using T = decltype(t);
            if (q.rows > 256) done = launch_tc<2, T>(q, 256, st);
            else done = launch_tc<1, T>(q, (int)(q.rows + 15) / 16 * 16, st);
        });
        if (rc != YGG_OK) return rc;
        if (done != YGG_OK) return done;
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

int ygg_linear_status(int device, void *stream, int *status_out) {
    if (!status_out) return YGG_E_ARG;
    OnDevice on(device);
    if (!on.ok) return YGG_E_DEVICE;
    int v = 0;
    const int none = 0;
    const cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e = cudaMemcpyFromSymbolAsync(&v, g_fault, sizeof v, 0, cudaMemcpyDeviceToHost, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e == cudaSuccess && v) e = cudaMemcpyToSymbolAsync(g_fault, &none, sizeof none, 0, cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e != cudaSuccess) return YGG_E_CUDA;
    *status_out = v ? YGG_E_TIMEOUT : YGG_OK;
    return YGG_OK;
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
