// Linear layers in 8-bit integers: rows of activations quantised as they come, weights quantised once.
//
// Row m of x (K values) has the scale s_m = max|x_m| / 127 and the codes c = rint(x 127 / max|x_m|), in [-127, 127];
// a weight row n (one output channel) has codes w and its scale s_n. Then
//   y[m][n] = (sum_k c[m][k] w[n][k]) s_m s_n + b[n],
// (the channel's factor first: a row's scale may be near the end of the type's range, where only a result beyond it may
// overflow), with the sum exact in int32 (K <= 131072 keeps |sum| below 127 127 2^17 < 2^31), one rounding to float, one for
// the channel's factor, one for the row's factor and the bias together, and one to the output's type. Integer sums have no
// order: a row's results repeat bit for bit, alone or among others.
// A row of zeros (or one so small that 127 / max|x_m| is beyond the type's range: below 3.73e-37) has scale 0 and codes 0; a row
// that holds NaN or infinity has scale NaN and codes 0, so that its outputs are NaN.
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
// Magnitudes compare as the integers of their bits, with NaN above infinity above the numbers.
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// The largest magnitude of a vector; 16-bit types compare in pairs.
__device__ __forceinline__ uint32_t magnitude_of(const uint4 &q, float) {
    return max(max(q.x & 0x7FFFFFFFu, q.y & 0x7FFFFFFFu), max(q.z & 0x7FFFFFFFu, q.w & 0x7FFFFFFFu));
}
__device__ __forceinline__ uint32_t magnitude_16(const uint4 &q) {
    const uint32_t m = __vmaxu2(__vmaxu2(q.x & 0x7FFF7FFFu, q.y & 0x7FFF7FFFu), __vmaxu2(q.z & 0x7FFF7FFFu, q.w & 0x7FFF7FFFu));
    return max(m & 0xFFFFu, m >> 16);
}
__device__ __forceinline__ uint32_t magnitude_of(const uint4 &q, __half) {
    const uint32_t m = magnitude_16(q);
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
}
__device__ __forceinline__ uint32_t magnitude_of(const uint4 &q, __nv_bfloat16) { return magnitude_16(q) << 16; }

// A code is the low byte of the sum: the product rounds once, and adding 1.5 2^23 rounds it to the nearest integer, ties
// to even. |x| inverse is at most 127 (1 + 2^-22), so no code is beyond 127.
// The sums are single instructions on purpose: as a pair (add.rn.f32x2) after the paired product they came out as if
// fused with it, rounded once, and codes at halves went the other way.
__device__ __forceinline__ uint2 code2(float a, float b, float inverse) {
    float x, y;
    asm("{\n\t.reg .b64 v, f;\n\t"
        "mov.b64 v, {%2, %3};\n\tmov.b64 f, {%4, %4};\n\tmul.rn.f32x2 v, v, f;\n\tmov.b64 {%0, %1}, v;\n\t}"
        : "=f"(x), "=f"(y)
        : "f"(a), "f"(b), "f"(inverse));
    return make_uint2(__float_as_uint(__fadd_rn(x, 12582912.0f)), __float_as_uint(__fadd_rn(y, 12582912.0f)));
}
__device__ __forceinline__ uint32_t code4(float a, float b, float c, float d, float inverse) {
    const uint2 x = code2(a, b, inverse), y = code2(c, d, inverse);
    return __byte_perm(__byte_perm(x.x, x.y, 0x0040), __byte_perm(y.x, y.y, 0x0040), 0x5410);
}
__device__ __forceinline__ void store_codes(int8_t *p, const float (&v)[4], float inverse) {
    *(uint32_t *)p = inverse == 0.0f ? 0u : code4(v[0], v[1], v[2], v[3], inverse);
}
__device__ __forceinline__ void store_codes(int8_t *p, const float (&v)[8], float inverse) {
    *(uint2 *)p = inverse == 0.0f ? make_uint2(0, 0)
                                  : make_uint2(code4(v[0], v[1], v[2], v[3], inverse), code4(v[4], v[5], v[6], v[7], inverse));
}

// The output of a sum: one expression for all kernels, so that a row's outputs have the same bits however many rows go with
// it and however the product is cut. (Rounded apart, product and bias gave other last bits in one of four float32 outputs.)
__device__ __forceinline__ float value_of(int sum, float scale, float row_scale, float bias) {
    return fmaf(__int2float_rn(sum) * scale, row_scale, bias);
}

// THREADS threads a row (32: eight rows a block, or the whole block of 256), the row in registers as VECS vectors of 16
// bytes a thread. Rows on 16-byte boundaries; what lies past k in a row's last vector is not the row's. Bound by HBM: 8192
// x 4096 bf16 16 us, 6.3 TB/s read and written; small calls by the launch (1.7 us).
template <typename T, int THREADS, int VECS>
__global__ void __launch_bounds__(256) quantize_kernel(const Quantize p) {
    constexpr int N = kPer<T>;
    __shared__ uint32_t part[8];
    const int64_t row = THREADS == 32 ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
    const int t = threadIdx.x & (THREADS - 1);
    wait_for_previous();
    let_next_begin();   // not before the wait: a product may read its weights before its own wait, and whoever wrote them
                        // has to be done by then
    if (row >= p.rows) return;
    const T *x = (const T *)p.x + row * p.stride;
    uint4 q[VECS];
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < VECS; i++) {
        const int j = (i * THREADS + t) * N;
        q[i] = make_uint4(0, 0, 0, 0);
        if (j < p.k) q[i] = load_stream(x + j);
    }
#pragma unroll
    for (int i = 0; i < VECS; i++) {
        const int j = (i * THREADS + t) * N;
        if (j < p.k && j + N > p.k) {   // the vector that holds the row's end
            uint32_t *w = (uint32_t *)&q[i];
#pragma unroll
            for (int e = 0; e < N; e++)
                if (j + e >= p.k) w[e * 4 / N] &= N == 4 ? 0u : 0xFFFFu << (e & 1 ? 0 : 16);
        }
        most = max(most, magnitude_of(q[i], T()));
    }
    most = __reduce_max_sync(~0u, most);
    if (THREADS > 32) {
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; w++) most = max(most, part[w]);
    }
    const Factors f = factors(__uint_as_float(most));
    int8_t *codes = p.codes + row * p.code_stride;
#pragma unroll
    for (int i = 0; i < VECS; i++) {
        const int j = (i * THREADS + t) * N;
        if (j >= p.padded) continue;
        float v[N];
        unpack(q[i], v, T());
        store_codes(codes + j, v, f.inverse);
    }
    if (t == 0) p.scale[row] = f.scale;
}

// Any k and any alignment: the row is read twice.
template <typename T> __global__ void __launch_bounds__(256) quantize_any_kernel(const Quantize p) {
    __shared__ uint32_t part[8];
    wait_for_previous();
    let_next_begin();
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T *x = (const T *)p.x + row * p.stride;
        uint32_t most = 0;
#pragma unroll 8
        for (int j = threadIdx.x; j < p.k; j += 256) most = max(most, magnitude(to_f(x[j])));
        most = __reduce_max_sync(~0u, most);
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = most;
        __syncthreads();
        for (int w = 0; w < 8; w++) most = max(most, part[w]);
        __syncthreads();
        const Factors f = factors(__uint_as_float(most));
        int8_t *codes = p.codes + row * p.code_stride;
#pragma unroll 4
        for (int j = 4 * threadIdx.x; j < p.padded; j += 1024) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = j + e < p.k ? to_f(x[j + e]) : 0.0f;
            store_codes(codes + j, v, f.inverse);
        }
        if (threadIdx.x == 0) p.scale[row] = f.scale;
    }
}

template <typename T> cudaError_t launch_quantize(const Quantize &p, cudaStream_t st) {
    constexpr int N = kPer<T>;
    cudaError_t e;
    const auto launch = [&](void (*kernel)(const Quantize), unsigned grid) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(grid);
        cfg.blockDim = dim3(256);
        cfg.stream = st;
        cudaLaunchAttribute attr[1];   // it may begin under the launch before it
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        return cudaLaunchKernelEx(&cfg, kernel, p);
    };
    const bool even = ((uintptr_t)p.x & 15) == 0 && (p.rows == 1 || p.stride % N == 0);
    const int vecs = (p.k + N - 1) / N;
    if (!even || vecs > 2048 || p.rows > INT32_MAX) {
        e = launch(quantize_any_kernel<T>, (unsigned)std::min<int64_t>(p.rows, 8 * sm_count()));
    } else if (vecs <= 256 && p.rows >= 8 * sm_count()) {   // enough rows to fill the SMs with a warp each
        const unsigned grid = (unsigned)((p.rows + 7) / 8);
        if (vecs <= 32) e = launch(quantize_kernel<T, 32, 1>, grid);
        else if (vecs <= 64) e = launch(quantize_kernel<T, 32, 2>, grid);
        else if (vecs <= 128) e = launch(quantize_kernel<T, 32, 4>, grid);
        else e = launch(quantize_kernel<T, 32, 8>, grid);
    } else {
        const unsigned grid = (unsigned)p.rows;
        if (vecs <= 256) e = launch(quantize_kernel<T, 256, 1>, grid);
        else if (vecs <= 512) e = launch(quantize_kernel<T, 256, 2>, grid);
        else if (vecs <= 1024) e = launch(quantize_kernel<T, 256, 4>, grid);
        else e = launch(quantize_kernel<T, 256, 8>, grid);
    }
    return e;
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
// Large products are bound by the tensor cores: 8192 x 4096 x 16384 bf16 342 us, 0.98 of the rate of a burst (393 with one
// CTA a tile), fewer rows by the weights (64 x 4096 x 16384 14 us, 4.8 TB/s), a small K by the epilogue (4096 x 64 x 16384
// bf16 41.6 us, twice its floor; fp32 51, 1.2 times).
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
    alignas(16) float row_scale[kEpilogueWarps][256];   // each warp its own: no barrier among them
    uint32_t tmem;
};

constexpr int kBand = 8;   // channel blocks that share the rows of x while they are in L2

__device__ __forceinline__ void tile_at(const Tiles &p, int t, int &cb, int &rb) {
    const int band = kBand * p.row_blocks, first = t / band * kBand, left = min(kBand, p.channel_blocks - first);
    t %= band;
    cb = first + t % left;
    rb = t / left;
}

// (Rows staged in shared memory and written in whole lines were slower: 4096 x 64 x 16384 bf16 47 to 52 us, 41.6 so.)
// 16 sums of one channel, of the rows whose scales are rs[0..16) (16-byte aligned): row j goes to out + j stride.
template <typename T>
__device__ __forceinline__ void write_rows(const uint32_t (&v)[16], const float *rs, float sn, float bn, T *out,
                                           int64_t stride, int rows) {
    float4 f[4];
#pragma unroll
    for (int j = 0; j < 4; j++) f[j] = ((const float4 *)rs)[j];
    const float *r = (const float *)f;
    if (rows >= 16) {
#pragma unroll
        for (int j = 0; j < 16; j++, out += stride) from_f(value_of((int)v[j], sn, r[j], bn), *out);
    } else {
#pragma unroll
        for (int j = 0; j < 16; j++, out += stride)
            if (j < rows) from_f(value_of((int)v[j], sn, r[j], bn), *out);
    }
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
            wait_for_previous();   // the codes
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
        wait_for_previous();       // the rows' scales
        for (int t = first; t < tiles; t += step, it++) {
            int cb, rb;
            tile_at(p, t, cb, rb);
            const int acc = it & 1;
            const int64_t row0 = (int64_t)rb * p.tn, ch = (int64_t)(cb * CTAS + rank) * 128 + quad * 32 + lane;
            const int rows = (int)min((int64_t)p.tn, p.rows - row0);
            __syncwarp();
            for (int c = lane; c < p.tn; c += 32) rs[c] = c < rows ? p.row_scale[row0 + c] : 0.0f;
            const bool live = ch < p.n;
            const float sn = live ? p.scale[ch] : 0.0f, bn = live && p.bias ? p.bias[ch] : 0.0f;
            if (!(ok = __all_sync(~0u, mbar_wait_bounded(smem_addr(&sh.done[acc]), (it >> 1) & 1)))) break;
            tmem_fence_after();
            const uint32_t d = tmem + acc * (p.tmem_cols / 2) + ((uint32_t)(quad * 32) << 16);
            T *out = (T *)p.out + row0 * p.out_stride + ch;
            const int span = p.tn >= 64 ? 32 : 16;   // columns a turn; small tiles give each half of the warps some
            for (int c = half * span; c < p.tn; c += 2 * span) {
                uint32_t v[16], w[16];
                const bool two = span == 32 && c + 16 < p.tn;
                __syncwarp();
                tmem_load16(d + c, v);
                if (two) tmem_load16(d + c + 16, w);
                tmem_loaded();
                if (live) {
                    write_rows(v, rs + c, sn, bn, out + c * p.out_stride, p.out_stride, rows - c);
                    if (two) write_rows(w, rs + c + 16, sn, bn, out + (c + 16) * p.out_stride, p.out_stride, rows - c - 16);
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

// Few tiles: the K of a tile is cut among the CTAs of a cluster (CTAS 1, one tile a cluster). Each sums its part in
// tensor memory; then the columns go round in chunks of 16, chunk q to CTA q mod the cluster's size, through distributed
// shared memory (the rings, once every CTA's products are done), and each CTA adds up and writes its chunks. Integer sums:
// the result does not depend on the cut. 16 x 4096 x 4096: 8.0 us with four parts, 11.0 with one; bound by latency.
struct SplitShared {
    uint64_t full[kMaxStages], empty[kMaxStages], done;
    uint32_t tmem;
};

template <typename T>
__global__ void __launch_bounds__(kTcThreads, 1)
    split_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, const Tiles p,
                 int ring_bytes, int parts) {
    extern __shared__ __align__(1024) uint8_t ring[];
    SplitShared &sh = *(SplitShared *)(ring + ring_bytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = (int)cluster_rank();
    const int tile = blockIdx.x / parts, cb = tile % p.channel_blocks, rb = tile / p.channel_blocks;
    const int k0 = (int)((int64_t)p.k_blocks * part / parts), k1 = (int)((int64_t)p.k_blocks * (part + 1) / parts);
    const int stage_bytes = 128 * kStageK + p.tn * kStageK;
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; s++) {
            mbar_init(smem_addr(&sh.full[s]), 1);
            mbar_init(smem_addr(&sh.empty[s]), 1);
        }
        mbar_init(smem_addr(&sh.done), 1);
        fence_mbar_init();
    }
    if (warp == kEpilogueWarps) tmem_alloc<1>(smem_addr(&sh.tmem), p.tmem_cols);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = *(volatile uint32_t *)&sh.tmem;
    bool ok = true;
    if (warp == kEpilogueWarps) {
        if (lane == 0) {
            int s = 0;
            uint32_t phase = 1;
            wait_for_previous();
            for (int kb = k0; kb < k1; kb++) {
                if (!(ok = mbar_wait_bounded(smem_addr(&sh.empty[s]), phase))) break;
                const uint32_t bar = smem_addr(&sh.full[s]), at = smem_addr(ring + s * stage_bytes);
                mbar_expect_tx(bar, stage_bytes);
                tma_load<1>(at, &wmap, kb * kStageK, cb * 128, bar);
                tma_load<1>(at + 128 * kStageK, &xmap, kb * kStageK, rb * p.tn, bar);
                if (++s == p.stages) s = 0, phase ^= 1;
            }
        }
    } else if (warp == kEpilogueWarps + 1) {
        if (lane == 0) {
            const uint32_t shape = product_s8(128, p.tn);
            int s = 0;
            uint32_t phase = 0;
            for (int kb = k0; kb < k1; kb++) {
                if (!(ok = mbar_wait_bounded(smem_addr(&sh.full[s]), phase))) break;
                tmem_fence_after();
                const uint32_t at = smem_addr(ring + s * stage_bytes);
                const uint64_t a = operand_128b(at), b = operand_128b(at + 128 * kStageK);
#pragma unroll
                for (int j = 0; j < kStageK / 32; j++) mma_s8<1>(tmem, a + 2 * j, b + 2 * j, shape, kb > k0 || j > 0);
                mma_commit<1>(smem_addr(&sh.empty[s]));
                if (++s == p.stages) s = 0, phase ^= 1;
            }
            if (ok) mma_commit<1>(smem_addr(&sh.done));
        }
    } else {
        wait_for_previous();
        ok = __all_sync(~0u, mbar_wait_bounded(smem_addr(&sh.done), 0));
        tmem_fence_after();
    }
    __syncwarp();
    cluster_sync();   // every ring is free
    const int quad = warp & 3, half = warp >> 2, chunks = p.tn / 16;
    const uint32_t mine = smem_addr(ring);
    if (warp < kEpilogueWarps) {
        for (int q = half; q < chunks; q += 2) {
            uint32_t v[16];
            tmem_load16(tmem + q * 16 + ((uint32_t)(quad * 32) << 16), v);
            tmem_loaded();
            const uint32_t to = at_rank(mine + ((q / parts) * parts + part) * 8192 + (quad * 32 + lane) * 4, q % parts);
#pragma unroll
            for (int j = 0; j < 16; j++)
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to + j * 512), "r"(v[j]) : "memory");
        }
    }
    tmem_fence_before();
    __syncwarp();
    cluster_sync();
    if (warp < kEpilogueWarps && ok) {
        const int64_t row0 = (int64_t)rb * p.tn, ch = (int64_t)cb * 128 + quad * 32 + lane;
        const bool live = ch < p.n;
        const float sn = live ? p.scale[ch] : 0.0f, bn = live && p.bias ? p.bias[ch] : 0.0f;
        T *out = (T *)p.out + row0 * p.out_stride + ch;
        const int rows = (int)min((int64_t)p.tn, p.rows - row0);
        for (int q = part; q < chunks && live; q += parts) {
            const int *from = (const int *)(ring + (q / parts) * parts * 8192) + quad * 32 + lane;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int c = half * 8 + j, r = q * 16 + c;
                if (r >= rows) break;
                int sum = 0;
                for (int i = 0; i < parts; i++) sum += from[i * 2048 + c * 128];
                from_f(value_of(sum, sn, p.row_scale[row0 + r], bn), out[(int64_t)r * p.out_stride]);
            }
        }
    }
    if (!ok) {
        *(volatile int *)&g_fault = 1;
        const long long t0 = clock64();
        while (clock64() - t0 < 50000000LL) {}
    }
    __syncwarp();
    __syncthreads();
    if (warp == kEpilogueWarps) tmem_free<1>(tmem, p.tmem_cols);
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

// The launch attributes of the tensor-core kernels: a cluster, and leave to begin under the launch before it.
struct Launch {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[2];
    Launch(int64_t blocks, int cluster, size_t smem, cudaStream_t st) {
        cfg.gridDim = dim3((unsigned)blocks);
        cfg.blockDim = dim3(kTcThreads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = st;
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = cluster;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
    }
};

Tiles tiles_of(const Linear &q, int ctas, int tn, int accumulators) {
    Tiles p{q.rows, q.n, (q.k + kStageK - 1) / kStageK, tn, 0, (int)((q.n + 128 * ctas - 1) / (128 * ctas)),
            (int)((q.rows + tn - 1) / tn), 32, q.row_scale, q.scale, q.bias, q.out, q.out_stride};
    while (p.tmem_cols < accumulators * tn) p.tmem_cols *= 2;
    return p;
}

template <int CTAS, typename T> int launch_tc(const Linear &q, int tn, cudaStream_t st) {
    static SmemLimits limits;
    const size_t smem = kRing + sizeof(TcShared);
    Tiles p = tiles_of(q, CTAS, tn, 2);
    p.stages = std::min(kMaxStages, kRing / ((128 + tn / CTAS) * kStageK));
    CUtensorMap wmap, xmap;
    if (!map_rows(&wmap, q.weight, q.n, q.weight_stride, q.k, 128) ||
        !map_rows(&xmap, q.codes, q.rows, q.code_stride, q.k, tn / CTAS) ||
        raise_smem_limit((const void *)tc_kernel<CTAS, T>, smem, limits) != cudaSuccess)
        return YGG_E_CUDA;
    const int64_t tiles = (int64_t)p.channel_blocks * p.row_blocks;
    Launch l(std::min<int64_t>(tiles, sm_count() / CTAS) * CTAS, CTAS, smem, st);
    return cudaLaunchKernelEx(&l.cfg, tc_kernel<CTAS, T>, wmap, xmap, p) == cudaSuccess ? YGG_OK : YGG_E_CUDA;
}

template <typename T> int launch_split(const Linear &q, int tn, int parts, cudaStream_t st) {
    static SmemLimits limits;
    Tiles p = tiles_of(q, 1, tn, 1);
    const int stage = (128 + tn) * kStageK, k_blocks = (p.k_blocks + parts - 1) / parts;
    // two CTAs an SM where a few stages fit half of its shared memory, else the whole ring
    p.stages = std::min(std::min(kMaxStages, k_blocks), (tn <= 128 ? kRing / 2 : kRing) / stage);
    const int chunks = (tn / 16 + parts - 1) / parts, ring = std::max(p.stages * stage, chunks * parts * 8192);
    const size_t smem = ring + sizeof(SplitShared);
    CUtensorMap wmap, xmap;
    if (!map_rows(&wmap, q.weight, q.n, q.weight_stride, q.k, 128) ||
        !map_rows(&xmap, q.codes, q.rows, q.code_stride, q.k, tn) ||
        raise_smem_limit((const void *)split_kernel<T>, smem, limits) != cudaSuccess)
        return YGG_E_CUDA;
    Launch l((int64_t)p.channel_blocks * p.row_blocks * parts, parts, smem, st);
    return cudaLaunchKernelEx(&l.cfg, split_kernel<T>, wmap, xmap, p, ring, parts) == cudaSuccess ? YGG_OK : YGG_E_CUDA;
}

// ---------------------------------------------------------------------------------------------------- few rows
//
// Up to 4 rows (from 5 on the tensor cores are faster: 5 x 4096 x 32768 in 26.3 us there, 27.8 us here; 4 rows in 26.6 and
// 25.0): the weights are read once and nothing else counts. A warp (or `split` warps, each a part of K) takes two
// channels at a time, 2048 bytes of each; the codes of the rows lie in shared memory. Short rows before few weights are
// quantised by every block itself, under its first loads.
constexpr int kFewRows = 4, kFewBlock = 2048;

struct Few {
    Linear q;
    const void *x;          // what to quantise, or null: q.codes
    int64_t x_stride;
    int out_dtype, split, k_room;   // k_room: bytes of a row in shared memory, a multiple of kFewBlock
    bool early;             // the weights may be read before the launch before this one ends
};

struct FewLoad { uint4 w[2][4]; };

__device__ __forceinline__ void few_load(FewLoad &l, const Linear &q, int64_t ch, int kb, int lane) {
#pragma unroll
    for (int c = 0; c < 2; c++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int at = kb * kFewBlock + i * 512 + lane * 16;
            l.w[c][i] = make_uint4(0, 0, 0, 0);
            if (at < q.k && ch + c < q.n) l.w[c][i] = load_stream(q.weight + (ch + c) * q.weight_stride + at);
        }
}

__device__ __forceinline__ void store_as(int dtype, void *out, int64_t at, float v) {
    if (dtype == YGG_DTYPE_FLOAT) ((float *)out)[at] = v;
    else if (dtype == YGG_DTYPE_HALF) ((__half *)out)[at] = __float2half_rn(v);
    else ((__nv_bfloat16 *)out)[at] = __float2bfloat16_rn(v);
}

// Blocks an SM. A warp has 4 KB of weights on their way while it sums nothing, so that the SM's warps cover for each other:
// 1 x 4096 x 32768 in 22.9 us with four blocks, 23.9 with two whose warps load the next 4 KB while they sum.
template <int ROWS> constexpr int kFewBlocks = ROWS < 4 ? 4 : 3;

// X: the type of the rows to quantise, or int8_t: codes.
template <typename X, int ROWS> __global__ void __launch_bounds__(256, kFewBlocks<ROWS>) few_kernel(const Few p) {
    extern __shared__ __align__(16) uint8_t room[];   // [ROWS][k_room] codes
    __shared__ uint32_t most[ROWS][8];
    __shared__ float row_scale[ROWS];
    __shared__ int sums[2][8][2 * ROWS];
    const Linear &q = p.q;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rows = (int)q.rows;
    const int teams = 8 / p.split, team = warp / p.split, part = warp - team * p.split;
    const int64_t groups = (q.n + 1) / 2, all = (int64_t)gridDim.x * teams, id = (int64_t)blockIdx.x * teams + team;
    const int64_t g0 = groups * id / all, g1 = groups * (id + 1) / all;
    const int blocks = p.k_room / kFewBlock;
    FewLoad cur;
    if (!p.early) wait_for_previous();
    if (g0 < g1) few_load(cur, q, 2 * g0, part, lane);
    if constexpr (sizeof(X) > 1) {
        const X *x = (const X *)p.x;
        for (int r = 0; r < rows; r++) {
            uint32_t m = 0;
#pragma unroll 4
            for (int j = threadIdx.x; j < q.k; j += 256) m = max(m, magnitude(to_f(x[r * p.x_stride + j])));
            m = __reduce_max_sync(~0u, m);
            if (lane == 0) most[r][warp] = m;
        }
        __syncthreads();
        for (int r = 0; r < rows; r++) {
            uint32_t m = 0;
            for (int w = 0; w < 8; w++) m = max(m, most[r][w]);
            const Factors f = factors(__uint_as_float(m));
            if (threadIdx.x == 0) row_scale[r] = f.scale;
#pragma unroll 2
            for (int j = 4 * threadIdx.x; j < p.k_room; j += 1024) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = j + e < q.k ? to_f(x[r * p.x_stride + j + e]) : 0.0f;
                store_codes((int8_t *)room + r * p.k_room + j, v, f.inverse);
            }
        }
    } else {
        if (p.early) wait_for_previous();
        for (int i = threadIdx.x; i < rows * (p.k_room / 16); i += 256) {
            const int r = i / (p.k_room / 16), at = (i - r * (p.k_room / 16)) * 16;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (at < q.k) v = *(const uint4 *)(q.codes + r * q.code_stride + at);
            if (at + 16 > q.k) {   // bytes past k are not the row's
                uint32_t *w = (uint32_t *)&v;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int left = q.k - at - 4 * e;
                    if (left < 4) w[e] = left <= 0 ? 0u : w[e] & ((1u << (8 * left)) - 1);
                }
            }
            *(uint4 *)(room + r * p.k_room + at) = v;
        }
        if (threadIdx.x < rows) row_scale[threadIdx.x] = q.row_scale[threadIdx.x];
    }
    __syncthreads();
    int turn = 0;
    for (int64_t g = g0; g < g1; g++, turn ^= 1) {
        int acc[2][ROWS] = {};
        for (int kb = part; kb < blocks; kb += p.split) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint8_t *at = room + kb * kFewBlock + i * 512 + lane * 16;
#pragma unroll
                for (int r = 0; r < ROWS; r++) {
                    if (r >= rows) break;
                    const uint4 c = *(const uint4 *)(at + r * p.k_room);
#pragma unroll
                    for (int ch = 0; ch < 2; ch++) acc[ch][r] = dot16(cur.w[ch][i], c, acc[ch][r]);
                }
            }
            if (kb + p.split < blocks) few_load(cur, q, 2 * g, kb + p.split, lane);
            else if (g + 1 < g1) few_load(cur, q, 2 * (g + 1), part, lane);
        }
        int mine = 0;   // lane ch ROWS + r keeps the sum of channel ch and row r
#pragma unroll
        for (int ch = 0; ch < 2; ch++)
#pragma unroll
            for (int r = 0; r < ROWS; r++) {
                const int sum = __reduce_add_sync(~0u, acc[ch][r]);
                if (lane == ch * ROWS + r) mine = sum;
            }
        if (p.split > 1) {
            if (lane < 2 * ROWS) sums[turn][warp][lane] = mine;
            asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(p.split * 32) : "memory");
            if (part) continue;
            mine = 0;
            if (lane < 2 * ROWS)
                for (int w = 0; w < p.split; w++) mine += sums[turn][warp + w][lane];
        }
        const int64_t ch = 2 * g + lane / ROWS;
        const int r = lane % ROWS;
        if (lane < 2 * ROWS && r < rows && ch < q.n) {
            store_as(p.out_dtype, q.out, r * q.out_stride + ch,
                     value_of(mine, q.scale[ch], row_scale[r], q.bias ? q.bias[ch] : 0.0f));
        }
    }
}

int few_room(int k) { return (k + kFewBlock - 1) / kFewBlock * kFewBlock; }
bool is_few(int64_t rows, int k) { return rows <= kFewRows && rows * few_room(k) <= 192 * 1024; }

template <typename X, int ROWS> cudaError_t launch_few_rows(Few p, cudaStream_t st) {
    static SmemLimits limits;
    const size_t smem = (size_t)p.q.rows * p.k_room;
    cudaError_t e = raise_smem_limit((const void *)few_kernel<X, ROWS>, smem, limits);
    if (e != cudaSuccess) return e;
    const int64_t groups = (p.q.n + 1) / 2, fit = (int64_t)kFewBlocks<ROWS> * sm_count();
    const int blocks = p.k_room / kFewBlock;
    p.split = 1;
    while (p.split < 8 && 2 * p.split <= blocks && 2 * p.split * groups <= 8 * fit) p.split *= 2;
    Launch l(std::min<int64_t>((groups * p.split + 7) / 8, fit), 1, smem, st);
    l.cfg.blockDim = dim3(256);
    if (sizeof(X) > 1) l.cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&l.cfg, few_kernel<X, ROWS>, p);
}

template <typename X> int launch_few(const Few &p, cudaStream_t st) {
    const int64_t rows = p.q.rows;
    const cudaError_t e = rows == 1 ? launch_few_rows<X, 1>(p, st) : rows == 2 ? launch_few_rows<X, 2>(p, st)
                                                                               : launch_few_rows<X, 4>(p, st);
    return e == cudaSuccess ? YGG_OK : YGG_E_CUDA;
}

int padded_of(int64_t k) { return (int)((k + 15) / 16 * 16); }

bool rows_ok(int64_t rows, int64_t k) { return rows >= 0 && rows < ((int64_t)1 << 40) && k >= 1; }

int quantize(int dtype, const Quantize &p, cudaStream_t st) {
    cudaError_t e = cudaSuccess;
    const int rc = by_type(dtype, [&](auto t) { e = launch_quantize<decltype(t)>(p, st); });
    return rc != YGG_OK ? rc : e == cudaSuccess ? YGG_OK : YGG_E_CUDA;
}

// How a product is cut: CTAs a product, rows a tile, CTAs that share the K of a tile. The least of what the cuts are
// expected to take, in ns, by a model fitted to sweeps on a B200 (us, measured):
//   a launch costs 2500; 128 bytes of K of a tile 240, or its bytes at 115 a ns where those take longer (a pair of
//   256 x 256: 410, bound by the tensor cores); the epilogue 550 and 9 a column (a pair 3600), under the next tile's
//   products.
//   512 x 4096 x 4096: tn 128 12.1, 256 15.6; 1024 x 4096 x 4096: tn 256 16.0, 128 20.5;
//   8192 x 4096 x 16384: pair 342, one CTA 393; 4096 x 64 x 16384: tn 256 42.1, 128 49.7, 32 105.9, pair 51.2.
//   Sharing K costs 1650 and 16 a column more: 16 x 4096 x 4096 8.0 with 4 parts, 11.0 with one; 512 x 1024 x 4096
//   (tn 256) 15.5 with two, 7.2 with one.
struct Shape { int ctas, tn, parts; };
Shape shape_for(int64_t rows, int64_t n, int k) {
    const int64_t sms = sm_count(), k_blocks = (k + kStageK - 1) / kStageK, channel_blocks = (n + 127) / 128;
    Shape best{1, 16, 1};
    int64_t least = INT64_MAX;
    auto consider = [&](int ctas, int tn, int parts) {
        const int64_t tiles = (channel_blocks + ctas - 1) / ctas * ((rows + tn - 1) / tn);
        if (parts > 1 && tiles * parts > sms) return;
        const int64_t waves = (tiles * ctas * parts + sms - 1) / sms;
        const int64_t block = ctas == 2 ? 410 : std::max(240, (128 + tn) * kStageK / 115);
        const int64_t epilogue = ctas == 2 ? 3600 : 550 + 9 * tn;
        int64_t t = 2500 + (k_blocks + parts - 1) / parts * block + epilogue + (parts > 1 ? 1650 + 16 * tn : 0);
        t += (waves - 1) * std::max(k_blocks * block, epilogue);
        if (t < least) {
            least = t;
            best = {ctas, tn, parts};
        }
    };
    const int64_t row_blocks = (rows + 255) / 256;
    const int even = (int)((rows + row_blocks - 1) / row_blocks + 15) / 16 * 16;   // the rows in equal tiles
    for (const int tn : {even, 16, 32, 64, 128, 256})
        if (tn == even || tn < even || rows > 256)
            for (int parts = 1; parts <= 8 && parts <= k_blocks; parts *= 2) consider(1, tn, parts);
    if (rows > 256) consider(2, 256, 1);
    return best;
}

// early: the launch before this one wrote the codes and nothing else that the product reads.
int linear(int out_dtype, const Linear &p, bool early, cudaStream_t st) {
    if (is_few(p.rows, p.k)) return launch_few<int8_t>({p, nullptr, 0, out_dtype, 1, few_room(p.k), early}, st);
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
            const Shape s = shape_for(q.rows, q.n, q.k);
            done = s.ctas == 2    ? launch_tc<2, T>(q, s.tn, st)
                   : s.parts == 1 ? launch_tc<1, T>(q, s.tn, st)
                                  : launch_split<T>(q, s.tn, s.parts, st);
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
    if (k > YGG_LINEAR_MAX_K || out_dtype < YGG_DTYPE_FLOAT || out_dtype > YGG_DTYPE_BFLOAT) return YGG_E_UNSUPPORTED;
    if (rows == 0) return YGG_OK;
    if (!d_codes || !d_row_scale || !d_weight || !d_scale || !d_out || !aligned16(d_codes, code_stride) ||
        !aligned16(d_weight, weight_stride) || code_stride < k || weight_stride < k)
        return YGG_E_ARG;
    OnDevice on(device);
    if (!on.ok) return YGG_E_DEVICE;
    const int rc = linear(out_dtype, {d_codes, d_weight, code_stride, weight_stride, d_row_scale, d_scale, d_bias, rows,
                                      n, (int)k, d_out, out_stride}, false, (cudaStream_t)stream);
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
    if (k > YGG_LINEAR_MAX_K || out_dtype < YGG_DTYPE_FLOAT || out_dtype > YGG_DTYPE_BFLOAT) return YGG_E_UNSUPPORTED;
    if (rows == 0) return YGG_OK;
    if (!d_workspace || ((uintptr_t)d_workspace & 15) || workspace_bytes < ygg_linear_workspace(rows, k)) return YGG_E_ARG;
    if (!d_x || !d_weight || !d_scale || !d_out || !aligned16(d_weight, weight_stride) || weight_stride < k)
        return YGG_E_ARG;
    OnDevice on(device);
    if (!on.ok) return YGG_E_DEVICE;
    const cudaStream_t st = (cudaStream_t)stream;
    const int64_t padded = padded_of(k);
    int8_t *codes = (int8_t *)d_workspace;
    float *scale = (float *)(codes + rows * padded);
    const Linear q{codes, d_weight, padded, weight_stride, scale, d_scale, d_bias, rows, n, (int)k, d_out, out_stride};
    int rc;
    // one launch: 1 x 1280 x 256 in 3.7 us against 4.1, 1 x 4096 x 4096 in 6.7 against 6.4 but 3 us less on the host, which
    // larger weights would hide (1 x 4096 x 32768: 24.5 against 24.1)
    if (rows * k <= 4096 && n * k <= (1 << 25) && is_few(rows, (int)k)) {
        int done = YGG_OK;
        rc = by_type(dtype, [&](auto t) {
            done = launch_few<decltype(t)>({q, d_x, row_stride, out_dtype, 1, few_room((int)k), true}, st);
        });
        if (rc == YGG_OK) rc = done;
    } else {
        rc = quantize(dtype, {d_x, rows, row_stride, (int)k, (int)padded, codes, padded, scale}, st);
        if (rc == YGG_OK) rc = linear(out_dtype, q, true, st);
    }
    return rc != YGG_OK ? rc : cudaGetLastError() == cudaSuccess ? YGG_OK : YGG_E_CUDA;
}

}  // extern "C"
