// The choice over beams and vocabulary, and the rows of a batch in its order.
//
// A prompt has H beams, each with a score and V logits. With lse_b = log sum_v e^(x_bv), the continuation of beam b by v is
// worth score_b + (x_bv - lse_b), in 64 bits; the best W of the H V continuations go on, ties by the lower b V + v. A beam
// that is done goes on with the token `end` alone, at no cost: the others are worth -inf, and a pick among them writes `end`
// too. -inf logits are worth -inf, a row of -inf alone is worth -inf everywhere; a row that holds NaN or +inf is worth NaN
// everywhere. NaN ranks as -inf and is written as it is.
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "ygg_ops.cuh"

namespace {

using namespace ygg;

struct Select {
    const void *logits;
    int64_t prompts, prompt_stride, beam_stride;
    int beams, vocab, width, end;   // end: -1 for none
    const void *scores;             // [prompts][beams] float, or double where `wide`
    bool wide;
    const uint8_t *done;            // [prompts][beams], or null
    void *out_scores;               // [prompts][width], as `scores`
    int32_t *tokens, *parents;
    uint8_t *out_done;              // or null
};

// What a beam's continuations are worth: score + (x - lse).
struct Beam {
    double score, lse;
    bool done;
};

template <typename T> __device__ __forceinline__ const T *row_of(const Select &p, int64_t prompt, int b) {
    return (const T *)p.logits + prompt * p.prompt_stride + b * p.beam_stride;
}

__device__ __forceinline__ double worth(const Beam &b, float x, int v, int end) {
    if (b.done) return v == end ? b.score : -INFINITY;
    return b.score + (b.lse == -INFINITY ? -INFINITY : (double)x - b.lse);
}
__device__ __forceinline__ double rank_of(double worth) { return isnan(worth) ? -INFINITY : worth; }

__device__ __forceinline__ void write_pick(const Select &p, int64_t prompt, int k, uint32_t at, double value, const Beam *beams) {
    const int64_t to = prompt * p.width + k;
    const int b = (int)(at / (uint32_t)p.vocab);
    const int token = beams[b].done ? p.end : (int)(at - (uint32_t)b * (uint32_t)p.vocab);
    if (p.wide) ((double *)p.out_scores)[to] = value;
    else ((float *)p.out_scores)[to] = (float)value;
    p.tokens[to] = token;
    p.parents[to] = b;
    if (p.out_done) p.out_done[to] = beams[b].done || token == p.end;
}

// A block a prompt; everything in 64 bits, the picks one after another.
template <typename T> __global__ void __launch_bounds__(256) plain_kernel(const Select p) {
    __shared__ Beam beams[YGG_BEAMS_MAX];
    __shared__ double part[256];
    __shared__ uint32_t part_at[256];
    const int t = threadIdx.x;
    const int64_t prompt = blockIdx.x;
    for (int b = 0; b < p.beams; b++) {
        const T *x = row_of<T>(p, prompt, b);
        double m = -INFINITY, s = 0.0;
        bool bad = false;
        for (int v = t; v < p.vocab; v += 256) {
            const float f = to_f(x[v]);
            bad |= isnan(f) || f == INFINITY;
            m = fmax(m, (double)f);
        }
        part[t] = m;
        bad = __syncthreads_or(bad);
        for (int d = 128; d; d >>= 1) {
            if (t < d) part[t] = fmax(part[t], part[t + d]);
            __syncthreads();
        }
        m = part[0];
        __syncthreads();
        for (int v = t; v < p.vocab && m > -INFINITY && !bad; v += 256) s += exp((double)to_f(x[v]) - m);
        part[t] = s;
        __syncthreads();
        for (int d = 128; d; d >>= 1) {
            if (t < d) part[t] += part[t + d];
            __syncthreads();
        }
        if (t == 0) {
            const int64_t at = prompt * p.beams + b;
            beams[b] = {p.wide ? ((const double *)p.scores)[at] : (double)((const float *)p.scores)[at],
                        bad ? (double)NAN : m == -INFINITY ? m : m + log(part[0]), p.done && p.done[at]};
        }
        __syncthreads();
    }
    double last = INFINITY;
    uint32_t last_at = 0;
    for (int k = 0; k < p.width; k++) {
        double best = -INFINITY;
        uint32_t best_at = ~0u;
        for (int b = 0; b < p.beams; b++) {
            const T *x = row_of<T>(p, prompt, b);
            for (int v = t; v < p.vocab; v += 256) {
                const double r = rank_of(worth(beams[b], to_f(x[v]), v, p.end));
                const uint32_t at = (uint32_t)b * (uint32_t)p.vocab + v;
                if (k > 0 && !(r < last || (r == last && at > last_at))) continue;
                if (r > best || (r == best && at < best_at)) best = r, best_at = at;
            }
        }
        part[t] = best;
        part_at[t] = best_at;
        __syncthreads();
        for (int d = 128; d; d >>= 1) {
            if (t < d && (part[t + d] > part[t] || (part[t + d] == part[t] && part_at[t + d] < part_at[t]))) {
                part[t] = part[t + d];
                part_at[t] = part_at[t + d];
            }
            __syncthreads();
        }
        last = part[0];
        last_at = part_at[0];
        if (t == 0) {
            const int b = (int)(last_at / (uint32_t)p.vocab), v = (int)(last_at - (uint32_t)b * (uint32_t)p.vocab);
            write_pick(p, prompt, k, last_at, worth(beams[b], to_f(row_of<T>(p, prompt, b)[v]), v, p.end), beams);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------------------------- rows

constexpr int kParts = YGG_REORDER_MAX, kUnits = 8;

struct Part {
    const uint8_t *from;
    uint8_t *to;
    int64_t units;        // of `unit` bytes, in all rows
    uint32_t per_row;     // of them in a row
    int unit;
    int64_t first;        // of its tasks
};
struct Reorder {
    const void *parents;
    int wide, beams, width, parts;
    int64_t tasks;
    Part part[kParts];
};

// A unit, 16 bytes or what the alignment leaves.
template <typename U>
__device__ __forceinline__ void copy_units(const Reorder &p, const Part &a, int64_t task, int lane) {
    U v[kUnits];
    bool live[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; i++) {
        const int64_t u = (task * kUnits + i) * 32 + lane;
        live[i] = u < a.units;
        if (!live[i]) continue;
        const int64_t row = u / a.per_row, at = u - row * a.per_row, prompt = row / p.width;
        const int64_t b = p.wide ? ((const int64_t *)p.parents)[row] : ((const int32_t *)p.parents)[row];
        v[i] = U{};
        if (b >= 0 && b < p.beams) v[i] = ((const U *)a.from)[(prompt * p.beams + b) * a.per_row + at];
    }
#pragma unroll
    for (int i = 0; i < kUnits; i++)
        if (live[i]) ((U *)a.to)[(task * kUnits + i) * 32 + lane] = v[i];
}

__global__ void __launch_bounds__(256) reorder_kernel(const __grid_constant__ Reorder p) {
    const int lane = threadIdx.x & 31;
    int64_t task = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (task >= p.tasks) return;
    int k = p.parts - 1;
    while (k && task < p.part[k].first) k--;
    const Part &a = p.part[k];
    task -= a.first;
    switch (a.unit) {
        case 16: copy_units<uint4>(p, a, task, lane); break;
        case 8: copy_units<uint2>(p, a, task, lane); break;
        case 4: copy_units<uint32_t>(p, a, task, lane); break;
        case 2: copy_units<uint16_t>(p, a, task, lane); break;
        default: copy_units<uint8_t>(p, a, task, lane);
    }
}

}  // namespace

extern "C" {

int ygg_beam_select(int device, int dtype, int64_t prompts, int64_t beams, int64_t vocab, const void *d_logits,
                    int64_t prompt_stride, int64_t beam_stride, int score_bytes, const void *d_scores, const uint8_t *d_done,
                    int64_t end, int64_t width, void *d_out_scores, int32_t *d_tokens, int32_t *d_parents,
                    uint8_t *d_out_done, void *stream) {
    if (prompts < 0 || beams < 1 || vocab < 1 || width < 1 || (score_bytes != 4 && score_bytes != 8)) return YGG_E_ARG;
    if (beams > YGG_BEAMS_MAX || width > YGG_BEAMS_MAX || prompts > INT32_MAX || vocab > INT32_MAX / beams) return YGG_E_UNSUPPORTED;
    if (width > beams * vocab || end < -1 || end >= vocab || (d_done && end < 0)) return YGG_E_ARG;
    if (prompts == 0) return YGG_OK;
    if (!d_logits || !d_scores || !d_out_scores || !d_tokens || !d_parents) return YGG_E_ARG;
    OnDevice on(device);
    if (!on.ok) return YGG_E_DEVICE;
    const Select p{d_logits, prompts, prompt_stride, beam_stride, (int)beams, (int)vocab, (int)width, (int)end, d_scores,
                   score_bytes == 8, d_done, d_out_scores, d_tokens, d_parents, d_out_done};
    const int rc = by_type(dtype, [&](auto t) {
        plain_kernel<decltype(t)><<<(unsigned)prompts, 256, 0, (cudaStream_t)stream>>>(p);
    });
    return rc != YGG_OK ? rc : cudaGetLastError() == cudaSuccess ? YGG_OK : YGG_E_CUDA;
}

int ygg_reorder(int device, int64_t prompts, int64_t beams, int64_t width, const void *d_parents, int parent_bytes,
                int count, const void *const *d_from, void *const *d_to, const int64_t *row_bytes, void *stream) {
    if (prompts < 0 || beams < 0 || width < 0 || beams > INT32_MAX || width > INT32_MAX || count < 0 ||
        count > YGG_REORDER_MAX || (parent_bytes != 4 && parent_bytes != 8) || (count && (!d_from || !d_to || !row_bytes)))
        return YGG_E_ARG;
    if (prompts > INT32_MAX || prompts * width > INT32_MAX) return YGG_E_UNSUPPORTED;
    Reorder p{d_parents, parent_bytes == 8, (int)beams, (int)width, 0, 0, {}};
    for (int i = 0; i < count; i++) {
        if (row_bytes[i] < 0 || row_bytes[i] > UINT32_MAX) return YGG_E_UNSUPPORTED;
        if (prompts * width * row_bytes[i] == 0) continue;
        if (!d_parents || !d_from[i] || !d_to[i]) return YGG_E_ARG;
        const uint64_t low = (uintptr_t)d_from[i] | (uintptr_t)d_to[i] | (uint64_t)row_bytes[i] | 16;
        const int unit = (int)(low & -low);
        const int64_t per_row = row_bytes[i] / unit, units = prompts * width * per_row;
        p.part[p.parts++] = {(const uint8_t *)d_from[i], (uint8_t *)d_to[i], units, (uint32_t)per_row, unit, p.tasks};
        p.tasks += (units + 32 * kUnits - 1) / (32 * kUnits);
    }
    if (!p.tasks) return YGG_OK;
    if (p.tasks > (int64_t)INT32_MAX * 8) return YGG_E_UNSUPPORTED;
    OnDevice on(device);
    if (!on.ok) return YGG_E_DEVICE;
    reorder_kernel<<<(unsigned)((p.tasks + 7) / 8), 256, 0, (cudaStream_t)stream>>>(p);
    return cudaGetLastError() == cudaSuccess ? YGG_OK : YGG_E_CUDA;
}

}  // extern "C"
