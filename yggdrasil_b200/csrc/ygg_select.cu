// The choice over beams and vocabulary, and the rows of a batch in its order.
//
// A prompt has H beams, each with a score and V logits. With lse_b = log sum_v e^(x_bv), the continuation of beam b by v is
// worth score_b + (x_bv - lse_b), in 64 bits; the best W of the H V continuations go on, ties by the lower b V + v. A beam
// that is done goes on with the token `end` alone, at no cost: the others are worth -inf, and a pick among them writes `end`
// too. -inf logits are worth -inf, a row of -inf alone is worth -inf everywhere; a row that holds NaN or +inf is worth NaN
// everywhere. NaN ranks as -inf and is written as it is.
//
// The logits are read once. A warp takes a piece of a row, adds up its exponentials in 32 bits and keeps the largest entry of each
// lane's part (a segment). With every row's lse known, the W-th best segment bounds the W-th best continuation from below, so that only
// the few segments that reach it are read again; their entries that reach it are ranked in 64 bits.
// An lse from float sums is off by at most kNear / 2 (below), which only matters between beams: where two of the chosen
// (or the last chosen and the next) of different beams are nearer than kNear, the lse of their rows is computed again in 64 bits. So the order is
// the exact one, for a second pass over a row in few calls (a prompt of 8 picks needs one about once in 5 000).
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "ygg_ops.cuh"
#include "ygg_rows.cuh"
#include "ygg_smem.h"

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
    int pieces, batches;            // pieces of a row, of `batches` times VECS vectors a lane
    float *tops;                    // [prompts][beams][pieces][32] largest entries of the segments, and
    float2 *sums;                   // [prompts][beams][pieces] largest entry m, sum of e^(x - m): between two launches
};

// Twice what an lse is off, at most: a term by 2^-22 of exp2 and 2^-23 |y| of its argument (y = x - m, rounded, times log2 e,
// rounded; weighted by e^y at most log V, 12: 1.4e-6); a chain of 8 + 3 + 4 + 5 additions by 2^-24 each (1.2e-6); three new references by
// 2^-22 and their argument (1.2e-6).
constexpr double kNear = 1e-5;

// What a beam's continuations are worth: score + (x - lse). m: the row's largest entry.
struct Beam {
    double score, lse;
    float m;
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
// Floats at or below the worth, in the order of integers; only what is -inf (or NaN) is kClosed.
constexpr int kClosed = (int)0x807FFFFF;
__device__ __forceinline__ int key_of(double worth) {
    const double r = rank_of(worth);
    return r == -INFINITY ? kClosed : order(fmaxf(__double2float_rd(r), -3.402823466e38f));
}

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

// ---------------------------------------------------------------------------------------------------- pieces of rows

// A warp's piece of a row: m and the sum of e^(x - m) over it (the same in every lane), and the largest entry of the lane's own.
template <typename T, int VECS>
__device__ __forceinline__ float2 sum_piece(const T *x, int vocab, int piece, int batches, int lane, float &top) {
    constexpr int N = kPer<T>;
    const uint32_t off = offset_of(x), end = off + (uint32_t)vocab;
    const T *from = x - off;
    const Pair l = pair(kLog2e, kLog2e);
    float m = -INFINITY, sum = 0.0f;
    top = -INFINITY;
    for (int b = 0; b < batches; b++) {
        const uint32_t u0 = (uint32_t)(piece * batches + b) * (VECS * 32 * N);
        if (u0 >= end) break;
        uint4 q[VECS];
        float mine = -INFINITY;
#pragma unroll
        for (int r = 0; r < VECS; r++) q[r] = load_run<T, true>(from, u0 + r * 32 * N, off, end, lane);
#pragma unroll
        for (int r = 0; r < VECS; r++) mine = fmaxf(mine, largest(q[r], T()));
        top = fmaxf(top, mine);
        const float most = unorder(__reduce_max_sync(~0u, order(mine)));
        if (most > m) {
            sum *= m == -INFINITY ? 0.0f : exp2_approx((m - most) * kLog2e);
            m = most;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        const Pair minus = pair(-ref, -ref);
        Pair s[4] = {};
#pragma unroll
        for (int r = 0; r < VECS; r++)
#pragma unroll
            for (int i = 0; i < N / 2; i++) s[(r * N / 2 + i) & 3] = add(s[(r * N / 2 + i) & 3], exp2_approx(mul(add(pair_of(q[r], i, T()), minus), l)));
        const float2 f = split(add(add(s[0], s[1]), add(s[2], s[3])));
        sum += f.x + f.y;
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
    return make_float2(m, sum);
}

// --------------------------------------------------------------------------------------------------------- the choice

// A team of threads chooses for a prompt: a warp (THREADS 32), or a block.
template <int THREADS> constexpr int kBeams = THREADS == 32 ? 16 : YGG_BEAMS_MAX;
template <int THREADS> constexpr int kRoom = THREADS == 32 ? 128 : 1024;   // candidates, and segments that are read again

template <int THREADS> struct Team {
    Beam beams[kBeams<THREADS>];
    double value[kRoom<THREADS>];
    uint32_t at[kRoom<THREADS>], list[kRoom<THREADS>];   // list: segments, then the candidates' order
    double part[THREADS / 32];
    uint32_t part_at[THREADS / 32];
    int count[3], candidates, segments;
    unsigned long long near;   // rows whose lse is wanted in 64 bits
};

template <int THREADS> __device__ __forceinline__ void sync() {
    if (THREADS == 32) __syncwarp();
    else __syncthreads();
}
__device__ __forceinline__ double shuffle_add(double v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
    return v;
}
__device__ __noinline__ double exp64(double x) { return exp(x); }

// lse of a row in 64 bits; the same in every thread.
template <typename T, int THREADS> __device__ __noinline__ void exact_lse(const Select &p, int64_t prompt, int b, int t, Team<THREADS> &sh) {
    const T *x = row_of<T>(p, prompt, b);
    const double m = sh.beams[b].m;
    double s = 0.0;
#pragma unroll 4
    for (int v = t; v < p.vocab; v += THREADS) s += exp64((double)to_f(x[v]) - m);
    s = shuffle_add(s);
    if (THREADS > 32) {
        if ((t & 31) == 0) sh.part[t >> 5] = s;
        __syncthreads();
        s = 0.0;
        for (int w = 0; w < THREADS / 32; w++) s += sh.part[w];
    }
    sync<THREADS>();
    if (t == 0) sh.beams[b].lse = m + log(s);
    sync<THREADS>();
}
// The rows of a set (one bit each) whose lse is a number.
template <typename T, int THREADS> __device__ __forceinline__ void exact_rows(const Select &p, int64_t prompt, unsigned long long rows, int t, Team<THREADS> &sh) {
    for (; rows; rows &= rows - 1) {
        const int b = __ffsll((long long)rows) - 1;
        if (!sh.beams[b].done && isfinite(sh.beams[b].lse)) exact_lse<T, THREADS>(p, prompt, b, t, sh);
    }
}

__device__ __forceinline__ bool better(double a, uint32_t a_at, double b, uint32_t b_at) { return a > b || (a == b && a_at < b_at); }

// The picks one after another, over all entries: where more reach the bound than there is room for (rows of equal logits).
template <typename T, int THREADS> __device__ __noinline__ void pick_slowly(const Select &p, int64_t prompt, int t, Team<THREADS> &sh) {
    exact_rows<T, THREADS>(p, prompt, ~0ull >> (64 - p.beams), t, sh);
    double last = INFINITY;
    uint32_t last_at = 0;
    for (int k = 0; k < p.width; k++) {
        double best = -INFINITY;
        uint32_t best_at = ~0u;
        for (int b = 0; b < p.beams; b++) {
            const T *x = row_of<T>(p, prompt, b);
            for (int v = t; v < p.vocab; v += THREADS) {
                const double r = rank_of(worth(sh.beams[b], to_f(x[v]), v, p.end));
                const uint32_t at = (uint32_t)b * (uint32_t)p.vocab + v;
                if ((k == 0 || better(last, last_at, r, at)) && better(r, at, best, best_at)) best = r, best_at = at;
            }
        }
        for (int d = 16; d; d >>= 1) {
            const double o = __shfl_xor_sync(~0u, best, d);
            const uint32_t o_at = __shfl_xor_sync(~0u, best_at, d);
            if (better(o, o_at, best, best_at)) best = o, best_at = o_at;
        }
        if (THREADS > 32) {
            __syncthreads();
            if ((t & 31) == 0) sh.part[t >> 5] = best, sh.part_at[t >> 5] = best_at;
            __syncthreads();
            for (int w = 0; w < THREADS / 32; w++)
                if (better(sh.part[w], sh.part_at[w], best, best_at)) best = sh.part[w], best_at = sh.part_at[w];
        }
        last = best;
        last_at = best_at;
        if (t == 0) {
            const int b = (int)(best_at / (uint32_t)p.vocab), v = (int)(best_at - (uint32_t)b * (uint32_t)p.vocab);
            write_pick(p, prompt, k, best_at, worth(sh.beams[b], to_f(row_of<T>(p, prompt, b)[v]), v, p.end), sh.beams);
        }
    }
}

// tops [beams][pieces][32] and sums [beams][pieces] of the prompt; keys: room for as many numbers as `tops` has, or kKeys (they may
// be the same memory where all fit). per: vectors of a segment.
constexpr int kKeys = 8192;
template <typename T, int THREADS>
__device__ void choose(const Select &p, int64_t prompt, int t, const float *tops, const float2 *sums, int *keys, int per, Team<THREADS> &sh) {
    constexpr int N = kPer<T>;
    const int lane = t & 31, row_segments = p.pieces * 32, segments = p.beams * row_segments;
    const bool fits = segments <= kKeys;
    // each row's lse
    for (int b = t >> 5; b < p.beams; b += THREADS / 32) {
        const int64_t row = prompt * p.beams + b;
        const bool done = p.done && p.done[row];
        float m = -INFINITY;
        double s = 0.0;
        if (!done) {
            for (int i = lane; i < p.pieces; i += 32) m = fmaxf(m, sums[b * p.pieces + i].x);
            m = unorder(__reduce_max_sync(~0u, order(m)));
            for (int i = lane; i < p.pieces; i += 32) {
                const float2 f = sums[b * p.pieces + i];
                s += p.pieces == 1 ? (double)f.y : f.x == -INFINITY ? (double)f.y : (double)f.y * exp64((double)f.x - (double)m);
            }
            s = shuffle_add(s);
        }
        if (lane == 0) {
            const double score = p.wide ? ((const double *)p.scores)[row] : (double)((const float *)p.scores)[row];
            sh.beams[b] = {score, isnan(s) ? (double)NAN : m == -INFINITY ? -INFINITY : (double)m + log(s), m, done};
        }
    }
    if (t == 0) sh.candidates = sh.segments = 0, sh.count[0] = sh.count[1] = sh.count[2] = 0, sh.near = 0;
    sync<THREADS>();

    // a bound that at least `width` segments reach
    const auto value_of = [&](int b, int i) {   // of a segment's largest entry; a done beam is one entry
        const Beam &beam = sh.beams[b];
        return beam.done ? (i ? -INFINITY : beam.score) : worth(beam, tops[b * row_segments + i], 0, -1);
    };
    int most = kClosed;
    for (int b = 0, j = t; b < p.beams; b++)
        for (; j < (b + 1) * row_segments; j += THREADS) {
            int k = key_of(value_of(b, j - b * row_segments));
            if (!fits && j >= kKeys) k = max(k, keys[j & (kKeys - 1)]);   // this thread's own: THREADS divides kKeys
            keys[fits ? j : j & (kKeys - 1)] = k;
            most = max(most, k);
        }
    const int held = min(segments, kKeys);
    most = __reduce_max_sync(~0u, most);
    if (THREADS > 32) {
        if (lane == 0) sh.list[t >> 5] = (uint32_t)most;
        __syncthreads();
        for (int w = 0; w < THREADS / 32; w++) most = max(most, (int)sh.list[w]);
    }
    sync<THREADS>();
    int round = 0;
    const auto reach = [&](int bound) {   // how many keys are at least the bound
        int n = 0;
        for (int j = t; j < held; j += THREADS) n += keys[j] >= bound;
        n = __reduce_add_sync(~0u, n);
        if (THREADS == 32) return n;
        if (lane == 0 && n) atomicAdd(&sh.count[round], n);
        if (t == 0) sh.count[round == 2 ? 0 : round + 1] = 0;
        __syncthreads();
        n = sh.count[round];
        round = round == 2 ? 0 : round + 1;
        return n;
    };
    bool open = false;   // no bound: all that is not closed
    int bound = kClosed + 1;
    if (most == kClosed || reach(bound) < p.width) {
        open = true;
    } else {
        int hi = most;
        const int guess = order(unorder(most) - 32.0f);
        if (guess > bound && guess < hi) {
            if (reach(guess) >= p.width) bound = guess;
            else hi = guess - 1;
        }
        while (bound < hi) {
            const int mid = bound + (int)(((unsigned)hi - (unsigned)bound + 1u) / 2u);
            const int n = reach(mid);
            if (n < p.width) {
                hi = mid - 1;
            } else {
                bound = mid;
                if (n <= p.width + p.width / 4) break;
            }
        }
        open = unorder(bound) < -1e38f;   // beyond what keys tell apart
    }
    const double least = open ? -INFINITY : (double)unorder(bound) - kNear;
    const int least_key = open ? kClosed + 1 : order(__double2float_rd(least));

    // the segments that reach it, and their entries that do
    const auto push = [&](double value, uint32_t at) {
        const int i = atomicAdd(&sh.candidates, 1);
        if (i < kRoom<THREADS>) sh.value[i] = value, sh.at[i] = at;
    };
    for (int b = 0, j = t; b < p.beams; b++)
        for (; j < (b + 1) * row_segments; j += THREADS) {
            if ((fits ? keys[j] : keys[j & (kKeys - 1)]) < least_key) continue;
            if (!fits && key_of(value_of(b, j - b * row_segments)) < least_key) continue;
            if (sh.beams[b].done) {
                push(sh.beams[b].score, (uint32_t)b * (uint32_t)p.vocab + (uint32_t)p.end);
            } else {
                const int i = atomicAdd(&sh.segments, 1);
                if (i < kRoom<THREADS>) sh.list[i] = (uint32_t)j;
            }
        }
    sync<THREADS>();
    const int listed = sh.segments;
    if (listed > kRoom<THREADS>) {
        pick_slowly<T, THREADS>(p, prompt, t, sh);
        return;
    }
    for (int item = t; item < listed * per; item += THREADS) {
        const int e = item / per, i = item - e * per, j = (int)sh.list[e], b = j / row_segments;
        const int piece = (j - b * row_segments) >> 5;
        const T *x = row_of<T>(p, prompt, b);
        const uint32_t off = offset_of(x), end = off + (uint32_t)p.vocab, u = (uint32_t)(piece * per + i) * (32 * N) + (j & 31) * N;
        if (u >= end) continue;
        float v[N];
        unpack(load_run<T, true>(x - off, u, off, end, 0), v, T());
        const Beam beam = sh.beams[b];
#pragma unroll
        for (int k = 0; k < N; k++) {
            const double w = worth(beam, v[k], 0, -1);
            if (open ? w > -INFINITY : w >= least) push(w, (uint32_t)b * (uint32_t)p.vocab + (u + k - off));
        }
    }
    sync<THREADS>();
    const int n = sh.candidates;
    if (n > kRoom<THREADS>) {
        pick_slowly<T, THREADS>(p, prompt, t, sh);
        return;
    }

    // their order
    const auto rank = [&] {
        for (int c = t; c < n; c += THREADS) {
            const double v = sh.value[c];
            const uint32_t at = sh.at[c];
            int r = 0;
            for (int i = 0; i < n; i++) r += better(sh.value[i], sh.at[i], v, at);
            sh.list[r] = c;
        }
        sync<THREADS>();
    };
    rank();
    const auto beam_of = [&](int r) { return (int)(sh.at[sh.list[r]] / (uint32_t)p.vocab); };
    for (int r = t + 1; r < n; r += THREADS) {   // with the one before, or, past the last pick, with that
        const int q = min(r, p.width) - 1, a = beam_of(q), b = beam_of(r);
        if (p.wide || (a != b && sh.value[sh.list[q]] - sh.value[sh.list[r]] < kNear))
            atomicOr(&sh.near, (1ull << a) | (1ull << b));
    }
    if (p.wide && t == 0 && n) atomicOr(&sh.near, 1ull << beam_of(0));
    sync<THREADS>();
    const unsigned long long near = sh.near;
    if (near) {
        exact_rows<T, THREADS>(p, prompt, near, t, sh);
        for (int c = t; c < n; c += THREADS) {
            const int b = (int)(sh.at[c] / (uint32_t)p.vocab), v = (int)(sh.at[c] - (uint32_t)b * (uint32_t)p.vocab);
            if (near >> b & 1) sh.value[c] = worth(sh.beams[b], to_f(row_of<T>(p, prompt, b)[v]), v, p.end);
        }
        sync<THREADS>();
        rank();
    }
    for (int k = t; k < min(n, p.width); k += THREADS) write_pick(p, prompt, k, sh.at[sh.list[k]], sh.value[sh.list[k]], sh.beams);
    if (n >= p.width || t >= 32) return;
    // fewer are open than are wanted: closed ones in their order
    const uint32_t all = (uint32_t)p.beams * (uint32_t)p.vocab;
    for (uint32_t first = 0, k = n; k < p.width && first < all; first += 32) {
        const uint32_t at = first + lane;
        double w = 0.0;
        if (at < all) {
            const int b = (int)(at / (uint32_t)p.vocab), v = (int)(at - (uint32_t)b * (uint32_t)p.vocab);
            w = worth(sh.beams[b], to_f(row_of<T>(p, prompt, b)[v]), v, p.end);
        }
        const unsigned closed = __ballot_sync(~0u, at < all && rank_of(w) == -INFINITY);
        const uint32_t to = k + __popc(closed & ((1u << lane) - 1));
        if ((closed >> lane & 1) && to < p.width) write_pick(p, prompt, to, at, w, sh.beams);
        k += __popc(closed);
    }
}

// A prompt to a team, in one launch; the team's warps share its rows' pieces. Dynamic shared memory: for each team [beams][pieces][32] largest entries
// (then their keys) and [beams][pieces] sums.
template <typename T, int VECS, int THREADS> __global__ void __launch_bounds__(256) small_kernel(const Select p) {
    extern __shared__ __align__(16) uint8_t room[];
    __shared__ Team<THREADS> teams[256 / THREADS];
    const int team = threadIdx.x / THREADS, t = threadIdx.x % THREADS, lane = t & 31, all = p.beams * p.pieces;
    const int64_t prompt = (int64_t)blockIdx.x * (256 / THREADS) + team;
    if (prompt >= p.prompts) return;   // a whole team
    float *tops = (float *)(room + (size_t)team * all * 136);
    float2 *sums = (float2 *)(tops + all * 32);
    for (int i = t >> 5; i < all; i += THREADS / 32) {
        const int b = i / p.pieces;
        if (p.done && p.done[prompt * p.beams + b]) continue;
        float top;
        const float2 s = sum_piece<T, VECS>(row_of<T>(p, prompt, b), p.vocab, i - b * p.pieces, 1, lane, top);
        tops[i * 32 + lane] = top;
        if (lane == 0) sums[i] = s;
    }
    sync<THREADS>();
    choose<T, THREADS>(p, prompt, t, tops, sums, (int *)tops, VECS, teams[team]);
}

// Pieces of rows over the whole GPU, then a block a prompt.
template <typename T> __global__ void __launch_bounds__(256) pieces_kernel(const Select p) {
    let_next_begin();
    const int lane = threadIdx.x & 31;
    const int64_t id = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), row = id / p.pieces, prompt = row / p.beams;
    if (row >= p.prompts * p.beams || (p.done && p.done[row])) return;
    float top;
    const float2 s = sum_piece<T, 8>(row_of<T>(p, prompt, (int)(row - prompt * p.beams)), p.vocab, (int)(id - row * p.pieces), p.batches, lane, top);
    p.tops[id * 32 + lane] = top;
    if (lane == 0) p.sums[id] = s;
}
constexpr int kChooseThreads = 512;
template <typename T> __global__ void __launch_bounds__(kChooseThreads) choose_kernel(const Select p) {
    extern __shared__ __align__(16) uint8_t room[];   // the keys
    __shared__ Team<kChooseThreads> team;
    wait_for_previous();
    const int64_t prompt = blockIdx.x, rows = prompt * p.beams;
    choose<T, kChooseThreads>(p, prompt, threadIdx.x, p.tops + rows * p.pieces * 32, p.sums + rows * p.pieces, (int *)room,
                              8 * p.batches, team);
}

// How a call is cut, by its sizes alone (aligned: every row begins on a 16-byte boundary).
struct Plan {
    int vecs, pieces, batches, team;   // team: threads of small_kernel's, or 0: two launches
};
constexpr int kSms = 148;
Plan plan_of(int size, bool aligned, int64_t prompts, int beams, int vocab, int width) {
    const int n = 16 / size;
    const int64_t vectors = ((int64_t)vocab + (aligned ? 0 : n - 1) + n - 1) / n;
    const int lanes = (int)((vectors + 31) / 32);   // vectors a lane
    Plan r{lanes <= 1 ? 1 : lanes <= 2 ? 2 : lanes <= 4 ? 4 : 8, 1, 1, 0};
    r.pieces = (lanes + r.vecs - 1) / r.vecs;
    const int all = beams * std::min(r.pieces, 1 << 20);
    if (all <= 16 && width <= 16 && prompts >= 4 * kSms) r.team = 32;
    else if (all <= 16 || (all <= 64 && prompts >= kSms)) r.team = 256;
    if (r.team) return r;
    r.vecs = 8;
    const int whole = (lanes + 7) / 8;
    for (r.batches = 4; r.batches > 1 && prompts * beams * ((whole + r.batches - 1) / r.batches) < 32 * kSms; r.batches /= 2) {}
    r.pieces = (whole + r.batches - 1) / r.batches;
    return r;
}
size_t room_of(const Plan &r, int64_t rows) { return r.team ? 0 : (size_t)rows * r.pieces * 136; }

template <typename T, int VECS, int THREADS> cudaError_t launch_small(const Select &p, cudaStream_t st) {
    static SmemLimits limits;
    const size_t smem = (size_t)(256 / THREADS) * p.beams * p.pieces * 136;
    const cudaError_t e = raise_smem_limit((const void *)small_kernel<T, VECS, THREADS>, smem, limits);
    if (e != cudaSuccess) return e;
    small_kernel<T, VECS, THREADS><<<(unsigned)((p.prompts + 256 / THREADS - 1) / (256 / THREADS)), 256, smem, st>>>(p);
    return cudaGetLastError();
}
template <typename T, int VECS> cudaError_t launch_team(const Select &p, int team, cudaStream_t st) {
    return team == 32 ? launch_small<T, VECS, 32>(p, st) : launch_small<T, VECS, 256>(p, st);
}
template <typename T> cudaError_t launch_select(Select p, bool aligned, void *room, cudaStream_t st) {
    const Plan r = plan_of(sizeof(T), aligned, p.prompts, p.beams, p.vocab, p.width);
    p.pieces = r.pieces;
    p.batches = r.batches;
    if (r.team)
        return r.vecs == 1 ? launch_team<T, 1>(p, r.team, st) : r.vecs == 2 ? launch_team<T, 2>(p, r.team, st)
               : r.vecs == 4 ? launch_team<T, 4>(p, r.team, st) : launch_team<T, 8>(p, r.team, st);
    const int64_t pieces = p.prompts * p.beams * p.pieces;
    p.tops = (float *)room;
    p.sums = (float2 *)(p.tops + pieces * 32);
    pieces_kernel<T><<<(unsigned)((pieces + 7) / 8), 256, 0, st>>>(p);
    static SmemLimits limits;
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) e = raise_smem_limit((const void *)choose_kernel<T>, 4 * kKeys, limits);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)p.prompts);
    cfg.blockDim = dim3(kChooseThreads);
    cfg.dynamicSmemBytes = 4 * std::min<int64_t>(kKeys, (int64_t)p.beams * p.pieces * 32);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, choose_kernel<T>, p);
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

size_t ygg_beam_workspace(int dtype, int64_t prompts, int64_t beams, int64_t vocab, int64_t width) {
    if (prompts < 0 || prompts > INT32_MAX || beams < 1 || beams > YGG_BEAMS_MAX || vocab < 1 || vocab > INT32_MAX / beams) return 0;
    const int size = dtype == YGG_DTYPE_FLOAT ? 4 : 2;
    size_t most = 0;
    for (const bool aligned : {false, true})
        most = std::max(most, room_of(plan_of(size, aligned, prompts, (int)beams, (int)vocab, (int)std::min<int64_t>(width, 64)), prompts * beams));
    return most;
}

int ygg_beam_select(int device, int dtype, int64_t prompts, int64_t beams, int64_t vocab, const void *d_logits,
                    int64_t prompt_stride, int64_t beam_stride, int score_bytes, const void *d_scores, const uint8_t *d_done,
                    int64_t end, int64_t width, void *d_out_scores, int32_t *d_tokens, int32_t *d_parents,
                    uint8_t *d_out_done, void *d_workspace, size_t workspace_bytes, void *stream) {
    if (prompts < 0 || beams < 1 || vocab < 1 || width < 1 || (score_bytes != 4 && score_bytes != 8)) return YGG_E_ARG;
    if (beams > YGG_BEAMS_MAX || width > YGG_BEAMS_MAX || prompts > INT32_MAX || vocab > INT32_MAX / beams) return YGG_E_UNSUPPORTED;
    if (width > beams * vocab || end < -1 || end >= vocab || (d_done && end < 0)) return YGG_E_ARG;
    if (dtype < YGG_DTYPE_FLOAT || dtype > YGG_DTYPE_BFLOAT) return YGG_E_UNSUPPORTED;
    if (prompts == 0) return YGG_OK;
    if (!d_logits || !d_scores || !d_out_scores || !d_tokens || !d_parents) return YGG_E_ARG;
    const size_t room = ygg_beam_workspace(dtype, prompts, beams, vocab, width);
    if (room && (!d_workspace || ((uintptr_t)d_workspace & 15) || workspace_bytes < room)) return YGG_E_ARG;
    OnDevice on(device);
    if (!on.ok) return YGG_E_DEVICE;
    const Select p{d_logits, prompts, prompt_stride, beam_stride, (int)beams, (int)vocab, (int)width, (int)end, d_scores,
                   score_bytes == 8, d_done, d_out_scores, d_tokens, d_parents, d_out_done, 0, 0, nullptr, nullptr};
    cudaError_t e = cudaSuccess;
    by_type(dtype, [&](auto t) {
        using T = decltype(t);
        const bool aligned = ((uintptr_t)d_logits & 15) == 0 && (prompts == 1 || prompt_stride % kPer<T> == 0) &&
                             (beams == 1 || beam_stride % kPer<T> == 0);
        e = launch_select<T>(p, aligned, d_workspace, (cudaStream_t)stream);
    });
    return e == cudaSuccess ? YGG_OK : YGG_E_CUDA;
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
