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
#include "ygg_rows.cuh"

namespace {

using namespace ygg;

constexpr float kFloor = -200.0f;   // e^-200 is 0 in 32 bits: y below it only has to stay finite

struct Rows {
    const void *logits;
    int64_t rows, vocab, stride;
    const void *tokens;   // int32 or int64
    int token_bytes, top;
    float *logprob, *entropy, *lse;
    int32_t *top_ids;
    float *top_logprobs;
    float4 *stats;        // m, log2 s (inf for an empty row), log s, H: what the gradient needs; or null
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

__device__ __forceinline__ int64_t token_of(const void *tokens, int bytes, int64_t row) {
    return bytes == 8 ? ((const int64_t *)tokens)[row] : (int64_t)((const int32_t *)tokens)[row];
}

// Adds the entries of vectors to sums whose m is at least the largest of them. y is cut off for the product alone: an entry of
// -inf has e = 0, and 0 times its y would be NaN (looking for NaN and going back instead cost 4 to 16 % more).
template <typename T, int RUNS> __device__ __forceinline__ void add_entries(Sums &a, const uint4 (&q)[RUNS]) {
    constexpr int N = kPer<T>;
    const float m = a.m == -INFINITY ? 0.0f : a.m;
    const Pair minus = pair(-m, -m), l = pair(kLog2e, kLog2e);
    Pair s = 0, t = 0;
#pragma unroll
    for (int r = 0; r < RUNS; r++)
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            const Pair y = add(pair_of(q[r], i, T()), minus), e = exp2_approx(mul(y, l));
            const float2 f = split(y);
            s = add(s, e);
            t = fma(e, pair(fmaxf(f.x, kFloor), fmaxf(f.y, kFloor)), t);
        }
    const float2 sf = split(s), tf = split(t);
    a.s += sf.x + sf.y;
    a.t += tf.x + tf.y;
}

using Key = unsigned long long;   // orders entries: value above, then the lower index
__device__ __forceinline__ Key key_of(float x, uint32_t j) {
    return ((Key)((unsigned)order(x) ^ 0x80000000u) << 32) | ~j;
}
__device__ __forceinline__ float value_of(Key k) { return unorder((int)((unsigned)(k >> 32) ^ 0x80000000u)); }
__device__ __forceinline__ int32_t index_of(Key k) { return (int32_t)~(unsigned)k; }
__device__ __forceinline__ Key warp_max(Key k) {
#pragma unroll
    for (int o = 16; o; o >>= 1) k = max(k, __shfl_xor_sync(~0u, k, o));
    return k;
}

// What a row's sums say.
struct Ends {
    float m, ls, h;
    bool empty;
    __device__ __forceinline__ explicit Ends(const Sums &a) {
        empty = a.s == 0.0f;
        m = empty ? 0.0f : a.m;
        ls = empty ? -INFINITY : logf(a.s);
        h = empty ? 0.0f : ls - a.t / a.s;
    }
    __device__ __forceinline__ float logprob(float x) const { return empty ? -INFINITY : (x - m) - ls; }
};
// The given token of a row and its logit; loaded before the row's sums are known, so that they do not wait for it.
struct Given {
    float x = 0.0f;
    int kind = 0;   // 0: padding, 1: a token, 2: one beyond the vocabulary
    template <typename T> __device__ __forceinline__ void load(const Rows &p, int64_t row, const T *logits) {
        const int64_t t = token_of(p.tokens, p.token_bytes, row);
        kind = t >= p.vocab ? 2 : t >= 0;
        if (kind == 1) x = to_f(logits[t]);
    }
};
__device__ __forceinline__ void write_row(const Rows &p, int64_t row, const Given &given, const Sums &a, const Ends &e) {
    p.logprob[row] = given.kind == 0 ? 0.0f : given.kind == 1 ? e.logprob(given.x) : NAN;
    p.entropy[row] = e.h;
    p.lse[row] = e.m + e.ls;
    if (p.stats) p.stats[row] = make_float4(e.m, e.empty ? INFINITY : log2f(a.s), e.empty ? 0.0f : e.ls, e.h);
}
__device__ __forceinline__ void write_top(const Rows &p, int64_t row, int k, float x, uint32_t index, const Ends &e) {
    p.top_ids[row * p.top + k] = (int32_t)index;
    p.top_logprobs[row * p.top + k] = e.logprob(x);
}
__device__ __forceinline__ void write_top(const Rows &p, int64_t row, int k, Key key, const Ends &e) {
    write_top(p, row, k, value_of(key), (uint32_t)index_of(key), e);
}

// The k-th largest of the lanes' values (k <= 32), a lower bound of the k-th largest entry that the lanes hold.
__device__ __forceinline__ int kth_of_lanes(int mine, int k) {
    int best;
    do {
        best = __reduce_max_sync(~0u, mine);
        const bool it = mine == best;
        k -= __popc(__ballot_sync(~0u, it));
        if (it) mine = INT32_MIN;
    } while (k > 0);
    return best;
}
__device__ __forceinline__ void order_down(int &a, int &b, int &c, int &d) {
    const auto order2 = [](int &x, int &y) {
        const int t = min(x, y);
        x = max(x, y);
        y = t;
    };
    order2(a, b), order2(c, d), order2(a, c), order2(b, d), order2(b, c);
}
// The same over four values a lane (k <= 128): a closer bound.
__device__ __forceinline__ int kth_of_lanes(int a, int b, int c, int d, int k) {
    order_down(a, b, c, d);
    int best;
    do {
        best = __reduce_max_sync(~0u, a);
        const bool it = a == best;
        k -= __popc(__ballot_sync(~0u, it));
        if (it) a = b, b = c, c = d, d = INT32_MIN;
    } while (k > 0);
    return best;
}
// A bound that k to 1.25 k of four values a lane reach (k <= 64; more only where they tie), by halving the range between
// the largest and one that 32 or 64 reach: some 5 rounds for logits, where the k-th itself takes k.
__device__ __forceinline__ int about_kth_of_lanes(int a, int b, int c, int d, int k, int largest) {
    order_down(a, b, c, d);
    int low = __reduce_min_sync(~0u, k <= 32 ? a : b);
    unsigned range = (unsigned)largest - (unsigned)low;   // the k-th lies in [low, low + range]
    while (range) {
        const unsigned half = range - range / 2;
        const int at = (int)((unsigned)low + half);
        const int n = __reduce_add_sync(~0u, (a >= at) + (b >= at) + (c >= at) + (d >= at));
        if (n < k) {
            range = half - 1;
        } else {
            low = at, range -= half;
            if (n <= k + k / 4) break;
        }
    }
    return low;
}

// Up to 8 entries: a thread a row (65536 x 5 fp32 2.1 us, a launch's time; a warp a row takes 12 for 65536 x 20).
template <typename T> __global__ void __launch_bounds__(128) tiny_kernel(const Rows p) {
    const int64_t row = (int64_t)blockIdx.x * 128 + threadIdx.x;
    if (row >= p.rows) return;
    const T *x = (const T *)p.logits + row * p.stride;
    float v[8];
    Sums a = none();
#pragma unroll
    for (int i = 0; i < 8; i++) {
        v[i] = i < p.vocab ? to_f(x[i]) : -INFINITY;
        a.m = fmaxf(a.m, v[i]);
    }
    const uint4 q[2] = {pack({v[0], v[1], v[2], v[3]}, 0.0f), pack({v[4], v[5], v[6], v[7]}, 0.0f)};
    add_entries<float>(a, q);
    const Ends e(a);
    Given given;
    given.load(p, row, x);
    write_row(p, row, given, a, e);
    if (p.top == 0) return;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        int above = 0;
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j != i) above += order(v[j]) + (j < i) > order(v[i]);
        if (i < p.vocab && above < p.top) write_top(p, row, above, v[i], i, e);
    }
}

// Short rows: a warp holds a row in registers, RUNS runs of 32 kPer places, and takes R rows one after another, so that
// what a row needs only once (the sums over the lanes, the logarithm, the token, the writes) is done for R rows by
// different lanes at once. Alternatives: the k-th largest of the lanes' maxima, or for more than 8 a value that about k
// of four maxima a lane reach (20 of 128 bins leave about 22 candidates, 20 of 32 about 31, 64 of 128 about 89), bounds
// the k-th largest entry from below, so the few entries at or above it are the candidates, and they are ranked by
// counting (65536 x 256 with 32 alternatives: fp32 69 us, 86 with the k-th of the bins itself; bf16 64, 128 with values
// and indices apart). Where ties make them more than the list holds, the equal ones that come too late are left out;
// where entries above the bound are too many, they are taken one at a time.
// Bound by instructions and the latency of the selection's chain: 65536 x 256 fp32 16.3 us (4.1 TB/s), 27.8 with 5
// alternatives; issue slots 58 % full, 40 warps an SM.
constexpr int kShortWarps = 4, kCandidates = 128, kList = kCandidates + 1;   // an odd pitch: lists begin in unlike banks
// WHOLE: rows of exactly RUNS runs, all on 16-byte boundaries.
template <typename T> struct List {
    int value[kList];        // order() of the candidates
    uint32_t index[kList];
    __device__ __forceinline__ void put(int at, float x, uint32_t j) { value[at] = order(x), index[at] = j; }
};
// 16-bit entries tie often: value and index in one word, the lower index above
struct HalfList {
    int value[kList];
    __device__ __forceinline__ uint32_t index_at(int i) const { return ~value[i] & 0xFFFF; }
};
template <> struct List<__nv_bfloat16> : HalfList {
    __device__ __forceinline__ void put(int at, float x, uint32_t j) { value[at] = (order(x) & 0xFFFF0000) | (~j & 0xFFFF); }
    __device__ __forceinline__ float value_at(int i) const {
        const int high = value[i] & 0xFFFF0000;
        return unorder(high < 0 ? high | 0xFFFF : high);
    }
};
template <> struct List<__half> : HalfList {
    __device__ __forceinline__ void put(int at, float x, uint32_t j) {
        const int b = (int16_t)__half_as_ushort(__float2half_rn(isnan(x) ? -INFINITY : x + 0.0f));
        value[at] = (int)((unsigned)(b >= 0 ? b : b ^ 0x7FFF) << 16 | (~j & 0xFFFF));
    }
    __device__ __forceinline__ float value_at(int i) const {
        const int b = value[i] >> 16;
        return __half2float(__ushort_as_half((unsigned short)(b >= 0 ? b : b ^ 0x7FFF)));
    }
};
// Place `bit` of a lane's, by selects.
template <int RUNS, int N> __device__ __forceinline__ float entry_at(const float (&v)[RUNS][N], int bit) {
    float w[RUNS * N];
#pragma unroll
    for (int i = 0; i < RUNS * N; i++) w[i] = v[i / N][i % N];
#pragma unroll
    for (int h = RUNS * N / 2; h; h /= 2)
#pragma unroll
        for (int i = 0; i < h; i++) w[i] = bit & h ? w[i + h] : w[i];
    return w[0];
}

// Blocks an SM for so many places a lane: the registers that keep the loads of enough rows in flight.
constexpr int blocks_for(int places) { return places <= 4 ? 11 : places <= 8 ? 10 : places <= 16 ? 8 : 5; }
template <typename T, int RUNS, int R, bool WHOLE>
__global__ void __launch_bounds__(kShortWarps * 32, blocks_for(RUNS * kPer<T>)) short_kernel(const Rows p) {
    constexpr int N = kPer<T>;
    __shared__ List<T> lists[kShortWarps][R];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row0 = ((int64_t)blockIdx.x * kShortWarps + warp) * R;
    if (row0 >= p.rows) return;
    const unsigned below = (1u << lane) - 1;
    float ms[R], sums[2 * R];
    int found[R];
    Given given;   // lane l serves row l mod R
    if (lane < R && row0 + lane < p.rows) given.load(p, row0 + lane, (const T *)p.logits + (row0 + lane) * p.stride);
#pragma unroll
    for (int w = 0; w < R; w++) {
        const int64_t row = min(row0 + w, p.rows - 1);   // rows past the last are the last once more, unseen
        const T *x = (const T *)p.logits + row * p.stride;
        const uint32_t off = WHOLE ? 0 : offset_of(x), end = WHOLE ? RUNS * 32 * N : (uint32_t)p.vocab + off;
        const T *from = x - off;
        uint4 q[RUNS];
        float v[RUNS][N];
        float most = -INFINITY;
#pragma unroll
        for (int r = 0; r < RUNS; r++) {
            q[r] = (WHOLE ? load_again(x + (r * 32 + lane) * N) : load_run<T, true>(from, r * 32 * N, off, end, lane));
            unpack(q[r], v[r], T());
        }
#pragma unroll
        for (int r = 0; r < RUNS; r++)
#pragma unroll
            for (int i = 0; i < N; i++) most = fmaxf(most, v[r][i]);
        const int mine = order(most);
        Sums a{unorder(__reduce_max_sync(~0u, mine)), 0.0f, 0.0f};
        add_entries<T>(a, q);
        ms[w] = a.m, sums[w] = a.s, sums[R + w] = a.t;
        found[w] = 0;
        if (p.top == 0) continue;
        List<T> &list = lists[warp][w];
        int n;
        {
            int kth;
            if (p.top <= 8) {
                kth = kth_of_lanes(mine, p.top);
            } else {
                float bin[4];
#pragma unroll
                for (int k = 0; k < 4; k++) bin[k] = v[0][k];
#pragma unroll
                for (int r = 0; r < RUNS; r++)
#pragma unroll
                    for (int i = 0; i < N; i++)
                        if (r || i >= 4) bin[i & 3] = fmaxf(bin[i & 3], v[r][i]);
                kth = about_kth_of_lanes(order(bin[0]), order(bin[1]), order(bin[2]), order(bin[3]), p.top, order(a.m));
            }
            const float bound = unorder(kth);
            unsigned in = 0;
#pragma unroll
            for (int r = 0; r < RUNS; r++)
#pragma unroll
                for (int i = 0; i < N; i++) in |= v[r][i] >= bound ? 1u << (r * N + i) : 0u;
            if (bound == -INFINITY) {   // every entry, NaN too, but not the places outside the row
                in = ~0u;
#pragma unroll
                for (int r = 0; r < RUNS; r++)
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        const uint32_t u = (r * 32 + lane) * N + i;
                        if (u - off >= end - off) in &= ~(1u << (r * N + i));
                    }
                if (RUNS * N < 32) in &= (1u << (RUNS * N & 31)) - 1;
            }
            n = __reduce_add_sync(~0u, __popc(in));
            if (n <= kCandidates) {
                unsigned who;
                for (int done = 0; (who = __ballot_sync(~0u, in != 0)) != 0; done += __popc(who)) {
                    if (in) {
                        const int bit = __ffs(in) - 1, u = (bit / N * 32 + lane) * N + bit % N;
                        // up to 8 places by selects: 28.3 us against 29.5 for 65536 x 256 fp32 with 5 alternatives
                        list.put(done + __popc(who & below), RUNS * N <= 8 ? entry_at(v, bit) : to_f(from[u]), u - off);
                        in &= in - 1;
                    }
                }
            } else {   // ties at the bound: the entries above it, and as many equal ones as are still wanted
                n = 0;
#pragma unroll
                for (int r = 0; r < RUNS; r++)
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        const bool more = v[r][i] > bound;
                        const unsigned who = __ballot_sync(~0u, more);
                        const int at = n + __popc(who & below);
                        if (more && at < kCandidates) list.put(at, v[r][i], (r * 32 + lane) * N + i - off);
                        n += __popc(who);
                    }
                // in the order of their indices: a lane's entries of a run lie side by side
#pragma unroll
                for (int r = 0; r < RUNS; r++) {
                    if (n >= p.top) break;
                    const unsigned mask = (N == 32 ? ~0u : (1u << N) - 1) << (r * N);
                    unsigned equal = in & mask;
#pragma unroll
                    for (int i = 0; i < N; i++)
                        if (v[r][i] > bound) equal &= ~(1u << (r * N + i));
                    const int own = __popc(equal);
                    int upto = own;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const int y = __shfl_up_sync(~0u, upto, o);
                        if (lane >= o) upto += y;
                    }
                    int at = n + upto - own;
#pragma unroll
                    for (int i = 0; i < N; i++)
                        if (equal >> (r * N + i) & 1) {
                            if (at < p.top) list.put(at, v[r][i], (r * 32 + lane) * N + i - off);
                            at++;
                        }
                    n = min(p.top, n + __shfl_sync(~0u, upto, 31));
                }
            }
        }
        if (n > kCandidates) {
            __syncwarp();   // other lanes wrote to the list
            Key last = ~0ull;
            for (int k = 0; k < p.top; k++) {
                Key best = 0;
#pragma unroll
                for (int r = 0; r < RUNS; r++)
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        const uint32_t u = (r * 32 + lane) * N + i;
                        const Key key = u - off < end - off ? key_of(v[r][i], u - off) : 0;
                        if (key < last && key > best) best = key;
                    }
                last = warp_max(best);
                if (lane == 0) list.put(k, value_of(last), (uint32_t)index_of(last));
            }
            n = p.top;
        }
        found[w] = n;
    }
    // lane l serves row l mod R: the sums of 2 R values over the lanes, halved with the values while there are several
#pragma unroll
    for (int half = R, o = 16; o; o >>= 1, half = half > 1 ? half / 2 : 0) {
        if (half) {
#pragma unroll
            for (int i = 0; i < half; i++) {
                const bool upper = lane & o;
                const float give = upper ? sums[i] : sums[half + i];
                sums[i] = (upper ? sums[half + i] : sums[i]) + __shfl_xor_sync(~0u, give, o);
            }
        } else {
            sums[0] += __shfl_xor_sync(~0u, sums[0], o);
        }
    }
    // value i of the 2 R is now in the lanes whose upper bits, first bit first, spell i
    const int mine = lane & (R - 1);
    constexpr int kStep = 16 / R;   // lanes of one value: t of a row lies 16 lanes above its s
    Sums a;
    a.m = ms[0];
    int n = found[0], most = found[0];
#pragma unroll
    for (int w = 1; w < R; w++) {
        if (mine == w) a.m = ms[w], n = found[w];
        most = max(most, found[w]);
    }
    a.s = __shfl_sync(~0u, sums[0], mine * kStep);
    a.t = __shfl_sync(~0u, sums[0], 16 + mine * kStep);
    const Ends e(a);
    const int64_t row = row0 + mine;
    if (row >= p.rows) n = 0;
    if (lane < R && row < p.rows) write_row(p, row, given, a, e);
    __syncwarp();
    if (p.top == 0) return;
    const List<T> &list = lists[warp][mine];
    if constexpr (sizeof(T) == 2) {
        for (int slot = lane / R; slot < n; slot += 32 / R) {
            const int value = list.value[slot];
            int above = 0;
            for (int i = 0; i < n; i++) above += list.value[i] > value;
            if (above < p.top) write_top(p, row, above, list.value_at(slot), list.index_at(slot), e);
        }
    } else {
        // ranks by the values alone; ties give ranks twice, which shows in the ranks' sum, and then the indices count too
        int wrong = 0;
        for (int slot = lane / R; slot < most; slot += 32 / R) {
            if (slot >= n) continue;
            const int value = list.value[slot];
            int above = 0;
            for (int i = 0; i < n; i++) above += list.value[i] > value;
            wrong += slot - above;   // a row's slots and ranks have one sum
            if (above < p.top) write_top(p, row, above, unorder(value), list.index[slot], e);
        }
        // (the rows' sums are looked at together: ranks are never above the true ones, so that no row makes up for another)
        if (__reduce_add_sync(~0u, wrong) == 0) return;
        __syncwarp();   // the ranks that tied are written over, by other lanes
        for (int slot = lane / R; slot < n; slot += 32 / R) {
            const int value = list.value[slot];
            const uint32_t index = list.index[slot];
            int above = 0;
            for (int i = 0; i < n; i++)
                above += list.value[i] > value || (list.value[i] == value && list.index[i] < index);
            if (above < p.top) write_top(p, row, above, unorder(value), index, e);
        }
    }
}

// Long rows: a cluster of up to 8 blocks a row. The row is cut into segments of 2^lg vectors of 16 bytes, 512 to 1024 of
// them (fewer in rows of fewer vectors), and the warps of the cluster take runs of 32 vectors in turn; a warp keeps its
// running sums and leaves the largest value of each segment. The first block joins the sums. Alternatives: the k-th
// largest of 128 bins' maxima (bin b: the segments b mod 128) bounds the k-th best entry from below, so the segments that
// reach it hold the k best entries: about 22 for 20, which are read again, and the entries that reach it are ranked by
// counting. Where ties at the bound make the segments too many, the equal ones beyond the k-th are left out, in the order
// of their indices. If the entries are too many (ties, masks, sorted rows), a second bound from the threads' best entries
// leaves fewer; if those are still more, they are taken one at a time.
// Bound by issue slots and the exponentials' pipe, then by waves of rows that end unevenly: 8192 x 32768 bf16 103 us (5.2
// TB/s, 0.8 of a copy's rate), 136 with 20 alternatives; fp32 4096 x 32768 82 us, a copy's rate.
// (Loading a warp's next batch while one is added up costs the registers of a block an SM and gained nothing: 8192 x 32768
// bf16 136 us with, 117 without, 7 x 100003 bf16 9.5 and 9.4.)
constexpr int kMaxSegments = 1024, kBins = 128, kMaxCluster = 8, kBatch = 4, kKeys = 256;
// segments above the bound: at most 63 bins' worth
constexpr int kMost = (YGG_TOP_MAX - 1) * (kMaxSegments / kBins);

template <int WARPS> struct LongShared {
    Sums part[kMaxCluster * WARPS];   // in the first block
    Sums all;
    uint16_t picked[kMost];           // segments
    Key keys[kKeys];
    Key best[WARPS];
    int count, picks, bound;
    alignas(16) int segment[];        // order() of the segments' largest values; in the first block of all
};

__device__ __forceinline__ uint32_t shared_at(const void *p, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ void put_remote(uint32_t at, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}

template <typename T, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) long_kernel(const Rows p, int cluster, int lg, int segments) {
    constexpr int N = kPer<T>, kThreads = WARPS * 32;
    extern __shared__ __align__(16) uint8_t raw[];
    LongShared<WARPS> &sh = *(LongShared<WARPS> *)raw;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = blockIdx.x / cluster;
    const int rank = blockIdx.x - (int)row * cluster;
    if (cluster > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // the first block runs
    const T *x = (const T *)p.logits + row * p.stride;
    const int shift = max(lg - 5, 0);
    const uint32_t off = offset_of(x), span = (32u * N) << shift, end = (uint32_t)p.vocab + off;
    const T *from = x - off;
    constexpr int kJoin = WARPS > 1;   // the warp that joins the sums
    Given given;
    if (rank == 0 && warp == kJoin && lane == 0) given.load(p, row, x);
    Sums a = none();
    const int w = rank * WARPS + warp, warps = cluster * WARPS;
    // batches of kBatch runs: with shift of one segment (2^shift is then >= kBatch), else of 2^(5 - lg) segments a run
    const int steps = shift ? 1 << (shift - 2) : 1, per = shift ? 1 : kBatch, cut = shift ? 0 : 5 - lg;
    const int units = segments >> cut;
    const auto load = [&](uint4(&q)[kBatch], uint32_t u0) {
        if (u0 >= off && u0 + kBatch * 32 * N <= end) {   // inside the row
#pragma unroll
            for (int b = 0; b < kBatch; b++) q[b] = load_stream(from + u0 + (b * 32 + lane) * N);
        } else {
#pragma unroll
            for (int b = 0; b < kBatch; b++) q[b] = load_run<T>(from, u0 + b * 32 * N, off, end, lane);
        }
    };
    for (int g0 = w * per; g0 < units; g0 += warps * per) {
        float top_of[kBatch];
        for (int step = 0; step < steps; step++) {
            uint4 q[kBatch];
            load(q, g0 * span + step * kBatch * 32 * N);
            float most = -INFINITY;
#pragma unroll
            for (int b = 0; b < kBatch; b++) {
                const float t = largest(q[b], T());
                top_of[b] = shift && step ? fmaxf(top_of[b], t) : t;
                most = fmaxf(most, t);
            }
            if (most > a.m) raise(a, most);
            add_entries<T>(a, q);
        }
        if (p.top == 0) continue;
        if (shift) {
            const float t = fmaxf(fmaxf(top_of[0], top_of[1]), fmaxf(top_of[2], top_of[3]));
            const int best = __reduce_max_sync(~0u, order(t));
            if (lane == 0) sh.segment[g0] = best;
        } else if (lg == 5) {
#pragma unroll
            for (int b = 0; b < kBatch; b++) {
                const int best = __reduce_max_sync(~0u, order(top_of[b]));
                if (lane == 0) sh.segment[g0 + b] = best;
            }
        } else {
            int best[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; b++) best[b] = order(top_of[b]);
            for (int o = 1; o < 1 << lg; o <<= 1)
#pragma unroll
                for (int b = 0; b < kBatch; b++) best[b] = max(best[b], __shfl_xor_sync(~0u, best[b], o));
            if ((lane & ((1 << lg) - 1)) == 0)
#pragma unroll
                for (int b = 0; b < kBatch; b++) sh.segment[((g0 + b) << cut) + (lane >> lg)] = best[b];
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1)
        join(a, Sums{__shfl_xor_sync(~0u, a.m, o), __shfl_xor_sync(~0u, a.s, o), __shfl_xor_sync(~0u, a.t, o)});
    if (rank == 0 && lane == 0) sh.part[warp] = a;
    if (cluster > 1) {
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        if (rank) {
            if (lane == 0) {
                const uint32_t at = shared_at(&sh.part[w], 0);
                put_remote(at, __float_as_uint(a.m));
                put_remote(at + 4, __float_as_uint(a.s));
                put_remote(at + 8, __float_as_uint(a.t));
            }
            if (p.top) {   // the warp's own segments
                __syncwarp();
                for (int g0 = w * per; g0 < units; g0 += warps * per)
                    for (int g = g0 << cut; g < (g0 + per) << cut; g += 32)
                        if (g + lane < (g0 + per) << cut)
                            put_remote(shared_at(&sh.segment[g + lane], 0), (uint32_t)sh.segment[g + lane]);
            }
        }
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (rank) return;
    }
    __syncthreads();
    if (warp == kJoin) {   // the sums, while the first warp looks for the best segments
        a = lane < warps ? sh.part[lane] : none();
        if (lane + 32 < warps) join(a, sh.part[lane + 32]);
#pragma unroll
        for (int o = 16; o; o >>= 1)
            join(a, Sums{__shfl_xor_sync(~0u, a.m, o), __shfl_xor_sync(~0u, a.s, o), __shfl_xor_sync(~0u, a.t, o)});
        if (lane == 0) {
            sh.all = a;
            write_row(p, row, given, a, Ends(a));
        }
    }
    if (p.top == 0) return;

    // the best segments, by one warp
    if (warp == 0) {
        int4 bin = make_int4(INT32_MIN, INT32_MIN, INT32_MIN, INT32_MIN);
        const auto each = [&](auto f) {   // four segments a lane
            for (int g = lane * 4; g < segments; g += kBins) f(*(const int4 *)(sh.segment + g), g);
        };
        each([&](int4 v, int) {
            bin = make_int4(max(bin.x, v.x), max(bin.y, v.y), max(bin.z, v.z), max(bin.w, v.w));
        });
        const int bound = kth_of_lanes(bin.x, bin.y, bin.z, bin.w, p.top);
        if (lane == 0) sh.picks = sh.count = 0, sh.bound = bound;
        __syncwarp();
        const auto pick = [&](int least) {
            const auto put = [&](int v, int g) {
                if (v < least) return;
                const int at = atomicAdd(&sh.picks, 1);
                if (at < kMost) sh.picked[at] = (uint16_t)g;
            };
            each([&](int4 v, int g) { put(v.x, g), put(v.y, g + 1), put(v.z, g + 2), put(v.w, g + 3); });
            __syncwarp();
        };
        pick(bound);
        if (sh.picks > kMost) {
            __syncwarp();
            if (lane == 0) sh.picks = 0;
            __syncwarp();
            if (bound < INT32_MAX) pick(bound + 1);
            int n = sh.picks;
            for (int g0 = 0; g0 < segments && n < p.top; g0 += 32) {
                const bool equal = g0 + lane < segments && sh.segment[g0 + lane] == bound;
                const unsigned who = __ballot_sync(~0u, equal);
                const int at = n + __popc(who & ((1u << lane) - 1));
                if (equal && at < p.top) sh.picked[at] = (uint16_t)(g0 + lane);
                n = min(p.top, n + __popc(who));
            }
            __syncwarp();
            if (lane == 0) sh.picks = n;
        }
    }
    __syncthreads();
    const Ends e(sh.all);
    const float bound = unorder(sh.bound);
    const int vectors = sh.picks << lg;   // in the picked segments
    // f(entry, its place) for the entries of the picked segments
    const auto entries = [&](auto f) {
        for (int q = threadIdx.x; q < vectors; q += kThreads) {
            const uint32_t u0 = (((uint32_t)sh.picked[q >> lg] << lg) + (q & ((1 << lg) - 1))) * N;
            float v[N];
            load_run<T>(from, u0, off, end, 0, v);
#pragma unroll
            for (int i = 0; i < N; i++)
                if (u0 + i - off < end - off) f(v[i], u0 + i - off);
        }
    };
    const auto keep = [&](Key key) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kKeys) sh.keys[at] = key;
    };
    entries([&](float v, uint32_t j) {
        if (!(v < bound)) keep(key_of(v, j));
    });
    __syncthreads();
    int n = sh.count;
    if (n > kKeys && p.top <= kThreads) {
        // ties, masks, sorted rows: the k-th best of the threads' best entries (by value and index) is a better bound
        Key mine = 0;
        entries([&](float v, uint32_t j) { mine = max(mine, key_of(v, j)); });
        __syncthreads();
        sh.keys[threadIdx.x] = mine;
        if (threadIdx.x == 0) sh.count = 0, sh.best[0] = 0;
        __syncthreads();
        int above = 0;
        for (int i = 0; i < kThreads; i++) above += sh.keys[i] > mine;
        if (mine && above == p.top - 1) sh.best[0] = mine;
        __syncthreads();
        const Key least = sh.best[0];
        entries([&](float v, uint32_t j) {
            const Key key = key_of(v, j);
            if (key >= least) keep(key);
        });
        __syncthreads();
        n = sh.count;
    }
    if (n <= kKeys) {
        for (int k = threadIdx.x; k < n; k += kThreads) {
            const Key key = sh.keys[k];
            int above = 0;
            for (int i = 0; i < n; i++) above += sh.keys[i] > key;
            if (above < p.top) write_top(p, row, above, key, e);
        }
        return;
    }
    Key last = ~0ull;
    for (int k = 0; k < p.top; k++) {
        Key best = 0;
        entries([&](float v, uint32_t j) {
            const Key key = key_of(v, j);
            if (key < last && key > best) best = key;
        });
        best = warp_max(best);
        __syncthreads();
        if (lane == 0) sh.best[warp] = best;
        __syncthreads();
        for (int i = 0; i < WARPS; i++) best = max(best, sh.best[i]);
        last = best;
        if (threadIdx.x == 0) write_top(p, row, k, last, e);
    }
}

// Blocks a row for the long kernel: as many as it takes to give the SMs work, up to 8, while each keeps a batch a warp.
constexpr int kFewWarps = 8;
int cluster_for(int64_t rows, int64_t runs, int sms) {
    int c = 1;
    while (c < kMaxCluster && rows * c < 2 * sms && runs >= 2 * c * kFewWarps * kBatch) c *= 2;
    return c;
}

template <typename T, int WARPS>
cudaError_t launch_long(const Rows &p, int cluster, int lg, int segments, cudaStream_t st) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(p.rows * cluster));
    cfg.blockDim = dim3(WARPS * 32);
    cfg.dynamicSmemBytes = sizeof(LongShared<WARPS>) + (p.top ? segments : 0) * sizeof(int);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1;
    return cudaLaunchKernelEx(&cfg, long_kernel<T, WARPS>, p, cluster, lg, segments);
}

// Four rows a warp as soon as they fill the SMs.
template <typename T, int RUNS> void launch_short(const Rows &p, bool even, cudaStream_t st) {
    const bool many = p.rows >= (int64_t)sm_count() * 64, whole = even && p.vocab == RUNS * 32 * kPer<T>;
    const int64_t per = kShortWarps * (many ? 4 : 1);
    const unsigned grid = (unsigned)((p.rows + per - 1) / per);
    if (!many) short_kernel<T, RUNS, 1, false><<<grid, kShortWarps * 32, 0, st>>>(p);
    else if (whole) short_kernel<T, RUNS, 4, true><<<grid, kShortWarps * 32, 0, st>>>(p);
    else short_kernel<T, RUNS, 4, false><<<grid, kShortWarps * 32, 0, st>>>(p);
}

template <typename T> cudaError_t launch_rows(const Rows &p, cudaStream_t st) {
    constexpr int N = kPer<T>;
    const bool even = ((uintptr_t)p.logits & 15) == 0 && (p.rows == 1 || p.stride % N == 0);   // every row on a boundary
    const int64_t runs = (p.vocab + (even ? 0 : N - 1) + 32 * N - 1) / (32 * N);
    if (p.vocab <= 8) {
        tiny_kernel<T><<<(unsigned)((p.rows + 127) / 128), 128, 0, st>>>(p);
        return cudaGetLastError();
    }
    if (runs <= 32 / N) {   // at most 32 places a lane
        if (runs <= 1) launch_short<T, 1>(p, even, st);
        else if (runs <= 2) launch_short<T, 2>(p, even, st);
        else if (runs <= 4) launch_short<T, 4>(p, even, st);
        else launch_short<T, 32 / N>(p, even, st);
        return cudaGetLastError();
    }
    int lg = 0;
    while (runs * 32 > (int64_t)kMaxSegments << lg) lg = lg == 3 ? 5 : lg == 5 ? 7 : lg + 1;   // a run's part, a run, or batches of runs
    // whole batches, and four segments a read: the last may lie beyond the row
    const int cut = 5 - std::min(lg, 5);
    const int segments = (int)(((lg > 5 ? (runs + (1 << (lg - 5)) - 1) >> (lg - 5) : runs) + kBatch - 1) / kBatch * kBatch) << cut;
    const int cluster = cluster_for(p.rows, runs, sm_count());
    if (cluster > 1) return launch_long<T, kFewWarps>(p, cluster, lg, segments, st);
    // about 20 warps an SM, with as few to a row as give that: what a row needs once, it needs of each of its warps
    // (8192 x 32768 bf16: 101 us with one, 117 with eight; 800 x 32768: 15.5 with four, 17.2 with eight, 20.5 with two;
    // 600 x 100003 fp32: 180 with one, 45 with eight), and no more warps than batches (600 x 2600 bf16: 6.8 with eight,
    // 4.4 with four). Long rows that would leave most of a second round of 32 warps an SM empty are shared by two
    // (5000 x 32768 bf16 65.6, 77.7 with one; 8192 x 32768 101.2 and 102.5).
    const int64_t sms = sm_count(), batches = (runs + kBatch - 1) / kBatch;
    int warps = 1;
    while (warps < kFewWarps && warps < batches && p.rows * warps < 20 * sms) warps *= 2;
    if (warps == 1 && batches >= 16 && p.rows > 32 * sms && p.rows < 48 * sms) warps = 2;
    if (warps == 1) return launch_long<T, 1>(p, 1, lg, segments, st);
    if (warps == 2) return launch_long<T, 2>(p, 1, lg, segments, st);
    if (warps == 4) return launch_long<T, 4>(p, 1, lg, segments, st);
    return launch_long<T, kFewWarps>(p, 1, lg, segments, st);
}

// What the gradient of a row needs: p (A + B y) everywhere, p = 2^(y log2 e - log2 s), and more at the given token and
// the alternatives.
struct RowGrad {
    float m, l2, A, B, given;
    int64_t token;   // -1: none
    __device__ __forceinline__ void load(const Grad &p, int64_t row) {
        const float4 st = p.stats[row];
        token = token_of(p.tokens, p.token_bytes, row);
        if (token >= p.vocab) token = -1;
        given = p.g_logprob && token >= 0 ? p.g_logprob[row] : 0.0f;
        const float gh = p.g_entropy ? p.g_entropy[row] : 0.0f;
        float c = (p.g_lse ? p.g_lse[row] : 0.0f) - given;
        if (p.g_top)
            for (int k = 0; k < p.top; k++) c -= p.g_top[row * p.top + k];
        m = st.x, l2 = st.y, A = c - gh * (st.w - st.z), B = -gh;
        if (l2 == INFINITY) A = B = given = 0.0f;   // an empty row's gradient is 0 whatever arrives: 0 times NaN is not
    }
    __device__ __forceinline__ float dense(float x) const {
        const float y = x - m;
        return exp2_approx(fmaf(y, kLog2e, -l2)) * fmaf(B, fmaxf(y, kFloor), A);
    }
    // The same for a vector, in pairs.
    template <int N> __device__ __forceinline__ void dense(float (&v)[N]) const {
        const Pair minus = pair(-m, -m), l = pair(kLog2e, kLog2e), s = pair(-l2, -l2), a = pair(A, A), b = pair(B, B);
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            const Pair y = add(pair(v[2 * i], v[2 * i + 1]), minus);
            const float2 f = split(y);
            const float2 g = split(mul(exp2_approx(fma(y, l, s)), fma(b, pair(fmaxf(f.x, kFloor), fmaxf(f.y, kFloor)), a)));
            v[2 * i] = g.x, v[2 * i + 1] = g.y;
        }
    }
};

__device__ __forceinline__ void store_stream(void *p, const uint4 &v) {
    asm volatile("st.global.cs.v4.u32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Up to 8 entries: a thread a row.
template <typename T> __global__ void __launch_bounds__(128) tiny_grad_kernel(const Grad p) {
    const int64_t row = (int64_t)blockIdx.x * 128 + threadIdx.x;
    if (row >= p.rows) return;
    const T *x = (const T *)p.logits + row * p.stride;
    T *g = (T *)p.grad + row * p.grad_stride;
    RowGrad d;
    d.load(p, row);
    float more[8] = {};
    if (p.g_top)
        for (int k = 0; k < p.top; k++) {
            const int j = p.top_ids[row * p.top + k];
            const float v = p.g_top[row * p.top + k];
#pragma unroll
            for (int i = 0; i < 8; i++) more[i] += i == j ? v : 0.0f;
        }
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (i < p.vocab) {
            const float v = d.dense(to_f(x[i]));
            from_f(d.l2 == INFINITY ? 0.0f : v + (i == d.token ? d.given : 0.0f) + more[i], g[i]);
        }
}

// A warp takes kGradRuns runs of 32 kPer places: a chunk of one row, or ROWS short rows whole. SAME: the logits and the
// gradient of a row lie alike to the 16-byte boundary, so that both move 16 bytes at a time. Bound by HBM: 8192 x 32768
// bf16 188 us, 5.7 TB/s read and written, 0.87 of a copy's rate.
constexpr int kGradRuns = 4;
template <typename T, bool SAME, int ROWS>
__global__ void __launch_bounds__(256) grad_kernel(const Grad p, unsigned chunks) {
    constexpr int N = kPer<T>, RUNS = kGradRuns / ROWS;
    const int lane = threadIdx.x & 31;
    const int64_t it = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int64_t row0 = ROWS > 1 ? it * ROWS : it < ((int64_t)1 << 32) ? (unsigned)it / chunks : it / chunks;
    if (row0 >= p.rows) return;
    const uint32_t u0 = ROWS > 1 ? 0 : (uint32_t)(it - row0 * chunks) * (kGradRuns * 32 * N);
    uint4 q[ROWS][RUNS];
#pragma unroll
    for (int w = 0; w < ROWS; w++) {
        const int64_t row = min(row0 + w, p.rows - 1);
        const T *x = (const T *)p.logits + row * p.stride;
        const uint32_t off = offset_of(x), end = (uint32_t)p.vocab + off;
#pragma unroll
        for (int r = 0; r < RUNS; r++) q[w][r] = load_run<T>(x - off, u0 + r * 32 * N, off, end, lane);
    }
    RowGrad ds[ROWS];
#pragma unroll
    for (int w = 0; w < ROWS; w++) ds[w].load(p, min(row0 + w, p.rows - 1));
#pragma unroll
    for (int w = 0; w < ROWS; w++) {
        const int64_t row = row0 + w;
        if (row >= p.rows) break;
        const RowGrad &d = ds[w];
        const T *x = (const T *)p.logits + row * p.stride;
        T *g = (T *)p.grad + row * p.grad_stride;
        const uint32_t off = offset_of(x), end = (uint32_t)p.vocab + off;
#pragma unroll
        for (int r = 0; r < RUNS; r++) {
            const uint32_t u = u0 + (r * 32 + lane) * N;
            if (u >= end) break;
            float v[N];
            unpack(q[w][r], v, T());
            d.dense(v);
            if (SAME && u >= off && u + N <= end) {
                store_stream(g + (int64_t)u - off, pack(v, T()));
            } else {
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (u + i - off < end - off) from_f(v[i], g[u + i - off]);
            }
        }
        __syncwarp();
        // the given token and the alternatives: written again, whole, so that they are rounded once
        if (d.l2 == INFINITY) continue;   // an empty row
        const int64_t j0 = (int64_t)u0 - off, j1 = min(j0 + RUNS * 32 * N, p.vocab);
        for (int k = lane; k <= (p.g_top ? p.top : 0); k += 32) {
            const int64_t j = k == 0 ? d.token : p.top_ids[row * p.top + k - 1];
            if (j < 0 || j < j0 || j >= j1 || (k > 0 && j == d.token)) continue;
            float more = k == 0 ? d.given : p.g_top[row * p.top + k - 1];
            if (k == 0 && p.g_top)
                for (int i = 0; i < p.top; i++)
                    if (p.top_ids[row * p.top + i] == j) more += p.g_top[row * p.top + i];
            from_f(d.dense(to_f(x[j])) + more, g[j]);
        }
    }
}

template <typename T> cudaError_t launch_grad(const Grad &p, cudaStream_t st) {
    constexpr int N = kPer<T>;
    const bool even = ((uintptr_t)p.logits & 15) == 0 && (p.rows == 1 || p.stride % N == 0);
    const bool same = (((uintptr_t)p.logits ^ (uintptr_t)p.grad) & 15) == 0 &&
                      (p.rows == 1 || (p.stride - p.grad_stride) % N == 0);
    const int64_t places = p.vocab + (even ? 0 : N - 1), chunk = kGradRuns * 32 * N, chunks = (places + chunk - 1) / chunk;
    const int64_t step = std::max<int64_t>(1, ((int64_t)1 << 33) / chunks);   // rows a launch: its grid is below 2^31
    for (int64_t r = 0; r < p.rows; r += step) {
        Grad q = p;
        q.rows = std::min(step, p.rows - r);
        q.logits = (const T *)p.logits + r * p.stride;
        q.grad = (T *)p.grad + r * p.grad_stride;
        q.tokens = (const char *)p.tokens + r * p.token_bytes;
        q.stats += r;
        if (q.top_ids) q.top_ids += r * p.top;
        if (q.g_logprob) q.g_logprob += r;
        if (q.g_entropy) q.g_entropy += r;
        if (q.g_lse) q.g_lse += r;
        if (q.g_top) q.g_top += r * p.top;
        if (p.vocab <= 8) {
            tiny_grad_kernel<T><<<(unsigned)((q.rows + 127) / 128), 128, 0, st>>>(q);
            continue;
        }
        const int64_t runs = (places + 32 * N - 1) / (32 * N);
        const int each = runs <= 1 ? 4 : runs <= 2 ? 2 : 1;   // rows a warp
        const unsigned grid = (unsigned)(((q.rows + each - 1) / each * chunks + 7) / 8);
        const auto launch = [&](auto k) { k<<<grid, 256, 0, st>>>(q, (unsigned)chunks); };
        if (each == 4) launch(same ? grad_kernel<T, true, 4> : grad_kernel<T, false, 4>);
        else if (each == 2) launch(same ? grad_kernel<T, true, 2> : grad_kernel<T, false, 2>);
        else launch(same ? grad_kernel<T, true, 1> : grad_kernel<T, false, 1>);
    }
    return cudaGetLastError();
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
    cudaError_t e = cudaSuccess;
    const int64_t step = (int64_t)1 << 26;   // rows of a launch: its grid stays below 2^31 blocks
    for (int64_t r = 0; r < rows && e == cudaSuccess; r += step) {
        Rows q = p;
        q.rows = std::min(step, rows - r);
        q.tokens = (const char *)d_tokens + r * token_bytes;
        q.logprob += r, q.entropy += r, q.lse += r;
        if (top) q.top_ids += r * top, q.top_logprobs += r * top;
        if (q.stats) q.stats += r;
        const int rc = by_type(dtype, [&](auto t) {
            using T = decltype(t);
            q.logits = (const T *)d_logits + r * row_stride;
            e = launch_rows<T>(q, (cudaStream_t)stream);
        });
        if (rc != YGG_OK) return rc;
    }
    return e == cudaSuccess ? YGG_OK : YGG_E_CUDA;
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
    cudaError_t e = cudaSuccess;
    const int rc = by_type(dtype, [&](auto t) { e = launch_grad<decltype(t)>(p, (cudaStream_t)stream); });
    if (rc != YGG_OK) return rc;
    return e == cudaSuccess ? YGG_OK : YGG_E_CUDA;
}

}  // extern "C"
