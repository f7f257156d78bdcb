// The pages of a cache of stream states: growing, forking, freeing, compacting, and copying in and out.
//
// A pool holds `count` pages of page_bytes each; a page is a stream's state at one point. table[s][0 .. length[s]) are
// the pages of stream s in order (-1 beyond), refs[p] the number of table entries that hold page p (0: free). The last
// page of a stream is its live state and belongs to it alone; the pages before it are snapshots and may be shared.
//   grow    a stream gets a new last page, a copy of its last one (zeros for its first)
//   fork    an empty child gets its parent's first d pages: the first d - 1 shared, the d-th copied into a new page
//   free    a stream lets go of its pages
//   compact with n pages live, the k-th free page below n takes over from the k-th live page at or above n
// New pages are the free ones of the call's beginning in ascending order, given in the order of the call's list: the
// result depends on nothing else. Parents are read as they were before the call, children must be empty. What cannot
// be done is left undone and reported in the status word: an index at or beyond the number of streams, a child that
// holds pages or is named twice (the first one counts), a pool or a table row without room. Negative indices are
// padding. Tables and counts come from the caller and need not fit together: a page beyond the pool, or one to be moved
// that nothing counts, is reported and never used as an address.
//
// Sources and destinations of one call's page copies never overlap: grow and fork write pages that were free, compact
// writes below n and reads at or above it.
#include <stdint.h>

#include <algorithm>

#include "ygg_ops.cuh"

namespace {

using namespace ygg;

enum : int { kBadIndex = 0, kNoRoom = 1, kTimeout = 2 };   // the words of Cache::status

struct Pools {
    const char *src;
    char *dst;
    int64_t src_count, dst_count, page_bytes;
};

struct Cache {
    char *pages;
    int64_t count, page_bytes;   // count < 2^31
    int32_t *table;
    int64_t streams;
    int per_stream;
    int32_t *length, *refs;
    int32_t *status;             // three words, set to 1 by plain stores: they may lie in mapped host memory
    unsigned long long *sync;    // in device memory: how often a block has come to a barrier
    __device__ __forceinline__ Pools pools() const { return {pages, pages, count, count, page_bytes}; }
};

// One page copy: source page (or none: zeros), destination page (or none: nothing to do).
struct Move { int32_t from, to; };

__device__ __forceinline__ void report(int32_t *status, int what) { *(volatile int32_t *)(status + what) = 1; }

constexpr int kPlan = 1024, kWarps = kPlan / 32, kMaxBlocks = 256;

// A barrier of all blocks of a cooperative launch. The cache's counter goes up by the number of blocks at each barrier and is
// never reset (its calls are ordered and their launches have one size), so that one look before the first barrier tells
// how far it will have come at each. The wait is bounded (false: it ran out, and the cache is reported as unusable). After
// one that ran out the counter no longer tells how many came, and a later barrier would open too early: its top bit is set
// then, at which every barrier gives up, this call's and those of the calls behind it.
constexpr unsigned long long kDead = 1ull << 63;
struct AllBlocks {
    unsigned long long *count, target = 0;
    int32_t *status;
    __device__ __forceinline__ explicit AllBlocks(const Cache &c) : count(c.sync), status(c.status) {
        if (gridDim.x > 1 && threadIdx.x == 0) target = look() / gridDim.x * gridDim.x;
    }
    __device__ __forceinline__ unsigned long long look() const {
        unsigned long long v;
        asm volatile("ld.acquire.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(count) : "memory");
        return v;
    }
    __device__ __forceinline__ bool meet() {
        __shared__ int fine;
        __syncthreads();
        if (gridDim.x == 1) return true;
        if (threadIdx.x == 0) {
            target += gridDim.x;
            asm volatile("red.release.gpu.global.add.u64 [%0], 1;" ::"l"(count) : "memory");
            const long long t0 = clock64();
            unsigned long long v;
            while (!((v = look()) & kDead) && v < target)
                if (clock64() - t0 > 2000000000LL) atomicOr(count, kDead);
            fine = !(v & kDead);
            if (!fine) report(status, kTimeout);
        }
        __syncthreads();
        return fine;
    }
};

// Exclusive prefix sum over the block's threads of v; `total` receives the sum.
__device__ __forceinline__ int block_scan(int v, int *scratch, int &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(~0u, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) scratch[warp] = x;
    __syncthreads();
    int w = scratch[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(~0u, w, o);
        if (lane >= o) w += y;
    }
    total = __shfl_sync(~0u, w, 31);
    return x - v + (warp ? __shfl_sync(~0u, w, warp - 1) : 0);
}
// How many of the block's threads have it set, and how many before this one.
__device__ __forceinline__ int block_count(bool v, int *scratch, int &before) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned who = __ballot_sync(~0u, v);
    __syncthreads();
    if (lane == 0) scratch[warp] = __popc(who);
    __syncthreads();
    int w = scratch[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(~0u, w, o);
        if (lane >= o) w += y;
    }
    before = __popc(who & ((1u << lane) - 1)) + (warp ? __shfl_sync(~0u, w, warp - 1) : 0);
    return __shfl_sync(~0u, w, 31);
}
// The sum of the blocks' counts (`own`: this block's), and of those before this block. They come from other blocks: past
// the L1.
__device__ __forceinline__ int over_blocks(const int *counts, int own, int *scratch, int &before) {
    if (gridDim.x == 1) {
        before = 0;
        return own;
    }
    int total;
    const int mine = threadIdx.x < gridDim.x ? __ldcg(counts + threadIdx.x) : 0;
    const int at = block_scan(mine, scratch, total);
    __shared__ int here;
    if (threadIdx.x == blockIdx.x) here = at;
    __syncthreads();
    before = here;
    return total;
}

// The block's share of n things, side by side.
struct Range { int64_t from, to; };
__device__ __forceinline__ Range share(int64_t n) {
    return {n * blockIdx.x / gridDim.x, n * (blockIdx.x + 1) / gridDim.x};
}

__device__ __forceinline__ int length_of(const Cache &c, int64_t s) {
    return max(0, min(c.length[s], c.per_stream));
}
__device__ __forceinline__ bool is_page(const Cache &c, int p) { return p >= 0 && p < c.count; }

// 2^ the result: the lanes of a row of a page of so many units.
__host__ __device__ constexpr int lanes_log(int64_t units) {
    return units > 16 ? 5 : units > 8 ? 4 : units > 4 ? 3 : units > 2 ? 2 : units > 1;
}
// Whole pages in units of V, `n` of them, by the threads of `all` from `thread` on; move(i) says which. A warp (part of it
// where a page has less units) copies a row of its lanes' units of a page, eight rows side by side at a time: where they
// lie, then all loads, then all stores. So one look at the list serves 4 KB, and 128 KB of an SM are in flight: 30 000 pages
// of 5 KB in 47 us inside a compact, the rate of a plain copy (58 with eight units a thread spread over the grid, each looked
// up).
template <typename V, int kRows = 8, typename F>
__device__ __forceinline__ void copy_moves(const Pools &c, int64_t n, int64_t thread, int64_t all, F move) {
    const int64_t units = c.page_bytes / (int64_t)sizeof(V);
    const int log = lanes_log(units), lanes = 1 << log, lane = threadIdx.x & (lanes - 1);
    const int64_t rows = (units + lanes - 1) >> log, items = n * rows, step = (all >> log) * kRows;
    for (int64_t q0 = (thread >> log) * kRows; q0 < items; q0 += step) {
        int64_t i = items < ((int64_t)1 << 32) ? (uint32_t)q0 / (uint32_t)rows : q0 / rows, r = q0 - i * rows;
        int64_t from[kRows], to[kRows];   // -1: zeros; nothing to do
        decltype(move(0)) m{-1, -1};
#pragma unroll
        for (int k = 0; k < kRows; k++) {
            if ((k == 0 || r == 0) && i < n) m = move(i);
            const int64_t u = r * lanes + lane;
            const bool go = i < n && u < units && m.to >= 0 && m.to < c.dst_count && m.from < c.src_count;
            to[k] = go ? (int64_t)m.to * c.page_bytes + u * (int64_t)sizeof(V) : -1;
            from[k] = go && m.from >= 0 ? (int64_t)m.from * c.page_bytes + u * (int64_t)sizeof(V) : -1;
            if (++r == rows) r = 0, i++;
        }
        V v[kRows];
#pragma unroll
        for (int k = 0; k < kRows; k++) {
            v[k] = V{};
            if (from[k] >= 0) v[k] = __ldcs((const V *)(c.src + from[k]));
        }
#pragma unroll
        for (int k = 0; k < kRows; k++)
            if (to[k] >= 0) __stcs((V *)(c.dst + to[k]), v[k]);
    }
}

constexpr int32_t kClaim = INT32_MIN;

// grow and fork, in three parts between barriers:
//   claims: a fork claims its (empty) child by the smallest index of the list in the child's first table entry, a grow its
//           stream in the entry after its last page (-1 before); the blocks count the free pages of their shares
//   order:  the free pages in ascending order, as many as may be wanted; the blocks count the claims that held
//   pages:  the k-th claim that held takes the k-th free page; table rows, counts, and the page's copy
// info[i]: the pages that entry i takes over, or -1: nothing to do.
// 65 536 forks of 512 B: 21 us, 11 of them the barriers and three rounds of dependent loads; 8 forks of 5 KB 6.7 us.
template <typename V>
__global__ void __launch_bounds__(kPlan, 1)
    fork_kernel(const Cache c, const int32_t *parents, const int32_t *children, const int32_t *depth, int64_t n,
                int32_t *info, int32_t *order, Move *moves, int *counts) {
    __shared__ int scratch[kWarps];
    AllBlocks blocks(c);
    const bool grow = children == nullptr;
    const Range mine = share(n), pages = share(c.count);
    int *const free_counts = counts, *const held_counts = counts + kMaxBlocks;
    const auto slot = [&](int64_t child, int taken) { return c.table + child * c.per_stream + (grow ? taken : 0); };
    // a thread's first entry stays in registers (all of them, up to 1024 a block); the others are read again
    int32_t parent0 = -1, child0 = -1;
    int taken0 = -1;

    const int64_t first_page = pages.from + threadIdx.x;
    const bool free0 = first_page < pages.to && c.refs[first_page] == 0;   // its load runs under the claims
    for (int64_t i = mine.from + threadIdx.x; i < mine.to; i += kPlan) {
        const int32_t parent = parents[i], child = grow ? parent : children[i];
        int taken = -1;
        if (parent >= 0 && child >= 0) {
            if (parent >= c.streams || child >= c.streams) {
                report(c.status, kBadIndex);
            } else {
                const int held = length_of(c, parent), other = grow ? 0 : length_of(c, child);
                if (grow) {
                    taken = held;
                    if (held >= c.per_stream) {
                        report(c.status, kNoRoom);
                        taken = -1;
                    }
                } else {
                    taken = depth ? min(depth[i], held) : held;
                    if (taken <= 0) {   // a parent without pages: a child without
                        taken = -1;
                    } else if (other != 0) {
                        report(c.status, kBadIndex);
                        taken = -1;
                    }
                }
            }
        }
        if (taken >= 0) atomicMin(slot(child, taken), kClaim + (int32_t)i);
        if (i < mine.from + kPlan) parent0 = parent, child0 = child, taken0 = taken;
        else info[i] = taken;
    }
    int free_here = __syncthreads_count(free0), before;
    for (int64_t p0 = pages.from + kPlan; p0 < pages.to; p0 += kPlan) {
        const int64_t p = p0 + threadIdx.x;
        free_here += __syncthreads_count(p < pages.to && c.refs[p] == 0);
    }
    if (threadIdx.x == 0) free_counts[blockIdx.x] = free_here;
    if (!blocks.meet()) return;

    const int32_t claim0 = taken0 >= 0 ? __ldcg(slot(child0, taken0)) : 0;   // its load runs under the free pages' list
    int free_before;
    const int available = over_blocks(free_counts, free_here, scratch, free_before);
    for (int64_t p0 = pages.from; p0 < pages.to && free_before < n; p0 += kPlan) {
        const int64_t p = p0 + threadIdx.x;
        const bool is_free = p0 == pages.from ? free0 : p < pages.to && c.refs[p] == 0;
        const int here = block_count(is_free, scratch, before);
        if (is_free && free_before + before < n) order[free_before + before] = (int32_t)p;
        free_before += here;
    }
    int held = 0;
    for (int64_t i0 = mine.from; i0 < mine.to; i0 += kPlan) {
        const int64_t i = i0 + threadIdx.x;
        const bool first = i0 == mine.from;
        const int taken = i >= mine.to ? -1 : first ? taken0 : info[i];
        bool holds = false;
        if (taken >= 0) {
            const int32_t claim = first ? claim0 : __ldcg(slot(grow ? parents[i] : children[i], taken));
            holds = claim == kClaim + (int32_t)i;
            if (!holds) {   // named twice
                report(c.status, kBadIndex);
                if (first) taken0 = -1;
                else info[i] = -1;
            }
        }
        held += __syncthreads_count(holds);
    }
    if (threadIdx.x == 0) held_counts[blockIdx.x] = held;
    // what the first entry will copy does not wait for its place
    const int32_t source0 = taken0 > 0 ? c.table[(int64_t)parent0 * c.per_stream + taken0 - 1] : -1;
    if (!blocks.meet()) return;

    int given;
    over_blocks(held_counts, held, scratch, given);
    for (int64_t i0 = mine.from; i0 < mine.to; i0 += kPlan) {
        const int64_t i = i0 + threadIdx.x;
        const bool first = i0 == mine.from;
        const int taken = i >= mine.to ? -1 : first ? taken0 : info[i];
        const int here = block_count(taken >= 0, scratch, before);
        Move m{-1, -1};
        if (taken >= 0) {
            const int64_t parent = first ? parent0 : parents[i], child = first ? child0 : grow ? parent : children[i];
            int32_t *row = c.table + child * c.per_stream;
            if (given + before < available) {
                const int32_t *from = c.table + parent * c.per_stream;
                m.to = __ldcg(order + given + before);
                m.from = first ? source0 : taken > 0 ? from[taken - 1] : -1;
                if (m.from >= c.count) {   // a table that names a page beyond the pool
                    report(c.status, kBadIndex);
                    m.from = -1;
                }
                if (!grow)
                    for (int j = 0; j < taken - 1; j++) {
                        const int32_t page = from[j];
                        row[j] = page;
                        if (is_page(c, page)) atomicAdd(&c.refs[page], 1);
                        else report(c.status, kBadIndex);
                    }
                row[grow ? taken : taken - 1] = m.to;
                c.refs[m.to] = 1;
                c.length[child] = grow ? taken + 1 : taken;
            } else {   // the claim is taken back
                report(c.status, kNoRoom);
                *slot(child, taken) = -1;
            }
        }
        if (i < mine.to) moves[i] = m;
        given += here;
    }
    __syncthreads();
    const Move *own = moves + mine.from;
    copy_moves<V>(c.pools(), mine.to - mine.from, threadIdx.x, kPlan, [&](int64_t i) { return own[i]; });
}

// A thread a stream: scattered words, a few us for 32 768 streams.
__global__ void __launch_bounds__(256) free_kernel(const Cache c, const int32_t *streams, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t s = streams[i];
        if (s < 0) continue;
        if (s >= c.streams) {
            report(c.status, kBadIndex);
            continue;
        }
        const int32_t first = c.table[s * c.per_stream];                   // its load runs under the exchange
        const int held = min(atomicExch(&c.length[s], 0), c.per_stream);   // a stream named twice is freed once
        for (int j = 0; j < held; j++) {
            const int32_t p = j ? c.table[s * c.per_stream + j] : first;
            if (is_page(c, p)) atomicSub(&c.refs[p], 1);
            else report(c.status, kBadIndex);
            c.table[s * c.per_stream + j] = -1;
        }
    }
}

// compact, in three parts between barriers. rank(p): the live pages before p.
//   count:  the live pages of the blocks' shares, n in all
//   lists:  holes[k], the k-th free page below n (k = p - rank(p)); movers[rank(p)] = p and ranks[p] = rank(p) for the live
//           pages at or above n, whose k is rank(p) less the live pages below n (ranks[p] = -1 for the free ones: a table
//           that names one is reported, and nothing is looked up for it)
//   moves:  tables, counts and pages
// Bound by the copies: 30 000 moves of 5 KB among 65 536 streams 60 us, 47 of them the copies; few streams 8.5 us, latency.
template <typename V>
__global__ void __launch_bounds__(kPlan, 1)
    compact_kernel(const Cache c, int32_t *live, int32_t *holes, int32_t *movers, int32_t *ranks, int *counts) {
    __shared__ int scratch[kWarps];
    AllBlocks blocks(c);
    const Range pages = share(c.count);
    int here = 0, before, rank0;
    for (int64_t p0 = pages.from; p0 < pages.to; p0 += kPlan) {
        const int64_t p = p0 + threadIdx.x;
        here += __syncthreads_count(p < pages.to && c.refs[p] > 0);
    }
    if (threadIdx.x == 0) counts[blockIdx.x] = here;
    if (!blocks.meet()) return;

    const int n = over_blocks(counts, here, scratch, rank0);
    int *const below = counts + kMaxBlocks;   // the live pages below n
    if (threadIdx.x == 0 && n == c.count && blockIdx.x == 0) *below = n;
    for (int64_t p0 = pages.from; p0 < pages.to; p0 += kPlan) {
        const int64_t p = p0 + threadIdx.x;
        const bool used = p < pages.to && c.refs[p] > 0;
        const int count = block_count(used, scratch, before);
        const int rank = rank0 + before;
        if (p < pages.to) {
            if (p == n) *below = rank;
            if (p < n && !used) holes[p - rank] = (int32_t)p;
            if (p >= n) ranks[p] = used ? rank : -1;
            if (p >= n && used) movers[rank] = (int32_t)p;
        }
        rank0 += count;
    }
    if (!blocks.meet()) return;

    const int low = __ldcg(below), moving = n - low;
    const int64_t thread = (int64_t)blockIdx.x * kPlan + threadIdx.x, all = (int64_t)gridDim.x * kPlan;
    if (thread == 0) *live = n;
    if (moving == 0) return;
    const int64_t entries = c.streams * c.per_stream;
    for (int64_t i = thread; i < entries; i += all) {
        const int32_t p = c.table[i];
        if (p < n) continue;
        const int rank = p < c.count ? __ldcg(ranks + p) : -1;
        if (rank >= 0) c.table[i] = __ldcg(holes + rank - low);
        else report(c.status, kBadIndex);   // a page beyond the pool, or one that nothing counts
    }
    for (int64_t k = thread; k < moving; k += all) {
        const int32_t from = __ldcg(movers + low + k), to = __ldcg(holes + k);
        c.refs[to] = c.refs[from];
        c.refs[from] = 0;
    }
    copy_moves<V>(c.pools(), moving, thread, all, [&](int64_t k) { return Move{__ldcg(movers + low + k), __ldcg(holes + k)}; });
}

// Copies of whole pages in units of V, bound by HBM: a read of 30 000 pages of 5 KB, found through tables, in 52 us, 0.9 of a
// copy's rate (the moves inside a compact take 47). Where from[i] and to[i] are is what Where says: pages outside their pool
// are skipped.
struct Where {
    const char *src;
    char *dst;
    int64_t src_count, dst_count;
    const int32_t *src_ids, *dst_ids;   // null: page i
    const int32_t *streams, *table, *length;   // the last pages of streams, on the side that `last` names
    int64_t stream_count;
    int per_stream, last;           // 0: none, 1: source, 2: destination
    int64_t n;
    int32_t *status;
};

struct WideMove { int64_t from, to; };
__device__ __forceinline__ WideMove resolve(const Where &w, int64_t i) {
    const WideMove none{-1, -1};
    int64_t from = w.src_ids ? w.src_ids[i] : i;
    int64_t to = w.dst_ids ? w.dst_ids[i] : i;
    if (w.last) {
        const int64_t s = w.streams[i];
        if (s >= w.stream_count) report(w.status, kBadIndex);
        int32_t p = -1;
        if (s >= 0 && s < w.stream_count) {
            const int n = min(w.length[s], w.per_stream);
            if (n > 0) p = w.table[s * w.per_stream + n - 1];
        }
        if (p >= (w.last == 1 ? w.src_count : w.dst_count)) {   // a table that names a page beyond the pool
            report(w.status, kBadIndex);
            p = -1;
        }
        (w.last == 1 ? from : to) = p;
        if (w.last == 1) return {from, to};   // a stream without pages reads as zeros
    } else if (from >= w.src_count || to >= w.dst_count) {
        report(w.status, kBadIndex);
    }
    return from >= 0 && from < w.src_count && to >= 0 && to < w.dst_count ? WideMove{from, to} : none;
}

template <typename V, int ROWS> __global__ void __launch_bounds__(256) copy_kernel(const Where w, int64_t page_bytes) {
    copy_moves<V, ROWS>({w.src, w.dst, w.src_count, w.dst_count, page_bytes}, w.n, (int64_t)blockIdx.x * 256 + threadIdx.x,
                  (int64_t)gridDim.x * 256, [&](int64_t i) { return resolve(w, i); });
}

int blocks_for(int64_t threads) { return (int)std::max<int64_t>(1, std::min<int64_t>((threads + 255) / 256, 148 * 16)); }

// f of a unit that pages at `mix` (addresses and sizes, or'ed) can be copied in.
template <typename F> auto by_unit(uintptr_t mix, F f) {
    return mix % 16 == 0 ? f(uint4()) : mix % 4 == 0 ? f(uint32_t()) : f(uint8_t());
}

int copy_pages(const Where &w, int64_t page_bytes, cudaStream_t st) {
    return by_unit((uintptr_t)w.src | (uintptr_t)w.dst | (uintptr_t)page_bytes, [&](auto v) {
        using V = decltype(v);
        const int64_t units = page_bytes / (int64_t)sizeof(V), lanes = 1 << lanes_log(units);
        const int64_t rows = w.n * ((units + lanes - 1) / lanes);
        // eight rows a warp once the rows fill the SMs: 30 000 pages of 5 KB 52 us, 72 with one; 8 pages 8.0 and 6.1
        if (rows * lanes >= (int64_t)sm_count() * 1024) copy_kernel<V, 8><<<blocks_for((rows + 7) / 8 * lanes), 256, 0, st>>>(w, page_bytes);
        else copy_kernel<V, 1><<<blocks_for(rows * lanes), 256, 0, st>>>(w, page_bytes);
        return cudaGetLastError() == cudaSuccess ? YGG_OK : YGG_E_CUDA;
    });
}

// One block where its own work is short, else a block an SM that meet at barriers.
template <typename... P, typename... A>
int launch_plan(void (*kernel)(P...), int64_t things, int64_t bytes, cudaStream_t st, A... args) {
    const bool small = things <= 4096 && bytes <= (128 << 10);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(small ? 1 : std::min(kMaxBlocks, sm_count()));
    cfg.blockDim = dim3(kPlan);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeCooperative;
    attr[0].val.cooperative = 1;
    cfg.attrs = attr;
    cfg.numAttrs = small ? 0 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? YGG_OK : YGG_E_CUDA;
}

int cache_of(const ygg_cache_t *h, Cache &c) {
    if (!h || !h->pages || !h->table || !h->length || !h->refs || !h->status || !h->sync || ((uintptr_t)h->sync & 7) || h->page_bytes < 1 || h->page_count < 1 ||
        h->page_count > INT32_MAX || h->streams < 1 || h->streams > INT32_MAX || h->per_stream < 1 ||
        h->page_bytes > ((int64_t)1 << 40))
        return YGG_E_ARG;
    c = {(char *)h->pages, h->page_count, h->page_bytes, h->table, h->streams, h->per_stream, h->length, h->refs,
         h->status, (unsigned long long *)h->sync};
    return YGG_OK;
}

int done() { return cudaGetLastError() == cudaSuccess ? YGG_OK : YGG_E_CUDA; }

int64_t rounded(int64_t v) { return (v + 3) / 4 * 4; }

}  // namespace

extern "C" {

size_t ygg_cache_workspace(const ygg_cache_t *h, int64_t n) {
    if (!h || n < 0 || h->page_count < 1) return 0;
    // counts; fork and grow: info [n], order [n], moves [n]; compact: holes, movers, ranks [count]
    return sizeof(int32_t) * (2 * kMaxBlocks + 4 * (size_t)rounded(std::max(n, h->page_count)));
}

int ygg_cache_fork(int device, const ygg_cache_t *h, int64_t n, const int32_t *d_parents, const int32_t *d_children,
                   const int32_t *d_depth, void *d_workspace, size_t workspace_bytes, void *stream) {
    Cache c;
    if (cache_of(h, c) != YGG_OK || n < 0 || n > INT32_MAX / 2) return YGG_E_ARG;
    if (n == 0) return YGG_OK;
    if (!d_parents || !d_workspace || ((uintptr_t)d_workspace & 15) || workspace_bytes < ygg_cache_workspace(h, n))
        return YGG_E_ARG;
    OnDevice on(device);
    if (!on.ok) return YGG_E_DEVICE;
    const cudaStream_t st = (cudaStream_t)stream;
    int *counts = (int *)d_workspace;
    int32_t *info = counts + 2 * kMaxBlocks, *order = info + rounded(n);
    Move *moves = (Move *)(order + rounded(n));
    return by_unit((uintptr_t)c.pages | (uintptr_t)c.page_bytes, [&](auto v) {
        return launch_plan(fork_kernel<decltype(v)>, std::max(n, c.count), n * c.page_bytes, st, c, d_parents, d_children,
                           d_depth, n, info, order, moves, counts);
    });
}

int ygg_cache_free(int device, const ygg_cache_t *h, int64_t n, const int32_t *d_streams, void *stream) {
    Cache c;
    if (cache_of(h, c) != YGG_OK || n < 0) return YGG_E_ARG;
    if (n == 0) return YGG_OK;
    if (!d_streams) return YGG_E_ARG;
    OnDevice on(device);
    if (!on.ok) return YGG_E_DEVICE;
    free_kernel<<<blocks_for(n), 256, 0, (cudaStream_t)stream>>>(c, d_streams, n);
    return done();
}

int ygg_cache_compact(int device, const ygg_cache_t *h, int32_t *d_live, void *d_workspace,
                      size_t workspace_bytes, void *stream) {
    Cache c;
    if (cache_of(h, c) != YGG_OK || !d_live || !d_workspace || ((uintptr_t)d_workspace & 15) ||
        workspace_bytes < ygg_cache_workspace(h, 0))
        return YGG_E_ARG;
    OnDevice on(device);
    if (!on.ok) return YGG_E_DEVICE;
    const cudaStream_t st = (cudaStream_t)stream;
    int *counts = (int *)d_workspace;
    int32_t *holes = counts + 2 * kMaxBlocks, *movers = holes + rounded(c.count), *ranks = movers + rounded(c.count);
    return by_unit((uintptr_t)c.pages | (uintptr_t)c.page_bytes, [&](auto v) {
        return launch_plan(compact_kernel<decltype(v)>, std::max(c.count, c.streams * c.per_stream),
                           c.count / 4 * c.page_bytes, st, c, d_live, holes, movers, ranks, counts);
    });
}

int ygg_cache_read(int device, const ygg_cache_t *h, int64_t n, const int32_t *d_streams, void *d_batch, void *stream) {
    Cache c;
    if (cache_of(h, c) != YGG_OK || n < 0) return YGG_E_ARG;
    if (n == 0) return YGG_OK;
    if (!d_streams || !d_batch) return YGG_E_ARG;
    OnDevice on(device);
    if (!on.ok) return YGG_E_DEVICE;
    Where w{c.pages, (char *)d_batch, c.count, n, nullptr, nullptr, d_streams, c.table, c.length, c.streams, c.per_stream, 1,
            n, c.status};
    return copy_pages(w, c.page_bytes, (cudaStream_t)stream);
}

int ygg_cache_write(int device, const ygg_cache_t *h, int64_t n, const int32_t *d_streams, const void *d_batch,
                    void *stream) {
    Cache c;
    if (cache_of(h, c) != YGG_OK || n < 0) return YGG_E_ARG;
    if (n == 0) return YGG_OK;
    if (!d_streams || !d_batch) return YGG_E_ARG;
    OnDevice on(device);
    if (!on.ok) return YGG_E_DEVICE;
    Where w{(const char *)d_batch, c.pages, n, c.count, nullptr, nullptr, d_streams, c.table, c.length, c.streams,
            c.per_stream, 2, n, c.status};
    return copy_pages(w, c.page_bytes, (cudaStream_t)stream);
}

int ygg_cache_copy(int device, const ygg_cache_t *h, int64_t n, const int32_t *d_from, const int32_t *d_to, void *stream) {
    Cache c;
    if (cache_of(h, c) != YGG_OK || n < 0) return YGG_E_ARG;
    if (n == 0) return YGG_OK;
    if (!d_from || !d_to) return YGG_E_ARG;
    OnDevice on(device);
    if (!on.ok) return YGG_E_DEVICE;
    Where w{c.pages, c.pages, c.count, c.count, d_from, d_to, nullptr, nullptr, nullptr, 0, 0, 0, n, c.status};
    return copy_pages(w, c.page_bytes, (cudaStream_t)stream);
}

}  // extern "C"
