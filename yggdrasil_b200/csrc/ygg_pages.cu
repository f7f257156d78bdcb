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
// padding.
//
// Sources and destinations of one call's page copies never overlap: grow and fork write pages that were free, compact
// writes below n and reads at or above it.
#include <stdint.h>

#include <algorithm>

#include "ygg_ops.cuh"

namespace {

using namespace ygg;

enum : int { kBadIndex = 0, kNoRoom = 1 };   // the words of Cache::status

struct Cache {
    char *pages;
    int64_t count, page_bytes;   // count < 2^31
    int32_t *table;
    int64_t streams;
    int per_stream;
    int32_t *length, *refs;
    int32_t *status;             // two words, set to 1 by plain stores: they may lie in mapped host memory
};

// One page copy: source page (or none: zeros), destination page (or none: nothing to do).
struct Move { int32_t from, to; };

__device__ __forceinline__ void report(int32_t *status, int what) { *(volatile int32_t *)(status + what) = 1; }

constexpr int kPlan = 1024;

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
    int before = 0;
    total = 0;
    for (int w = 0; w < kPlan / 32; w++) {
        if (w == warp) before = total;
        total += scratch[w];
    }
    return before + x - v;
}

__device__ __forceinline__ int length_of(const Cache &c, int64_t s) {
    return max(0, min(c.length[s], c.per_stream));
}
__device__ __forceinline__ bool is_page(const Cache &c, int p) { return p >= 0 && p < c.count; }

// What a grow or a fork does, before room is looked for: the pages taken over and whether it can be done at all.
struct Wish { int64_t parent, child; int taken; bool ok; };

__device__ __forceinline__ Wish wish(const Cache &c, const int32_t *parents, const int32_t *children,
                                     const int32_t *depth, int64_t i) {
    Wish w{parents[i], children ? children[i] : parents[i], 0, false};
    if (w.parent < 0 || w.child < 0) return w;
    if (w.parent >= c.streams || w.child >= c.streams) {
        report(c.status, kBadIndex);
        return w;
    }
    const int n = length_of(c, w.parent);
    if (!children) {
        w.taken = n;
        w.ok = true;
        return w;
    }
    w.taken = depth ? min(depth[i], n) : n;
    if (w.taken <= 0) return w;   // an empty parent: the child stays empty
    w.ok = true;
    return w;
}

constexpr int32_t kClaim = INT32_MIN;

// fork: the first of a child's forks claims it by the smallest index in its (empty) table row, -1 before.
// grow: likewise in the slot after its last page.
__device__ __forceinline__ int32_t *claim_slot(const Cache &c, const Wish &w, bool grow) {
    return c.table + w.child * c.per_stream + (grow ? w.taken : 0);
}

__global__ void __launch_bounds__(kPlan) plan_kernel(const Cache c, const int32_t *parents, const int32_t *children,
                                                     const int32_t *depth, int64_t n, int32_t *order, Move *moves) {
    __shared__ int scratch[kPlan / 32];
    __shared__ int found;
    const bool grow = children == nullptr;
    int total;
    // the free pages in ascending order, as many as may be wanted
    int free_before = 0;
    for (int64_t p0 = 0; p0 < c.count && free_before < n; p0 += kPlan) {
        const int64_t p = p0 + threadIdx.x;
        const bool is_free = p < c.count && c.refs[p] == 0;
        const int at = free_before + block_scan(is_free, scratch, total);
        if (is_free && at < n) order[at] = (int32_t)p;
        free_before += total;
    }
    const int available = (int)min((int64_t)free_before, n);
    if (threadIdx.x == 0) found = available;
    // claims
    for (int64_t i = threadIdx.x; i < n; i += kPlan) {
        const Wish w = wish(c, parents, children, depth, i);
        if (!w.ok) continue;
        if (grow ? w.taken >= c.per_stream : length_of(c, w.child) != 0) {
            report(c.status, grow ? kNoRoom : kBadIndex);
            continue;
        }
        atomicMin(claim_slot(c, w, grow), kClaim + (int32_t)i);
    }
    __syncthreads();
    // pages in the order of the list
    int given = 0;
    for (int64_t i0 = 0; i0 < n; i0 += kPlan) {
        const int64_t i = i0 + threadIdx.x;
        Wish w{};
        bool mine = false;
        if (i < n) {
            w = wish(c, parents, children, depth, i);
            if (w.ok && !(grow ? w.taken >= c.per_stream : length_of(c, w.child) != 0)) {
                mine = *(volatile int32_t *)claim_slot(c, w, grow) == kClaim + (int32_t)i;
                if (!mine) report(c.status, kBadIndex);   // named twice
            }
        }
        const int at = given + block_scan(mine, scratch, total);
        given += total;
        if (i < n) {
            Move m{-1, -1};
            if (mine && at < found) {
                m.to = order[at];
                m.from = w.taken > 0 ? c.table[w.parent * c.per_stream + w.taken - 1] : -1;
            } else if (mine) {
                report(c.status, kNoRoom);
            }
            moves[i] = m;
        }
    }
    __syncthreads();
    // the claims that got no page are taken back; the others become table rows
    for (int64_t i = threadIdx.x; i < n; i += kPlan) {
        const Move m = moves[i];
        const int64_t child = children ? children[i] : parents[i], parent = parents[i];
        if (child < 0 || parent < 0 || child >= c.streams || parent >= c.streams) continue;
        int32_t *row = c.table + child * c.per_stream;
        if (m.to < 0) {
            const Wish w = wish(c, parents, children, depth, i);
            if (w.ok && (grow ? w.taken < c.per_stream : true)) {
                int32_t *slot = claim_slot(c, w, grow);
                if (*slot == kClaim + (int32_t)i) *slot = -1;
            }
            continue;
        }
        const Wish w = wish(c, parents, children, depth, i);
        if (!grow) {
            const int32_t *from = c.table + parent * c.per_stream;
            for (int j = 0; j < w.taken - 1; j++) {
                row[j] = from[j];
                if (is_page(c, from[j])) atomicAdd(&c.refs[from[j]], 1);
            }
        }
        row[grow ? w.taken : w.taken - 1] = m.to;
        c.refs[m.to] = 1;
        c.length[child] = grow ? w.taken + 1 : w.taken;
    }
}

__global__ void __launch_bounds__(256) free_kernel(const Cache c, const int32_t *streams, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t s = streams[i];
        if (s < 0) continue;
        if (s >= c.streams) {
            report(c.status, kBadIndex);
            continue;
        }
        const int held = min(atomicExch(&c.length[s], 0), c.per_stream);   // a stream named twice is freed once
        for (int j = 0; j < held; j++) {
            const int32_t p = c.table[s * c.per_stream + j];
            if (is_page(c, p)) atomicSub(&c.refs[p], 1);
            c.table[s * c.per_stream + j] = -1;
        }
    }
}

// compact: the moves, and renumber[p] for each page.
__global__ void __launch_bounds__(kPlan) compact_plan_kernel(const Cache c, int32_t *live, int32_t *moved,
                                                             int32_t *renumber, Move *moves) {
    __shared__ int scratch[kPlan / 32];
    int total, n = 0;
    for (int64_t p0 = 0; p0 < c.count; p0 += kPlan) {
        const int64_t p = p0 + threadIdx.x;
        block_scan(p < c.count && c.refs[p] > 0, scratch, total);
        n += total;
    }
    int holes = 0, movers = 0;
    for (int64_t p0 = 0; p0 < c.count; p0 += kPlan) {
        const int64_t p = p0 + threadIdx.x;
        const bool used = p < c.count && c.refs[p] > 0;
        const bool hole = p < n && !used, mover = p >= n && used;
        int at = holes + block_scan(hole, scratch, total);
        holes += total;
        if (hole) moves[at].to = (int32_t)p;
        at = movers + block_scan(mover, scratch, total);
        movers += total;
        if (mover) moves[at].from = (int32_t)p;
        if (p < c.count) renumber[p] = (int32_t)p;
    }
    __syncthreads();
    for (int k = threadIdx.x; k < movers; k += kPlan) {
        const Move m = moves[k];
        renumber[m.from] = m.to;
        c.refs[m.to] = c.refs[m.from];
        c.refs[m.from] = 0;
    }
    if (threadIdx.x == 0) {
        *live = n;
        *moved = movers;
    }
}

__global__ void __launch_bounds__(256) renumber_kernel(const Cache c, const int32_t *renumber) {
    const int64_t n = c.streams * c.per_stream;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int32_t p = c.table[i];
        if (is_page(c, p) && renumber[p] != p) c.table[i] = renumber[p];
    }
}

// Copies of whole pages in units of V. Where from[i] and to[i] are is what Where says: pages outside their pool are
// skipped.
struct Where {
    const char *src;
    char *dst;
    int64_t src_count, dst_count;
    const Move *moves;              // or
    const int32_t *src_ids, *dst_ids;   // null: page i
    const int32_t *streams, *table, *length;   // the last pages of streams, on the side that `last` names
    int64_t stream_count;
    int per_stream, last;           // 0: none, 1: source, 2: destination
    const int32_t *n_of;            // the number of copies on the device, or null
    int64_t n;
    int32_t *status;
};

__device__ __forceinline__ bool resolve(const Where &w, int64_t i, bool first, int64_t &from, int64_t &to) {
    if (w.moves) {
        from = w.moves[i].from;
        to = w.moves[i].to;
        return to >= 0 && to < w.dst_count && from < w.src_count;   // from < 0: zeros
    }
    from = w.src_ids ? w.src_ids[i] : i;
    to = w.dst_ids ? w.dst_ids[i] : i;
    if (w.last) {
        const int64_t s = w.streams[i];
        if (s >= w.stream_count && first) report(w.status, kBadIndex);
        int32_t p = -1;
        if (s >= 0 && s < w.stream_count) {
            const int n = min(w.length[s], w.per_stream);
            if (n > 0) p = w.table[s * w.per_stream + n - 1];
        }
        (w.last == 1 ? from : to) = p;
        if (w.last == 1) return from < w.src_count;                 // a stream without pages reads as zeros
    } else if (first && (from >= w.src_count || to >= w.dst_count)) {
        report(w.status, kBadIndex);
    }
    return from >= 0 && from < w.src_count && to >= 0 && to < w.dst_count;
}

template <typename V> __global__ void __launch_bounds__(256) copy_kernel(const Where w, int64_t page_bytes) {
    const int64_t units = page_bytes / sizeof(V), n = w.n_of ? *w.n_of : w.n, all = n * units;
    for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < all; u += (int64_t)gridDim.x * 256) {
        const int64_t i = u / units, at = u - i * units;
        int64_t from, to;
        if (!resolve(w, i, at == 0, from, to)) continue;
        V v{};
        if (from >= 0) v = ((const V *)(w.src + from * page_bytes))[at];
        ((V *)(w.dst + to * page_bytes))[at] = v;
    }
}

int blocks_for(int64_t threads) { return (int)std::max<int64_t>(1, std::min<int64_t>((threads + 255) / 256, 148 * 16)); }

void copy_pages(const Where &w, int64_t page_bytes, int64_t most, cudaStream_t st) {
    const uintptr_t mix = (uintptr_t)w.src | (uintptr_t)w.dst | (uintptr_t)page_bytes;
    if (mix % 16 == 0) copy_kernel<uint4><<<blocks_for(most * (page_bytes / 16)), 256, 0, st>>>(w, page_bytes);
    else if (mix % 4 == 0) copy_kernel<uint32_t><<<blocks_for(most * (page_bytes / 4)), 256, 0, st>>>(w, page_bytes);
    else copy_kernel<uint8_t><<<blocks_for(most * page_bytes), 256, 0, st>>>(w, page_bytes);
}

int cache_of(const ygg_cache_t *h, Cache &c) {
    if (!h || !h->pages || !h->table || !h->length || !h->refs || !h->status || h->page_bytes < 1 || h->page_count < 1 ||
        h->page_count > INT32_MAX || h->streams < 1 || h->streams > INT32_MAX || h->per_stream < 1 ||
        h->page_bytes > ((int64_t)1 << 40))
        return YGG_E_ARG;
    c = {(char *)h->pages, h->page_count, h->page_bytes, h->table, h->streams, h->per_stream, h->length, h->refs,
         h->status};
    return YGG_OK;
}

int done() { return cudaGetLastError() == cudaSuccess ? YGG_OK : YGG_E_CUDA; }

int64_t rounded(int64_t v) { return (v + 3) / 4 * 4; }

}  // namespace

extern "C" {

size_t ygg_cache_workspace(const ygg_cache_t *h, int64_t n) {
    if (!h || n < 0 || h->page_count < 1) return 0;
    // fork and grow: order [n], moves [n]; compact: renumber [count], moves [count]
    return sizeof(int32_t) * (size_t)(3 * rounded(std::max(n, h->page_count)) + 4);
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
    int32_t *order = (int32_t *)d_workspace;
    Move *moves = (Move *)(order + rounded(n));
    plan_kernel<<<1, kPlan, 0, st>>>(c, d_parents, d_children, d_depth, n, order, moves);
    Where w{};
    w.src = w.dst = c.pages;
    w.src_count = w.dst_count = c.count;
    w.moves = moves;
    w.n = n;
    copy_pages(w, c.page_bytes, n, st);
    return done();
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
    int32_t *counts = (int32_t *)d_workspace, *renumber = counts + 4;
    Move *moves = (Move *)(renumber + rounded(c.count));
    compact_plan_kernel<<<1, kPlan, 0, st>>>(c, d_live, counts, renumber, moves);
    renumber_kernel<<<blocks_for(c.streams * c.per_stream), 256, 0, st>>>(c, renumber);
    Where w{};
    w.src = w.dst = c.pages;
    w.src_count = w.dst_count = c.count;
    w.moves = moves;
    w.n_of = counts;
    copy_pages(w, c.page_bytes, c.count / 2 + 1, st);
    return done();
}

int ygg_cache_read(int device, const ygg_cache_t *h, int64_t n, const int32_t *d_streams, void *d_batch, void *stream) {
    Cache c;
    if (cache_of(h, c) != YGG_OK || n < 0) return YGG_E_ARG;
    if (n == 0) return YGG_OK;
    if (!d_streams || !d_batch) return YGG_E_ARG;
    OnDevice on(device);
    if (!on.ok) return YGG_E_DEVICE;
    Where w{c.pages, (char *)d_batch, c.count, n, nullptr, nullptr, nullptr, d_streams, c.table, c.length, c.streams,
            c.per_stream, 1, nullptr, n, c.status};
    copy_pages(w, c.page_bytes, n, (cudaStream_t)stream);
    return done();
}

int ygg_cache_write(int device, const ygg_cache_t *h, int64_t n, const int32_t *d_streams, const void *d_batch,
                    void *stream) {
    Cache c;
    if (cache_of(h, c) != YGG_OK || n < 0) return YGG_E_ARG;
    if (n == 0) return YGG_OK;
    if (!d_streams || !d_batch) return YGG_E_ARG;
    OnDevice on(device);
    if (!on.ok) return YGG_E_DEVICE;
    Where w{(const char *)d_batch, c.pages, n, c.count, nullptr, nullptr, nullptr, d_streams, c.table, c.length,
            c.streams, c.per_stream, 2, nullptr, n, c.status};
    copy_pages(w, c.page_bytes, n, (cudaStream_t)stream);
    return done();
}

int ygg_cache_copy(int device, const ygg_cache_t *h, int64_t n, const int32_t *d_from, const int32_t *d_to, void *stream) {
    Cache c;
    if (cache_of(h, c) != YGG_OK || n < 0) return YGG_E_ARG;
    if (n == 0) return YGG_OK;
    if (!d_from || !d_to) return YGG_E_ARG;
    OnDevice on(device);
    if (!on.ok) return YGG_E_DEVICE;
    Where w{c.pages, c.pages, c.count, c.count, nullptr, d_from, d_to, nullptr, nullptr, nullptr, 0, 0, 0, nullptr, n,
            c.status};
    copy_pages(w, c.page_bytes, n, (cudaStream_t)stream);
    return done();
}

}  // extern "C"
