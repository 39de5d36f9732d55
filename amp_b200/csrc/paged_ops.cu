// paged_ops.cu -- bookkeeping of the paged KV cache on the device: copying, forking,
// extending, compacting and freeing pages.
//
// AMP's scheduler keeps a sequence's pages in a host list (Sequence::kv_page_ids,
// include/scheduler.hpp:61) and frees them through a host free list
// (src/pool_fast.cpp:31-60).  Here the block table and the context lengths, which
// the attention kernels read on the device anyway, are the whole truth: page p is
// in use iff some row b names it among its first ceil(ctx_lens[b] / 16) entries.
// There is no reference count that could drift, nothing is copied to the host,
// and every call can be captured into a graph.
//
// Each operation is a plan and a move.  The plan (a cluster of eight blocks) marks
// the pages in use in bitmaps in shared memory; one block turns them into a list of free
// pages, lowest first, by a scan over the bitmap's words, and hands pages out in
// the order of the request, so the result does not depend on the scheduling of
// any atomic.  The move copies the pages that the plan listed in every layer and
// rewrites table rows; it is one grid, launched while the plan runs (programmatic
// dependent launch), and is HBM-bound: a page is read and written once.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "runtime.h"
#include "tc_common.cuh"

namespace cg = cooperative_groups;

namespace ampb {
namespace {

constexpr int kPage = 16;
constexpr int kPlanThreads = 1024;
constexpr int kCluster = 8;   // blocks that mark pages for one plan
constexpr int kMoveThreads = 256;
// The bitmaps take 2 bits a page, of the 227 KB that a block may have.
constexpr int kMaxPages = 768 * 1024;
constexpr int kMaxRows = 64 * 1024;

// The plan's results in the workspace.
struct Moves {
    int* count;     // [0] pairs; [1] fork: rows are staged
    int* src;       // [cap] page to read, or -1: skip
    int* dst;       // [cap]
    int* aux;       // what the operation needs besides
};
inline size_t moves_bytes(int64_t cap, int64_t aux) { return 64 + (2 * cap + aux) * sizeof(int); }
inline Moves moves_at(void* ws, int64_t cap) {
    int* p = static_cast<int*>(ws);
    return {p, p + 16, p + 16 + cap, p + 16 + 2 * cap};
}

struct Table {
    int* table;     // [rows][width]
    int* ctx;       // [rows]
    int rows, width, num_pages;
    int* status;
};

__device__ __forceinline__ int named(const Table& t, int ctx) {   // entries that stand for tokens
    return ctx <= 0 ? 0 : min((ctx - 1) / kPage + 1, t.width);
}
__device__ __forceinline__ bool bit(const unsigned* map, int i) { return map[i >> 5] >> (i & 31) & 1; }
__device__ __forceinline__ bool set_bit(unsigned* map, int i) {   // true if it was set
    const unsigned m = 1u << (i & 31);
    return atomicOr(&map[i >> 5], m) & m;
}
__device__ __forceinline__ void bad_index(int* status) {
    status[kStatusBadIndexInt] = AMP_DEV_ERR_BAD_INDEX;
}

// Marks the pages of the rows that `counts` accepts in this block's bitmaps; `twice` (may be
// null) gets those that are named more than once.  The rows are shared out among the warps of
// the cluster, a row among several where there are fewer rows than warps; four entries a
// lane are in flight.
template <typename F>
__device__ __forceinline__ void mark_used(const Table& t, unsigned* used, unsigned* twice, F counts) {
    constexpr int kWarps = kCluster * kPlanThreads / 32;
    const int lane = threadIdx.x & 31;
    const int split = max(1, kWarps / t.rows);   // warps of a row
    const int tasks = t.rows * split;
    for (int task = blockIdx.x * (kPlanThreads / 32) + (threadIdx.x >> 5); task < tasks; task += kWarps) {
        const int r = task / split, seg = task - r * split;
        if (!counts(r)) continue;
        const int n = named(t, t.ctx[r]);
        const int* row = t.table + (int64_t)r * t.width;
        for (int e0 = seg * 128; e0 < n; e0 += split * 128) {
            int p[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int e = e0 + i * 32 + lane;
                if (e < n) p[i] = row[e];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (e0 + i * 32 + lane >= n) continue;
                if (p[i] < 0 || p[i] >= t.num_pages) bad_index(t.status);
                else if (set_bit(used, p[i]) && twice) set_bit(twice, p[i]);
            }
        }
    }
}

// Joins the cluster's bitmaps in its first block, each block taking a part of the words; true
// for that block, which goes on alone.  (What bounds a plan is marking: a shared-memory atomic
// takes about as many cycles as a warp has lanes, 12 thousand entries of 256 rows took one
// block 11 us, eight blocks 3 us with the two waits of the cluster.)
__device__ __forceinline__ bool join_marks(unsigned* used, unsigned* twice, int words) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const int each = (words + kCluster - 1) / kCluster;
    const int w0 = (int)blockIdx.x * each, w1 = min(w0 + each, words);
    for (int w = w0 + (int)threadIdx.x; w < w1; w += kPlanThreads) {
        unsigned once = 0, more = 0;
#pragma unroll
        for (int c = 0; c < kCluster; ++c) {
            const unsigned u = *cluster.map_shared_rank(used + w, c);
            if (twice) more |= (once & u) | *cluster.map_shared_rank(twice + w, c);
            once |= u;
        }
        *cluster.map_shared_rank(used + w, 0) = once;
        if (twice) *cluster.map_shared_rank(twice + w, 0) = more;
    }
    cluster.sync();
    return blockIdx.x == 0;
}

// Writes the lowest free pages, ascending, into list[0 .. most) and returns how many pages
// are free in all.  Each thread takes a run of the bitmap's words.
__device__ __forceinline__ int list_free(const unsigned* used, int num_pages, int* list, int most,
                                         int* part) {
    const int words = (num_pages + 31) / 32;
    const int each = (words + kPlanThreads - 1) / kPlanThreads;
    const int w0 = min(threadIdx.x * each, words), w1 = min(w0 + each, words);
    auto free_bits = [&](int w) {
        const int left = num_pages - w * 32;
        return ~used[w] & (left >= 32 ? 0xffffffffu : (1u << left) - 1);
    };
    int n = 0;
    for (int w = w0; w < w1; ++w) n += __popc(free_bits(w));
    const int end = block_scan(n, part);
    const int total = part[31];
    int rank = end - n;
    for (int w = w0; w < w1 && rank < most; ++w)
        for (unsigned m = free_bits(w); m && rank < most; m &= m - 1)
            list[rank++] = w * 32 + __ffs(m) - 1;
    __syncthreads();   // the list is complete
    return total;
}

// ------------------------------------------------------------------ the move
// 16 KB pieces of the listed pages, in every layer, of both pools.
struct Pools {
    uint4 *k, *v;             // [layers][num_pages][page16]
    int layers, num_pages;
    int page16;               // 16-byte words of a page
};

// `pair(i, src, dst)`: the i-th pair, src < 0 to skip; all threads of a block call it with one i.
template <typename P>
__device__ __forceinline__ void move_pages(const Pools& pl, int count, P pair_at) {
    constexpr int kUnroll = 4, kPiece = kMoveThreads * kUnroll;
    const int pieces = (pl.page16 + kPiece - 1) / kPiece;
    const int64_t total = (int64_t)count * pl.layers * 2 * pieces;
    for (int64_t w = blockIdx.x; w < total; w += gridDim.x) {
        int64_t r = w;
        const int piece = (int)(r % pieces);
        r /= pieces;
        const int pool = (int)(r & 1);
        r >>= 1;
        const int layer = (int)(r % pl.layers);
        const int pair = (int)(r / pl.layers);
        int src, dst;
        pair_at(pair, src, dst);
        if (src < 0) continue;
        uint4* base = (pool ? pl.v : pl.k) + (int64_t)layer * pl.num_pages * pl.page16;
        const uint4* s = base + (int64_t)src * pl.page16;
        uint4* d = base + (int64_t)dst * pl.page16;
        uint4 x[kUnroll];
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) {
            const int e = piece * kPiece + i * kMoveThreads + threadIdx.x;
            if (e < pl.page16) x[i] = s[e];
        }
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) {
            const int e = piece * kPiece + i * kMoveThreads + threadIdx.x;
            if (e < pl.page16) d[e] = x[i];
        }
    }
}
__device__ __forceinline__ void move_pages(const Pools& pl, const Moves& mv, int count) {
    move_pages(pl, count, [&](int i, int& src, int& dst) {
        src = mv.src[i];
        dst = mv.dst[i];
    });
}

// ------------------------------------------------------------------ copy
// Pairs with one target, or a pair whose source another one writes, would make the result
// depend on the order: they are skipped and reported.  A negative number
// and a page onto itself are nothing to do.
__device__ __forceinline__ bool real_pair(int s, int d, int num_pages) {
    return s >= 0 && d >= 0 && s != d && s < num_pages && d < num_pages;
}

// Up to kDirectPairs pairs each block compares its pair with all others itself, for every piece that
// it copies, which saves the plan's launch (inside a graph, planned -> direct: 38 pairs of 32 KB pages,
// one layer 3.5 -> 2.5 us, 32 layers 30.0 -> 28.8; 1024 pairs 24.2 -> 24.0 and 741 -> 726).  With pages of
// less than half a piece the comparisons outweigh the copying once there are more than about 1024
// pieces a pool (2 KB pages, one layer: 512 pairs 4.1 -> 3.4; 32 layers: 38 pairs 5.5 -> 5.6, 256 pairs
// 21.8 -> 32.0, 1024 pairs 93.7 -> 157; 8 KB pages, 32 layers: 1024 pairs 188 -> 173).
constexpr int kDirectPairs = 1024;
bool copies_direct(const Pools& pl, int n) {
    return n <= kDirectPairs && (pl.page16 >= kMoveThreads * 2 || (int64_t)n * pl.layers <= 1024);
}
__global__ void __launch_bounds__(kMoveThreads)
    k_copy_direct(Pools pl, const int* src, const int* dst, int n, int* status) {
    pdl_wait();
    move_pages(pl, n, [&](int i, int& s, int& d) {
        s = src[i];
        d = dst[i];
        const bool real = real_pair(s, d, pl.num_pages);
        bool clash = false;
        if (real)
            for (int j = threadIdx.x; j < n; j += kMoveThreads)
                clash |= j != i && (dst[j] == d || dst[j] == s) && real_pair(src[j], dst[j], pl.num_pages);
        clash = __syncthreads_or(clash);
        if (threadIdx.x == 0 && (clash || s >= pl.num_pages || d >= pl.num_pages)) bad_index(status);
        if (!real || clash) s = -1;
    });
}

__global__ void __launch_bounds__(kPlanThreads)
    k_copy_plan(const int* src, const int* dst, int n, int num_pages, Moves mv, int* status) {
    extern __shared__ unsigned seen[];
    const int words = (num_pages + 31) / 32;
    unsigned* twice = seen + words;
    pdl_wait();
    pdl_trigger();
    for (int i = threadIdx.x; i < 2 * words; i += kPlanThreads) seen[i] = 0;
    __syncthreads();
    auto real = [&](int s, int d) { return real_pair(s, d, num_pages); };
    for (int i = threadIdx.x; i < n; i += kPlanThreads)
        if (real(src[i], dst[i]) && set_bit(seen, dst[i])) set_bit(twice, dst[i]);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kPlanThreads) {
        const int s = src[i], d = dst[i];
        const bool ok = real(s, d) && !bit(twice, d) && !bit(seen, s);
        if (s >= num_pages || d >= num_pages || (real(s, d) && !ok)) bad_index(status);
        mv.src[i] = ok ? s : -1;
        mv.dst[i] = d;
    }
    if (threadIdx.x == 0) mv.count[0] = n;
}

__global__ void __launch_bounds__(kMoveThreads) k_move(Pools pl, Moves mv) {
    pdl_wait();
    move_pages(pl, mv, mv.count[0]);
}

// ------------------------------------------------------------------ fork
// aux: [n] entry of the child: the rank of its fresh page, kShare (no page needed), kFailed
// (none left) or kSkip; [n] new context; [n * width] parents' rows, when a parent is a child too
constexpr int kShare = -1, kFailed = -2, kSkip = -3;

__global__ void __cluster_dims__(kCluster) __launch_bounds__(kPlanThreads)
    k_fork_plan(Table t, const int* parents, const int* children, int n, int* done, Moves mv) {
    extern __shared__ unsigned used[];
    __shared__ int part[32];
    __shared__ int chained;
    const int words = (t.num_pages + 31) / 32, row_words = (t.rows + 31) / 32;
    unsigned *child = used + words, *again = child + row_words, *parent = again + row_words;
    int *entry = mv.aux, *new_ctx = mv.aux + n, *stage = mv.aux + 2 * (int64_t)n;
    pdl_wait();
    pdl_trigger();
    for (int i = threadIdx.x; i < words + 3 * row_words; i += kPlanThreads) used[i] = 0;
    if (threadIdx.x == 0) chained = 0;
    __syncthreads();
    auto in_range = [&](int i) {
        return parents[i] >= 0 && parents[i] < t.rows && children[i] >= 0 && children[i] < t.rows;
    };
    for (int i = threadIdx.x; i < n; i += kPlanThreads) {
        if (!in_range(i)) bad_index(t.status);   // every block looks: row flags are the block's own
        else if (set_bit(child, children[i])) set_bit(again, children[i]);
    }
    __syncthreads();
    // a row named twice as a child: none of its forks is done
    auto valid = [&](int i) { return in_range(i) && !bit(again, children[i]); };
    for (int i = threadIdx.x; i < n; i += kPlanThreads) {
        if (valid(i)) set_bit(parent, parents[i]);
        else if (in_range(i)) bad_index(t.status);
    }
    __syncthreads();
    auto replaced = [&](int r) { return bit(child, r) && !bit(again, r); };
    mark_used(t, used, nullptr, [&](int r) { return !replaced(r) || bit(parent, r); });
    if (!join_marks(used, nullptr, words)) return;
    // the fresh pages, in dst: the k-th goes to the k-th fork that needs one
    const int free = list_free(used, t.num_pages, mv.dst, n, part);
    int carry = 0;
    for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
        const int i = i0 + threadIdx.x;
        int e = kSkip, ctx = 0;
        if (i < n) {
            if (valid(i)) {
                ctx = max(t.ctx[parents[i]], 0);
                e = parents[i] == children[i] ? kSkip : kShare;
                if (e == kShare && bit(child, parents[i])) chained = 1;
            }
        }
        const bool fresh = e == kShare && ctx % kPage != 0 && (ctx - 1) / kPage < t.width;
        const int rank = carry + block_scan(fresh ? 1 : 0, part) - 1;
        carry += part[31];
        if (fresh) {
            e = rank < free ? rank : kFailed;
            if (e >= 0) {
                const int old = t.table[(int64_t)parents[i] * t.width + (ctx - 1) / kPage];
                mv.src[e] = old >= 0 && old < t.num_pages ? old : -1;
            } else {
                ctx = 0;
            }
        }
        if (i < n) {
            entry[i] = e;
            new_ctx[i] = ctx;
            done[i] = valid(i) && e != kFailed;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        mv.count[0] = min(carry, free);
        mv.count[1] = chained;
    }
    if (chained) {   // rows that are read and replaced in one call: read them all first
        for (int64_t w = threadIdx.x; w < (int64_t)n * t.width; w += kPlanThreads) {
            const int i = (int)(w / t.width);
            if (entry[i] >= kShare) stage[w] = t.table[(int64_t)parents[i] * t.width + w % t.width];
        }
    }
    for (int i = threadIdx.x; i < n; i += kPlanThreads)
        if (entry[i] != kSkip) t.ctx[children[i]] = new_ctx[i];
}

__global__ void __launch_bounds__(kMoveThreads)
    k_fork_move(Pools pl, Moves mv, Table t, const int* parents, const int* children, int n) {
    pdl_wait();
    const int *entry = mv.aux, *new_ctx = mv.aux + n, *stage = mv.aux + 2 * (int64_t)n;
    const bool staged = mv.count[1] != 0;
    for (int i = blockIdx.x; i < n; i += gridDim.x) {
        const int e = entry[i];
        if (e == kSkip) continue;
        const int need = named(t, new_ctx[i]);
        const int* from = staged ? stage + (int64_t)i * t.width : t.table + (int64_t)parents[i] * t.width;
        int* to = t.table + (int64_t)children[i] * t.width;
        for (int c = threadIdx.x; c < t.width; c += kMoveThreads)
            to[c] = e == kFailed || c >= need ? -1 : (e >= 0 && c == need - 1 ? mv.dst[e] : from[c]);
    }
    move_pages(pl, mv, mv.count[0]);
}

// ------------------------------------------------------------------ extend
// aux: [num_pages] free pages; [rows] where a row's pages begin in that list; [rows] how many
// (0: none, or not extended); [rows] its entries so far, less one if its last page is replaced
__global__ void __cluster_dims__(kCluster) __launch_bounds__(kPlanThreads)
    k_extend_plan(Table t, const int* add, int* ctx_out, int* done, Moves mv) {
    extern __shared__ unsigned used[];
    __shared__ int part[32];
    const int words = (t.num_pages + 31) / 32;
    unsigned* twice = used + words;
    int *list = mv.aux, *first = list + t.num_pages, *count = first + t.rows, *at_entry = count + t.rows;
    pdl_wait();
    pdl_trigger();
    for (int i = threadIdx.x; i < 2 * words; i += kPlanThreads) used[i] = 0;
    __syncthreads();
    mark_used(t, used, twice, [](int) { return true; });
    if (!join_marks(used, twice, words)) return;
    // Pages that row r needs: new ones, and one for a partly filled last page that another
    // row names too (the next token must not be written into the other's cache).
    auto plan_row = [&](int r, int& ctx, int& have, bool& own, bool& ok) {
        ctx = max(t.ctx[r], 0);
        have = named(t, ctx);
        own = false;
        const int n = add[r];
        ok = n >= 0 && (int64_t)ctx + n <= (int64_t)t.width * kPage;
        if (n <= 0 || !ok) return 0;
        int more = (int)(((int64_t)ctx + n - 1) / kPage + 1) - have;
        if (ctx % kPage != 0) {
            const int tail = t.table[(int64_t)r * t.width + have - 1];
            own = tail >= 0 && tail < t.num_pages && bit(twice, tail);
            more += own;
        }
        return min(more, t.num_pages + 1);   // more than there are is as bad as one too many
    };
    int carry = 0;
    for (int r0 = 0; r0 < t.rows; r0 += kPlanThreads) {
        const int r = r0 + threadIdx.x;
        int ctx, have = 0, more = 0;
        bool own = false, ok;
        if (r < t.rows) more = plan_row(r, ctx, have, own, ok);
        const int end = carry + block_scan(more, part);
        carry = min(carry + part[31], 1 << 30);   // far past any pool: stays below 2^31
        if (r < t.rows) {
            first[r] = end - more;
            count[r] = more;
            at_entry[r] = have - own;
            // for now: kept, or kept only if its pages are there
            ctx_out[r] = ok ? ctx + add[r] : t.ctx[r];
            done[r] = ok;
        }
    }
    const int free = list_free(used, t.num_pages, list, min(carry, t.num_pages), part);
    int copies = 0;
    for (int r0 = 0; r0 < t.rows; r0 += kPlanThreads) {
        const int r = r0 + threadIdx.x;
        bool own = false;
        if (r < t.rows && count[r] > 0) {
            // in order: once the pool cannot hold a row's pages, that row and all later ones
            // that need any fail
            const int new_ctx = ctx_out[r], have = named(t, new_ctx - add[r]);
            if (first[r] + count[r] > free) {
                count[r] = 0;
                ctx_out[r] = new_ctx - add[r];
                done[r] = 0;
            } else {
                own = at_entry[r] < have;
            }
        }
        const int at = copies + block_scan(own ? 1 : 0, part) - 1;
        copies += part[31];
        if (own) {
            mv.src[at] = t.table[(int64_t)r * t.width + at_entry[r]];
            mv.dst[at] = list[first[r]];
        }
    }
    if (threadIdx.x == 0) mv.count[0] = copies;
}

__global__ void __launch_bounds__(kMoveThreads) k_extend_move(Pools pl, Moves mv, Table t) {
    pdl_wait();
    const int *list = mv.aux, *first = list + t.num_pages, *count = first + t.rows,
              *at_entry = count + t.rows;
    // a warp a row: most rows get one page or none
    for (int r = blockIdx.x * (kMoveThreads / 32) + threadIdx.x / 32; r < t.rows;
         r += gridDim.x * (kMoveThreads / 32)) {
        const int n = count[r];
        int* to = t.table + (int64_t)r * t.width + at_entry[r];
        for (int i = threadIdx.x & 31; i < n; i += 32) to[i] = list[first[r] + i];
    }
    move_pages(pl, mv, mv.count[0]);
}

// ------------------------------------------------------------------ compact
// With L pages in use, those at L and above move to the free ones below L, both in
// ascending order; aux[p] is where page p >= L goes.
__global__ void __cluster_dims__(kCluster) __launch_bounds__(kPlanThreads) k_compact_plan(Table t, int* used_out, Moves mv) {
    extern __shared__ unsigned used[];
    __shared__ int part[32];
    const int words = (t.num_pages + 31) / 32;
    pdl_wait();
    pdl_trigger();
    for (int i = threadIdx.x; i < words; i += kPlanThreads) used[i] = 0;
    __syncthreads();
    mark_used(t, used, nullptr, [](int) { return true; });
    if (!join_marks(used, nullptr, words)) return;
    const int each = (words + kPlanThreads - 1) / kPlanThreads;
    const int w0 = min((int)threadIdx.x * each, words), w1 = min(w0 + each, words);
    int n = 0;
    for (int w = w0; w < w1; ++w) n += __popc(used[w]);
    const int end = block_scan(n, part);
    const int live = part[31];
    // free pages below `live`: page p is free number p - (used pages before p)
    int before = end - n;
    for (int w = w0; w < w1; ++w) {
        for (int b = 0; b < 32; ++b) {
            const int p = w * 32 + b;
            if (p >= live) break;
            if (used[w] >> b & 1) ++before;
            else mv.dst[p - before] = p;
        }
    }
    __syncthreads();
    // used pages from `live` on, in order
    n = 0;
    for (int w = w0; w < w1; ++w) {
        unsigned m = used[w];
        if (w * 32 < live) m &= w * 32 + 32 <= live ? 0u : ~((1u << (live - w * 32)) - 1);
        n += __popc(m);
    }
    const int high = block_scan(n, part);
    int rank = high - n;
    const int moves = part[31];
    for (int w = w0; w < w1; ++w) {
        unsigned m = used[w];
        if (w * 32 < live) m &= w * 32 + 32 <= live ? 0u : ~((1u << (live - w * 32)) - 1);
        for (; m; m &= m - 1, ++rank) {
            const int p = w * 32 + __ffs(m) - 1;
            mv.src[rank] = p;
            mv.aux[p] = mv.dst[rank];
        }
    }
    if (threadIdx.x == 0) {
        mv.count[0] = moves;
        mv.count[1] = live;
        *used_out = live;
    }
}

__global__ void __launch_bounds__(kMoveThreads) k_compact_move(Pools pl, Moves mv, Table t, int* out) {
    pdl_wait();
    const int live = mv.count[1];
    for (int r = blockIdx.x; r < t.rows; r += gridDim.x) {
        const int need = named(t, t.ctx[r]);
        for (int c = threadIdx.x; c < t.width; c += kMoveThreads) {
            const int64_t i = (int64_t)r * t.width + c;
            int p = c < need ? t.table[i] : -1;
            if (p >= t.num_pages) p = -1;
            out[i] = p < live ? max(p, -1) : mv.aux[p];
        }
    }
    move_pages(pl, mv, mv.count[0]);
}

// ------------------------------------------------------------------ free
__global__ void __launch_bounds__(kMoveThreads) k_free(Table t, const int* seqs, int n) {
    pdl_wait();
    for (int i = blockIdx.x; i < n; i += gridDim.x) {
        const int r = seqs[i];
        if (r < 0 || r >= t.rows) {
            if (threadIdx.x == 0) bad_index(t.status);
            continue;
        }
        for (int c = threadIdx.x; c < t.width; c += kMoveThreads) t.table[(int64_t)r * t.width + c] = -1;
        if (threadIdx.x == 0) t.ctx[r] = 0;
    }
}

// ------------------------------------------------------------------ host side
int make_pools(Pools& pl, void* k, void* v, int layers, int num_pages, int Hkv, int D) {
    AMPB_REQUIRE(k && v, AMP_ERR_INVALID, "NULL pool");
    AMPB_REQUIRE(aligned16(k) && aligned16(v), AMP_ERR_INVALID, "the pools must be 16-byte aligned");
    AMPB_REQUIRE(layers > 0 && num_pages > 0 && Hkv > 0 && D > 0, AMP_ERR_INVALID,
                 "pool sizes must be positive");
    AMPB_REQUIRE(num_pages <= kMaxPages, AMP_ERR_UNSUPPORTED, "pools of more than %d pages not supported",
                 kMaxPages);
    AMPB_REQUIRE((int64_t)Hkv * D <= (1 << 24), AMP_ERR_UNSUPPORTED, "page too large");
    pl = {static_cast<uint4*>(k), static_cast<uint4*>(v), layers, num_pages, Hkv * kPage * D * 2 / 16};
    return AMP_OK;
}

int make_table(Table& t, int32_t* table, int32_t* ctx, int rows, int width, int num_pages) {
    AMPB_REQUIRE(table && ctx, AMP_ERR_INVALID, "NULL table or context lengths");
    AMPB_REQUIRE(rows > 0 && width > 0, AMP_ERR_INVALID, "table sizes must be positive");
    AMPB_REQUIRE(rows <= kMaxRows && width <= (1 << 24), AMP_ERR_UNSUPPORTED,
                 "tables of more than %d rows or 2^24 entries a row not supported", kMaxRows);
    t = {table, ctx, rows, width, num_pages, nullptr};   // status: once all arguments are checked
    return AMP_OK;
}

int check_ws(const void* ws, size_t have, size_t need) {
    AMPB_REQUIRE(ws && aligned16(ws), AMP_ERR_INVALID, "workspace must be 16-byte aligned");
    AMPB_REQUIRE(have >= need, AMP_ERR_INVALID, "workspace too small: %zu < %zu", have, need);
    return AMP_OK;
}

// (two bitmaps of the pages, or one and three of the rows)
constexpr size_t kMaxPlanSmem = std::max(2 * kMaxPages / 8, kMaxPages / 8 + 3 * kMaxRows / 8);

template <auto kern, typename... A>
int launch_plan(int blocks, int smem_words, cudaStream_t st, A... args) {
    const size_t smem = (size_t)smem_words * 4;
    static std::atomic<uint64_t> allowed{0};
    AMPB_CHECK_CUDA(allow_smem_once(allowed, kern, kMaxPlanSmem));
    AMPB_CHECK_CUDA(launch_pdl(kern, dim3(blocks), dim3(kPlanThreads), smem, st, args...));
    return AMP_OK;
}

// One block a 16 KB piece up to eight blocks a multiprocessor, which then walk the rest.
unsigned move_grid(const Pools& pl, int64_t most_pairs, int64_t rows) {
    const int64_t pieces = (pl.page16 + kMoveThreads * 4 - 1) / (kMoveThreads * 4);
    const int64_t want = std::max(most_pairs * pl.layers * 2 * pieces, rows);
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>(want, (int64_t)sm_count() * 8));
}

}  // namespace
}  // namespace ampb

using namespace ampb;

extern "C" {

size_t amp_paged_copy_workspace_bytes(int n) { return n >= 0 ? moves_bytes(n, 0) : 0; }
size_t amp_paged_fork_workspace_bytes(int n, int max_pages_per_seq) {
    return n >= 0 && max_pages_per_seq > 0 ? moves_bytes(n, (int64_t)n * (2 + (int64_t)max_pages_per_seq)) : 0;
}
size_t amp_paged_extend_workspace_bytes(int rows, int num_pages) {
    return rows > 0 && num_pages > 0 ? moves_bytes(rows, num_pages + 3 * (int64_t)rows) : 0;
}
size_t amp_paged_compact_workspace_bytes(int num_pages) {
    return num_pages > 0 ? moves_bytes(num_pages, num_pages) : 0;
}

int amp_paged_copy_pages_dev(void* k_pool, void* v_pool, int layers, int num_pages, int Hkv,
                             int head_dim, const int32_t* src, const int32_t* dst, int n,
                             void* workspace, size_t workspace_bytes, void* stream) {
    Pools pl;
    int rc = make_pools(pl, k_pool, v_pool, layers, num_pages, Hkv, head_dim);
    if (rc) return rc;
    AMPB_REQUIRE(n >= 0, AMP_ERR_INVALID, "copy: n must be >= 0");
    if (n == 0) return AMP_OK;
    AMPB_REQUIRE(src && dst, AMP_ERR_INVALID, "copy: NULL page numbers");
    if ((rc = check_ws(workspace, workspace_bytes, amp_paged_copy_workspace_bytes(n)))) return rc;
    int* status = nullptr;
    if ((rc = device_status(&status))) return rc;
    cudaStream_t st = as_stream(stream);
    if (copies_direct(pl, n)) {
        AMPB_CHECK_CUDA(launch_pdl(k_copy_direct, dim3(move_grid(pl, n, 1)), dim3(kMoveThreads), 0, st, pl, src,
                                   dst, n, status));
        return AMP_OK;
    }
    const Moves mv = moves_at(workspace, n);
    if ((rc = launch_plan<k_copy_plan>(1, 2 * ((num_pages + 31) / 32), st, src, dst, n, num_pages, mv, status)))
        return rc;
    AMPB_CHECK_CUDA(launch_pdl(k_move, dim3(move_grid(pl, n, 1)), dim3(kMoveThreads), 0, st, pl, mv));
    return AMP_OK;
}

int amp_paged_fork_dev(void* k_pool, void* v_pool, int layers, int num_pages, int Hkv, int head_dim,
                       int32_t* block_table, int32_t* ctx_lens, int rows, int max_pages_per_seq,
                       const int32_t* parents, const int32_t* children, int n, int32_t* done,
                       void* workspace, size_t workspace_bytes, void* stream) {
    Pools pl;
    Table t;
    int rc = make_pools(pl, k_pool, v_pool, layers, num_pages, Hkv, head_dim);
    if (rc) return rc;
    if ((rc = make_table(t, block_table, ctx_lens, rows, max_pages_per_seq, num_pages))) return rc;
    AMPB_REQUIRE(n >= 0, AMP_ERR_INVALID, "fork: n must be >= 0");
    if (n == 0) return AMP_OK;
    AMPB_REQUIRE(parents && children && done, AMP_ERR_INVALID, "fork: NULL rows or result");
    if ((rc = check_ws(workspace, workspace_bytes, amp_paged_fork_workspace_bytes(n, max_pages_per_seq))))
        return rc;
    if ((rc = device_status(&t.status))) return rc;
    const Moves mv = moves_at(workspace, n);
    cudaStream_t st = as_stream(stream);
    const int words = (num_pages + 31) / 32 + 3 * ((rows + 31) / 32);
    if ((rc = launch_plan<k_fork_plan>(kCluster, words, st, t, parents, children, n, done, mv))) return rc;
    AMPB_CHECK_CUDA(launch_pdl(k_fork_move, dim3(move_grid(pl, n, n)), dim3(kMoveThreads), 0, st, pl, mv, t,
                               parents, children, n));
    return AMP_OK;
}

int amp_paged_extend_dev(void* k_pool, void* v_pool, int layers, int num_pages, int Hkv, int head_dim,
                         int32_t* block_table, const int32_t* ctx_lens, int rows,
                         int max_pages_per_seq, const int32_t* add, int32_t* ctx_out, int32_t* done,
                         void* workspace, size_t workspace_bytes, void* stream) {
    Pools pl;
    Table t;
    int rc = make_pools(pl, k_pool, v_pool, layers, num_pages, Hkv, head_dim);
    if (rc) return rc;
    if ((rc = make_table(t, block_table, const_cast<int32_t*>(ctx_lens), rows, max_pages_per_seq, num_pages)))
        return rc;
    AMPB_REQUIRE(add && ctx_out && done, AMP_ERR_INVALID, "extend: NULL counts or result");
    // the plan reads add again after it has written lengths and done
    AMPB_REQUIRE(add != ctx_out && add != done && ctx_out != done && ctx_lens != done, AMP_ERR_INVALID,
                 "extend: the results may share memory with ctx_lens only, and done with nothing");
    if ((rc = check_ws(workspace, workspace_bytes, amp_paged_extend_workspace_bytes(rows, num_pages)))) return rc;
    if ((rc = device_status(&t.status))) return rc;
    const Moves mv = moves_at(workspace, rows);
    cudaStream_t st = as_stream(stream);
    if ((rc = launch_plan<k_extend_plan>(kCluster, 2 * ((num_pages + 31) / 32), st, t, add, ctx_out, done, mv))) return rc;
    // pages are copied only where rows share a partly filled one: a block a multiprocessor is enough.
    // (As few blocks as rows were not: two rows, 32 layers of 32 KB pages 68 -> 9 us; 64 rows 109 -> 64.)
    AMPB_CHECK_CUDA(launch_pdl(k_extend_move, dim3(std::min(move_grid(pl, rows, 1), (unsigned)sm_count())),
                               dim3(kMoveThreads), 0, st, pl, mv, t));
    return AMP_OK;
}

int amp_paged_compact_dev(void* k_pool, void* v_pool, int layers, int num_pages, int Hkv, int head_dim,
                          const int32_t* block_table, const int32_t* ctx_lens, int rows,
                          int max_pages_per_seq, int32_t* table_out, int32_t* used,
                          void* workspace, size_t workspace_bytes, void* stream) {
    Pools pl;
    Table t;
    int rc = make_pools(pl, k_pool, v_pool, layers, num_pages, Hkv, head_dim);
    if (rc) return rc;
    if ((rc = make_table(t, const_cast<int32_t*>(block_table), const_cast<int32_t*>(ctx_lens), rows,
                         max_pages_per_seq, num_pages)))
        return rc;
    AMPB_REQUIRE(table_out && used, AMP_ERR_INVALID, "compact: NULL result");
    if ((rc = check_ws(workspace, workspace_bytes, amp_paged_compact_workspace_bytes(num_pages)))) return rc;
    if ((rc = device_status(&t.status))) return rc;
    const Moves mv = moves_at(workspace, num_pages);
    cudaStream_t st = as_stream(stream);
    if ((rc = launch_plan<k_compact_plan>(kCluster, (num_pages + 31) / 32, st, t, used, mv))) return rc;
    AMPB_CHECK_CUDA(launch_pdl(k_compact_move, dim3(move_grid(pl, num_pages / 2, rows)), dim3(kMoveThreads), 0,
                               st, pl, mv, t, table_out));
    return AMP_OK;
}

int amp_paged_free_dev(int32_t* block_table, int32_t* ctx_lens, int rows, int max_pages_per_seq,
                       const int32_t* seqs, int n, void* stream) {
    Table t;
    int rc = make_table(t, block_table, ctx_lens, rows, max_pages_per_seq, 0);
    if (rc) return rc;
    AMPB_REQUIRE(n >= 0, AMP_ERR_INVALID, "free: n must be >= 0");
    if (n == 0) return AMP_OK;
    AMPB_REQUIRE(seqs, AMP_ERR_INVALID, "free: NULL rows");
    if ((rc = device_status(&t.status))) return rc;
    AMPB_CHECK_CUDA(launch_pdl(k_free, dim3((unsigned)std::min(n, sm_count() * 8)), dim3(kMoveThreads), 0,
                               as_stream(stream), t, seqs, n));
    return AMP_OK;
}

}  // extern "C"
