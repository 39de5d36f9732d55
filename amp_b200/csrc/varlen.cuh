// varlen.cuh -- work lists of the packed-sequence attention kernels.
//
// Packed tensors hold the tokens of B sequences one after another: sequence b is
// rows cu[b] .. cu[b+1] of [total, heads, D].  Lengths are known on the device
// only, so the attention kernels' CTAs turn them into items themselves (up to 32
// sequences) or take them from lists that a one-CTA kernel (varlen_plan.cu) made:
// the sequences ordered by length, longest first, and the running number of items
// before each.  An item's index is turned back into (sequence, head, tile) by a
// warp-wide search of that prefix.  CTAs draw items from a global counter: with
// lengths that differ by a factor of a hundred no fixed assignment is balanced
// (25 sequences of up to 16384 tokens: 9.4 ms dealt out in turn, 8.8 ms drawn),
// and taking the longest first leaves only small items for the end.
#pragma once
#include <cuda_runtime.h>
#include <cstddef>
#include <cstdint>

#include "common.cuh"
#include "tc_common.cuh"

namespace ampb {

struct VarlenSeq {
    int q_off, q_len, k_off, k_len;
};

// Number of 128-row tiles of a sequence.
__host__ __device__ __forceinline__ int varlen_tiles(int len) { return (len + 127) / 128; }

// Items of one sequence in each list.
//   forward: pairs of (query tile, query head) of one kv head, times `splits`
//   dK/dV:   key tiles of one kv head, times `parts`;  dQ: query tiles of one query head
__host__ __device__ __forceinline__ int varlen_fwd_pairs(int q_len, int group) {
    return (varlen_tiles(q_len) * group + 1) / 2;
}

// The most pairs that B sequences of total_q tokens in all can have: a sequence has at most one
// tile more than its tokens fill, and with an odd group half a pair more for a kv head.
inline int64_t varlen_most_pairs(int B, int total_q, int Hq, int Hkv) {
    const int64_t tiles = (int64_t)total_q / 128 + B, group = Hq / Hkv;
    return Hkv * ((tiles * group + (group % 2 ? B : 0)) / 2);
}

// A pair of the forward: its two (query tile, query head) of one kv head, `pair` counting in
// the order tile major, then the heads; and the K/V tiles that each of them visits.
struct VarlenPair {
    int row0[2], head[2];   // first query row; head within the group
    int n[2];               // n[1] >= n[0] >= 1
};
__device__ __forceinline__ VarlenPair varlen_pair(const VarlenSeq& s, int pair, int group, bool causal) {
    const int tiles = varlen_tiles(s.q_len), n_all = varlen_tiles(s.k_len);
    VarlenPair r;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int sub = 2 * pair + t;
        const bool none = sub >= tiles * group;   // the last pair's second half
        r.row0[t] = none ? tiles * 128 : sub / group * 128;
        r.head[t] = none ? r.head[0] : sub % group;
        r.n[t] = none ? 0 : n_all;
        if (!none && causal) {
            const int last = r.row0[t] + 127 + s.k_len - s.q_len;
            r.n[t] = last < 0 ? 0 : min(n_all, last / 128 + 1);
        }
    }
    r.n[0] = max(r.n[0], 1);
    r.n[1] = max(r.n[1], r.n[0]);
    return r;
}
// K/V tiles of one split of n, where a pair's tiles are shared out among at most `splits`
// items: an item outside its steps takes as long as four of them.
__device__ __forceinline__ int varlen_chunk(int n, int splits) { return max((n + splits - 1) / splits, 4); }

// The lists in the caller's workspace:
//   next   int [16]     items drawn beyond the first of each CTA, one count a list
//   seqs   VarlenSeq [B], longest first
//   first  int [B + 1]  items before sequence r, for list 0 (forward or dK/dV) and 1 (dQ)
inline size_t varlen_plan_bytes(int B) {
    return 64 + (size_t)B * sizeof(VarlenSeq) + 2 * ((size_t)B + 1) * sizeof(int);
}

struct VarlenPlan {
    void* ws;
    bool lists, counted;             // which of the ways of VarlenDraw
    const int *cu_q, *cu_kv;         // the offsets themselves
    int B, total_q, total_kv;
    int most[2];                     // items that each list can have while no two sequences overlap
    __device__ int* next() const { return static_cast<int*>(ws); }
    __device__ VarlenSeq* seqs() const {
        return reinterpret_cast<VarlenSeq*>(static_cast<uint8_t*>(ws) + 64);
    }
    __device__ int* first(int list) const { return reinterpret_cast<int*>(seqs() + B) + list * (B + 1); }

    // Sequence b.  One whose bounds are not within its tensor, in order, counts as empty.
    __device__ __forceinline__ VarlenSeq load(int b, int* status) const {
        const int q0 = cu_q[b], q1 = cu_q[b + 1], k0 = cu_kv[b], k1 = cu_kv[b + 1];
        const bool ok = q0 >= 0 && q1 >= q0 && q1 <= total_q && k0 >= 0 && k1 >= k0 && k1 <= total_kv;
        if (!ok) {
            status[kStatusBadIndexInt] = AMP_DEV_ERR_BAD_INDEX;
            return {0, 0, 0, 0};
        }
        return {q0, q1 - q0, k0, k1 - k0};
    }
};

// Chooses how the CTAs get their items, and enqueues what that needs: the plan kernel
// (`backward` selects which lists it fills), or, where `zero` is true, the zeroing of the
// counters.  most0, most1: the most items of list 0 and 1, which is all that the host knows; offsets
// that name more (sequences that overlap) get none, so that a call's work is bounded by its sizes.
// parts: items of a key tile of a kv head in the dK/dV list, or of a pair in the forward's.
int varlen_make_plan(VarlenPlan& plan, int64_t most0, int64_t most1, int Hq, int Hkv, bool backward,
                     int parts, bool zero, cudaStream_t st);

// Warp-wide (all lanes call it): the sequence r whose items hold `item`, i.e. the
// last r with first[r] <= item, where first[] ascends and first[0] <= item < first[B];
// sequences without items are never returned.  Whatever first[] holds, the result is
// in [0, B).
__device__ __forceinline__ int varlen_find(const int* first, int B, int item) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = B;                 // the answer is in [lo, lo + n)
    while (n > 1) {
        const int step = (n + 31) / 32;
        const int at = lo + lane * step;
        const bool le = lane * step < n && first[at] <= item;
        const int k = max(__popc(__ballot_sync(0xffffffffu, le)) - 1, 0);
        n = min(step, n - k * step);
        lo += k * step;
    }
    return lo;
}

// Warp-wide (all lanes call it, with one t): the sequence that row t of q (kKeys: of k and v)
// belongs to, or an empty one.  Ascending offsets are searched; where that finds no sequence with
// the row, it is a row of none or the offsets are out of order, and every sequence is looked at.
template <bool kKeys>
__device__ __forceinline__ VarlenSeq varlen_owner(const VarlenPlan& plan, int t, int* status) {
    auto holds = [&](const VarlenSeq& s) {
        return t >= (kKeys ? s.k_off : s.q_off) && t < (kKeys ? s.k_off + s.k_len : s.q_off + s.q_len);
    };
    const VarlenSeq found = plan.load(varlen_find(kKeys ? plan.cu_kv : plan.cu_q, plan.B, t), status);
    if (holds(found)) return found;
    const int lane = threadIdx.x & 31;
    for (int b0 = 0; b0 < plan.B; b0 += 32) {
        const bool mine = b0 + lane < plan.B && holds(plan.load(b0 + lane, status));
        const unsigned who = __ballot_sync(0xffffffffu, mine);
        if (who) return plan.load(b0 + __ffs(who) - 1, status);
    }
    return {0, 0, 0, 0};
}

// How a CTA's drawing warp gets its items.
//   lists    (more than 32 sequences) the sequences by length and the items before each come
//            from the plan kernel; otherwise lane r holds the r-th longest sequence, which
//            saves the plan's launch.
//   counted  the first item is the CTA's index, the rest come from the counter; otherwise
//            (few items) they are dealt out forth and back, so that a CTA whose first was
//            long gets a short one.
struct VarlenDraw {
    const VarlenPlan& plan;
    int list, total;
    VarlenSeq mine;
    int first;

    template <typename F>
    __device__ __forceinline__ VarlenDraw(const VarlenPlan& p, int list_, F items, int* status)
        : plan(p), list(list_), mine{0, 0, 0, 0}, first(0) {
        if (plan.lists) {
            total = plan.first(list)[plan.B];
            return;
        }
        const int lane = threadIdx.x & 31;
        VarlenSeq s = {0, 0, 0, 0};
        if (lane < plan.B) s = plan.load(lane, status);
        mine = s;
        number(items(mine));
        if (total > plan.most[list]) {   // sequences overlap
            status[kStatusBadIndexInt] = AMP_DEV_ERR_BAD_INDEX;
            total = 0;
        }
        if (total <= (int)gridDim.x) return;   // an item a CTA: any order will do
        const int key = s.q_len > s.k_len ? s.q_len : s.k_len;
        int rank = 0, from = 0;
        for (int i = 0; i < 32; ++i) {
            const int other = __shfl_sync(0xffffffffu, key, i);
            rank += other > key || (other == key && i < lane);
        }
        for (int i = 0; i < 32; ++i)
            if (__shfl_sync(0xffffffffu, rank, i) == lane) from = i;
        mine.q_off = __shfl_sync(0xffffffffu, s.q_off, from);
        mine.q_len = __shfl_sync(0xffffffffu, s.q_len, from);
        mine.k_off = __shfl_sync(0xffffffffu, s.k_off, from);
        mine.k_len = __shfl_sync(0xffffffffu, s.k_len, from);
        number(items(mine));
    }
    // the lanes' running numbers of items
    __device__ __forceinline__ void number(int n) {
        const int lane = threadIdx.x & 31;
        int end = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, end, o);
            if (lane >= o) end = add_counts(end, t);
        }
        first = end - n;
        total = __shfl_sync(0xffffffffu, end, 31);
    }
    // the CTA's k-th item, k = 0, 1, ...; at or past `total`: no more
    __device__ __forceinline__ int next(int k) const {
        const int grid = (int)gridDim.x, cta = (int)blockIdx.x;
        if (!plan.counted) return k * grid + (k & 1 ? grid - 1 - cta : cta);
        if (k == 0) return cta;
        int item = 0;
        if ((threadIdx.x & 31) == 0) item = grid + atomicAdd(plan.next() + list, 1);
        return __shfl_sync(0xffffffffu, item, 0);
    }
    // the sequence of an item, and the item's number within it
    __device__ __forceinline__ int find(int item, VarlenSeq& s) const {
        if (plan.lists) {
            const int r = varlen_find(plan.first(list), plan.B, item);
            s = plan.seqs()[r];
            return item - plan.first(list)[r];
        }
        const int r = __popc(__ballot_sync(0xffffffffu, first <= item)) - 1;
        s.q_off = __shfl_sync(0xffffffffu, mine.q_off, r);
        s.q_len = __shfl_sync(0xffffffffu, mine.q_len, r);
        s.k_off = __shfl_sync(0xffffffffu, mine.k_off, r);
        s.k_len = __shfl_sync(0xffffffffu, mine.k_len, r);
        return item - __shfl_sync(0xffffffffu, first, r);
    }
};

}  // namespace ampb
