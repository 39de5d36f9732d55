// varlen.cuh -- work lists of the packed-sequence attention kernels.
//
// Packed tensors hold the tokens of B sequences one after another: sequence b is
// rows cu[b] .. cu[b+1] of [total, heads, D].  Lengths are known on the device
// only, so a one-CTA kernel (varlen_plan.cu) turns them into a list that the
// attention kernels' CTAs draw items from: the sequences ordered by length,
// longest first, and the running number of items before each.  An item's index
// is turned back into (sequence, head, tile) by a warp-wide search of that
// prefix.  CTAs draw items from a global counter: with lengths that differ by a
// factor of a hundred no fixed assignment is balanced, and taking the longest
// first leaves only small items for the end.
#pragma once
#include <cuda_runtime.h>
#include <cstddef>
#include <cstdint>

namespace ampb {

struct VarlenSeq {
    int q_off, q_len, k_off, k_len;
};

// Number of 128-row tiles of a sequence.
__host__ __device__ __forceinline__ int varlen_tiles(int len) { return (len + 127) / 128; }

// Items of one sequence in each list.
//   forward: pairs of (query tile, query head) of one kv head
//   dK/dV:   key tiles of one kv head;  dQ: query tiles of one query head
__host__ __device__ __forceinline__ int varlen_fwd_pairs(int q_len, int group) {
    return (varlen_tiles(q_len) * group + 1) / 2;
}

// The lists, in the caller's workspace.
struct VarlenPlan {
    int* next;            // [2] items drawn so far beyond the first of each CTA
    VarlenSeq* seqs;      // [B] longest first
    int* first[2];        // [B + 1] items before sequence r: list 0 (forward or dK/dV), list 1 (dQ)
    int B;
};

inline size_t varlen_plan_bytes(int B) {
    return 64 + (size_t)B * sizeof(VarlenSeq) + 2 * ((size_t)B + 1) * sizeof(int);
}

inline VarlenPlan varlen_plan_at(void* ws, int B) {
    uint8_t* p = static_cast<uint8_t*>(ws);
    VarlenPlan pl;
    pl.next = reinterpret_cast<int*>(p);
    pl.seqs = reinterpret_cast<VarlenSeq*>(p + 64);
    pl.first[0] = reinterpret_cast<int*>(pl.seqs + B);
    pl.first[1] = pl.first[0] + B + 1;
    pl.B = B;
    return pl;
}

// Enqueues the plan kernel; `backward` selects which lists it fills.
int varlen_make_plan(const VarlenPlan& plan, const int* cu_q, const int* cu_kv, int total_q,
                     int total_kv, int Hq, int Hkv, bool backward, cudaStream_t st);

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

}  // namespace ampb
