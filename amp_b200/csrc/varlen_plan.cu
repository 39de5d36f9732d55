// varlen_plan.cu -- orders the sequences of a packed batch for the attention
// kernels (varlen.cuh): longest first by a counting sort on the length's leading
// bits, with the running number of work items before each.
//
// One CTA: the work is 16 bytes a sequence, and a grid-wide sort would cost more
// launches than it saves.  The order within one bucket follows from the
// scheduling of the atomics; it decides only which CTA computes an item.
#include <algorithm>

#include "common.cuh"
#include "runtime.h"
#include "tc_common.cuh"
#include "varlen.cuh"

namespace ampb {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kBuckets = 1024;   // == kPlanThreads: one bucket a thread in the scan

// Buckets descend with the length: 5 leading mantissa bits and the exponent of
// the length as a float (31 octaves * 32 < 1024).
__device__ __forceinline__ int length_bucket(int len) {
    if (len <= 0) return kBuckets - 1;
    const unsigned u = __float_as_uint((float)len) >> 18;
    return kBuckets - 2 - (int)(u - (0x3f800000u >> 18));
}

__global__ void __launch_bounds__(kPlanThreads)
    k_varlen_plan(VarlenPlan pl, int Hq, int Hkv, int backward, int parts, int* status) {
    __shared__ int at[kBuckets];
    __shared__ int part[32];
    const int tid = threadIdx.x;
    at[tid] = 0;
    pdl_wait();
    pdl_trigger();   // the attention kernel's CTAs set up meanwhile
    if (tid < 2) pl.next()[tid] = 0;
    __syncthreads();
    for (int b = tid; b < pl.B; b += kPlanThreads) {
        const VarlenSeq s = pl.load(b, status);
        atomicAdd(&at[length_bucket(max(s.q_len, s.k_len))], 1);
    }
    __syncthreads();
    const int mine = at[tid];
    const int end = block_scan(mine, part);
    at[tid] = end - mine;
    __syncthreads();
    for (int b = tid; b < pl.B; b += kPlanThreads) {
        const VarlenSeq s = pl.load(b, status);
        pl.seqs()[atomicAdd(&at[length_bucket(max(s.q_len, s.k_len))], 1)] = s;
    }
    __syncthreads();
    const int group = Hq / Hkv;
    int carry0 = 0, carry1 = 0;
    for (int r0 = 0; r0 < pl.B; r0 += kPlanThreads) {
        const int r = r0 + tid;
        int n0 = 0, n1 = 0;
        if (r < pl.B) {
            const VarlenSeq s = pl.seqs()[r];
            n0 = (backward ? varlen_tiles(s.k_len) : varlen_fwd_pairs(s.q_len, group)) * Hkv * parts;
            n1 = backward ? varlen_tiles(s.q_len) * Hq : 0;
        }
        const int e0 = add_counts(carry0, block_scan(n0, part));
        const int last0 = part[31];
        if (r < pl.B) pl.first(0)[r] = e0 - n0;
        carry0 = add_counts(carry0, last0);
        if (backward) {
            const int e1 = add_counts(carry1, block_scan(n1, part));
            const int last1 = part[31];
            if (r < pl.B) pl.first(1)[r] = e1 - n1;
            carry1 = add_counts(carry1, last1);
        }
    }
    if (tid == 0) {
        const bool over = carry0 > pl.most[0] || carry1 > pl.most[1];   // sequences overlap: no items
        if (over) status[kStatusBadIndexInt] = AMP_DEV_ERR_BAD_INDEX;
        pl.first(0)[pl.B] = over ? 0 : carry0;
        pl.first(1)[pl.B] = over ? 0 : carry1;
    }
}

}  // namespace

int varlen_make_plan(VarlenPlan& plan, int64_t most0, int64_t most1, int Hq, int Hkv, bool backward,
                     int parts, bool zero, cudaStream_t st) {
    AMPB_REQUIRE(most0 <= INT32_MAX / 2 && most1 <= INT32_MAX / 2, AMP_ERR_UNSUPPORTED,
                 "packed attention too large");
    plan.most[0] = (int)most0;
    plan.most[1] = (int)most1;
    // 32 sequences fit a warp.  Up to four items a CTA, dealing them out in turn loses less than
    // the counter's zeroing and its latency cost (forward of 8 prompts of 22 to 200 tokens:
    // 16.4 -> 12.4 us; forward and backward of 17 sequences of up to 700: 65.4 -> 61.7 us); with
    // more, lengths decide (25 sequences of up to 16384 tokens: 9.4 ms dealt, 8.8 counted; 20
    // documents of up to 8192, forward and backward: 10.0 ms dealt, 8.7 counted).
    plan.lists = plan.B > 32;
    plan.counted = plan.lists || std::max(most0, most1) > 4 * sm_count();
    if (!plan.lists) {
        if (plan.counted && zero) AMPB_CHECK_CUDA(cudaMemsetAsync(plan.ws, 0, 64, st));
        return AMP_OK;
    }
    int* status = nullptr;
    int rc = device_status(&status);
    if (rc) return rc;
    AMPB_CHECK_CUDA(launch_pdl(k_varlen_plan, dim3(1), dim3(kPlanThreads), 0, st, plan, Hq, Hkv,
                               backward ? 1 : 0, parts, status));
    return AMP_OK;
}

}  // namespace ampb
