// flash_attn_bwd.cu -- FlashAttention-2 backward on tcgen05: the lse consumer.
//
// The reference has no backward; its forward documents lse as "required for
// the backward pass" (kernels/flash_attn.cuh:48).  Given Q, K, V, O, dO and the
// forward's lse (natural log):
//   Delta = rowsum(dO * O)                                   k_fa_bwd_delta
//     (packed, rows of few keys: rowsum(P * dP)              k_fa_bwd_few)
//   P = exp(scale Q K^T - lse),  dP = dO V^T,  dS = P * (dP - Delta)
//   dV = P^T dO,  dK = scale dS^T Q,  dQ = scale dS K
// in two passes shaped like the forward, so every product is one of its MMA
// forms (SS, K-major x K-major; TS with P / dS in TMEM and an MN-major B):
//   k_fa_bwd_dkdv  per (batch * kv head, 128-key tile), on persistent CTAs (one
//                  per SM) that walk pairs of such tiles.  S^T = K Q^T and
//                  dP^T = V dO^T put keys on the TMEM lanes; P^T and dS^T go
//                  back over them as bf16; dV += P^T dO and dK += dS^T Q
//                  accumulate in TMEM over every query tile of every query head
//                  that shares the kv head (GQA).
//   k_fa_bwd_dq    per (batch * query head, 128-query tile), on persistent
//                  CTAs (one per SM) that walk pairs of such tiles.  S = Q K^T,
//                  dP = dO V^T with queries on the lanes; dS back over dP;
//                  dQ += dS K over the visible key tiles.
// Steps overlap: the element-wise warps write P (or P^T) first and dS after, so
// the tensor core takes the next step's S^T while dS^T is computed (dK/dV pass:
// dV_t, S^T_{t+1}, dK_t, dP^T_{t+1}); the dQ pass keeps two S buffers in TMEM
// (S_{j+1}, dQ_j, dP_{j+1}).
// Each pass recomputes P from lse, so there are no atomics and no fp32 dQ
// accumulator in global memory.
// Packed mode, few key tiles: an item sums over the query tiles of all query heads of its kv
// head, so a short batch with large groups leaves most CTAs idle behind a few long items
// (one kv head for 8 query heads, 2000 tokens: 16 items of up to 128 steps).  There the query
// heads are shared out among items of their own, which leave fp32 sums that k_fa_bwd_join
// adds in order (no atomics; the same bits every time).
// Packed mode (sequences of different lengths one after another, varlen.cuh): both
// passes draw their tiles from lists of the sequences, longest first, most steps first;
// warp 3 decodes items ahead into a two-slot ring.  A tile that runs past its sequence
// brings rows of the next one.  Where those rows would be summed over (Q and dO in the
// dK/dV pass, K and V in the dQ pass) warp 2 zeroes them in shared memory before the
// MMAs may read them; where they are rows of the output they are just not stored.
// Measured: 20 documents of up to 8192 tokens (46763 in all, 32 / 8 heads, D 128), forward and
// backward, 8.7 ms = 741 TFLOP/s, the dense passes' rate.
// Both kernels: 384 threads; warp 0 TMA, warp 1
// TMEM + MMA issue (warps 2-3 only lend their registers, setmaxnreg 72 / 216);
// warps 4-11 the element-wise work, two warps per TMEM lane quadrant (one row
// per thread), each taking one 64-column half of the 128-column tile.
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "common.cuh"
#include "runtime.h"
#include "tc_common.cuh"
#include "varlen.cuh"

namespace ampb {

int fa_make_tmap_3d(CUtensorMap* m, const void* base, int64_t d, int64_t s, int64_t bh);
int fa_make_tmap_packed(CUtensorMap* m, const void* base, int64_t d, int64_t tokens, int64_t heads,
                        int64_t tok_stride, int64_t head_stride);
int varlen_check(int B, int total_q, int total_kv, int Hq, int Hkv, int D, const int* cu_q,
                 const int* cu_kv, const int64_t* strides, int n_strides, const void* ws,
                 size_t ws_bytes, size_t need);

namespace {

constexpr int BT = 128;                 // rows per query / key tile
constexpr int kThreads = 384;      // 3 warpgroups
// Register split: 128 * 72 + 256 * 216 == 384 * 168, the launch's allocation
// (__launch_bounds__(384, 1) compiles for exactly 168).
constexpr int kRegCtl = 72, kRegEw = 216;
constexpr int SLAB_BYTES = 128 * 128;   // [128 rows x 128 bytes] swizzled slab
constexpr float kLog2e = 1.4426950408889634f;

template <int D>
struct BwdCfg {
    static constexpr int SLABS = D / 64;
    static constexpr int TILE = SLABS * SLAB_BYTES;          // 128 rows x D bf16
    // tiles, lse and Delta columns, alignment, barriers with the packed items
    static constexpr int SMEM_KV = 6 * TILE + 2 * 2 * BT * 4 + 1024 + 384;
    static constexpr int SMEM_Q = 6 * TILE + 1024 + 384;
    static constexpr uint32_t IDESC_SS = make_idesc(1, 1, 0, 0, BT, BT);
    static constexpr uint32_t IDESC_TS = make_idesc(1, 1, 0, 1, BT, D);
};

struct BwdParams {
    int B, Hq, Hkv, S_q, S_kv;
    int causal, causal_offset;   // key j visible for query i iff j <= i + causal_offset
    float scale, scale_log2;
    const float* lse;            // [B*Hq][S_q], natural log (forward output)
    const float* delta;          // [B*Hq][S_q]
    void* dq;                    // [B*Hq][S_q][D] bf16
    void* dk;                    // [B*Hkv][S_kv][D] bf16
    void* dv;
    int* status;
    // packed mode: rows of the whole Q (lse, delta are [Hq][total_q]), strides of the
    // gradients in elements, the work lists
    int total_q, total_kv, after_dkdv;
    // the query heads of a kv head are summed in so many parts, each [total_kv][Hkv][D] of
    // dK, then of dV, in `sums`
    int parts;
    float* sums;
    int64_t dq_tok, dq_head, dk_tok, dk_head, dv_tok, dv_head;
    VarlenPlan plan;
};

// One item: a 128-row tile of one head of one sequence (dense: of one batch entry).
struct BwdItem {
    int live;                   // packed: 0 ends the list
    int b, head, tile;          // head: kv head (dK/dV) or query head (dQ) within b
    int g0, heads, part;        // dK/dV: query heads of the group that it sums, and its part
    int q_tok, k_tok;           // packed: the sequence's first rows
    int S_q, S_kv;
    int coff;                   // key j visible for query i iff j <= i + coff
};

// Packed mode, warp 3: draws item after item of its list and publishes it.  It and warp 2
// sleep in their waits: polling would take issue slots from the element-wise warps.
template <bool kKeys>
__device__ __forceinline__ void draw_items(const BwdParams& p, BwdItem* items, uint64_t* it_full,
                                           uint64_t* it_empty) {
    const int lane = threadIdx.x & 31;
    VarlenDraw draw(p.plan, kKeys ? 0 : 1, [&](const VarlenSeq& s) {
        return kKeys ? varlen_tiles(s.k_len) * p.Hkv * p.parts : varlen_tiles(s.q_len) * p.Hq;
    }, p.status);
    for (int k = 0;; ++k) {
        if (k >= 2 && !mbar_wait_warp<true, kItemLimits>(&it_empty[k & 1], ((k >> 1) & 1) ^ 1, p.status)) return;
        const int item = draw.next(k);
        BwdItem it = {};
        if (item < draw.total) {
            VarlenSeq sq;
            int w = draw.find(item, sq);   // number within its sequence
            const int n = varlen_tiles(kKeys ? sq.k_len : sq.q_len);
            if constexpr (kKeys) {
                const int group = p.Hq / p.Hkv;
                it.part = w % p.parts;
                w /= p.parts;
                it.g0 = it.part * group / p.parts;
                it.heads = (it.part + 1) * group / p.parts - it.g0;
            }
            it.live = 1;
            it.head = w / n;
            // under a causal mask the first keys and the last queries have the most steps
            it.tile = kKeys ? w % n : n - 1 - w % n;
            it.q_tok = sq.q_off;
            it.k_tok = sq.k_off;
            it.S_q = sq.q_len;
            it.S_kv = sq.k_len;
        }
        if (lane == 0) {
            items[k & 1] = it;
            mbar_arrive(&it_full[k & 1]);
        }
        __syncwarp();
        if (item >= draw.total) return;
    }
}

// Reads the k-th published item; false at the end (or when a wait ran out).  What comes out of
// shared memory is not known to be the same in every lane, and what is derived from it would be
// converted for every MMA; a shuffle from lane 0 makes it known.
template <typename Who>
__device__ __forceinline__ bool read_item(int k, const BwdItem* items, uint64_t* it_full,
                                          int* status, BwdItem& it) {
    if (!Who::wait(&it_full[k & 1], (k >> 1) & 1, status)) return false;
    const BwdItem& src = items[k & 1];
    it.live = same_in<Who>(src.live);
    it.b = 0;
    it.head = same_in<Who>(src.head);
    it.tile = same_in<Who>(src.tile);
    it.g0 = same_in<Who>(src.g0);
    it.heads = same_in<Who>(src.heads);
    it.part = same_in<Who>(src.part);
    it.q_tok = same_in<Who>(src.q_tok);
    it.k_tok = same_in<Who>(src.k_tok);
    it.S_q = same_in<Who>(src.S_q);
    it.S_kv = same_in<Who>(src.S_kv);
    it.coff = it.S_kv - it.S_q;
    return it.live != 0;
}

// Packed mode, warp 2: once the tile has landed, zeroes its rows from `valid` on (one
// or two tiles of `slabs` slabs each) and passes it on to the MMA warp.
__device__ __forceinline__ bool zero_tail(uint64_t* raw, uint32_t parity, uint64_t* full,
                                          uint8_t* tile0, uint8_t* tile1, int slabs, int valid,
                                          int* status) {
    if (!mbar_wait_warp<true, kItemLimits>(raw, parity, status)) return false;
    const int lane = threadIdx.x & 31;
    for (int i = valid * 8 + lane; i < BT * 8; i += 32)
        for (int sl = 0; sl < slabs; ++sl) {
            *reinterpret_cast<uint4*>(tile0 + sl * SLAB_BYTES + i * 16) = make_uint4(0u, 0u, 0u, 0u);
            if (tile1)
                *reinterpret_cast<uint4*>(tile1 + sl * SLAB_BYTES + i * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(full);
    return true;
}

// SS product of two 128-row K-major tiles over D: acc[128 x 128] (+)= A B^T
template <int D>
__device__ __forceinline__ void mma_ss(uint32_t acc, uint32_t a_addr, uint32_t b_addr) {
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
        const uint32_t off = (kk >> 2) * SLAB_BYTES + (kk & 3) * 32;
        tc_mma_f16(acc, smem_desc_sw128(a_addr + off, 16, 1024),
                   smem_desc_sw128(b_addr + off, 16, 1024), BwdCfg<D>::IDESC_SS, kk != 0);
    }
}
// TS product: acc[128 x D] (+)= T[128 x 128] (bf16 in TMEM) x B[128 rows x D] (MN-major).
// T is packed two bf16 per column in two halves: its columns 0-63 at TMEM
// columns [t_col, t_col + 32), 64-127 at [t_col + 96, t_col + 128) -- where the
// two element-wise warps of a lane quadrant write them (see the element-wise code).
template <int D>
__device__ __forceinline__ void mma_ts(uint32_t acc, uint32_t t_col, uint32_t b_addr,
                                       bool accumulate) {
#pragma unroll
    for (int kk = 0; kk < BT / 16; ++kk)
        tc_mma_f16_ts(acc, t_col + kk * 8 + (kk >= BT / 32 ? BT / 2 : 0),
                      smem_desc_sw128(b_addr + kk * 16 * 128, SLAB_BYTES, 1024),
                      BwdCfg<D>::IDESC_TS, (accumulate || kk != 0) ? 1u : 0u);
}

// ---------------------------------------------------------------- Delta
// Delta[row] = sum_d dO[row][d] * O[row][d] in fp32.  HBM-bound (reads O and dO
// once): D/8 lanes per row with 16-byte loads, kDeltaLoads rows per lane group in
// flight, and the row's partial sums reduced within its lane group.
constexpr int kDeltaLoads = 4;
// Packed: row r is head r % H of token r / H (the order in which a contiguous
// [total, H, D] lies in memory), read through the strides and stored at [head][token].
struct DeltaStrides {
    int64_t o_tok, o_head, do_tok, do_head;
    int H, total;
    int* next;   // the two passes' counters to zero, or null
};
template <int D, bool kPacked = false>
__global__ void __launch_bounds__(256) k_fa_bwd_delta(const __nv_bfloat16* __restrict__ O,
                                                      const __nv_bfloat16* __restrict__ dO,
                                                      float* __restrict__ delta, int64_t rows,
                                                      DeltaStrides st = {}) {
    pdl_wait();
    pdl_trigger();
    if (kPacked && st.next && blockIdx.x == 0 && threadIdx.x < 2) st.next[threadIdx.x] = 0;
    constexpr int LPR = D / 8;            // lanes per row, 8 bf16 (16 bytes) each
    constexpr int RPW = 32 / LPR;         // rows per warp-wide load
    constexpr int ROWS = RPW * kDeltaLoads;
    static_assert(LPR >= 1 && LPR <= 32 && (LPR & (LPR - 1)) == 0, "D/8 lanes per row");
    const int lane = threadIdx.x & 31;
    const int sub = lane / LPR, col = (lane % LPR) * 8;
    const int64_t nwarps = (int64_t)gridDim.x * 8;
    for (int64_t r0 = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * ROWS; r0 < rows;
         r0 += nwarps * ROWS) {
        uint4 o[kDeltaLoads], g[kDeltaLoads];
        // packed: token and head of this lane's rows, by one division for all of them (one a
        // row made the pass issue-bound: 45 -> 36 us, 6.2 TB/s, for 13609 tokens x 32 heads x 128)
        int t[kDeltaLoads], h[kDeltaLoads];
        if constexpr (kPacked) {
            t[0] = (int)(r0 + sub) / st.H;
            h[0] = (int)(r0 + sub) - t[0] * st.H;
#pragma unroll
            for (int u = 1; u < kDeltaLoads; ++u) {
                t[u] = t[u - 1];
                h[u] = h[u - 1] + RPW;
                while (h[u] >= st.H) {
                    h[u] -= st.H;
                    ++t[u];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kDeltaLoads; ++u) {
            const int64_t r = r0 + u * RPW + sub;
            if (r < rows) {
                if constexpr (kPacked) {
                    o[u] = *reinterpret_cast<const uint4*>(O + t[u] * st.o_tok + h[u] * st.o_head + col);
                    g[u] = *reinterpret_cast<const uint4*>(dO + t[u] * st.do_tok + h[u] * st.do_head + col);
                } else {
                    o[u] = *reinterpret_cast<const uint4*>(O + r * D + col);
                    g[u] = *reinterpret_cast<const uint4*>(dO + r * D + col);
                }
            } else {
                o[u] = make_uint4(0u, 0u, 0u, 0u);
                g[u] = o[u];
            }
        }
#pragma unroll
        for (int u = 0; u < kDeltaLoads; ++u) {
            const uint32_t ow[4] = {o[u].x, o[u].y, o[u].z, o[u].w};
            const uint32_t gw[4] = {g[u].x, g[u].y, g[u].z, g[u].w};
            float acc = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                acc = fmaf(bf16_lo(ow[i]), bf16_lo(gw[i]), acc);
                acc = fmaf(bf16_hi(ow[i]), bf16_hi(gw[i]), acc);
            }
#pragma unroll
            for (int m = LPR / 2; m > 0; m >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, m);
            const int64_t r = r0 + u * RPW + sub;
            if (lane % LPR == 0 && r < rows) {
                if constexpr (kPacked)
                    delta[(int64_t)h[u] * st.total + t[u]] = acc;
                else
                    delta[r] = acc;
            }
        }
    }
}

// ------------------------------------------------------- Delta of rows of few keys
// Queries of a sequence that see few keys (1 to kFewKeys): row0 .. row0 + n.  O is rounded to
// bf16, and in a row of n keys that moves Delta by about 1 / sqrt(n) of what rounding dS does, all
// entries of the row together; beyond 32 keys there is little left to gain.  Error
// of dQ and dK against fp64, with Delta from O -> with these rows' Delta from the unrounded
// P and dP (both passes' sum of P dP): sequences of 8 tokens 0.0034 -> 0.0023, of 20 0.0030 -> 0.0024,
// of up to 700 0.0026 -> 0.0024; outputs and dS rounded alone: 0.0024.
constexpr int kFewKeys = 32;
struct FewRows {
    int row0, n;
};
__device__ __forceinline__ FewRows few_rows(const VarlenSeq& s, int causal) {
    if (!causal) return {0, s.k_len >= 1 && s.k_len <= kFewKeys ? s.q_len : 0};
    // query i sees i + 1 + (k_len - q_len) keys
    const int first = max(0, s.q_len - s.k_len);
    const int64_t end = (int64_t)kFewKeys + s.q_len - s.k_len;
    return {first, (int)max((int64_t)0, min((int64_t)s.q_len, end) - first)};
}

struct Frag4 { uint32_t x[4]; };
struct Frag2 { uint32_t x[2]; };
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], const Frag4& a, const Frag2& b) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
                 "{%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a.x[0]), "r"(a.x[1]), "r"(a.x[2]), "r"(a.x[3]), "r"(b.x[0]), "r"(b.x[1]));
}

struct FewParams {
    const __nv_bfloat16 *q, *k, *v, *d_o;
    int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, do_tok, do_head;
    const float* lse;
    float* delta;
    int Hq, Hkv, causal, strips;   // strips: warps of a (sequence, head)
    float scale_log2;
    int* status;
    VarlenPlan plan;
};

// Delta of 16 such rows (from row0 on, below row_end) of one head by one warp: the scores and dP
// of up to 32 keys are 16 x 8 tiles of mma.sync, whose few products end before operands for tcgen05
// would be staged.  A lane loads 16 bytes of a row, 8 neighbouring elements, and gives them to the
// MMA as the columns that it has to bring in two steps: a dot product may be summed in any order,
// as long as both operands keep one.
// Measured, whole backward without -> with these rows: 17 sequences of up to 700 tokens (8 heads, D 64)
// 46 -> 46 us, 20 documents of up to 8192 unchanged; 200 sequences of 30 tokens 80 -> 87; 1000 of 30
// (32 / 8 heads, D 128) 1464 -> 1640, where nearly all rows see few keys and what it adds is
// reading q, k, v and dO once more.  (4-byte loads in the MMA's own order: 2080; all 32 keys at once
// in 160 registers: 1708; 80 registers: 1678; in the Delta kernel's own blocks, whose rows then have
// to be looked up: 1686.)
template <int D>
__device__ __forceinline__ float2 few_tile(const FewParams& st, const VarlenSeq& s, int row0, int row_end, int h) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = (lane & 3) * 8;
    // (a row or key past the end is read as the last one: MMA rows and columns do not mix)
    const __nv_bfloat16 *qp[2], *op[2];
    // as the passes take it; a row that sees no key, or is none, takes no part
    int seen[2];
    float nl2[2], acc[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int row = row0 + g + i * 8;
        const int64_t tok = s.q_off + min(row, row_end - 1);
        qp[i] = st.q + tok * st.q_tok + h * st.q_head + c;
        op[i] = st.d_o + tok * st.do_tok + h * st.do_head + c;
        seen[i] = row >= row_end ? 0 : st.causal ? row + 1 + s.k_len - s.q_len : s.k_len;
        const float lse = seen[i] > 0 ? st.lse[(int64_t)h * st.plan.total_q + tok] : -INFINITY;
        nl2[i] = lse == -INFINITY ? -INFINITY : -lse * kLog2e;
    }
    const int keys = st.causal ? min(row0 + 16, row_end) + s.k_len - s.q_len : s.k_len;   // seen by the last row
    const int hk = h / (st.Hq / st.Hkv);
    auto eight = [](const __nv_bfloat16* p) { return *reinterpret_cast<const uint4*>(p); };
    constexpr int kTiles = 2;   // of 8 keys at a time
#pragma unroll 1
    for (int n0 = 0; n0 < keys; n0 += kTiles * 8) {
        const __nv_bfloat16 *kp[kTiles], *vp[kTiles];
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
            const int64_t tok = s.k_off + min(n0 + n * 8 + g, keys - 1);
            kp[n] = st.k + tok * st.k_tok + hk * st.k_head + c;
            vp[n] = st.v + tok * st.v_tok + hk * st.v_head + c;
        }
        float sc[kTiles][4] = {}, dp[kTiles][4] = {};
#pragma unroll 1
        for (int e = 0; e < D; e += 32) {
            const uint4 q0 = eight(qp[0] + e), q1 = eight(qp[1] + e), o0 = eight(op[0] + e), o1 = eight(op[1] + e);
            uint4 kv[kTiles], vv[kTiles];
#pragma unroll
            for (int n = 0; n < kTiles; ++n) kv[n] = eight(kp[n] + e), vv[n] = eight(vp[n] + e);
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
                mma_16x8x16(sc[n], {q0.x, q1.x, q0.y, q1.y}, {kv[n].x, kv[n].y});
                mma_16x8x16(dp[n], {o0.x, o1.x, o0.y, o1.y}, {vv[n].x, vv[n].y});
                mma_16x8x16(sc[n], {q0.z, q1.z, q0.w, q1.w}, {kv[n].z, kv[n].w});
                mma_16x8x16(dp[n], {o0.z, o1.z, o0.w, o1.w}, {vv[n].z, vv[n].w});
            }
        }
        const int col = n0 + (lane & 3) * 2;
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (col + n * 8 + (i & 1) < seen[i >> 1])
                    acc[i >> 1] = fmaf(ex2_approx(fmaf(sc[n][i], st.scale_log2, nl2[i >> 1])), dp[n][i], acc[i >> 1]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], 1);
        acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], 2);
    }
    return make_float2(acc[0], acc[1]);   // of rows g and g + 8, in every lane of four
}

// A warp takes a (sequence, head)'s tiles of 16 rows: one of at most two under a causal mask, every
// strips-th of all rows of a sequence with few keys under a full one.  Runs beside k_fa_bwd_delta,
// which forms Delta of every row: only the store has to wait for that kernel's end.  What this one
// reads is there before: each of that kernel's blocks waited for it before it let this one launch.
template <int D>
__global__ void __launch_bounds__(256, 2) k_fa_bwd_few(const __grid_constant__ FewParams p) {
    pdl_trigger();
    const int lane = threadIdx.x & 31, g = lane >> 2;
    bool waited = false;
    // (B * Hq is below 2^30: varlen_check.)  Sequences that the plan refused (varlen_make_plan) get no
    // work here either.
    const bool none = p.plan.lists && p.plan.first(0)[p.plan.B] == 0;
    const unsigned total = none ? 0u : (unsigned)p.plan.B * p.Hq * p.strips;
    for (unsigned w = blockIdx.x * 8 + (threadIdx.x >> 5); w < total; w += gridDim.x * 8) {
        // heads first: the warps of a block share keys
        const unsigned bs = w / (unsigned)p.Hq;
        const int h = (int)(w - bs * p.Hq), strip = (int)(bs % (unsigned)p.strips);
        const VarlenSeq s = p.plan.load((int)(bs / (unsigned)p.strips), p.status);
        const FewRows rows = few_rows(s, p.causal);
        for (int r = strip * 16; r < rows.n; r += p.strips * 16) {
            const int row0 = rows.row0 + r, end = rows.row0 + rows.n;
            const float2 d = few_tile<D>(p, s, row0, end, h);
            if (!waited) pdl_wait();
            waited = true;
            float* at = p.delta + (int64_t)h * p.plan.total_q + s.q_off + row0 + g;
            if ((lane & 3) == 0 && row0 + g < end) at[0] = d.x;
            if ((lane & 3) == 0 && row0 + g + 8 < end) at[8] = d.y;
        }
    }
    if (!waited) pdl_wait();
}

// The P that dS = P (dP - Delta) multiplies with.  Dense: as rounded to bf16 for P^T dO.
// Packed: as computed, in fp32 (dQ and dK then carry two roundings to bf16, of dS and their
// own, instead of three: an error of 0.0024 instead of 0.0030 relative to fp64; the outputs'
// rounding alone is 0.0017).  dS is rounded because the tensor core multiplies 16-bit operands.
// Delta is formed from O as the forward rounded it, the only O there is, except in rows of few
// keys, where that rounding is felt (few_rows).
template <bool kExact>
struct Probs {
    float v[kExact ? 64 : 1];
    __device__ __forceinline__ void keep(int e, float p0, float p1) {
        if constexpr (kExact) v[e] = p0, v[e + 1] = p1;
    }
    __device__ __forceinline__ uint64_t pair(int e, const uint32_t* rounded) const {
        if constexpr (kExact) return f2pack(v[e], v[e + 1]);
        else return f2pack(bf16_lo(rounded[e >> 1]), bf16_hi(rounded[e >> 1]));
    }
};

// store columns [half * D/2, half * D/2 + D/2) of one 128 x D fp32 TMEM
// accumulator row (this thread's lane) as bf16 * mul
template <int D>
__device__ __forceinline__ void store_row(uint32_t lane_addr, float mul, __nv_bfloat16* row,
                                          bool ok, int half) {
    __syncwarp();
#pragma unroll
    for (int ocl = 0; ocl < D / 64; ++ocl) {
        const int oc = half * (D / 64) + ocl;
        uint32_t v[32];
        tmem_ld_32x32b_x32(lane_addr + oc * 32, v);
        tmem_ld_wait();
        if (ok) {
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
                uint4 w;
                w.x = f32x2_to_bf16x2(__uint_as_float(v[e]) * mul, __uint_as_float(v[e + 1]) * mul);
                w.y = f32x2_to_bf16x2(__uint_as_float(v[e + 2]) * mul, __uint_as_float(v[e + 3]) * mul);
                w.z = f32x2_to_bf16x2(__uint_as_float(v[e + 4]) * mul, __uint_as_float(v[e + 5]) * mul);
                w.w = f32x2_to_bf16x2(__uint_as_float(v[e + 6]) * mul, __uint_as_float(v[e + 7]) * mul);
                *reinterpret_cast<uint4*>(row + oc * 32 + e) = w;
            }
        }
    }
}

template <int D>
__device__ __forceinline__ void store_zero_row(__nv_bfloat16* row, int half) {
#pragma unroll
    for (int e = half * (D / 2); e < (half + 1) * (D / 2); e += 8)
        *reinterpret_cast<uint4*>(row + e) = make_uint4(0u, 0u, 0u, 0u);
}

// the same as fp32, for the parts of dK and dV
template <int D>
__device__ __forceinline__ void store_sums(uint32_t lane_addr, float mul, float* row, bool ok, int half) {
    __syncwarp();
#pragma unroll
    for (int ocl = 0; ocl < D / 64; ++ocl) {
        const int oc = half * (D / 64) + ocl;
        uint32_t v[32];
        tmem_ld_32x32b_x32(lane_addr + oc * 32, v);
        tmem_ld_wait();
        if (ok) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
                *reinterpret_cast<float4*>(row + oc * 32 + e) =
                    make_float4(__uint_as_float(v[e]) * mul, __uint_as_float(v[e + 1]) * mul,
                                __uint_as_float(v[e + 2]) * mul, __uint_as_float(v[e + 3]) * mul);
        }
    }
}
template <int D>
__device__ __forceinline__ void store_zero_sums(float* row, int half) {
#pragma unroll
    for (int e = half * (D / 2); e < (half + 1) * (D / 2); e += 4)
        *reinterpret_cast<float4*>(row + e) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
}

// Adds the parts up, in order, and rounds once: a warp a token of some sequence, four
// elements a lane (the parts of a row are total_kv rows apart).
template <int D>
__global__ void __launch_bounds__(256) k_fa_bwd_join(BwdParams p) {
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int per_row = p.Hkv * (D / 4);
    const int64_t part = (int64_t)p.total_kv * p.Hkv * D;
    for (int t = blockIdx.x * 8 + (threadIdx.x >> 5); t < p.total_kv; t += gridDim.x * 8) {
        if (varlen_owner<true>(p.plan, t, p.status).k_len == 0) continue;   // a token of no sequence
        for (int i = lane; i < 2 * per_row; i += 32) {
            const bool v = i >= per_row;
            const int c = v ? i - per_row : i;   // four elements c * 4 of the token's heads
            const float* src = p.sums + (v ? p.parts * part : 0) + (int64_t)t * p.Hkv * D + c * 4;
            float4 a = *reinterpret_cast<const float4*>(src);
            for (int z = 1; z < p.parts; ++z) {
                const float4 b = *reinterpret_cast<const float4*>(src + z * part);
                a = make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
            }
            const int h = c / (D / 4), e = c % (D / 4) * 4;
            __nv_bfloat16* dst = v ? static_cast<__nv_bfloat16*>(p.dv) + t * p.dv_tok + h * p.dv_head
                                   : static_cast<__nv_bfloat16*>(p.dk) + t * p.dk_tok + h * p.dk_head;
            uint2 w;
            w.x = f32x2_to_bf16x2(a.x, a.y);
            w.y = f32x2_to_bf16x2(a.z, a.w);
            *reinterpret_cast<uint2*>(dst + e) = w;
        }
    }
}

// ---------------------------------------------------------------- dK, dV
template <int D, bool kPacked = false>
__global__ void __launch_bounds__(kThreads, 1)
    k_fa_bwd_dkdv(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmdO,
                  const BwdParams p) {
    pdl_wait();
    pdl_trigger();
    using CF = BwdCfg<D>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~uintptr_t(1023));
    uint8_t* k_s = smem;                          // K_j
    uint8_t* v_s = k_s + CF::TILE;                // V_j
    uint8_t* q_s = v_s + CF::TILE;                // [2][Q_i]
    uint8_t* o_s = q_s + 2 * CF::TILE;            // [2][dO_i]
    float* cols = reinterpret_cast<float*>(o_s + 2 * CF::TILE);   // [2][2][128] lse2, Delta
    uint64_t* bars = reinterpret_cast<uint64_t*>(cols + 2 * 2 * BT);
    uint64_t* kv_full = bars;
    uint64_t* qs_full = bars + 1;     // [2]
    uint64_t* qs_empty = bars + 3;    // [2]
    uint64_t* s_full = bars + 5;      // S^T of the step in TMEM
    uint64_t* dp_full = bars + 6;     // dP^T of the step in TMEM
    uint64_t* p_full = bars + 7;      // P^T written back (8 warps)
    uint64_t* ds_full = bars + 8;     // dS^T written back (8 warps)
    // bars + 9: unused (S^T_{t+1} follows dV_t in MMA issue order, no barrier between)
    uint64_t* dk_done = bars + 10;    // dK has read dS^T: dP^T may be rewritten
    uint64_t* drain = bars + 11;
    uint64_t* cols_ready = bars + 12; // [2]: the 256 element-wise threads posted the step
    uint64_t* kv_empty = bars + 14;   // the item's last MMA reading K / V has completed
    uint64_t* dkv_free = bars + 15;   // the item's epilogue has read dK, dV out of TMEM
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 16);
    uint64_t* it_full = bars + 17;    // [2] packed items
    uint64_t* it_empty = bars + 19;   // [2] load, MMA and zeroing warps, 8 element-wise warps
    uint64_t* qs_raw = bars + 21;     // [2] Q / dO loaded, rows past the end not yet zeroed
    BwdItem* items = reinterpret_cast<BwdItem*>(bars + 23);   // [2]

    const int lane = threadIdx.x & 31;
    const int warp = kPacked ? same_in<WholeWarp<false>>(threadIdx.x >> 5) : threadIdx.x >> 5;
    const int G = p.Hq / p.Hkv;
    const int n_kt = (p.S_kv + BT - 1) / BT;
    // Persistent: unit u = blockIdx.x + (k/2) * gridDim.x pairs key tile n_kt-1-q with
    // key tile q of one kv head (under a causal mask they see the fewest and the most
    // query tiles), so the units of a causal square problem carry the same work.
    const int half_units = (n_kt + 1) / 2;
    const int units = p.B * p.Hkv * half_units;
    // k-th item of this CTA: 0 = no more, 1 = item (bh_kv, jt), 2 = empty slot
    auto item_at = [&](int k, int& bh_kv, int& jt) -> int {
        const int u = (int)blockIdx.x + (k >> 1) * (int)gridDim.x;
        if (u >= units) return 0;
        bh_kv = u / half_units;
        const int q = u % half_units;
        jt = (k & 1) ? q : n_kt - 1 - q;
        return ((k & 1) && q == n_kt - 1 - q) ? 2 : 1;
    };
    // the same with the item's geometry; packed: from the ring, released with it_done
    auto next_item = [&](int k, BwdItem& it, auto who) -> int {
        if constexpr (kPacked) {
            return read_item<decltype(who)>(k, items, it_full, p.status, it) ? 1 : 0;
        } else {
            int bh_kv, jt;
            const int st = item_at(k, bh_kv, jt);
            if (st == 1) {
                it.b = bh_kv / p.Hkv;
                it.head = bh_kv % p.Hkv;
                it.g0 = it.part = 0;
                it.heads = G;
                it.tile = jt;
                it.q_tok = it.k_tok = 0;
                it.S_q = p.S_q;
                it.S_kv = p.S_kv;
                it.coff = p.causal_offset;
            }
            return st;
        }
    };
    auto it_done = [&](int k) {
        if constexpr (kPacked) mbar_arrive(&it_empty[k & 1]);
    };
    // first query tile with a query that sees a key of the item's tile
    auto first_tile = [&](const BwdItem& it) {
        int i_lo = 0;
        if (p.causal) {
            const int first_q = it.tile * BT - it.coff;
            i_lo = first_q <= 0 ? 0 : first_q / BT;
        }
        return i_lo;
    };
    auto q_tiles = [&](const BwdItem& it) { return (it.S_q + BT - 1) / BT; };

    if (threadIdx.x == 0) {
        mbar_init(kv_full, 1);
        mbar_init(kv_empty, 1);
        mbar_init(dkv_free, 8);
        for (int s = 0; s < 2; ++s) {
            mbar_init(&qs_full[s], 1);
            mbar_init(&qs_empty[s], 1);
        }
        mbar_init(s_full, 1);
        mbar_init(dp_full, 1);
        mbar_init(p_full, 8);
        mbar_init(ds_full, 8);
        mbar_init(dk_done, 1);
        mbar_init(drain, 1);
        mbar_init(&cols_ready[0], 256);
        mbar_init(&cols_ready[1], 256);
        if constexpr (kPacked) {
            for (int i = 0; i < 2; ++i) {
                mbar_init(&it_full[i], 1);
                mbar_init(&it_empty[i], 11);
                mbar_init(&qs_raw[i], 1);
            }
        }
        fence_barrier_init();
        fence_proxy_async_smem();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = kPacked ? 0u : *tmem_slot;   // all 512 columns start at column 0
    const uint32_t T_S = tmem, T_dP = tmem + BT, T_dV = tmem + 2 * BT, T_dK = tmem + 2 * BT + D;

    if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegCtl));
    if (warp == 0) {
        if (lane == 0) {
            tma_prefetch_desc(&tmQ);
            tma_prefetch_desc(&tmdO);
            int g = 0, li = 0;   // Q/dO tiles loaded (ring stage g & 1); items with work
            bool ok = true;
            for (int k = 0; ok; ++k) {
                BwdItem it;
                const int st = next_item(k, it, OneLane{});
                if (st == 0) break;
                if (st == 2) continue;
                it_done(k);
                const int i_lo = first_tile(it);
                const int per_head = max(0, q_tiles(it) - i_lo);
                const int steps = it.heads * per_head;
                if (steps == 0) continue;
                const int b = it.b, hk = it.head, bh_kv = b * p.Hkv + hk;
                const int k_row = it.k_tok + it.tile * BT;
                // K_j / V_j once the previous item's last MMA reading them has completed
                if (li > 0 && !mbar_wait(kv_empty, (li - 1) & 1, p.status)) break;
                mbar_arrive_expect_tx(kv_full, 2 * CF::TILE);
#pragma unroll
                for (int sl = 0; sl < CF::SLABS; ++sl) {
                    tma_load_3d(k_s + sl * SLAB_BYTES, &tmK, kv_full, sl * 64, k_row, bh_kv);
                    tma_load_3d(v_s + sl * SLAB_BYTES, &tmV, kv_full, sl * 64, k_row, bh_kv);
                }
                for (int t = 0; t < steps; ++t, ++g) {
                    const int s = g & 1;
                    if (!mbar_wait(&qs_empty[s], ((g >> 1) & 1) ^ 1, p.status)) { ok = false; break; }
                    const int gq = it.g0 + t / per_head, qt = i_lo + t % per_head;
                    const int bh_q = b * p.Hq + hk * G + gq;
                    // packed: a tile past the sequence's end goes to warp 2 first
                    uint64_t* bar = kPacked && (qt + 1) * BT > it.S_q ? &qs_raw[s] : &qs_full[s];
                    mbar_arrive_expect_tx(bar, 2 * CF::TILE);
#pragma unroll
                    for (int sl = 0; sl < CF::SLABS; ++sl) {
                        tma_load_3d(q_s + s * CF::TILE + sl * SLAB_BYTES, &tmQ, bar, sl * 64,
                                    it.q_tok + qt * BT, bh_q);
                        tma_load_3d(o_s + s * CF::TILE + sl * SLAB_BYTES, &tmdO, bar, sl * 64,
                                    it.q_tok + qt * BT, bh_q);
                    }
                }
                ++li;
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            // tensor-core order per step t:  dV_t, S^T_{t+1}, dK_t, dP^T_{t+1} -- so the
            // next step's S^T runs while the element-wise warps compute dS^T_t
            const uint32_t ka0 = smem_u32(k_s), va0 = smem_u32(v_s);
            auto qa = [&](int g) { return opaque_u32(smem_u32(q_s + (g & 1) * CF::TILE)); };
            auto oa = [&](int g) { return opaque_u32(smem_u32(o_s + (g & 1) * CF::TILE)); };
            int g = 0, li = 0;   // steps before this item; items with work before it
            bool ok = true;
            for (int k = 0; ok; ++k) {
                BwdItem it;
                const int st = next_item(k, it, OneLane{});
                if (st == 0) break;
                if (st == 2) continue;
                it_done(k);
                const int steps = it.heads * max(0, q_tiles(it) - first_tile(it));
                if (steps == 0) continue;
                const uint32_t ka = opaque_u32(ka0), va = opaque_u32(va0);
                if (!(mbar_wait(kv_full, li & 1, p.status) &&
                      mbar_wait(&qs_full[g & 1], (g >> 1) & 1, p.status)))
                    break;
                // S^T held the previous item's last P^T, read by its dV; dP^T its last
                // dS^T, read by its dK: both were issued before
                tc_fence_after();
                mma_ss<D>(T_S, ka, qa(g));     // S^T_0 = K Q_0^T
                tc_commit(s_full);
                mma_ss<D>(T_dP, va, oa(g));    // dP^T_0 = V dO_0^T
                tc_commit(dp_full);
                if (steps == 1) tc_commit(kv_empty);
                for (int t = 0; ok && t < steps; ++t) {
                    const int gt = g + t;
                    const bool more = t + 1 < steps;
                    if (!mbar_wait(p_full, gt & 1, p.status)) { ok = false; break; }
                    // the item's first dV / dK overwrite the accumulators: the previous
                    // item's epilogue must have read them
                    if (t == 0 && li > 0 && !mbar_wait(dkv_free, (li - 1) & 1, p.status)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    mma_ts<D>(T_dV, T_S, oa(gt), t != 0);    // dV += P^T dO
                    if (more) {
                        // S^T_{t+1} overwrites P^T_t, which dV_t reads: tcgen05.mma operations
                        // issued by one thread execute in issue order, so no wait is needed
                        if (!mbar_wait(&qs_full[(gt + 1) & 1], ((gt + 1) >> 1) & 1, p.status)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        mma_ss<D>(T_S, ka, qa(gt + 1));
                        tc_commit(s_full);
                    }
                    if (!mbar_wait(ds_full, gt & 1, p.status)) { ok = false; break; }
                    tc_fence_after();
                    mma_ts<D>(T_dK, T_dP, qa(gt), t != 0);   // dK += dS^T Q
                    tc_commit(dk_done);
                    tc_commit(&qs_empty[gt & 1]);
                    if (more) {   // dP^T_{t+1} over dS^T_t, after dK_t in issue order
                        mma_ss<D>(T_dP, va, oa(gt + 1));
                        tc_commit(dp_full);
                        if (t + 2 == steps) tc_commit(kv_empty);   // the item's last S^T / dP^T
                    }
                }
                g += steps;
                ++li;
            }
            tc_commit(drain);
            mbar_wait(drain, 0, p.status);
        }
    } else if (kPacked && warp == 2) {
        // rows of Q and dO past the sequence's end: zeroed in shared memory
        int g = 0;                           // tiles loaded before this item
        uint32_t phase0 = 0, phase1 = 0;     // qs_raw phases used
        bool ok = true;
        for (int k = 0; ok; ++k) {
            BwdItem it;
            const bool any = read_item<WholeWarp<true>>(k, items, it_full, p.status, it);
            if (!any) break;
            __syncwarp();
            if (lane == 0) it_done(k);
            const int per_head = max(0, q_tiles(it) - first_tile(it));
            const int valid = it.S_q - (q_tiles(it) - 1) * BT;   // rows of the last tile
            if (per_head > 0 && valid < BT)
                for (int gq = 0; ok && gq < it.heads; ++gq) {    // the last tile of each head
                    const int s = (g + gq * per_head + per_head - 1) & 1;
                    ok = zero_tail(&qs_raw[s], (s ? phase1 : phase0) & 1, &qs_full[s],
                                   q_s + s * CF::TILE, o_s + s * CF::TILE, CF::SLABS, valid,
                                   p.status);
                    if (s) ++phase1; else ++phase0;
                }
            g += it.heads * per_head;
        }
    } else if (kPacked && warp == 3) {
        draw_items<true>(p, items, it_full, it_empty);
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegEw));
        // ---------------------------------------------------- element-wise
        // Two warps per lane quadrant: `half` takes query columns [64 half, 64 half + 64)
        // of the tile.  P^T / dS^T of half 0 are packed into TMEM columns [0, 32) of
        // their region, of half 1 into [96, 128), so each half overwrites only columns
        // it has already read itself (mma_ts reads that layout).
        const int quad = warp & 3, half = (warp - 4) >> 2;
        const int tid = threadIdx.x - 128;            // 0..255
        const int kr = quad * 32 + lane;              // key row == TMEM lane
        const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
        const uint32_t src_col = half * 64, dst_col = half ? 96 : 0;
        const uint64_t c2 = f2pack(p.scale_log2, p.scale_log2);
        int gs = 0;   // steps before this item
        bool ok = true;
        for (int k = 0; ok; ++k) {
        BwdItem item;
        const int st = next_item(k, item, WholeWarp<false>{});
        if (st == 0) break;
        if (st == 2) continue;
        const int b = item.b, hk = item.head, bh_kv = b * p.Hkv + hk;
        const int kj = item.tile * BT + kr;
        const int i_lo = first_tile(item);
        const int per_head = max(0, q_tiles(item) - i_lo);
        const int steps = item.heads * per_head;
        const bool row_ok = kj < item.S_kv;
        const int64_t dense_row = ((int64_t)bh_kv * p.S_kv + (row_ok ? kj : 0)) * D;
        const int64_t tok = item.k_tok + (row_ok ? kj : 0);
        __nv_bfloat16* dk_row = static_cast<__nv_bfloat16*>(p.dk) +
                                (kPacked ? tok * p.dk_tok + hk * p.dk_head : dense_row);
        __nv_bfloat16* dv_row = static_cast<__nv_bfloat16*>(p.dv) +
                                (kPacked ? tok * p.dv_tok + hk * p.dv_head : dense_row);
        // packed, in parts: fp32 sums of the part's query heads
        const bool parted = kPacked && p.parts > 1;
        float* dk_sum = nullptr;
        float* dv_sum = nullptr;
        if (parted) {
            dk_sum = p.sums + (((int64_t)item.part * p.total_kv + tok) * p.Hkv + hk) * D;
            dv_sum = dk_sum + (int64_t)p.parts * p.total_kv * p.Hkv * D;
        }
        if (steps == 0) {   // no query sees these keys: dK = dV = 0, no barriers
            if (row_ok && parted) {
                store_zero_sums<D>(dk_sum, half);
                store_zero_sums<D>(dv_sum, half);
            } else if (row_ok) {
                store_zero_row<D>(dk_row, half);
                store_zero_row<D>(dv_row, half);
            }
            if constexpr (kPacked) {
                __syncwarp();
                if (lane == 0) it_done(k);
            }
            continue;
        }
        // -lse2 / -Delta of query `tid` of step t's tile (threads tid < 128)
        auto fetch = [&](int t, float& nl2, float& ndl) {
            const int gq = item.g0 + t / per_head, qt = i_lo + t % per_head;
            const int q = qt * BT + tid;
            const int64_t row = (int64_t)(b * p.Hq + hk * G + gq) * (kPacked ? p.total_q : p.S_q) +
                                item.q_tok + q;
            const float lse = q < item.S_q ? p.lse[row] : -INFINITY;
            nl2 = lse == -INFINITY ? -INFINITY : -lse * kLog2e;   // -inf: the column's P is 0
            ndl = q < item.S_q ? -p.delta[row] : 0.0f;
        };
        float nl2 = 0.0f, ndl = 0.0f;
        if (tid < BT) fetch(0, nl2, ndl);
        for (int t = 0; t < steps; ++t) {
            const int gt = gs + t;
            // [-lse2 | -Delta] of this step's query tile; a buffer is rewritten two
            // steps later, after all 256 threads have posted the step in between (so
            // every thread has finished reading this one)
            float* cl = cols + (gt & 1) * 2 * BT;
            if (tid < BT) {
                cl[tid] = nl2;
                cl[BT + tid] = ndl;
            }
            mbar_arrive(&cols_ready[gt & 1]);
            if (!mbar_wait_warp(&cols_ready[gt & 1], (gt >> 1) & 1, p.status)) { ok = false; break; }
            if (t + 1 < steps && tid < BT) fetch(t + 1, nl2, ndl);
            // key kj sees query q iff kj <= q + causal_offset: this half's columns
            // e < lo are masked (q = q0 + e)
            const int q0 = (i_lo + t % per_head) * BT + half * 64;
            int lo = 0;
            if (!row_ok) lo = 64;
            else if (p.causal) lo = min(64, max(0, kj - item.coff - q0));
            const bool dense = __all_sync(0xffffffffu, lo == 0);
            const float* hcl = cl + half * 64;
            // phase P (needs S^T only): P^T = exp2(S^T c - lse2), kept as bf16 pairs
            if (!mbar_wait_warp(s_full, gt & 1, p.status)) { ok = false; break; }
            tc_fence_after();
            uint32_t sv[2][32];
            __syncwarp();
            tmem_ld_32x32b_x32(T_S + lane_base + src_col, sv[0]);
            tmem_ld_32x32b_x32(T_S + lane_base + src_col + 32, sv[1]);
            tmem_ld_wait();
            uint32_t pw[32];
            Probs<kPacked> pf;
#pragma unroll
            for (int e = 0; e < 64; e += 4) {
                const float4 l4 = *reinterpret_cast<const float4*>(hcl + e);
#pragma unroll
                for (int u = 0; u < 4; u += 2) {
                    const int ee = e + u;
                    const uint64_t x2 = ffma2(f2pack(__uint_as_float(sv[ee >> 5][ee & 31]),
                                                     __uint_as_float(sv[ee >> 5][(ee & 31) + 1])),
                                              c2, u ? f2pack(l4.z, l4.w) : f2pack(l4.x, l4.y));
                    float x0, x1;
                    f2unpack(x2, x0, x1);
                    if (!dense) {
                        x0 = ee >= lo ? x0 : -INFINITY;
                        x1 = ee + 1 >= lo ? x1 : -INFINITY;
                    }
                    const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
                    pw[ee >> 1] = f32x2_to_bf16x2(p0, p1);
                    pf.keep(ee, p0, p1);
                }
            }
            tmem_st_32x32b_x32(T_S + lane_base + dst_col, pw);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full);
            // phase dS (needs dP^T): dS^T = P^T (dP^T - Delta) back over dP^T
            if (!mbar_wait_warp(dp_full, gt & 1, p.status)) { ok = false; break; }
            tc_fence_after();
            __syncwarp();
            tmem_ld_32x32b_x32(T_dP + lane_base + src_col, sv[0]);
            tmem_ld_32x32b_x32(T_dP + lane_base + src_col + 32, sv[1]);
            tmem_ld_wait();
            uint32_t dw[32];
#pragma unroll
            for (int e = 0; e < 64; e += 4) {
                const float4 d4 = *reinterpret_cast<const float4*>(hcl + BT + e);
#pragma unroll
                for (int u = 0; u < 4; u += 2) {
                    const int ee = e + u;
                    const uint64_t pp = pf.pair(ee, pw);
                    const uint64_t g2 = fadd2(f2pack(__uint_as_float(sv[ee >> 5][ee & 31]),
                                                     __uint_as_float(sv[ee >> 5][(ee & 31) + 1])),
                                              u ? f2pack(d4.z, d4.w) : f2pack(d4.x, d4.y));
                    float d0, d1;
                    f2unpack(fmul2(pp, g2), d0, d1);
                    dw[ee >> 1] = f32x2_to_bf16x2(d0, d1);
                }
            }
            tmem_st_32x32b_x32(T_dP + lane_base + dst_col, dw);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(ds_full);
        }

        // epilogue: dK = scale * acc, dV = acc (each half stores half of the columns)
        if (ok && !mbar_wait_warp(dk_done, (gs + steps - 1) & 1, p.status)) ok = false;
        if (!ok) break;
        tc_fence_after();
        if (parted) {
            store_sums<D>(T_dK + lane_base, p.scale, dk_sum, row_ok, half);
            store_sums<D>(T_dV + lane_base, 1.0f, dv_sum, row_ok, half);
        } else {
            store_row<D>(T_dK + lane_base, p.scale, dk_row, row_ok, half);
            store_row<D>(T_dV + lane_base, 1.0f, dv_row, row_ok, half);
        }
        // both accumulators are read out of TMEM: the next item's dV / dK may run
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
            mbar_arrive(dkv_free);
            it_done(k);
        }
        gs += steps;
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ---------------------------------------------------------------- dQ
// One persistent CTA per SM walks units of two (batch * query head, 128-query tile)
// items of one head: tile n_qt-1-q (the heaviest under a causal mask) and tile q, so
// units of a causal square problem carry the same work.  K/V tiles, S buffers and
// the per-step barriers count on across items (step g of the CTA: ring stage and
// S buffer g & 1); Q/dO reload once the item's last dP has been issued (q_empty),
// and an item's first dQ MMA waits for the previous item's epilogue to have read
// dQ out of TMEM (dq_free).
template <int D, bool kPacked = false>
__global__ void __launch_bounds__(kThreads, 1)
    k_fa_bwd_dq(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmdO,
                const BwdParams p) {
    // Packed, after a dK/dV pass: nothing here needs what that pass writes, so a CTA starts as
    // soon as one of its CTAs leaves the SM, and waits for the pass to be complete (the next
    // kernel in the stream relies on it) only at the end.  Delta and the counters are there:
    // every dK/dV CTA waited for them before it let this kernel launch.
    if (!kPacked || !p.after_dkdv) pdl_wait();
    pdl_trigger();
    using CF = BwdCfg<D>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~uintptr_t(1023));
    uint8_t* q_s = smem;                          // Q_i
    uint8_t* o_s = q_s + CF::TILE;                // dO_i
    uint8_t* k_s = o_s + CF::TILE;                // [2][K_j]
    uint8_t* v_s = k_s + 2 * CF::TILE;            // [2][V_j]
    uint64_t* bars = reinterpret_cast<uint64_t*>(v_s + 2 * CF::TILE);
    uint64_t* q_full = bars;
    uint64_t* k_full = bars + 1;      // [2]
    uint64_t* k_empty = bars + 3;     // [2]
    uint64_t* v_full = bars + 5;      // [2]
    uint64_t* v_empty = bars + 7;     // [2]
    uint64_t* s_full = bars + 9;      // [2]: S of step g in TMEM buffer g & 1
    uint64_t* dp_full = bars + 11;
    uint64_t* ds_full = bars + 12;
    uint64_t* dq_done = bars + 13;    // dQ has read dS: dP may be rewritten
    uint64_t* drain = bars + 14;
    uint64_t* q_empty = bars + 15;    // the item's last MMA reading Q / dO has completed
    uint64_t* dq_free = bars + 16;    // the item's epilogue has read dQ out of TMEM
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 17);
    uint64_t* it_full = bars + 18;    // [2] packed items
    uint64_t* it_empty = bars + 20;   // [2] load, MMA and zeroing warps, 8 element-wise warps
    uint64_t* k_raw = bars + 22;      // [2] loaded, rows past the end not yet zeroed
    uint64_t* v_raw = bars + 24;      // [2]
    BwdItem* items = reinterpret_cast<BwdItem*>(bars + 26);   // [2]

    const int lane = threadIdx.x & 31;
    const int warp = kPacked ? same_in<WholeWarp<false>>(threadIdx.x >> 5) : threadIdx.x >> 5;
    const int n_qt = (p.S_q + BT - 1) / BT;
    const int half_units = (n_qt + 1) / 2;
    const int units = p.B * p.Hq * half_units;
    // k-th item of this CTA: 0 = no more, 1 = item (bh, it), 2 = empty slot
    auto item_at = [&](int k, int& bh, int& it) -> int {
        const int u = (int)blockIdx.x + (k >> 1) * (int)gridDim.x;
        if (u >= units) return 0;
        bh = u / half_units;
        const int q = u % half_units;
        it = (k & 1) ? q : n_qt - 1 - q;
        return ((k & 1) && q == n_qt - 1 - q) ? 2 : 1;
    };
    // the same with the item's geometry; packed: from the ring, released with it_done
    auto next_item = [&](int k, BwdItem& it, auto who) -> int {
        if constexpr (kPacked) {
            return read_item<decltype(who)>(k, items, it_full, p.status, it) ? 1 : 0;
        } else {
            int bh, tile;
            const int st = item_at(k, bh, tile);
            if (st == 1) {
                it.b = bh / p.Hq;
                it.head = bh % p.Hq;
                it.tile = tile;
                it.q_tok = it.k_tok = 0;
                it.S_q = p.S_q;
                it.S_kv = p.S_kv;
                it.coff = p.causal_offset;
            }
            return st;
        }
    };
    auto it_done = [&](int k) {
        if constexpr (kPacked) mbar_arrive(&it_empty[k & 1]);
    };
    auto kv_tiles = [&](const BwdItem& it) {
        int n_kv = (it.S_kv + BT - 1) / BT;
        if (p.causal) {
            const int last = it.tile * BT + BT - 1 + it.coff;
            n_kv = min(n_kv, last < 0 ? 0 : last / BT + 1);
        }
        return n_kv;
    };

    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        mbar_init(dq_free, 8);
        for (int s = 0; s < 2; ++s) {
            mbar_init(&k_full[s], 1);
            mbar_init(&k_empty[s], 1);
            mbar_init(&v_full[s], 1);
            mbar_init(&v_empty[s], 1);
        }
        mbar_init(&s_full[0], 1);
        mbar_init(&s_full[1], 1);
        mbar_init(dp_full, 1);
        mbar_init(ds_full, 8);
        mbar_init(dq_done, 1);
        mbar_init(drain, 1);
        if constexpr (kPacked) {
            for (int i = 0; i < 2; ++i) {
                mbar_init(&it_full[i], 1);
                mbar_init(&it_empty[i], 11);
                mbar_init(&k_raw[i], 1);
                mbar_init(&v_raw[i], 1);
            }
        }
        fence_barrier_init();
        fence_proxy_async_smem();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = kPacked ? 0u : *tmem_slot;   // all 512 columns start at column 0
    // two S buffers, so that the next step's S = Q K^T runs during this step
    const uint32_t T_S = tmem, T_dP = tmem + 2 * BT, T_dQ = tmem + 3 * BT;

    if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegCtl));
    if (warp == 0) {
        if (lane == 0) {
            tma_prefetch_desc(&tmK);
            tma_prefetch_desc(&tmV);
            int g = 0, li = 0;   // K/V tiles loaded; items with work loaded
            bool ok = true;
            for (int k = 0; ok; ++k) {
                BwdItem it;
                const int st = next_item(k, it, OneLane{});
                if (st == 0) break;
                if (st == 1) it_done(k);
                const int n_kv = st == 1 ? kv_tiles(it) : 0;
                if (n_kv == 0) continue;
                const int b = it.b, h = it.head, bh = b * p.Hq + h;
                const int bh_kv = b * p.Hkv + h / (p.Hq / p.Hkv);
                const int q_row = it.q_tok + it.tile * BT;
                if (li > 0 && !mbar_wait(q_empty, (li - 1) & 1, p.status)) break;
                mbar_arrive_expect_tx(q_full, 2 * CF::TILE);
#pragma unroll
                for (int sl = 0; sl < CF::SLABS; ++sl) {
                    tma_load_3d(q_s + sl * SLAB_BYTES, &tmQ, q_full, sl * 64, q_row, bh);
                    tma_load_3d(o_s + sl * SLAB_BYTES, &tmdO, q_full, sl * 64, q_row, bh);
                }
                for (int j = 0; j < n_kv; ++j, ++g) {
                    const int s = g & 1;
                    const uint32_t ph = ((g >> 1) & 1) ^ 1;
                    // packed: a tile past the sequence's end goes to warp 2 first
                    const bool raw = kPacked && (j + 1) * BT > it.S_kv;
                    uint64_t* kb = raw ? &k_raw[s] : &k_full[s];
                    uint64_t* vb = raw ? &v_raw[s] : &v_full[s];
                    if (!mbar_wait(&k_empty[s], ph, p.status)) { ok = false; break; }
                    mbar_arrive_expect_tx(kb, CF::TILE);
#pragma unroll
                    for (int sl = 0; sl < CF::SLABS; ++sl)
                        tma_load_3d(k_s + s * CF::TILE + sl * SLAB_BYTES, &tmK, kb, sl * 64,
                                    it.k_tok + j * BT, bh_kv);
                    if (!mbar_wait(&v_empty[s], ph, p.status)) { ok = false; break; }
                    mbar_arrive_expect_tx(vb, CF::TILE);
#pragma unroll
                    for (int sl = 0; sl < CF::SLABS; ++sl)
                        tma_load_3d(v_s + s * CF::TILE + sl * SLAB_BYTES, &tmV, vb, sl * 64,
                                    it.k_tok + j * BT, bh_kv);
                }
                ++li;
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            // tensor-core order per step j:  S_{j+1}, dQ_j, dP_{j+1}
            const uint32_t qa0 = smem_u32(q_s), oa0 = smem_u32(o_s);
            auto ka = [&](int g) { return opaque_u32(smem_u32(k_s + (g & 1) * CF::TILE)); };
            auto va = [&](int g) { return opaque_u32(smem_u32(v_s + (g & 1) * CF::TILE)); };
            int g = 0, li = 0;   // steps before this item; items with work before it
            bool ok = true;
            for (int k = 0; ok; ++k) {
                BwdItem it;
                const int st = next_item(k, it, OneLane{});
                if (st == 0) break;
                if (st == 1) it_done(k);
                const int n_kv = st == 1 ? kv_tiles(it) : 0;
                if (n_kv == 0) continue;
                const uint32_t qa = opaque_u32(qa0), oa = opaque_u32(oa0);
                const int s0 = g & 1;
                const uint32_t ph0 = (g >> 1) & 1;
                if (!(mbar_wait(q_full, li & 1, p.status) && mbar_wait(&k_full[s0], ph0, p.status) &&
                      mbar_wait(&v_full[s0], ph0, p.status)))
                    break;
                // S buffer s0 held S of step g-2, read before ds_full(g-2); dP held the
                // previous item's last dS, read by its dQ, issued before
                tc_fence_after();
                mma_ss<D>(T_S + s0 * BT, qa, ka(g));     // S_0 = Q K_0^T
                tc_commit(&s_full[s0]);
                mma_ss<D>(T_dP, oa, va(g));              // dP_0 = dO V_0^T
                tc_commit(&v_empty[s0]);
                tc_commit(dp_full);
                if (n_kv == 1) tc_commit(q_empty);
                for (int j = 0; ok && j < n_kv; ++j) {
                    const int gj = g + j;
                    const bool more = j + 1 < n_kv;
                    const int n1 = (gj + 1) & 1;
                    const uint32_t ph1 = ((gj + 1) >> 1) & 1;
                    if (more) {   // S buffer n1 held S of step gj-1, read before ds_full(gj-1)
                        if (!mbar_wait(&k_full[n1], ph1, p.status)) { ok = false; break; }
                        tc_fence_after();
                        mma_ss<D>(T_S + n1 * BT, qa, ka(gj + 1));
                        tc_commit(&s_full[n1]);
                    }
                    if (!mbar_wait(ds_full, gj & 1, p.status)) { ok = false; break; }
                    // the item's first dQ overwrites the accumulator: the previous
                    // item's epilogue must have read it
                    if (j == 0 && li > 0 && !mbar_wait(dq_free, (li - 1) & 1, p.status)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    mma_ts<D>(T_dQ, T_dP, ka(gj), j != 0);   // dQ += dS K
                    tc_commit(dq_done);
                    tc_commit(&k_empty[gj & 1]);
                    if (more) {   // dP_{j+1} over dS_j, after dQ_j in issue order
                        if (!mbar_wait(&v_full[n1], ph1, p.status)) { ok = false; break; }
                        tc_fence_after();
                        mma_ss<D>(T_dP, oa, va(gj + 1));
                        tc_commit(&v_empty[n1]);
                        tc_commit(dp_full);
                        if (j + 2 == n_kv) tc_commit(q_empty);   // the item's last dP
                    }
                }
                g += n_kv;
                ++li;
            }
            tc_commit(drain);
            mbar_wait(drain, 0, p.status);
        }
    } else if (kPacked && warp == 2) {
        // rows of K and V past the sequence's end: zeroed in shared memory
        int g = 0;                           // tiles loaded before this item
        uint32_t phase0 = 0, phase1 = 0;     // k_raw / v_raw phases used
        bool ok = true;
        for (int k = 0; ok; ++k) {
            BwdItem it;
            const bool any = read_item<WholeWarp<true>>(k, items, it_full, p.status, it);
            if (!any) break;
            __syncwarp();
            if (lane == 0) it_done(k);
            const int n_kv = kv_tiles(it);
            const int valid = it.S_kv - (n_kv - 1) * BT;   // rows of the last tile
            if (n_kv > 0 && valid < BT) {
                const int s = (g + n_kv - 1) & 1;
                const uint32_t ph = (s ? phase1++ : phase0++) & 1;
                ok = zero_tail(&k_raw[s], ph, &k_full[s], k_s + s * CF::TILE, nullptr, CF::SLABS,
                               valid, p.status) &&
                     zero_tail(&v_raw[s], ph, &v_full[s], v_s + s * CF::TILE, nullptr, CF::SLABS,
                               valid, p.status);
            }
            g += n_kv;
        }
    } else if (kPacked && warp == 3) {
        draw_items<false>(p, items, it_full, it_empty);
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegEw));
        // ---------------------------------------------------- element-wise
        // Two warps per lane quadrant: `half` takes key columns [64 half, 64 half + 64);
        // dS of half 0 is packed into TMEM columns [0, 32) of the dP region, of half 1
        // into [96, 128) (the layout mma_ts reads).
        const int quad = warp & 3, half = (warp - 4) >> 2;
        const int r = quad * 32 + lane;               // query row == TMEM lane
        const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
        const uint32_t src_col = half * 64, dst_col = half ? 96 : 0;
        const uint64_t c2 = f2pack(p.scale_log2, p.scale_log2);
        int g = 0;   // steps before this item
        bool ok = true;
        for (int k = 0; ok; ++k) {
        BwdItem item;
        const int st = next_item(k, item, WholeWarp<false>{});
        if (st == 0) break;
        if (st == 2) continue;
        const int bh = item.b * p.Hq + item.head;
        const int n_kv = kv_tiles(item);
        const int qi = item.tile * BT + r;
        const bool row_ok = qi < item.S_q;
        const int64_t row = (int64_t)bh * (kPacked ? p.total_q : p.S_q) + item.q_tok + qi;
        __nv_bfloat16* dq_row =
            static_cast<__nv_bfloat16*>(p.dq) +
            (kPacked ? (int64_t)(item.q_tok + (row_ok ? qi : 0)) * p.dq_tok + item.head * p.dq_head
                     : ((int64_t)bh * p.S_q + (row_ok ? qi : 0)) * D);
        if (n_kv == 0) {   // no visible key: dQ = 0, no barriers
            if (row_ok) store_zero_row<D>(dq_row, half);
            if constexpr (kPacked) {
                __syncwarp();
                if (lane == 0) it_done(k);
            }
            continue;
        }
        const float lse = row_ok ? p.lse[row] : -INFINITY;
        const float nl2 = lse == -INFINITY ? -INFINITY : -lse * kLog2e;   // -inf: P = 0
        const float ndl = row_ok ? -p.delta[row] : 0.0f;
        const uint64_t nl2x2 = f2pack(nl2, nl2), ndlx2 = f2pack(ndl, ndl);
        const int vis_hi = p.causal ? min(item.S_kv - 1, qi + item.coff) : item.S_kv - 1;
        for (int j = 0; j < n_kv; ++j) {
            const int gj = g + j;
            // this half's key columns e > hi are masked
            const int hi = vis_hi - (j * BT + half * 64);
            const bool dense = __all_sync(0xffffffffu, hi >= 63);
            // phase P (needs S only), kept in registers as bf16 pairs
            if (!mbar_wait_warp(&s_full[gj & 1], (gj >> 1) & 1, p.status)) { ok = false; break; }
            tc_fence_after();
            const uint32_t sb = T_S + (gj & 1) * BT;
            uint32_t sv[2][32];
            __syncwarp();
            tmem_ld_32x32b_x32(sb + lane_base + src_col, sv[0]);
            tmem_ld_32x32b_x32(sb + lane_base + src_col + 32, sv[1]);
            tmem_ld_wait();
            uint32_t pw[32];
            Probs<kPacked> pf;
#pragma unroll
            for (int e = 0; e < 64; e += 2) {
                const uint64_t x2 = ffma2(f2pack(__uint_as_float(sv[e >> 5][e & 31]),
                                                 __uint_as_float(sv[e >> 5][(e & 31) + 1])),
                                          c2, nl2x2);
                float x0, x1;
                f2unpack(x2, x0, x1);
                if (!dense) {
                    x0 = e <= hi ? x0 : -INFINITY;
                    x1 = e + 1 <= hi ? x1 : -INFINITY;
                }
                const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
                if constexpr (!kPacked) pw[e >> 1] = f32x2_to_bf16x2(p0, p1);
                pf.keep(e, p0, p1);
            }
            // phase dS (needs dP): dS = P (dP - Delta) back over dP
            if (!mbar_wait_warp(dp_full, gj & 1, p.status)) { ok = false; break; }
            tc_fence_after();
            __syncwarp();
            tmem_ld_32x32b_x32(T_dP + lane_base + src_col, sv[0]);
            tmem_ld_32x32b_x32(T_dP + lane_base + src_col + 32, sv[1]);
            tmem_ld_wait();
            uint32_t dw[32];
#pragma unroll
            for (int e = 0; e < 64; e += 2) {
                const uint64_t pp = pf.pair(e, pw);
                const uint64_t g2 = fadd2(f2pack(__uint_as_float(sv[e >> 5][e & 31]),
                                                 __uint_as_float(sv[e >> 5][(e & 31) + 1])),
                                          ndlx2);
                float d0, d1;
                f2unpack(fmul2(pp, g2), d0, d1);
                dw[e >> 1] = f32x2_to_bf16x2(d0, d1);
            }
            tmem_st_32x32b_x32(T_dP + lane_base + dst_col, dw);   // dS over dP
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(ds_full);
        }
        if (ok && !mbar_wait_warp(dq_done, (g + n_kv - 1) & 1, p.status)) ok = false;
        if (!ok) break;
        tc_fence_after();
        store_row<D>(T_dQ + lane_base, p.scale, dq_row, row_ok, half);
        // store_row has read this half of dQ out of TMEM: the next item's dQ may run
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
            mbar_arrive(dq_free);
            it_done(k);
        }
        g += n_kv;
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
    if constexpr (kPacked) pdl_wait();
}

template <int D>
int launch_bwd(const void* Q, const void* K, const void* V, const void* O, const void* dO,
               const float* lse, void* dQ, void* dK, void* dV, float* delta, int B, int Hq,
               int Hkv, int S_q, int S_kv, int causal, float scale, cudaStream_t st) {
    using CF = BwdCfg<D>;
    CUtensorMap tq, tk, tv, to;
    int rc;
    if ((rc = fa_make_tmap_3d(&tq, Q, D, S_q, (int64_t)B * Hq))) return rc;
    if ((rc = fa_make_tmap_3d(&to, dO, D, S_q, (int64_t)B * Hq))) return rc;
    if ((rc = fa_make_tmap_3d(&tk, K, D, S_kv, (int64_t)B * Hkv))) return rc;
    if ((rc = fa_make_tmap_3d(&tv, V, D, S_kv, (int64_t)B * Hkv))) return rc;
    int* status = nullptr;
    if ((rc = device_status(&status))) return rc;
    BwdParams p = {};
    p.B = B;
    p.Hq = Hq;
    p.Hkv = Hkv;
    p.S_q = S_q;
    p.S_kv = S_kv;
    p.causal = causal;
    p.causal_offset = 0;
    p.scale = scale;
    p.scale_log2 = scale * kLog2e;
    p.lse = lse;
    p.delta = delta;
    p.dq = dQ;
    p.dk = dK;
    p.dv = dV;
    p.status = status;
    const int64_t rows = (int64_t)B * Hq * S_q;
    const int64_t delta_rows_per_block = 8 * (32 / (D / 8)) * kDeltaLoads;
    const int dgrid = (int)std::min<int64_t>((rows + delta_rows_per_block - 1) / delta_rows_per_block,
                                             (int64_t)sm_count() * 8);
    AMPB_CHECK_CUDA(launch_pdl(k_fa_bwd_delta<D>, dim3(dgrid), dim3(256), 0, st,
                               static_cast<const __nv_bfloat16*>(O),
                               static_cast<const __nv_bfloat16*>(dO), delta, rows,
                               DeltaStrides{}));
    constexpr int SMEM_KV = CF::SMEM_KV, SMEM_Q = CF::SMEM_Q;
    static std::atomic<uint64_t> attr_done{0};
    int dev = 0;
    AMPB_CHECK_CUDA(cudaGetDevice(&dev));
    if (dev >= 64 || !(attr_done.load() >> dev & 1)) {
        AMPB_CHECK_CUDA(cudaFuncSetAttribute(k_fa_bwd_dkdv<D>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_KV));
        AMPB_CHECK_CUDA(cudaFuncSetAttribute(k_fa_bwd_dq<D>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_Q));
        if (dev < 64) attr_done.fetch_or(1ull << dev);
    }
    // dK/dV: one persistent CTA per SM over units of two key tiles (k_fa_bwd_dkdv)
    const int64_t kv_units = (int64_t)B * Hkv * (((S_kv + BT - 1) / BT + 1) / 2);
    AMPB_REQUIRE(kv_units <= INT32_MAX / 2, AMP_ERR_UNSUPPORTED, "attention too large");
    AMPB_CHECK_CUDA(launch_pdl(k_fa_bwd_dkdv<D>, dim3((unsigned)std::min<int64_t>(kv_units, sm_count())),
                               dim3(kThreads), SMEM_KV, st, tq, tk, tv, to, p));
    // dQ: one persistent CTA per SM over units of two query tiles (k_fa_bwd_dq)
    const int64_t dq_units = (int64_t)B * Hq * (((S_q + BT - 1) / BT + 1) / 2);
    AMPB_REQUIRE(dq_units <= INT32_MAX / 2, AMP_ERR_UNSUPPORTED, "attention too large");
    AMPB_CHECK_CUDA(launch_pdl(k_fa_bwd_dq<D>, dim3((unsigned)std::min<int64_t>(dq_units, sm_count())),
                               dim3(kThreads), SMEM_Q, st, tq, tk, tv, to, p));
    return AMP_OK;
}

// Parts of the dK/dV pass's sums over a group: as many as six items a CTA allow, none larger
// than it must be.  A part costs 8 bytes an element, written and read again, and the dQ pass
// fills idle SMs anyway, so groups under 6 are shared out only where half of the CTAs would
// have no item, and with an item for every CTA a part keeps four steps.  Forward and backward,
// whole -> shared out: 8 / 1 heads, 2000 tokens 311 -> 114 us, 10 sequences of 200 to 8000
// tokens 1396 -> 1006; 28 / 4 heads, 8192 tokens 2325 -> 2175.  What the limits leave out:
// 32 / 8 heads, 2000 tokens 300 -> 315; 32 / 4 heads, 30 sequences of under 200 tokens 112 -> 174.
int fa_bwd_parts(int B, int total_kv, int Hq, int Hkv) {
    const int64_t items = ((int64_t)total_kv / BT + B) * Hkv;   // at most
    const int64_t sms = sm_count(), group = Hq / Hkv;
    if (group < 6 && items > sms / 2) return 1;
    int64_t most = std::min(group, 6 * sms / items);
    if (items > sms) most = std::min(most, group * total_kv / BT / B / 4);
    most = std::max<int64_t>(1, most);
    const int64_t size = (group + most - 1) / most;
    return (int)((group + size - 1) / size);
}
size_t fa_bwd_sums_at(int B, int Hq, int total_q) {
    return ((varlen_plan_bytes(B) + 15) / 16 * 16 + (size_t)Hq * total_q * 4 + 15) / 16 * 16;
}

struct PackedBwdArgs {
    const void *Q, *K, *V, *O, *dO;
    const float* lse;
    void *dQ, *dK, *dV;
    const int *cu_q, *cu_kv;
    int B, total_q, total_kv, Hq, Hkv, causal;
    const int64_t* strides;   // token and head stride of Q, K, V, O, dO, dQ, dK, dV
    float scale;
    void* ws;
};

template <int D>
int launch_bwd_packed(const PackedBwdArgs& a, cudaStream_t st) {
    using CF = BwdCfg<D>;
    const int64_t* s = a.strides;
    CUtensorMap tq, tk, tv, to;
    int rc;
    if (a.total_q > 0) {
        if ((rc = fa_make_tmap_packed(&tq, a.Q, D, a.total_q, a.Hq, s[0], s[1]))) return rc;
        if ((rc = fa_make_tmap_packed(&to, a.dO, D, a.total_q, a.Hq, s[8], s[9]))) return rc;
    }
    if (a.total_kv > 0) {
        if ((rc = fa_make_tmap_packed(&tk, a.K, D, a.total_kv, a.Hkv, s[2], s[3]))) return rc;
        if ((rc = fa_make_tmap_packed(&tv, a.V, D, a.total_kv, a.Hkv, s[4], s[5]))) return rc;
    }
    // with no query or no key at all every item is one without steps: no load is issued
    if (a.total_q == 0) tq = to = tk;
    if (a.total_kv == 0) tk = tv = tq;
    BwdParams p = {};
    if ((rc = device_status(&p.status))) return rc;
    p.B = a.B;
    p.Hq = a.Hq;
    p.Hkv = a.Hkv;
    p.causal = a.causal;
    p.scale = a.scale;
    p.scale_log2 = a.scale * kLog2e;
    p.lse = a.lse;
    p.dq = a.dQ;
    p.dk = a.dK;
    p.dv = a.dV;
    p.total_q = a.total_q;
    p.total_kv = a.total_kv;
    p.parts = fa_bwd_parts(a.B, a.total_kv, a.Hq, a.Hkv);
    p.sums = reinterpret_cast<float*>(static_cast<uint8_t*>(a.ws) + fa_bwd_sums_at(a.B, a.Hq, a.total_q));
    p.after_dkdv = a.total_kv > 0;
    p.dq_tok = s[10];
    p.dq_head = s[11];
    p.dk_tok = s[12];
    p.dk_head = s[13];
    p.dv_tok = s[14];
    p.dv_head = s[15];
    p.plan = {a.ws, false, false, a.cu_q, a.cu_kv, a.B, a.total_q, a.total_kv, {}};
    float* delta = reinterpret_cast<float*>(static_cast<uint8_t*>(a.ws) +
                                            (varlen_plan_bytes(a.B) + 15) / 16 * 16);
    p.delta = delta;
    // no more CTAs than there can be items
    const int64_t most_kv = ((int64_t)a.total_kv / BT + a.B) * a.Hkv * p.parts;
    const int64_t most_q = ((int64_t)a.total_q / BT + a.B) * a.Hq;
    const int64_t rows = (int64_t)a.total_q * a.Hq;
    if ((rc = varlen_make_plan(p.plan, most_kv, most_q, a.Hq, a.Hkv, true, p.parts, rows == 0, st)))
        return rc;
    if (rows > 0) {
        const int64_t per_block = 8 * (32 / (D / 8)) * kDeltaLoads;
        const DeltaStrides ds = {s[6], s[7], s[8], s[9], a.Hq, a.total_q,
                                 p.plan.lists ? nullptr : static_cast<int*>(a.ws)};
        AMPB_CHECK_CUDA(launch_pdl(k_fa_bwd_delta<D, true>,
                                   dim3((unsigned)std::min<int64_t>((rows + per_block - 1) / per_block,
                                                                    (int64_t)sm_count() * 8)),
                                   dim3(256), 0, st, static_cast<const __nv_bfloat16*>(a.O),
                                   static_cast<const __nv_bfloat16*>(a.dO), delta, rows, ds));
    }
    if (rows > 0 && a.total_kv > 0) {
        FewParams f = {static_cast<const __nv_bfloat16*>(a.Q), static_cast<const __nv_bfloat16*>(a.K),
                       static_cast<const __nv_bfloat16*>(a.V), static_cast<const __nv_bfloat16*>(a.dO),
                       s[0], s[1], s[2], s[3], s[4], s[5], s[8], s[9], a.lse, delta, a.Hq, a.Hkv, a.causal,
                       kFewKeys / 16, p.scale_log2, p.status, p.plan};
        // full mask: as many warps a head as fill the GPU, if the rows are there
        if (!a.causal)
            f.strips = (int)std::max<int64_t>(1, std::min<int64_t>((a.total_q + 15) / 16,
                                                                   sm_count() * 16ll / ((int64_t)a.B * a.Hq)));
        const int64_t blocks = ((int64_t)a.B * a.Hq * f.strips + 7) / 8;
        AMPB_CHECK_CUDA(launch_pdl(k_fa_bwd_few<D>, dim3((unsigned)std::min<int64_t>(blocks, sm_count() * 8ll)),
                                   dim3(256), 0, st, f));
    }
    static std::atomic<uint64_t> allowed_kv{0}, allowed_q{0};
    AMPB_CHECK_CUDA(allow_smem_once(allowed_kv, k_fa_bwd_dkdv<D, true>, CF::SMEM_KV));
    AMPB_CHECK_CUDA(allow_smem_once(allowed_q, k_fa_bwd_dq<D, true>, CF::SMEM_Q));
    if (a.total_kv > 0) {
        AMPB_CHECK_CUDA(launch_pdl(k_fa_bwd_dkdv<D, true>,
                                   dim3((unsigned)std::min<int64_t>(most_kv, sm_count())),
                                   dim3(kThreads), CF::SMEM_KV, st, tq, tk, tv, to, p));
    }
    if (a.total_q > 0) {
        AMPB_CHECK_CUDA(launch_pdl(k_fa_bwd_dq<D, true>,
                                   dim3((unsigned)std::min<int64_t>(most_q, sm_count())),
                                   dim3(kThreads), CF::SMEM_Q, st, tq, tk, tv, to, p));
    }
    if (a.total_kv > 0 && p.parts > 1)
        AMPB_CHECK_CUDA(launch_pdl(k_fa_bwd_join<D>,
                                   dim3((unsigned)std::min((a.total_kv + 7) / 8, sm_count() * 8)), dim3(256), 0,
                                   st, p));
    return AMP_OK;
}

}  // namespace

size_t fa_bwd_ws_bytes(int B, int Hq, int S_q) { return (size_t)B * Hq * S_q * 4 + 256; }

int flash_attn_bwd_dev(const void* Q, const void* K, const void* V, const void* O, const void* dO,
                       const float* lse, void* dQ, void* dK, void* dV, int B, int Hq, int Hkv,
                       int S_q, int S_kv, int D, int causal, float scale, void* ws,
                       size_t ws_bytes, cudaStream_t st) {
    AMPB_REQUIRE(B > 0 && Hq > 0 && Hkv > 0 && S_q > 0 && S_kv > 0, AMP_ERR_INVALID,
                 "attention sizes must be positive");
    AMPB_REQUIRE(Hq % Hkv == 0, AMP_ERR_INVALID, "num_q_heads (%d) must be a multiple of "
                 "num_kv_heads (%d)", Hq, Hkv);
    AMPB_REQUIRE(Q && K && V && O && dO && lse && dQ && dK && dV && ws, AMP_ERR_INVALID,
                 "NULL tensor");
    AMPB_REQUIRE(aligned16(Q) && aligned16(K) && aligned16(V) && aligned16(O) && aligned16(dO) &&
                     aligned16(dQ) && aligned16(dK) && aligned16(dV),
                 AMP_ERR_INVALID, "tensors must be 16-byte aligned");
    AMPB_REQUIRE(!causal || S_q == S_kv, AMP_ERR_UNSUPPORTED,
                 "causal backward needs S_q == S_kv (top-left aligned mask)");
    AMPB_REQUIRE((int64_t)B * Hq <= 65535, AMP_ERR_UNSUPPORTED, "B*Hq must be <= 65535");
    AMPB_REQUIRE(ws_bytes >= fa_bwd_ws_bytes(B, Hq, S_q), AMP_ERR_INVALID,
                 "workspace too small: %zu < %zu", ws_bytes, fa_bwd_ws_bytes(B, Hq, S_q));
    AMPB_REQUIRE((reinterpret_cast<uintptr_t>(ws) & 15u) == 0, AMP_ERR_INVALID,
                 "workspace must be 16-byte aligned");
    if (!(scale > 0.0f)) scale = 1.0f / sqrtf((float)D);
    float* delta = static_cast<float*>(ws);
    switch (D) {
        case 128:
            return launch_bwd<128>(Q, K, V, O, dO, lse, dQ, dK, dV, delta, B, Hq, Hkv, S_q, S_kv,
                                   causal, scale, st);
        case 64:
            return launch_bwd<64>(Q, K, V, O, dO, lse, dQ, dK, dV, delta, B, Hq, Hkv, S_q, S_kv,
                                  causal, scale, st);
        default:
            set_error(AMP_ERR_UNSUPPORTED, "flash_attn backward: head_dim %d not supported (64, 128)", D);
            return AMP_ERR_UNSUPPORTED;
    }
}

}  // namespace ampb

using namespace ampb;

extern "C" {

size_t amp_flash_attn_varlen_bwd_workspace_bytes(int B, int Hq, int Hkv, int total_q, int total_kv,
                                                 int head_dim) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || total_q < 0 || total_kv < 0 || head_dim <= 0) return 0;
    const int parts = fa_bwd_parts(B, total_kv, Hq, Hkv);
    return fa_bwd_sums_at(B, Hq, total_q) +
           (parts > 1 ? (size_t)parts * 2 * total_kv * Hkv * head_dim * sizeof(float) : 0);
}

int amp_flash_attn_varlen_bwd_bf16_dev(const void* Q, const void* K, const void* V, const void* O,
                                       const void* dO, const float* lse, void* dQ, void* dK,
                                       void* dV, const int32_t* cu_seqlens_q,
                                       const int32_t* cu_seqlens_kv, int B, int total_q,
                                       int total_kv, int Hq, int Hkv, int head_dim,
                                       const int64_t* strides, int causal, float scale,
                                       void* workspace, size_t workspace_bytes, void* stream) {
    int rc = varlen_check(B, total_q, total_kv, Hq, Hkv, head_dim, cu_seqlens_q, cu_seqlens_kv,
                          strides, 16, workspace, workspace_bytes,
                          amp_flash_attn_varlen_bwd_workspace_bytes(B, Hq, Hkv, total_q, total_kv,
                                                                    head_dim));
    if (rc) return rc;
    if (total_q == 0 && total_kv == 0) return AMP_OK;
    AMPB_REQUIRE((total_q == 0 || (Q && O && dO && lse && dQ)) && (total_kv == 0 || (K && V && dK && dV)),
                 AMP_ERR_INVALID, "NULL tensor");
    AMPB_REQUIRE(aligned16(Q) && aligned16(K) && aligned16(V) && aligned16(O) && aligned16(dO) &&
                     aligned16(dQ) && aligned16(dK) && aligned16(dV),
                 AMP_ERR_INVALID, "tensors must be 16-byte aligned");
    // the passes overlap: what one has written the other may still have to read
    const void *grads[3] = {dQ, dK, dV}, *inputs[5] = {Q, K, V, O, dO};
    for (int i = 0; i < 3; ++i) {
        for (const void* x : inputs)
            AMPB_REQUIRE(!grads[i] || grads[i] != x, AMP_ERR_INVALID,
                         "packed attention: a gradient shares memory with an input");
        AMPB_REQUIRE(!grads[i] || grads[i] != grads[(i + 1) % 3], AMP_ERR_INVALID,
                     "packed attention: two gradients share memory");
    }
    if (!(scale > 0.0f)) scale = 1.0f / sqrtf((float)head_dim);
    const PackedBwdArgs a = {Q,  K,  V,       O,        dO, lse, dQ,     dK,      dV,   cu_seqlens_q,
                             cu_seqlens_kv, B, total_q, total_kv, Hq, Hkv, causal, strides, scale,
                             workspace};
    return head_dim == 128 ? launch_bwd_packed<128>(a, as_stream(stream))
                           : launch_bwd_packed<64>(a, as_stream(stream));
}

size_t amp_flash_attn_bwd_workspace_bytes(int B, int Hq, int S_q) {
    return fa_bwd_ws_bytes(B, Hq, S_q);
}

int amp_flash_attn_bwd_bf16_dev(const void* Q, const void* K, const void* V, const void* O,
                                const void* dO, const float* lse, void* dQ, void* dK, void* dV,
                                int B, int Hq, int Hkv, int S_q, int S_kv, int head_dim,
                                int causal, float scale, void* workspace, size_t workspace_bytes,
                                void* stream) {
    return flash_attn_bwd_dev(Q, K, V, O, dO, lse, dQ, dK, dV, B, Hq, Hkv, S_q, S_kv, head_dim,
                              causal, scale, workspace, workspace_bytes, as_stream(stream));
}

}  // extern "C"
