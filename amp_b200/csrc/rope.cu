// rope.cu -- rotary positions with one or more axes, and their fusion with the
// paged cache's append.
//
// Pair i of a head's first R = 2 * pairs elements is turned by
//   phi = pos[axis(i)][token] * inv_freq[i]:   (x, y) -> (x cos - y sin, y cos + x sin)
// (the backward pass by -phi).  Pairs are (i, i + R/2), or (2i, 2i + 1) when
// interleaved; elements from R on pass through.  axis(i) comes from the sections:
// the first sections[0] pairs follow axis 0 (time), the next sections[1] axis 1
// (height), and so on.  The reference has no positional encoding.
//
// HBM-bound: every element is read and written once.  A warp takes a token and walks
// its heads (of q, k and v in turn): a lane holds a unit, two vectors of VE elements
// with VE pairs (or 2 VE elements that pass through), 32 / units heads at a time.  The token's angles are computed once a warp
// into its own shared memory, behind the first loads, and a lane keeps the VE it
// needs in registers for all heads; nothing waits for another warp.
//
// The angle is reduced in 64 bits (turns = pos * inv_freq / 2 pi, less the nearest
// whole number): in 32 bits a position of 10^5 is off by 2^-7 of a radian.  The
// rotation itself is fp32, rounded once to the tensor's type.
//
// Append mode writes k (turned) and v of each new token into its page of the
// cache instead of an output tensor.  Token t belongs to the sequence b with
// cu[b] <= t < cu[b+1] and is number ctx[b] - len(b) + (t - cu[b]) of its context
// (ctx counts the new tokens, as paged prefill expects).  One warp per token
// searches cu while the rows are being loaded.
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "runtime.h"
#include "tc_common.cuh"
#include "varlen.cuh"

namespace ampb {
namespace {

constexpr int kRopeThreads = 256, kRopeWarps = kRopeThreads / 32;
// Two steps of loads (64 bytes a lane) in flight and 64 registers, for 32 warps a
// multiprocessor: on 32768 tokens x 40 heads x 128 (forward and backward, 1.34 GB) 294 us;
// four steps at 16 warps 367, one step at 40 warps 274, and 223 us (6.0 TB/s) for two steps
// with the streaming hint on both sides (below): rows are read and written once, and
// without it the lines written push out those that neighbouring warps are reading.
constexpr int kSteps = 2, kBlocksPerSM = 4;
constexpr int kMaxAxes = 4;
constexpr int kPage = 16;

struct RopeTensor {
    const void* in;
    void* out;
    int64_t in_tok, in_head, out_tok, out_head;   // strides in elements
};

struct RopeParams {
    RopeTensor x[3];       // q, k, v (append: k and v have no `out`)
    int heads[3];
    int T, H, D;           // H: heads of all tensors
    int pairs;             // R / 2
    int units;             // of a head: D / (2 VE)
    int lanes_heads;       // heads of a step: 32 / units, 1 if a head has more units than lanes
    int steps;             // of a token: H / lanes_heads, rounded up
    int steps_warp, splits;   // steps that one warp takes; warps of a token
    float sign;            // -1: backward
    const int* pos;        // [axes][T]
    int64_t pos_stride;
    int axis_end[kMaxAxes - 1];   // first pair of axes 1, 2, 3
    const float* inv_freq;
    // append
    void *k_pool, *v_pool;        // [pages][heads][16][D]
    const int *block_table, *ctx_lens, *cu;
    int B, num_pages, max_pages;
    int* status;
};

template <typename T, int VE>
struct alignas(sizeof(T) * VE) Vec {
    T v[VE];
};

template <typename V>
__device__ __forceinline__ void load_once(V& v, const void* p) {
    if constexpr (sizeof(V) == 16) *reinterpret_cast<uint4*>(&v) = __ldcs(static_cast<const uint4*>(p));
    else v = *static_cast<const V*>(p);
}
template <typename V>
__device__ __forceinline__ void store_once(void* p, const V& v) {
    if constexpr (sizeof(V) == 16) __stcs(static_cast<uint4*>(p), *reinterpret_cast<const uint4*>(&v));
    else *static_cast<V*>(p) = v;
}

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x) {
    if constexpr (std::is_same<T, float>::value) return x;
    else return __float2bfloat16_rn(x);
}

__device__ __forceinline__ float2 angle(const RopeParams& p, int t, int i) {
    int axis = 0;
#pragma unroll
    for (int a = 0; a < kMaxAxes - 1; ++a) axis += i >= p.axis_end[a];
    const double turns = (double)p.pos[axis * p.pos_stride + t] * (double)p.inv_freq[i] *
                         0.15915494309189533577;   // 1 / (2 pi)
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    return make_float2(c, s * p.sign);
}

constexpr int64_t kNoSequence = -1, kNoPage = -2;

// Append: where token t's row of head 0 starts in the pools, in elements, or one of the
// two above.  All lanes of a warp call it.
__device__ __forceinline__ int64_t cache_row(const RopeParams& p, int t, int Hkv) {
    const int b = varlen_find(p.cu, p.B, t);
    const int q0 = p.cu[b], q1 = p.cu[b + 1];
    if (t < q0 || t >= q1) return kNoSequence;
    const int64_t at = (int64_t)p.ctx_lens[b] - (q1 - q0) + (t - q0);
    int page = -1;
    if (at >= 0 && at / kPage < p.max_pages)
        page = p.block_table[(int64_t)b * p.max_pages + at / kPage];
    if (page < 0 || page >= p.num_pages) {
        if ((threadIdx.x & 31) == 0) p.status[kStatusBadIndexInt] = AMP_DEV_ERR_BAD_INDEX;
        return kNoPage;
    }
    return ((int64_t)page * Hkv * kPage + at % kPage) * p.D;
}

template <typename T, int VE, bool kInter, bool kAppend>
__global__ void __launch_bounds__(kRopeThreads, kBlocksPerSM) k_rope(const __grid_constant__ RopeParams p) {
    using V = Vec<T, VE>;
    // cos, sin [warp][VE][pairs / VE]: the lanes of a head read neighbours
    extern __shared__ float2 trig_all[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float2* trig = trig_all + warp * p.pairs;
    pdl_wait();
    const int64_t task = (int64_t)blockIdx.x * kRopeWarps + warp;
    if (task >= (int64_t)p.T * p.splits) return;
    const int t = (int)(task / p.splits);
    const int step0 = (int)(task - (int64_t)t * p.splits) * p.steps_warp;
    const int step1 = min(step0 + p.steps_warp, p.steps);
    const int chunks = p.pairs / VE;
    const bool narrow = p.units <= 32;
    const int sub = narrow ? lane / p.units : 0;
    int64_t row = 0;
    bool ready = false;
    for (int c0 = 0; c0 < p.units; c0 += 32) {
        const int c = narrow ? lane - sub * p.units : c0 + lane;
        const bool live = sub < p.lanes_heads && c < p.units;
        const bool turned = c < chunks;
        const int off_a = turned && !kInter ? c * VE : c * 2 * VE;
        const int off_b = turned && !kInter ? p.pairs + c * VE : c * 2 * VE + VE;
        float2 cs[VE];
        bool loaded = false;
        for (int s0 = step0; s0 < step1; s0 += kSteps) {
            V a[kSteps], b[kSteps];
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const int h = (s0 + i) * p.lanes_heads + sub;
                if (!live || s0 + i >= step1 || h >= p.H) continue;
                const int x = (h >= p.heads[0]) + (h >= p.heads[0] + p.heads[1]);
                const int hx = h - (x > 0 ? p.heads[0] : 0) - (x > 1 ? p.heads[1] : 0);
                const T* src = static_cast<const T*>(x == 0 ? p.x[0].in : x == 1 ? p.x[1].in : p.x[2].in) +
                               t * (x == 0 ? p.x[0].in_tok : x == 1 ? p.x[1].in_tok : p.x[2].in_tok) +
                               hx * (x == 0 ? p.x[0].in_head : x == 1 ? p.x[1].in_head : p.x[2].in_head);
                load_once(a[i], src + off_a);
                load_once(b[i], src + off_b);
            }
            if (!ready) {
                ready = true;
                for (int i = lane; i < p.pairs; i += 32) trig[i % VE * chunks + i / VE] = angle(p, t, i);
                if constexpr (kAppend) row = cache_row(p, t, p.heads[1]);
                __syncwarp();
                if (kAppend && row == kNoSequence) return;
            }
            if (!loaded && turned && live) {
#pragma unroll
                for (int e = 0; e < VE; ++e) cs[e] = trig[e * chunks + c];
            }
            loaded = true;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const int h = (s0 + i) * p.lanes_heads + sub;
                if (!live || s0 + i >= step1 || h >= p.H) continue;
                const int x = (h >= p.heads[0]) + (h >= p.heads[0] + p.heads[1]);
                const int hx = h - (x > 0 ? p.heads[0] : 0) - (x > 1 ? p.heads[1] : 0);
                if (turned && !(kAppend && x == 2)) {
#pragma unroll
                    for (int e = 0; e < VE; ++e) {
                        // pair e: elements e of both vectors, or neighbours within the two
                        T& u = kInter ? (2 * e < VE ? a[i].v[(2 * e) % VE] : b[i].v[(2 * e) % VE]) : a[i].v[e];
                        T& v = kInter ? (2 * e + 1 < VE ? a[i].v[(2 * e + 1) % VE] : b[i].v[(2 * e + 1) % VE])
                                      : b[i].v[e];
                        const float fu = to_f32(u), fv = to_f32(v);
                        // the fused product is named, so that every vector width gives the same bits
                        u = from_f32<T>(__fmaf_rn(fu, cs[e].x, -__fmul_rn(fv, cs[e].y)));
                        v = from_f32<T>(__fmaf_rn(fv, cs[e].x, __fmul_rn(fu, cs[e].y)));
                    }
                }
                T* dst;
                if (kAppend && x > 0) {
                    if (row < 0) continue;
                    dst = static_cast<T*>(x == 1 ? p.k_pool : p.v_pool) + row + (int64_t)hx * kPage * p.D;
                } else {
                    dst = static_cast<T*>(x == 0 ? p.x[0].out : p.x[1].out) +
                          t * (x == 0 ? p.x[0].out_tok : p.x[1].out_tok) +
                          hx * (x == 0 ? p.x[0].out_head : p.x[1].out_head);
                }
                store_once(dst + off_a, a[i]);
                store_once(dst + off_b, b[i]);
            }
        }
    }
}

template <typename T, int VE, bool kInter, bool kAppend>
int launch_rope_as(RopeParams& p, cudaStream_t st) {
    p.units = p.D / (2 * VE);
    p.lanes_heads = std::max(1, 32 / p.units);
    p.steps = (p.H + p.lanes_heads - 1) / p.lanes_heads;
    // A warp takes all of a token's heads, so that its angles are computed once, unless that
    // leaves multiprocessors idle (a decode step): then the heads are shared out.
    const int64_t fill = (int64_t)sm_count() * kRopeWarps;
    p.splits = (int)std::min<int64_t>(p.steps, std::max<int64_t>(1, fill / std::max(p.T, 1)));
    p.steps_warp = (p.steps + p.splits - 1) / p.splits;
    p.splits = (p.steps + p.steps_warp - 1) / p.steps_warp;
    const size_t smem = (size_t)kRopeWarps * p.pairs * sizeof(float2);
    const int64_t blocks = ((int64_t)p.T * p.splits + kRopeWarps - 1) / kRopeWarps;
    AMPB_REQUIRE(blocks <= INT32_MAX, AMP_ERR_UNSUPPORTED, "rope: too large");
    AMPB_CHECK_CUDA(launch_pdl(k_rope<T, VE, kInter, kAppend>, dim3((unsigned)blocks), dim3(kRopeThreads),
                               smem, st, p));
    return AMP_OK;
}

// The widest vector that divides the pairs, the rest of the head, every stride and every
// address: 16 bytes for the usual head sizes, one element for the odd ones.
template <typename T, bool kAppend>
int launch_rope(RopeParams& p, bool interleaved, cudaStream_t st) {
    auto fits = [&](int ve) {
        bool ok = p.pairs % ve == 0 && (p.D - 2 * p.pairs) % (2 * ve) == 0;
        const size_t bytes = ve * sizeof(T);
        auto address = [&](const void* q) { return reinterpret_cast<uintptr_t>(q) % bytes == 0; };
        for (int i = 0; i < 3; ++i)
            if (p.heads[i] > 0)
                ok = ok && address(p.x[i].in) && address(p.x[i].out) && p.x[i].in_tok % ve == 0 &&
                     p.x[i].in_head % ve == 0 && p.x[i].out_tok % ve == 0 && p.x[i].out_head % ve == 0;
        return ok && address(p.k_pool) && address(p.v_pool);
    };
    constexpr int kWide = 16 / sizeof(T);
    if (fits(kWide))
        return interleaved ? launch_rope_as<T, kWide, true, kAppend>(p, st)
                           : launch_rope_as<T, kWide, false, kAppend>(p, st);
    if (kWide > 4 && fits(4))
        return interleaved ? launch_rope_as<T, 4, true, kAppend>(p, st)
                           : launch_rope_as<T, 4, false, kAppend>(p, st);
    return interleaved ? launch_rope_as<T, 1, true, kAppend>(p, st)
                       : launch_rope_as<T, 1, false, kAppend>(p, st);
}

// Positions, sections and frequencies into p; `heads` and D are set.
int set_angles(RopeParams& p, const int32_t* positions, int64_t pos_stride, int n_axes,
               const int32_t* sections, const float* inv_freq) {
    AMPB_REQUIRE(n_axes >= 0 && n_axes <= kMaxAxes, AMP_ERR_UNSUPPORTED,
                 "rope: %d axes not supported (at most %d)", n_axes, kMaxAxes);
    AMPB_REQUIRE(n_axes == 0 || sections, AMP_ERR_INVALID, "rope: NULL sections");
    int64_t pairs = 0;
    for (int a = 0; a < n_axes; ++a) {
        AMPB_REQUIRE(sections[a] >= 0, AMP_ERR_INVALID, "rope: section %d is negative", a);
        pairs += sections[a];
        if (a < kMaxAxes - 1) p.axis_end[a] = (int)std::min<int64_t>(pairs, INT32_MAX);
    }
    // pairs past the last axis do not exist: later ends are never reached
    for (int a = std::max(n_axes - 1, 0); a < kMaxAxes - 1; ++a) p.axis_end[a] = INT32_MAX;
    // an empty tensor's address is NULL: no tokens have no positions, no pairs no frequencies
    AMPB_REQUIRE((n_axes == 0 || p.T == 0 || positions) && (pairs == 0 || inv_freq), AMP_ERR_INVALID,
                 "rope: NULL positions or inv_freq");
    AMPB_REQUIRE(2 * pairs <= p.D, AMP_ERR_INVALID, "rope: sections name %lld pairs, head_dim is %d",
                 (long long)pairs, p.D);
    AMPB_REQUIRE(n_axes <= 1 || pos_stride >= p.T || pos_stride == 0, AMP_ERR_INVALID,
                 "rope: the axes' positions overlap (stride %lld < %d tokens)", (long long)pos_stride,
                 p.T);
    p.pairs = (int)pairs;
    p.pos = positions;
    p.pos_stride = pos_stride;
    p.inv_freq = inv_freq;
    return AMP_OK;
}

int set_tensor(RopeParams& p, int i, const void* in, void* out, int heads, const int64_t* in_strides,
               const int64_t* out_strides, bool has_out) {
    p.heads[i] = heads;
    if (heads == 0) return AMP_OK;
    AMPB_REQUIRE(in && (out || !has_out), AMP_ERR_INVALID, "rope: NULL tensor");
    for (int s = 0; s < 2; ++s)
        AMPB_REQUIRE(in_strides[s] > 0 && (!has_out || out_strides[s] > 0), AMP_ERR_INVALID,
                     "rope: strides must be positive");
    AMPB_REQUIRE(!has_out || in != out || (in_strides[0] == out_strides[0] && in_strides[1] == out_strides[1]),
                 AMP_ERR_INVALID, "rope: in place, the output's strides must be the input's");
    p.x[i] = {in, out, in_strides[0], in_strides[1], has_out ? out_strides[0] : 0,
              has_out ? out_strides[1] : 0};
    return AMP_OK;
}

// An output may be its own input, not another tensor's place (NULL: no tensor).
int check_apart(const void* out, const void* other) {
    AMPB_REQUIRE(!out || out != other, AMP_ERR_INVALID, "rope: an output shares memory with another tensor");
    return AMP_OK;
}

int check_sizes(int T, int Hq, int Hk, int D) {
    AMPB_REQUIRE(T >= 0 && Hq >= 0 && Hk >= 0 && D > 0, AMP_ERR_INVALID, "rope: negative size");
    AMPB_REQUIRE(D % 2 == 0 && D <= 1024 && Hq <= 4096 && Hk <= 4096, AMP_ERR_UNSUPPORTED,
                 "rope: head_dim %d (even, at most 1024) or %d + %d heads (at most 4096 each) not "
                 "supported", D, Hq, Hk);
    return AMP_OK;
}

}  // namespace
}  // namespace ampb

using namespace ampb;

extern "C" int amp_rope_dev(const void* q, void* q_out, const void* k, void* k_out, int dtype, int T,
                            int Hq, int Hk, int head_dim, const int64_t* strides,
                            const int32_t* positions, int64_t pos_stride, int n_axes,
                            const int32_t* sections, const float* inv_freq, int interleaved,
                            int backward, void* stream) {
    RopeParams p = {};
    int rc = check_sizes(T, Hq, Hk, head_dim);
    if (rc) return rc;
    AMPB_REQUIRE(dtype == AMP_DTYPE_BF16 || dtype == AMP_DTYPE_F32, AMP_ERR_UNSUPPORTED,
                 "rope: dtype %d not supported (bf16, fp32)", dtype);
    AMPB_REQUIRE(strides, AMP_ERR_INVALID, "rope: NULL strides");
    p.T = T;
    p.D = head_dim;
    p.H = Hq + Hk;
    p.sign = backward ? -1.0f : 1.0f;
    if ((rc = set_angles(p, positions, pos_stride, n_axes, sections, inv_freq))) return rc;
    if (T == 0 || p.H == 0) return AMP_OK;
    if ((rc = set_tensor(p, 0, q, q_out, Hq, strides, strides + 2, true))) return rc;
    if ((rc = set_tensor(p, 1, k, k_out, Hk, strides + 4, strides + 6, true))) return rc;
    if (Hq > 0 && Hk > 0 &&
        ((rc = check_apart(q_out, k)) || (rc = check_apart(k_out, q)) || (rc = check_apart(q_out, k_out))))
        return rc;
    return dtype == AMP_DTYPE_BF16
               ? launch_rope<__nv_bfloat16, false>(p, interleaved != 0, as_stream(stream))
               : launch_rope<float, false>(p, interleaved != 0, as_stream(stream));
}

extern "C" int amp_paged_rope_append_bf16_dev(
    const void* q, void* q_out, const void* k, const void* v, int T, int Hq, int Hkv, int head_dim,
    const int64_t* strides, const int32_t* positions, int64_t pos_stride, int n_axes,
    const int32_t* sections, const float* inv_freq, int interleaved, void* k_pool, void* v_pool,
    const int32_t* block_table, const int32_t* ctx_lens, const int32_t* cu_seqlens, int B,
    int num_pages, int max_pages_per_seq, void* stream) {
    RopeParams p = {};
    int rc = check_sizes(T, Hq, Hkv, head_dim);
    if (rc) return rc;
    AMPB_REQUIRE(strides, AMP_ERR_INVALID, "append: NULL strides");
    AMPB_REQUIRE(B > 0 && Hkv > 0 && num_pages > 0 && max_pages_per_seq > 0, AMP_ERR_INVALID,
                 "append: sizes must be positive");
    p.T = T;
    p.D = head_dim;
    p.H = Hq + 2 * Hkv;
    p.sign = 1.0f;
    if ((rc = set_angles(p, positions, pos_stride, n_axes, sections, inv_freq))) return rc;
    AMPB_REQUIRE(k_pool && v_pool && block_table && ctx_lens && cu_seqlens, AMP_ERR_INVALID,
                 "append: NULL pool or table");
    if (T == 0) return AMP_OK;
    if ((rc = set_tensor(p, 0, q, q_out, Hq, strides, strides + 2, true))) return rc;
    if ((rc = set_tensor(p, 1, k, nullptr, Hkv, strides + 4, nullptr, false))) return rc;
    if ((rc = set_tensor(p, 2, v, nullptr, Hkv, strides + 6, nullptr, false))) return rc;
    if (Hq > 0 && ((rc = check_apart(q_out, k)) || (rc = check_apart(q_out, v)))) return rc;
    p.k_pool = k_pool;
    p.v_pool = v_pool;
    p.block_table = block_table;
    p.ctx_lens = ctx_lens;
    p.cu = cu_seqlens;
    p.B = B;
    p.num_pages = num_pages;
    p.max_pages = max_pages_per_seq;
    if ((rc = device_status(&p.status))) return rc;
    return launch_rope<__nv_bfloat16, true>(p, interleaved != 0, as_stream(stream));
}
