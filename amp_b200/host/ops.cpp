// ops.cpp -- the Python entry points of the packed-sequence attention, the rotary
// positions and the paged cache's bookkeeping: argument checks, output allocation and
// the call of the C ABI (include/amp_b200.h), for torch tensors.
//
// A decode step makes these calls on a few kilobytes, where the kernels take 2 to 10 us.
// Checked and called through ctypes, a call cost 18 to 28 us of host time (20 to 25
// converted arguments, four attribute reads a tensor); here it costs 2.5 to 7, and 13 for the
// backward's three results and four kernels.  The rest of the package calls the C ABI through ctypes (_lib.py); both use the same library: bind()
// receives the addresses of its functions.
//
// Every entry takes its arguments by position -- the keywords, defaults and documentation
// are in attention.py, rope.py and paged.py.  A bad argument raises ValueError, a nonzero
// status _lib.AmpError.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <sstream>
#include <string>
#include <vector>

#include "amp_b200.h"

namespace {

#define AMP_FUNCTIONS(X)                       \
    X(amp_last_error)                          \
    X(amp_flash_attn_varlen_workspace_bytes)   \
    X(amp_flash_attn_varlen_fwd_bf16_dev)      \
    X(amp_flash_attn_varlen_bwd_workspace_bytes) \
    X(amp_flash_attn_varlen_bwd_bf16_dev)      \
    X(amp_rope_dev)                            \
    X(amp_paged_rope_append_bf16_dev)          \
    X(amp_paged_copy_workspace_bytes)          \
    X(amp_paged_copy_pages_dev)                \
    X(amp_paged_fork_workspace_bytes)          \
    X(amp_paged_fork_dev)                      \
    X(amp_paged_extend_workspace_bytes)        \
    X(amp_paged_extend_dev)                    \
    X(amp_paged_compact_workspace_bytes)       \
    X(amp_paged_compact_dev)                   \
    X(amp_paged_free_dev)

struct Functions {
#define X(name) decltype(&::name) name = nullptr;
    AMP_FUNCTIONS(X)
#undef X
} F;

PyObject* g_amp_error = nullptr;   // _lib.AmpError

struct Raised {};   // a Python exception is set

template <typename... A>
[[noreturn]] void bad(const A&... parts) {
    std::ostringstream s;
    (s << ... << parts);
    PyErr_SetString(PyExc_ValueError, s.str().c_str());
    throw Raised{};
}

// ------------------------------------------------------------------ arguments
struct Args {
    const char* fn;
    PyObject* const* v;
    Py_ssize_t n;

    const at::Tensor& tensor(int i, const char* name) const {
        if (!THPVariable_Check(v[i])) bad(fn, ": ", name, " must be a tensor");
        return THPVariable_Unpack(v[i]);
    }
    // the tensor, or an undefined one for None
    at::Tensor maybe(int i, const char* name) const {
        return v[i] == Py_None ? at::Tensor() : tensor(i, name);
    }
    bool truth(int i) const {
        const int t = PyObject_IsTrue(v[i]);
        if (t < 0) throw Raised{};
        return t != 0;
    }
    float number(int i) const {
        const double d = PyFloat_AsDouble(v[i]);
        if (d == -1.0 && PyErr_Occurred()) throw Raised{};
        return (float)d;
    }
};

void check_cuda(const at::Tensor& t, const char* name) {
    if (!t.is_cuda()) bad(name, ": expected a CUDA tensor, got one on ", t.device());
}

// Token and head stride in elements of a [tokens, heads, D] tensor with a contiguous last
// dimension; tokens or heads < 0: any.  `multiple`: what the strides must divide by.
void packed(const at::Tensor& t, const char* name, const at::Device& dev, at::ScalarType type,
            int64_t tokens, int64_t heads, int64_t D, int64_t multiple, int64_t* strides) {
    if (t.dim() != 3 || t.scalar_type() != type || t.device() != dev || t.size(2) != D ||
        (tokens >= 0 && t.size(0) != tokens) || (heads >= 0 && t.size(1) != heads))
        bad(name, ": expected a ", type, " tensor [", tokens < 0 ? std::string("tokens") : std::to_string(tokens),
            ", ", heads < 0 ? std::string("heads") : std::to_string(heads), ", ", D, "] on ", dev, ", got ",
            t.scalar_type(), " ", t.sizes(), " on ", t.device());
    // the stride of a dimension of one element says nothing
    const int64_t head = t.size(1) <= 1 ? D : t.stride(1);
    const int64_t tok = t.size(0) <= 1 ? std::max<int64_t>(1, t.size(1)) * D : t.stride(0);
    if ((D > 1 && t.stride(2) != 1) || tok <= 0 || head <= 0 || tok % multiple || head % multiple)
        bad(name, ": the last dimension must be contiguous and the other strides positive multiples of ",
            multiple, " elements, got ", t.strides());
    strides[0] = tok;
    strides[1] = head;
}

// A contiguous int32 tensor of `dims` dimensions on dev; sizes < 0: any.
int32_t* ints(const at::Tensor& t, const char* name, const at::Device& dev, int64_t n0, int64_t n1 = -2) {
    const bool two = n1 != -2;
    if (t.dim() != (two ? 2 : 1) || t.scalar_type() != at::kInt || t.device() != dev || !t.is_contiguous() ||
        (n0 >= 0 && t.size(0) != n0) || (two && n1 >= 0 && t.size(1) != n1))
        bad(name, ": expected a contiguous int32 tensor [", n0, two ? ", " : "", two ? std::to_string(n1) : "",
            "] on ", dev, " (-1: any size), got ", t.scalar_type(), " ", t.sizes(), " on ", t.device());
    return t.data_ptr<int32_t>();
}

int narrow(int64_t x, const char* name) {
    if (x > INT32_MAX) bad(name, ": ", x, " is more than 2^31 - 1");
    return (int)x;
}

// Straight from the caching allocator (dev's current stream), without the dispatcher.
at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const at::Device& dev) {
    return at::detail::empty_cuda(sizes, type, dev, std::nullopt);
}

at::Tensor scratch(at::Tensor ws, size_t bytes, const at::Device& dev) {
    if (!ws.defined()) return empty({(int64_t)bytes}, at::kByte, dev);
    if (ws.device() != dev || ws.scalar_type() != at::kByte || !ws.is_contiguous() ||
        (size_t)ws.numel() < bytes)
        bad("workspace: expected a contiguous uint8 tensor of >= ", bytes, " bytes on ", dev);
    return ws;
}

// Without the interpreter lock while it lives; an exception passes with the lock held again.
struct Unlocked {
    PyThreadState* state = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(state); }
};

// Runs `call(stream)`, which calls no Python, with the tensors' device current and its current stream, without the
// interpreter lock, and raises AmpError for a nonzero status.
template <typename C>
void run(const at::Device& dev, const char* name, C call) {
    int rc = 0;
    std::string message;
    {
        c10::cuda::OptionalCUDAGuard guard;
        if (c10::cuda::current_device() != dev.index()) guard.set_device(dev);
        void* stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
        const Unlocked unlocked;
        rc = call(stream);
        if (rc) message = F.amp_last_error();
    }
    if (rc == 0) return;
    PyObject* e = PyObject_CallFunction(g_amp_error, "sis", name, rc, message.c_str());
    if (e) {
        PyErr_SetObject(g_amp_error, e);
        Py_DECREF(e);
    }
    throw Raised{};
}

PyObject* wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }

PyObject* tuple(std::initializer_list<at::Tensor> ts) {
    PyObject* out = PyTuple_New((Py_ssize_t)ts.size());
    if (!out) throw Raised{};
    Py_ssize_t i = 0;
    for (const at::Tensor& t : ts) {
        PyObject* o = THPVariable_Wrap(t);
        if (!o) {
            Py_DECREF(out);
            throw Raised{};
        }
        PyTuple_SET_ITEM(out, i++, o);
    }
    return out;
}

// ------------------------------------------------------- packed attention
struct Packed {
    int T, Tk, Hq, Hkv, D, B;
    const int32_t *cu, *cu_kv;
    at::Device dev{at::kCUDA};
};

Packed packed_shapes(const at::Tensor& q, const at::Tensor& k, const at::Tensor& cu, const at::Tensor& cu_kv) {
    Packed p;
    check_cuda(q, "q");
    if (q.dim() != 3 || k.dim() != 3) bad("q, k, v: expected packed tensors [tokens, heads, head_dim]");
    p.dev = q.device();
    p.T = narrow(q.size(0), "q");
    p.Hq = narrow(q.size(1), "q");
    p.D = narrow(q.size(2), "q");
    p.Tk = narrow(k.size(0), "k");
    p.Hkv = narrow(k.size(1), "k");
    p.cu = ints(cu, "cu_seqlens", p.dev, -1);
    p.B = narrow(cu.numel() - 1, "cu_seqlens");
    if (p.B < 1) bad("cu_seqlens: expected one offset more than there are sequences, got ", cu.numel());
    p.cu_kv = cu_kv.defined() ? ints(cu_kv, "cu_seqlens_kv", p.dev, cu.numel()) : p.cu;
    return p;
}

float* check_lse(const at::Tensor& lse, const Packed& p) {
    if (lse.scalar_type() != at::kFloat || lse.dim() != 2 || lse.size(0) != p.Hq || lse.size(1) != p.T ||
        lse.device() != p.dev || !lse.is_contiguous())
        bad("lse: expected a contiguous float32 tensor [", p.Hq, ", ", p.T, "] on ", p.dev);
    return lse.data_ptr<float>();
}

// (q, k, v, cu_seqlens, cu_seqlens_kv, causal, scale, out, lse, workspace) -> (out, lse)
PyObject* varlen_fwd(const Args& a) {
    const at::Tensor &q = a.tensor(0, "q"), &k = a.tensor(1, "k"), &v = a.tensor(2, "v");
    const Packed p = packed_shapes(q, k, a.tensor(3, "cu_seqlens"), a.maybe(4, "cu_seqlens_kv"));
    const bool causal = a.truth(5);
    const float scale = a.number(6);
    at::Tensor out = a.maybe(7, "out"), lse = a.maybe(8, "lse");
    int64_t st[8];
    packed(q, "q", p.dev, at::kBFloat16, p.T, p.Hq, p.D, 8, st);
    packed(k, "k", p.dev, at::kBFloat16, p.Tk, p.Hkv, p.D, 8, st + 2);
    packed(v, "v", p.dev, at::kBFloat16, p.Tk, p.Hkv, p.D, 8, st + 4);
    if (!out.defined()) out = empty({p.T, p.Hq, p.D}, at::kBFloat16, p.dev);
    packed(out, "out", p.dev, at::kBFloat16, p.T, p.Hq, p.D, 8, st + 6);
    if (!lse.defined()) lse = empty({p.Hq, p.T}, at::kFloat, p.dev);
    float* l = check_lse(lse, p);
    const at::Tensor ws = scratch(a.maybe(9, "workspace"),
                                  F.amp_flash_attn_varlen_workspace_bytes(p.B, p.Hq, p.Hkv, p.T, p.Tk, p.D), p.dev);
    run(p.dev, "amp_flash_attn_varlen_fwd_bf16_dev", [&](void* stream) {
        return F.amp_flash_attn_varlen_fwd_bf16_dev(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), l,
                                                    p.cu, p.cu_kv, p.B, p.T, p.Tk, p.Hq, p.Hkv, p.D, st, causal,
                                                    scale, ws.data_ptr(), ws.numel(), stream);
    });
    return tuple({out, lse});
}

// (q, k, v, o, do, lse, cu_seqlens, cu_seqlens_kv, causal, scale, dq, dk, dv, workspace) -> (dq, dk, dv)
PyObject* varlen_bwd(const Args& a) {
    const at::Tensor &q = a.tensor(0, "q"), &k = a.tensor(1, "k"), &v = a.tensor(2, "v"), &o = a.tensor(3, "o"),
                     &d_o = a.tensor(4, "do"), &lse = a.tensor(5, "lse");
    const Packed p = packed_shapes(q, k, a.tensor(6, "cu_seqlens"), a.maybe(7, "cu_seqlens_kv"));
    const bool causal = a.truth(8);
    const float scale = a.number(9);
    at::Tensor dq = a.maybe(10, "dq"), dk = a.maybe(11, "dk"), dv = a.maybe(12, "dv");
    if (!dq.defined()) dq = empty({p.T, p.Hq, p.D}, at::kBFloat16, p.dev);
    if (!dk.defined()) dk = empty({p.Tk, p.Hkv, p.D}, at::kBFloat16, p.dev);
    if (!dv.defined()) dv = empty({p.Tk, p.Hkv, p.D}, at::kBFloat16, p.dev);
    int64_t st[16];
    const struct { const at::Tensor& t; const char* name; bool keys; } all[8] = {
        {q, "q", false}, {k, "k", true},    {v, "v", true},   {o, "o", false},
        {d_o, "do", false}, {dq, "dq", false}, {dk, "dk", true}, {dv, "dv", true}};
    for (int i = 0; i < 8; ++i)
        packed(all[i].t, all[i].name, p.dev, at::kBFloat16, all[i].keys ? p.Tk : p.T,
               all[i].keys ? p.Hkv : p.Hq, p.D, 8, st + 2 * i);
    const float* l = check_lse(lse, p);
    const at::Tensor ws = scratch(a.maybe(13, "workspace"),
                                  F.amp_flash_attn_varlen_bwd_workspace_bytes(p.B, p.Hq, p.Hkv, p.T, p.Tk, p.D),
                                  p.dev);
    run(p.dev, "amp_flash_attn_varlen_bwd_bf16_dev", [&](void* stream) {
        return F.amp_flash_attn_varlen_bwd_bf16_dev(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), d_o.data_ptr(), l, dq.data_ptr(),
            dk.data_ptr(), dv.data_ptr(), p.cu, p.cu_kv, p.B, p.T, p.Tk, p.Hq, p.Hkv, p.D, st, causal, scale,
            ws.data_ptr(), ws.numel(), stream);
    });
    return tuple({dq, dk, dv});
}

// ------------------------------------------------------------------ rotary
struct Angles {
    const int32_t* pos = nullptr;
    int64_t stride = 0;
    int axes = 0;
    int32_t sections[4] = {0, 0, 0, 0};
    const float* inv_freq = nullptr;
};

// positions int32 [T] or [axes, T], inv_freq fp32 [pairs], sections a sequence or None
Angles angles(const at::Tensor& pos, const at::Tensor& inv_freq, PyObject* sections, const at::Device& dev,
              int64_t T) {
    Angles g;
    if (pos.device() != dev || pos.scalar_type() != at::kInt || (pos.dim() != 1 && pos.dim() != 2) ||
        pos.size(-1) != T || (T > 1 && pos.stride(-1) != 1))
        bad("positions: expected int32 [", T, "] or [axes, ", T, "] on ", dev, ", got ", pos.scalar_type(), " ",
            pos.sizes(), " on ", pos.device());
    const int64_t axes = pos.dim() == 1 ? 1 : pos.size(0);
    if (inv_freq.device() != dev || inv_freq.scalar_type() != at::kFloat || inv_freq.dim() != 1 ||
        !inv_freq.is_contiguous())
        bad("inv_freq: expected a contiguous float32 vector on ", dev);
    if (axes < 1 || axes > 4) bad("positions: 1 to 4 axes, got ", axes);
    int64_t sum = 0, n = 0;
    if (sections == Py_None) {
        n = 1;
        sum = inv_freq.numel();
        g.sections[0] = narrow(sum, "inv_freq");
    } else {
        PyObject* seq = PySequence_Fast(sections, "sections: expected a sequence of counts");
        if (!seq) throw Raised{};
        n = PySequence_Fast_GET_SIZE(seq);
        for (int64_t i = 0; i < n && i < 4; ++i) {
            const long x = PyLong_AsLong(PySequence_Fast_GET_ITEM(seq, i));
            if (x == -1 && PyErr_Occurred()) {
                Py_DECREF(seq);
                throw Raised{};
            }
            if (x < 0 || x > INT32_MAX) {
                Py_DECREF(seq);
                bad("sections: ", x, " pairs");
            }
            g.sections[i] = (int32_t)x;
            sum += x;
        }
        Py_DECREF(seq);
    }
    if (n != axes || sum != inv_freq.numel())
        bad("sections: one count of pairs for each of ", axes, " axes, ", inv_freq.numel(),
            " (the entries of inv_freq) in all; got ", n, " counts, ", sum, " pairs");
    g.axes = (int)axes;
    g.stride = pos.dim() == 2 && axes > 1 ? pos.stride(0) : T;
    g.pos = pos.data_ptr<int32_t>();
    g.inv_freq = inv_freq.data_ptr<float>();
    return g;
}

// (q, k, positions, inv_freq, sections, interleaved, out_q, out_k, backward) -> (out_q, out_k)
PyObject* rope(const Args& a) {
    const at::Tensor& q = a.tensor(0, "q");
    const at::Tensor k = a.maybe(1, "k");
    check_cuda(q, "q");
    const at::ScalarType type = q.scalar_type();
    if (q.dim() != 3 || (type != at::kBFloat16 && type != at::kFloat))
        bad("q: expected a bfloat16 or float32 tensor [tokens, heads, head_dim]");
    const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2);
    const at::Device dev = q.device();
    const Angles g = angles(a.tensor(2, "positions"), a.tensor(3, "inv_freq"), a.v[4], dev, T);
    const bool interleaved = a.truth(5), backward = a.truth(8);
    at::Tensor out_q = a.maybe(6, "out_q"), out_k = a.maybe(7, "out_k");
    int64_t st[8] = {1, 1, 1, 1, 1, 1, 1, 1}, Hk = 0;
    packed(q, "q", dev, type, T, Hq, D, 1, st);
    if (!out_q.defined()) out_q = empty({T, Hq, D}, type, dev);
    packed(out_q, "out_q", dev, type, T, Hq, D, 1, st + 2);
    if (k.defined()) {
        packed(k, "k", dev, type, T, -1, D, 1, st + 4);
        Hk = k.size(1);
        if (!out_k.defined()) out_k = empty({T, Hk, D}, type, dev);
        packed(out_k, "out_k", dev, type, T, Hk, D, 1, st + 6);
    } else {
        out_k = at::Tensor();
    }
    const int t = narrow(T, "q"), hq = narrow(Hq, "q"), hk = narrow(Hk, "k"), d = narrow(D, "q");
    run(dev, "amp_rope_dev", [&](void* stream) {
        return F.amp_rope_dev(q.data_ptr(), out_q.data_ptr(), k.defined() ? k.data_ptr() : nullptr,
                              k.defined() ? out_k.data_ptr() : nullptr,
                              type == at::kFloat ? AMP_DTYPE_F32 : AMP_DTYPE_BF16, t, hq, hk, d, st, g.pos,
                              g.stride, g.axes, g.sections, g.inv_freq, interleaved, backward, stream);
    });
    return tuple({out_q, out_k});   // an undefined tensor becomes None
}

// (q | None, k, v, k_pool, v_pool, block_table, ctx_lens, cu_seqlens, positions, inv_freq, sections,
//  interleaved, out_q) -> out_q; without q: no turn, positions and the rest None
PyObject* append(const Args& a) {
    const at::Tensor q = a.maybe(0, "q");
    const at::Tensor &k = a.tensor(1, "k"), &v = a.tensor(2, "v"), &kp = a.tensor(3, "k_pool"),
                     &vp = a.tensor(4, "v_pool"), &bt = a.tensor(5, "block_table"),
                     &ctx = a.tensor(6, "ctx_lens"), &cu = a.tensor(7, "cu_seqlens");
    check_cuda(kp, "k_pool");
    const at::Device dev = kp.device();
    for (const at::Tensor* t : {&kp, &vp})
        if (t->dim() != 4 || t->scalar_type() != at::kBFloat16 || !t->is_contiguous() || t->size(2) != 16 ||
            t->sizes() != kp.sizes() || t->device() != dev)
            bad(t == &kp ? "k_pool" : "v_pool", ": expected contiguous bfloat16 pools [pages, Hkv, 16, D] on one "
                "device, got ", t->sizes());
    const int64_t pages = kp.size(0), Hkv = kp.size(1), D = kp.size(3);
    if (k.dim() != 3) bad("k: expected a tensor [tokens, Hkv, D]");
    const int64_t T = k.size(0);
    int64_t st[8] = {1, 1, 1, 1, 1, 1, 1, 1}, Hq = 0;
    at::Tensor out = a.maybe(12, "out_q");
    Angles g;
    if (q.defined()) {
        packed(q, "q", dev, at::kBFloat16, T, -1, D, 1, st);
        Hq = q.size(1);
        g = angles(a.tensor(8, "positions"), a.tensor(9, "inv_freq"), a.v[10], dev, T);
        if (!out.defined()) out = empty({T, Hq, D}, at::kBFloat16, dev);
        packed(out, "out_q", dev, at::kBFloat16, T, Hq, D, 1, st + 2);
    }
    packed(k, "k", dev, at::kBFloat16, T, Hkv, D, 1, st + 4);
    packed(v, "v", dev, at::kBFloat16, T, Hkv, D, 1, st + 6);
    const bool interleaved = a.truth(11);
    const int32_t* offsets = ints(cu, "cu_seqlens", dev, -1);
    const int64_t B = cu.numel() - 1;
    if (B < 1) bad("cu_seqlens: expected one offset more than there are sequences, got ", cu.numel());
    int32_t *table = ints(bt, "block_table", dev, -1, -1), *lens = ints(ctx, "ctx_lens", dev, -1);
    if (bt.size(0) < B || ctx.numel() < B) bad("block_table [>= ", B, ", pages] and ctx_lens [>= ", B, "] expected");
    const int t = narrow(T, "k"), hq = narrow(Hq, "q"), hkv = narrow(Hkv, "k"), d = narrow(D, "k"),
              b = narrow(B, "cu_seqlens"), np = narrow(pages, "k_pool"), width = narrow(bt.size(1), "block_table");
    run(dev, "amp_paged_rope_append_bf16_dev", [&](void* stream) {
        return F.amp_paged_rope_append_bf16_dev(
            q.defined() ? q.data_ptr() : nullptr, q.defined() ? out.data_ptr() : nullptr, k.data_ptr(),
            v.data_ptr(), t, hq, hkv, d, st, g.pos, g.stride, g.axes, g.sections, g.inv_freq, interleaved,
            kp.data_ptr(), vp.data_ptr(), table, lens, offsets, b, np, width, stream);
    });
    return wrap(out);   // None without q
}

// -------------------------------------------------------- cache bookkeeping
struct Cache {
    void *k, *v;
    int layers, pages, Hkv, D;
    at::Device dev{at::kCUDA};
};

Cache pools(const at::Tensor& k, const at::Tensor& v) {
    check_cuda(k, "k_pool");
    if (k.sizes() != v.sizes() || k.device() != v.device()) bad("k_pool and v_pool shapes or devices differ");
    for (const at::Tensor* t : {&k, &v})
        if (t->scalar_type() != at::kBFloat16 || !t->is_contiguous() || (t->dim() != 4 && t->dim() != 5) ||
            t->size(-2) != 16)
            bad(t == &k ? "k_pool" : "v_pool", ": expected a contiguous bfloat16 tensor [(layers,) pages, Hkv, 16, D], "
                "got ", t->scalar_type(), " ", t->sizes());
    Cache c;
    c.dev = k.device();
    c.layers = k.dim() == 5 ? narrow(k.size(0), "k_pool") : 1;
    c.pages = narrow(k.size(-4), "k_pool");
    c.Hkv = narrow(k.size(-3), "k_pool");
    c.D = narrow(k.size(-1), "k_pool");
    c.k = k.data_ptr();
    c.v = v.data_ptr();
    return c;
}

struct TableArgs {
    int32_t *table, *ctx;
    int rows, width;
};

TableArgs table(const at::Tensor& bt, const at::Tensor& ctx, const at::Device& dev) {
    TableArgs t;
    t.table = ints(bt, "block_table", dev, -1, -1);
    t.rows = narrow(bt.size(0), "block_table");
    t.width = narrow(bt.size(1), "block_table");
    t.ctx = ints(ctx, "ctx_lens", dev, t.rows);
    return t;
}

// (k_pool, v_pool, src, dst, workspace) -> None
PyObject* copy_pages(const Args& a) {
    const Cache c = pools(a.tensor(0, "k_pool"), a.tensor(1, "v_pool"));
    const at::Tensor& src = a.tensor(2, "src");
    const int32_t* s = ints(src, "src", c.dev, -1);
    const int n = narrow(src.numel(), "src");
    const int32_t* d = ints(a.tensor(3, "dst"), "dst", c.dev, n);
    const at::Tensor ws = scratch(a.maybe(4, "workspace"), F.amp_paged_copy_workspace_bytes(n), c.dev);
    run(c.dev, "amp_paged_copy_pages_dev", [&](void* stream) {
        return F.amp_paged_copy_pages_dev(c.k, c.v, c.layers, c.pages, c.Hkv, c.D, s, d, n, ws.data_ptr(),
                                          ws.numel(), stream);
    });
    Py_RETURN_NONE;
}

// (k_pool, v_pool, block_table, ctx_lens, parents, children, workspace) -> done
PyObject* fork_sequences(const Args& a) {
    const Cache c = pools(a.tensor(0, "k_pool"), a.tensor(1, "v_pool"));
    const TableArgs t = table(a.tensor(2, "block_table"), a.tensor(3, "ctx_lens"), c.dev);
    const at::Tensor& parents = a.tensor(4, "parents");
    const int32_t* p = ints(parents, "parents", c.dev, -1);
    const int n = narrow(parents.numel(), "parents");
    const int32_t* ch = ints(a.tensor(5, "children"), "children", c.dev, n);
    at::Tensor done = empty({n}, at::kInt, c.dev);
    const at::Tensor ws = scratch(a.maybe(6, "workspace"), F.amp_paged_fork_workspace_bytes(n, t.width), c.dev);
    run(c.dev, "amp_paged_fork_dev", [&](void* stream) {
        return F.amp_paged_fork_dev(c.k, c.v, c.layers, c.pages, c.Hkv, c.D, t.table, t.ctx, t.rows, t.width, p, ch,
                                    n, done.data_ptr<int32_t>(), ws.data_ptr(), ws.numel(), stream);
    });
    return wrap(done);
}

// (k_pool, v_pool, block_table, ctx_lens, add, out, workspace) -> (ctx_lens', done)
PyObject* extend_sequences(const Args& a) {
    const Cache c = pools(a.tensor(0, "k_pool"), a.tensor(1, "v_pool"));
    const TableArgs t = table(a.tensor(2, "block_table"), a.tensor(3, "ctx_lens"), c.dev);
    const int32_t* add = ints(a.tensor(4, "add"), "add", c.dev, t.rows);
    at::Tensor out = a.maybe(5, "out");
    if (!out.defined()) out = empty({t.rows}, at::kInt, c.dev);
    int32_t* o = ints(out, "out", c.dev, t.rows);
    at::Tensor done = empty({t.rows}, at::kInt, c.dev);
    const at::Tensor ws = scratch(a.maybe(6, "workspace"), F.amp_paged_extend_workspace_bytes(t.rows, c.pages), c.dev);
    run(c.dev, "amp_paged_extend_dev", [&](void* stream) {
        return F.amp_paged_extend_dev(c.k, c.v, c.layers, c.pages, c.Hkv, c.D, t.table, t.ctx, t.rows, t.width, add,
                                      o, done.data_ptr<int32_t>(), ws.data_ptr(), ws.numel(), stream);
    });
    return tuple({out, done});
}

// (k_pool, v_pool, block_table, ctx_lens, out, workspace) -> (table', used)
PyObject* compact_pages(const Args& a) {
    const Cache c = pools(a.tensor(0, "k_pool"), a.tensor(1, "v_pool"));
    const TableArgs t = table(a.tensor(2, "block_table"), a.tensor(3, "ctx_lens"), c.dev);
    at::Tensor out = a.maybe(4, "out");
    if (!out.defined()) out = empty({t.rows, t.width}, at::kInt, c.dev);
    int32_t* o = ints(out, "out", c.dev, t.rows, t.width);
    at::Tensor used = empty({1}, at::kInt, c.dev);
    const at::Tensor ws = scratch(a.maybe(5, "workspace"), F.amp_paged_compact_workspace_bytes(c.pages), c.dev);
    run(c.dev, "amp_paged_compact_dev", [&](void* stream) {
        return F.amp_paged_compact_dev(c.k, c.v, c.layers, c.pages, c.Hkv, c.D, t.table, t.ctx, t.rows, t.width, o,
                                       used.data_ptr<int32_t>(), ws.data_ptr(), ws.numel(), stream);
    });
    return tuple({out, used});
}

// (block_table, ctx_lens, seqs) -> None
PyObject* free_sequences(const Args& a) {
    const at::Tensor& bt = a.tensor(0, "block_table");
    check_cuda(bt, "block_table");
    const TableArgs t = table(bt, a.tensor(1, "ctx_lens"), bt.device());
    const at::Tensor& seqs = a.tensor(2, "seqs");
    const int32_t* s = ints(seqs, "seqs", bt.device(), -1);
    const int n = narrow(seqs.numel(), "seqs");
    run(bt.device(), "amp_paged_free_dev", [&](void* stream) {
        return F.amp_paged_free_dev(t.table, t.ctx, t.rows, t.width, s, n, stream);
    });
    Py_RETURN_NONE;
}

// ------------------------------------------------------------------ module
template <PyObject* (*body)(const Args&), int count>
PyObject* entry(PyObject*, PyObject* const* v, Py_ssize_t n) {
    if (n != count) return PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", count, n);
    if (!F.amp_last_error) {
        PyErr_SetString(PyExc_RuntimeError, "the library's functions are not bound");
        return nullptr;
    }
    try {
        return body(Args{"amp_b200", v, n});
    } catch (const Raised&) {
        return nullptr;
    } catch (const std::exception& e) {   // c10::Error: out of memory, for one
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// bind(addresses: dict[str, int], AmpError)
PyObject* bind(PyObject*, PyObject* const* v, Py_ssize_t n) {
    if (n != 2 || !PyDict_Check(v[0])) {
        PyErr_SetString(PyExc_TypeError, "bind(addresses, error)");
        return nullptr;
    }
    Functions f;
#define X(name)                                                                             \
    {                                                                                       \
        PyObject* p = PyDict_GetItemString(v[0], #name);                                    \
        void* address = p ? PyLong_AsVoidPtr(p) : nullptr;                                  \
        if (!address) return PyErr_Format(PyExc_KeyError, "%s has no address", #name);      \
        f.name = reinterpret_cast<decltype(f.name)>(address);                               \
    }
    AMP_FUNCTIONS(X)
#undef X
    F = f;
    Py_INCREF(v[1]);
    Py_XSETREF(g_amp_error, v[1]);
    Py_RETURN_NONE;
}

PyObject* names(PyObject*, PyObject*) {
    std::vector<const char*> all = {
#define X(name) #name,
        AMP_FUNCTIONS(X)
#undef X
    };
    PyObject* out = PyTuple_New((Py_ssize_t)all.size());
    for (size_t i = 0; out && i < all.size(); ++i) PyTuple_SET_ITEM(out, i, PyUnicode_FromString(all[i]));
    return out;
}

// what this file was compiled against (_lib.host_abi)
PyObject* built_for(PyObject*, PyObject*) { return PyUnicode_FromString(AMP_HOST_ABI); }

#define ENTRY(name, count) \
    {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<name, count>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&bind)), METH_FASTCALL, nullptr},
    {"names", names, METH_NOARGS, nullptr},
    {"built_for", built_for, METH_NOARGS, nullptr},
    ENTRY(varlen_fwd, 10),
    ENTRY(varlen_bwd, 14),
    ENTRY(rope, 9),
    ENTRY(append, 13),
    ENTRY(copy_pages, 5),
    ENTRY(fork_sequences, 7),
    ENTRY(extend_sequences, 7),
    ENTRY(compact_pages, 6),
    ENTRY(free_sequences, 3),
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops(void) { return PyModule_Create(&module); }
