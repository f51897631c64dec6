// tsb_pyserving.cpp - the CPython side of the serving-step operators: argument checks, output and workspace tensors and the
// call into the C ABI, natively.  A decode step makes these calls between launches of a few microseconds, and the same
// work through ctypes took 7 to 16 us a call (a launch itself takes 3 to 4); tinystrata_b200/serving.py has the documented
// functions over it.  Every function runs on its tensors' device and that device's current stream, and raises TsbError
// (given to init) for what it or the C ABI refuses.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "../../include/tsb_moe.h"

namespace {

PyObject* g_error = nullptr;   // tinystrata_b200.TsbError

struct Refused {
    std::string text;
};
struct Raised {};              // a Python exception is set already

[[noreturn]] void refuse(const std::string& s) { throw Refused{s}; }
void need(bool ok, const char* what) {
    if (!ok) refuse(what);
}
std::string list(c10::IntArrayRef v) {
    std::string s = "[";
    for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
    return s + "]";
}
[[noreturn]] void bad(const at::Tensor& t, const char* what, const std::string& want) {
    const std::string got = t.defined() ? list(t.sizes()) + " " + c10::toString(t.scalar_type()) + " on " + t.device().str() + ", strides " + list(t.strides())
                                        : std::string("None");
    refuse(std::string(what) + ": " + want + " wanted, got " + got);
}
void status(int rc, const char* what) {
    if (rc != 0) refuse(std::string(what) + ": status " + std::to_string(rc) + ": " + tsb_last_error());
}

const at::Tensor& tensor(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) refuse(std::string(what) + ": a tensor wanted");
    return THPVariable_Unpack(o);
}
at::Tensor maybe(PyObject* o, const char* what) { return o == Py_None ? at::Tensor() : tensor(o, what); }
int64_t integer(PyObject* o) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Raised{};
    return v;
}
int int32(PyObject* o, const char* what) {
    const int64_t v = integer(o);
    need(v >= INT32_MIN && v <= INT32_MAX, what);
    return (int) v;
}
double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised{};
    return v;
}

int elem(at::ScalarType t, const char* what) {
    if (t == at::kFloat) return 0;
    if (t == at::kHalf) return 1;
    if (t == at::kBFloat16) return 30;
    refuse(std::string(what) + ": float32, float16 or bfloat16");
}
const char* name_of(at::ScalarType t) { return c10::toString(t); }

void on(const at::Tensor& t, at::ScalarType type, int64_t dims, const c10::Device& dev, const char* what) {
    if (!t.defined() || t.scalar_type() != type || t.dim() != dims || t.device() != dev)
        bad(t, what, std::to_string(dims) + "-dimensional " + name_of(type) + " on " + dev.str());
}
// at least n contiguous values
void flat(const at::Tensor& t, at::ScalarType type, int64_t n, const c10::Device& dev, const char* what) {
    on(t, type, 1, dev, what);
    if (t.size(0) < n || (n > 1 && t.stride(0) != 1)) bad(t, what, "at least " + std::to_string(n) + " contiguous values");
}
// [n, heads, dim] rows of one type, the innermost dimension contiguous
void rows(const at::Tensor& t, int64_t n, int64_t heads, int64_t dim, at::ScalarType type, const c10::Device& dev, const char* what) {
    on(t, type, 3, dev, what);
    if (t.size(0) != n || t.size(1) != heads || t.size(2) != dim || (dim > 1 && t.stride(2) != 1))
        bad(t, what, "[" + std::to_string(n) + ", " + std::to_string(heads) + ", " + std::to_string(dim) + "] with a contiguous innermost dimension");
}
// An output whose elements are all its own: strides, smallest first, step past what the smaller dimensions span.
void own_memory(const at::Tensor& t, const char* what) {
    int order[8];
    const int n = (int) t.dim();
    for (int i = 0; i < n; ++i) order[i] = i;
    std::sort(order, order + n, [&](int a, int b) { return t.stride(a) < t.stride(b); });
    int64_t span = 1;
    for (int i = 0; i < n; ++i) {
        if (t.size(order[i]) <= 1) continue;
        if (t.stride(order[i]) < span) bad(t, what, "elements that do not share memory");
        span += (t.size(order[i]) - 1) * t.stride(order[i]);
    }
}
// The operators have no backward pass: a tensor that asks for gradients would get outputs without them.
void no_grad(std::initializer_list<const at::Tensor*> tensors, const char* what) {
    if (!c10::GradMode::is_enabled()) return;
    for (const at::Tensor* t : tensors)
        if (t->defined() && t->requires_grad())
            refuse(std::string(what) + ": a tensor requires gradients, and there is no backward pass: call it under torch.no_grad() or detach the tensor");
}
// A tensor that the call writes: what autograd saved of it before is out of date.
void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
c10::Device cuda_of(const at::Tensor& t, const char* what) {
    if (!t.is_cuda()) bad(t, what, "a tensor on a CUDA device");
    return t.device();
}
void* stream_of(const c10::Device& d) { return (void*) c10::cuda::getCurrentCUDAStream(d.index()).stream(); }
void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
at::Tensor bytes(uint64_t n, const c10::Device& dev) {
    return n ? at::empty({(int64_t) n}, at::TensorOptions().dtype(at::kByte).device(dev)) : at::Tensor();
}

template <class F>
PyObject* guarded(F f) {
    HANDLE_TH_ERRORS
    try {
        return f();
    } catch (const Refused& e) {
        PyErr_SetString(g_error, e.text.c_str());
    } catch (const Raised&) {
    }
    return nullptr;
    END_HANDLE_TH_ERRORS
}
void count(Py_ssize_t got, Py_ssize_t want) {
    if (got != want) refuse("wrong number of arguments");
}

PyObject* init(PyObject*, PyObject* error) {
    Py_INCREF(error);
    Py_XDECREF(g_error);
    g_error = error;
    Py_RETURN_NONE;
}

// (lens, n_new, table, free, n_free, block_size, cap_tokens, done) -> (lens, cu, slots, n_free)
PyObject* block_tables(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        count(n, 8);
        const at::Tensor &lens = tensor(a[0], "block_tables: lens"), &add = tensor(a[1], "block_tables: n_new"),
                         &table = tensor(a[2], "block_tables: table"), &stack = tensor(a[3], "block_tables: free"),
                         &n_free = tensor(a[4], "block_tables: n_free"), done = maybe(a[7], "block_tables: done");
        const int bs = int32(a[5], "block_tables: block_size");
        const int64_t cap = integer(a[6]);
        const c10::Device dev = cuda_of(lens, "block_tables: lens");
        on(lens, at::kInt, 1, dev, "block_tables: lens");
        const int64_t R = lens.size(0);
        flat(lens, at::kInt, R, dev, "block_tables: lens");
        flat(add, at::kInt, R, dev, "block_tables: n_new");
        on(table, at::kInt, 2, dev, "block_tables: table");
        on(stack, at::kInt, 1, dev, "block_tables: free");
        flat(stack, at::kInt, stack.size(0), dev, "block_tables: free");
        flat(n_free, at::kInt, 1, dev, "block_tables: n_free");
        if (done.defined()) flat(done, at::kByte, R, dev, "block_tables: done");
        const int64_t width = table.size(1), blocks = stack.size(0);
        if (table.size(0) < R || (width > 1 && table.stride(1) != 1)) bad(table, "block_tables: table", "a contiguous row for every request");
        // the call writes every request's row: rows that share memory would be one another's
        if (R > 1 && table.stride(0) < width) bad(table, "block_tables: table", "rows that do not overlap");
        need(cap >= 0, "block_tables: cap_tokens");
        need(R <= INT32_MAX && width <= INT32_MAX && blocks <= INT32_MAX, "block_tables: sizes");
        const c10::cuda::CUDAGuard guard(dev);
        at::Tensor after = at::empty({R}, lens.options()), cu = at::empty({R + 1}, lens.options()), left = at::empty({1}, lens.options()),
                   slots = at::empty({cap}, lens.options().dtype(at::kLong));
        written(table), written(stack);
        status(tsb_block_tables((const int32_t*) ptr(lens), (const int32_t*) ptr(add), (const uint8_t*) ptr(done), (int) R,
                                (int32_t*) ptr(table), R > 1 ? table.stride(0) : width, (int) width, (int32_t*) ptr(stack), (int) blocks,
                                (const int32_t*) ptr(n_free), bs, (int32_t*) ptr(after), (int32_t*) ptr(cu), (int64_t*) ptr(slots), cap,
                                (int32_t*) ptr(left), stream_of(dev)),
               "block_tables");
        PyObject* out = PyTuple_New(4);
        if (!out) throw Raised{};
        PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(after));
        PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(cu));
        PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(slots));
        PyTuple_SET_ITEM(out, 3, THPVariable_Wrap(left));
        return out;
    });
}

// The cache as its four tensors; they are looked at in every call, so that nothing outlives a change to them.
struct Pools {
    tsb_kv8 c;
    c10::Device dev;
    const at::Tensor &k, &v, &ks, &vs;
};
Pools pools(PyObject* o) {
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) refuse("KV8Cache: (k, v, k_scale, v_scale)");
    const at::Tensor &k = tensor(PyTuple_GET_ITEM(o, 0), "KV8Cache: k"), &v = tensor(PyTuple_GET_ITEM(o, 1), "KV8Cache: v"),
                     &ks = tensor(PyTuple_GET_ITEM(o, 2), "KV8Cache: k_scale"), &vs = tensor(PyTuple_GET_ITEM(o, 3), "KV8Cache: v_scale");
    const c10::Device dev = cuda_of(k, "KV8Cache: k");
    on(k, at::kChar, 4, dev, "KV8Cache: k");
    on(v, at::kChar, 4, dev, "KV8Cache: v");
    on(ks, at::kFloat, 2, dev, "KV8Cache: k_scale");
    on(vs, at::kFloat, 2, dev, "KV8Cache: v_scale");
    if (!k.is_contiguous()) bad(k, "KV8Cache: k", "contiguous codes");
    if (!v.is_contiguous() || v.sizes() != k.sizes()) bad(v, "KV8Cache: v", "contiguous codes of k's shape");
    for (const at::Tensor* s : {&ks, &vs})
        if (!s->is_contiguous() || s->size(0) != k.size(0) || s->size(1) != k.size(1))
            bad(*s, "KV8Cache: scales", "contiguous [n_blocks, n_kv_heads]");
    need(k.size(0) <= INT32_MAX && k.size(1) <= INT32_MAX, "KV8Cache: sizes");
    return Pools{tsb_kv8{sizeof(tsb_kv8), (int32_t) k.size(0), (int32_t) k.size(2), (int32_t) k.size(1), (int32_t) k.size(3),
                         (int8_t*) ptr(k), (int8_t*) ptr(v), (float*) ptr(ks), (float*) ptr(vs)},
                 dev, k, v, ks, vs};
}

// (cache, k, v, slots)
PyObject* kv8_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        count(n, 4);
        const Pools p = pools(a[0]);
        const at::Tensor &k = tensor(a[1], "kv8_append: k"), &v = tensor(a[2], "kv8_append: v"), &slots = tensor(a[3], "kv8_append: slots");
        const int e = elem(k.scalar_type(), "kv8_append");
        on(k, k.scalar_type(), 3, p.dev, "kv8_append: k");
        const int64_t T = k.size(0);
        rows(k, T, p.c.n_kv_heads, p.c.head_dim, k.scalar_type(), p.dev, "kv8_append: k");
        rows(v, T, p.c.n_kv_heads, p.c.head_dim, k.scalar_type(), p.dev, "kv8_append: v");
        flat(slots, at::kLong, T, p.dev, "kv8_append: slots");
        no_grad({&k, &v, &p.ks, &p.vs}, "kv8_append");
        const c10::cuda::CUDAGuard guard(p.dev);
        if (T)
            for (const at::Tensor* t : {&p.k, &p.v, &p.ks, &p.vs}) written(*t);
        status(tsb_kv8_append(&p.c, ptr(k), ptr(v), e, k.stride(0), k.stride(1), v.stride(0), v.stride(1), (const int64_t*) ptr(slots), T,
                              stream_of(p.dev)),
               "kv8_append");
        Py_RETURN_NONE;
    });
}

// (cache, slots, dtype of a tensor or None) -> (k, v)
PyObject* kv8_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        count(n, 3);
        const Pools p = pools(a[0]);
        const at::Tensor& slots = tensor(a[1], "kv8_read: slots");
        on(slots, at::kLong, 1, p.dev, "kv8_read: slots");
        const int64_t T = slots.size(0);
        flat(slots, at::kLong, T, p.dev, "kv8_read: slots");
        no_grad({&p.ks, &p.vs}, "kv8_read");
        const int e = int32(a[2], "kv8_read: dtype");
        const at::ScalarType type = e == 0 ? at::kFloat : e == 1 ? at::kHalf : at::kBFloat16;
        const c10::cuda::CUDAGuard guard(p.dev);
        const auto opt = at::TensorOptions().dtype(type).device(p.dev);
        at::Tensor k = at::empty({T, p.c.n_kv_heads, p.c.head_dim}, opt), v = at::empty({T, p.c.n_kv_heads, p.c.head_dim}, opt);
        status(tsb_kv8_read(&p.c, (const int64_t*) ptr(slots), T, ptr(k), ptr(v), e, stream_of(p.dev)), "kv8_read");
        PyObject* out = PyTuple_New(2);
        if (!out) throw Raised{};
        PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(k));
        PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(v));
        return out;
    });
}

// (cache, q, table, lens, cu_q, max_q or None, window, scale or None, out or None) -> out
PyObject* kv8_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        count(n, 9);
        const Pools p = pools(a[0]);
        const at::Tensor &q = tensor(a[1], "kv8_attention: q"), &table = tensor(a[2], "kv8_attention: table"),
                         &lens = tensor(a[3], "kv8_attention: lens"), cu = maybe(a[4], "kv8_attention: cu_q");
        at::Tensor out = maybe(a[8], "kv8_attention: out");
        tsb_kv8_attn d{};
        d.struct_size = sizeof d;
        d.elem_type = elem(q.scalar_type(), "kv8_attention");
        on(q, q.scalar_type(), 3, p.dev, "kv8_attention: q");
        const int64_t T = q.size(0), heads = q.size(1);
        rows(q, T, heads, p.c.head_dim, q.scalar_type(), p.dev, "kv8_attention: q");
        on(table, at::kInt, 2, p.dev, "kv8_attention: table");
        const int64_t R = table.size(0), width = table.size(1);
        if (width > 1 && table.stride(1) != 1) bad(table, "kv8_attention: table", "contiguous rows");
        flat(lens, at::kInt, R, p.dev, "kv8_attention: lens");
        if (cu.defined()) flat(cu, at::kInt, R + 1, p.dev, "kv8_attention: cu_q");
        need(R <= INT32_MAX && heads <= INT32_MAX && width <= INT32_MAX, "kv8_attention: sizes");
        no_grad({&q, &out, &p.ks, &p.vs}, "kv8_attention");
        const c10::cuda::CUDAGuard guard(p.dev);
        if (out.defined()) rows(out, T, heads, p.c.head_dim, q.scalar_type(), p.dev, "kv8_attention: out"), own_memory(out, "kv8_attention: out"), written(out);
        else out = at::empty({T, heads, p.c.head_dim}, q.options());
        d.n_req = (int32_t) R, d.q_heads = (int32_t) heads, d.table_width = (int32_t) width;
        if (a[5] != Py_None) d.max_q = int32(a[5], "kv8_attention: max_q");
        else d.max_q = cu.defined() ? (int32_t) std::min<int64_t>(T, INT32_MAX) : 1;
        d.window = int32(a[6], "kv8_attention: window");
        d.scale = a[7] == Py_None ? (float) (1.0 / std::sqrt((double) p.c.head_dim)) : (float) number(a[7]);
        d.n_tok = T, d.q_tok = q.stride(0), d.q_head = q.stride(1), d.o_tok = out.stride(0), d.o_head = out.stride(1);
        d.table_stride = R > 1 ? table.stride(0) : width;   // requests may share a row (an expanded table)
        const uint64_t size = tsb_kv8_attention_workspace_bytes(&p.c, &d);
        const at::Tensor ws = bytes(size, p.dev);
        status(tsb_kv8_attention(&p.c, &d, ptr(q), (const int32_t*) ptr(table), (const int32_t*) ptr(lens), (const int32_t*) ptr(cu),
                                 ptr(out), ptr(ws), size, stream_of(p.dev)),
               "kv8_attention");
        return THPVariable_Wrap(out);
    });
}

// (q, k, v, g, beta, state, cu_seqlens, max_len or None, state_idx, state_out, scale or None, qk_norm, eps, out or None)
// -> (out, state_out)
PyObject* gated_delta(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        count(n, 14);
        const at::Tensor &q = tensor(a[0], "gated_delta: q"), &k = tensor(a[1], "gated_delta: k"), &v = tensor(a[2], "gated_delta: v"),
                         &g = tensor(a[3], "gated_delta: g"), &beta = tensor(a[4], "gated_delta: beta"),
                         &state = tensor(a[5], "gated_delta: state"), cu = maybe(a[6], "gated_delta: cu_seqlens"),
                         idx = maybe(a[8], "gated_delta: state_idx");
        const at::Tensor& after = a[9] == Py_None ? state : tensor(a[9], "gated_delta: state_out");
        at::Tensor out = maybe(a[13], "gated_delta: out");
        const c10::Device dev = cuda_of(q, "gated_delta: q");
        const at::ScalarType type = q.scalar_type();
        tsb_delta_desc d{};
        d.struct_size = sizeof d;
        d.elem_type = elem(type, "gated_delta");
        on(q, type, 3, dev, "gated_delta: q");
        on(v, type, 3, dev, "gated_delta: v");
        const int64_t T = q.size(0), hk = q.size(1), dk = q.size(2), hv = v.size(1), dv = v.size(2);
        rows(q, T, hk, dk, type, dev, "gated_delta: q");
        rows(k, T, hk, dk, type, dev, "gated_delta: k");
        rows(v, T, hv, dv, type, dev, "gated_delta: v");
        for (const at::Tensor* t : {&g, &beta}) {
            on(*t, at::kFloat, 2, dev, "gated_delta: g, beta");
            if (t->size(0) != T || t->size(1) != hv || (hv > 1 && t->stride(1) != 1) || (T > 1 && t->stride(0) != g.stride(0)))
                bad(*t, "gated_delta: g, beta", "[tokens, v_heads], rows contiguous and of one stride,");
        }
        on(state, at::kFloat, 4, dev, "gated_delta: state");
        on(after, at::kFloat, 4, dev, "gated_delta: state_out");
        if (state.size(1) != hv || state.size(2) != dk || state.size(3) != dv || !state.is_contiguous())
            bad(state, "gated_delta: state", "contiguous [n_states, v_heads, dim_k, dim_v]");
        if (after.sizes() != state.sizes() || !after.is_contiguous()) bad(after, "gated_delta: state_out", "contiguous, as state,");
        const char *s0 = (const char*) ptr(state), *s1 = (const char*) ptr(after);
        if (s0 != s1 && s0 < s1 + after.nbytes() && s1 < s0 + state.nbytes())
            bad(after, "gated_delta: state_out", "state itself or memory of its own");
        no_grad({&q, &k, &v, &g, &beta, &state, &after, &out}, "gated_delta");
        const int64_t max_len = a[7] == Py_None ? T : integer(a[7]), slots = state.size(0);
        int64_t B;
        if (cu.defined()) {
            on(cu, at::kInt, 1, dev, "gated_delta: cu_seqlens");
            B = cu.size(0) - 1;
            need(B >= 0, "gated_delta: cu_seqlens needs its first bound");
            flat(cu, at::kInt, B + 1, dev, "gated_delta: cu_seqlens");
        } else {
            B = max_len > 0 ? T / max_len : 0;
            if (B * max_len != T) refuse("gated_delta: " + std::to_string(T) + " tokens are not sequences of " + std::to_string(max_len));
        }
        if (idx.defined()) flat(idx, at::kInt, B, dev, "gated_delta: state_idx");
        else need(slots >= B, "gated_delta: a state for every sequence");
        need(max_len >= 0 && max_len <= INT32_MAX && B <= INT32_MAX && slots <= INT32_MAX && hv <= INT32_MAX && dv <= INT32_MAX, "gated_delta: sizes");
        const c10::cuda::CUDAGuard guard(dev);
        if (out.defined()) rows(out, T, hv, dv, type, dev, "gated_delta: out"), own_memory(out, "gated_delta: out"), written(out);
        else out = at::empty({T, hv, dv}, q.options());
        d.n_seq = (int32_t) B, d.max_len = (int32_t) max_len, d.k_heads = (int32_t) hk, d.v_heads = (int32_t) hv;
        d.dim_k = (int32_t) dk, d.dim_v = (int32_t) dv, d.n_states = (int32_t) slots;
        const int norm = PyObject_IsTrue(a[11]);
        if (norm < 0) throw Raised{};
        d.qk_norm = norm;
        d.scale = a[10] == Py_None ? (float) (1.0 / std::sqrt((double) std::max<int64_t>(dk, 1))) : (float) number(a[10]);
        d.eps = (float) number(a[12]);
        d.n_tok = T, d.q_tok = q.stride(0), d.q_head = q.stride(1), d.k_tok = k.stride(0), d.k_head = k.stride(1);
        d.v_tok = v.stride(0), d.v_head = v.stride(1), d.o_tok = out.stride(0), d.o_head = out.stride(1), d.gb_tok = g.stride(0);
        written(after);
        const uint64_t size = tsb_gated_delta_workspace_bytes(&d);
        const at::Tensor ws = bytes(size, dev);
        status(tsb_gated_delta(&d, ptr(q), ptr(k), ptr(v), (const float*) ptr(g), (const float*) ptr(beta), (const float*) ptr(state),
                               (float*) ptr(after), (const int32_t*) ptr(idx), (const int32_t*) ptr(cu), ptr(out), ptr(ws), size, stream_of(dev)),
               "gated_delta");
        PyObject* res = PyTuple_New(2);
        if (!res) throw Raised{};
        PyTuple_SET_ITEM(res, 0, THPVariable_Wrap(out));
        PyTuple_SET_ITEM(res, 1, THPVariable_Wrap(after));
        return res;
    });
}

PyMethodDef g_methods[] = {
    {"init", (PyCFunction) init, METH_O, nullptr},
    {"block_tables", (PyCFunction) (void (*)()) block_tables, METH_FASTCALL, nullptr},
    {"kv8_append", (PyCFunction) (void (*)()) kv8_append, METH_FASTCALL, nullptr},
    {"kv8_read", (PyCFunction) (void (*)()) kv8_read, METH_FASTCALL, nullptr},
    {"kv8_attention", (PyCFunction) (void (*)()) kv8_attention, METH_FASTCALL, nullptr},
    {"gated_delta", (PyCFunction) (void (*)()) gated_delta, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" PyMODINIT_FUNC PyInit__serving() { return PyModule_Create(&g_module); }
