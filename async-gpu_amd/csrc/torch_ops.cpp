// The operators of ops.py in native code: argument checks, output allocation, context lookup and the call through the
// C ABI.  A decode-sized kernel runs 2 - 6 us; the same steps through ctypes took 9 us of host time per call, so a
// program that composes operators waited for the interpreter and not for the GPU.
//
// The library stays independent of torch: this module resolves the entry points at run time in the copy of
// libagpu_hip.so that _lib.py has loaded (bind()), and torch is only the allocator of the outputs, as in ops.py.
#include <Python.h>

#include <dlfcn.h>

#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <string>
#include <vector>

#include "../../include/agpu.h"
#include "paged.h"

namespace {

// ---- the library, its errors and its contexts ---------------------------------------------

#define AGPU_OPS(X)                                                                                                          \
    X(agpu_int4_linear) X(agpu_ln_int4_linear) X(agpu_layer_norm) X(agpu_add_layer_norm_dual) X(agpu_gelu)                    \
    X(agpu_add_inplace) X(agpu_bias_add) X(agpu_softmax_rows) X(agpu_embedding) X(agpu_argmax_rows) X(agpu_split_qkv)         \
    X(agpu_concat_heads) X(agpu_attention) X(agpu_kv_append) X(agpu_gemm_f32) X(agpu_last_error_string)          \
    X(agpu_paged_plan) X(agpu_paged_kv_append) X(agpu_paged_attention) X(agpu_paged_attention_shared)                        \
    X(agpu_paged_attention_weights) X(agpu_paged_evict) X(agpu_paged_trim) X(agpu_sample)
struct Lib {
#define X(f) decltype(&f) f##_ = nullptr;
    AGPU_OPS(X)
#undef X
} lib;

PyObject *g_error = nullptr, *g_context = nullptr, *g_ptr = nullptr;  // AgpuError, ops.context, _lib.ptr

// One entry per (device, stream) that has been used; the Context object is kept alive by ops.py.
struct Ctx {
    int device;
    hipStream_t stream;
    agpu_ctx *handle;
};
std::vector<Ctx> g_ctx;  // under the GIL

struct PyFail {};  // a Python error is set

[[noreturn]] void shape_err(const std::string &expected, const std::string &actual) {
    const std::string m = "shape mismatch: expected " + expected + ", got " + actual;
    PyObject *e = PyObject_CallFunction(g_error, "is", AGPU_ERR_SHAPE_MISMATCH, m.c_str());
    if (e) PyErr_SetObject(g_error, e);
    Py_XDECREF(e);
    throw PyFail();
}

std::string str(int64_t v) { return std::to_string(v); }
std::string str(at::IntArrayRef s) {
    std::string r = "(";
    for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + str(s[i]);
    return r + (s.size() == 1 ? ",)" : ")");
}

agpu_ctx *context(const at::Tensor &t) {
    const int device = t.device().has_index() ? t.device().index() : 0;
    const hipStream_t stream = c10::hip::getCurrentHIPStream(device).stream();
    for (size_t i = 0; i < g_ctx.size(); ++i)
        if (g_ctx[i].device == device && g_ctx[i].stream == stream) {
            const Ctx c = g_ctx[i];
            if (i) std::swap(g_ctx[i], g_ctx[0]);
            return c.handle;
        }
    PyObject *c = PyObject_CallFunction(g_context, "i", device);
    PyObject *h = c ? PyObject_GetAttrString(c, "handle") : nullptr;
    PyObject *v = h ? PyObject_GetAttrString(h, "value") : nullptr;
    void *p = v ? PyLong_AsVoidPtr(v) : nullptr;
    Py_XDECREF(v);
    Py_XDECREF(h);
    Py_XDECREF(c);
    if (PyErr_Occurred()) throw PyFail();
    g_ctx.insert(g_ctx.begin(), Ctx{device, stream, static_cast<agpu_ctx *>(p)});
    return static_cast<agpu_ctx *>(p);
}

template <class F, class... A>
void call(F fn, agpu_ctx *c, A... a) {
    PyThreadState *s = PyEval_SaveThread();
    const int32_t rc = fn(c, a...);
    PyEval_RestoreThread(s);
    if (rc == AGPU_OK) return;
    PyObject *e = PyObject_CallFunction(g_error, "is", rc, lib.agpu_last_error_string_(c));
    if (e) PyErr_SetObject(g_error, e);
    Py_XDECREF(e);
    throw PyFail();
}

// ---- arguments and results ----------------------------------------------------------------

const at::Tensor &tensor(PyObject *o) {
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "expects a torch tensor, got %s", Py_TYPE(o)->tp_name);
        throw PyFail();
    }
    return THPVariable_Unpack(o);
}

const at::Tensor &f32(PyObject *o) {
    const at::Tensor &t = tensor(o);
    if (t.scalar_type() != at::kFloat || !t.is_cuda() || !t.is_contiguous()) {
        PyErr_SetString(PyExc_AssertionError, "expects contiguous fp32 device tensors");
        throw PyFail();
    }
    return t;
}

// What _lib.ptr takes: a tensor, an address or None, and anything else through _lib.ptr itself.  A tensor that is written to is
// asked for a pointer to write through: one that shares its memory with a lazy clone gets memory of its own first.
void *address(PyObject *o, bool written = false) {
    if (o == Py_None) return nullptr;
    if (THPVariable_Check(o)) {
        const at::Tensor &t = THPVariable_Unpack(o);
        return written ? t.mutable_data_ptr() : const_cast<void *>(t.const_data_ptr());
    }
    if (PyLong_Check(o)) {
        void *p = PyLong_AsVoidPtr(o);
        if (PyErr_Occurred()) throw PyFail();
        return p;
    }
    PyObject *r = PyObject_CallFunctionObjArgs(g_ptr, o, nullptr);
    if (!r) throw PyFail();
    void *p = r == Py_None ? nullptr : PyLong_AsVoidPtr(r);
    Py_DECREF(r);
    if (PyErr_Occurred()) throw PyFail();
    return p;
}
const float *fp(PyObject *o) { return static_cast<const float *>(address(o)); }
const float *data(const at::Tensor &t) { return static_cast<const float *>(t.const_data_ptr()); }
float *written(const at::Tensor &t) { return static_cast<float *>(t.mutable_data_ptr()); }

int64_t integer(PyObject *o) {
    PyObject *n = PyNumber_Index(o);
    if (!n) throw PyFail();
    const long long v = PyLong_AsLongLong(n);
    Py_DECREF(n);
    if (v == -1 && PyErr_Occurred()) throw PyFail();
    return v;
}
// An argument of 32 bits of the C ABI; what does not fit is an error and not cut off.
int32_t i32(int64_t v) {
    if (v < INT32_MIN || v > INT32_MAX) {
        PyErr_Format(PyExc_OverflowError, "%lld does not fit the library's 32-bit arguments", (long long)v);
        throw PyFail();
    }
    return (int32_t)v;
}
int32_t i32(PyObject *o) { return i32(integer(o)); }
float real(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw PyFail();
    return (float)v;
}
int64_t last(const at::Tensor &t) {
    if (t.dim() == 0) shape_err("at least one dimension", "()");
    return t.size(-1);
}
void rank(const at::Tensor &t, int64_t dims, const char *what) {
    if (t.dim() != dims) shape_err(what, str(t.sizes()));
}

at::Tensor empty(at::IntArrayRef sizes, const at::Tensor &like, at::ScalarType type = at::kFloat) {
    return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}
PyObject *wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }
PyObject *same(PyObject *o) {
    Py_INCREF(o);
    return o;
}

// ---- the operators: positional arguments in the order of ops.py ----------------------------

// x, packed, scales, bias, residual, group, flags, ln, out
PyObject *int4_linear(PyObject *const *a) {
    const at::Tensor &x = tensor(a[0]);
    const int64_t K = last(x);
    int64_t kp, N;
    if (THPVariable_Check(a[1])) {
        const at::Tensor &packed = THPVariable_Unpack(a[1]);
        rank(packed, 2, "packed weights [K/8, N]");
        kp = packed.size(0), N = packed.size(1);
    } else {
        PyObject *s = PyObject_GetAttrString(a[1], "shape");
        long long n0 = 0, n1 = 0;
        const bool ok = s && PyArg_ParseTuple(s, "LL", &n0, &n1);
        Py_XDECREF(s);
        if (!ok) throw PyFail();
        kp = n0, N = n1;
    }
    if (K != kp * 8) shape_err("last dim = " + str(kp * 8), "last dim = " + str(K));
    f32(a[0]);
    const int64_t M = x.numel() ? x.numel() / K : 0;
    agpu_ctx *c = context(x);
    PyObject *out = a[8];
    at::Tensor y;
    if (out == Py_None) {
        if (x.dim() <= 2) {
            y = empty({M, N}, x);
        } else {
            std::vector<int64_t> s = x.sizes().vec();
            s.back() = N;
            y = empty(s, x);
        }
    }
    float *yp = out == Py_None ? written(y) : static_cast<float *>(address(out, true));
    const auto *pk = static_cast<const uint32_t *>(address(a[1]));
    const int32_t m = i32(M), n = i32(N), k = i32(K), group = i32(a[5]);
    const uint32_t flags = (uint32_t)integer(a[6]);
    if (a[7] == Py_None) {
        call(lib.agpu_int4_linear_, c, data(x), pk, fp(a[2]), fp(a[3]), fp(a[4]), yp, m, n, k, group, flags);
    } else {
        PyObject *ln = PySequence_Fast(a[7], "ln is (gamma, beta, eps)");
        if (!ln) throw PyFail();
        struct Drop {
            PyObject *o;
            ~Drop() { Py_DECREF(o); }
        } drop{ln};
        if (PySequence_Fast_GET_SIZE(ln) < 3) {
            PyErr_SetString(PyExc_IndexError, "ln is (gamma, beta, eps)");
            throw PyFail();
        }
        PyObject **l = PySequence_Fast_ITEMS(ln);
        call(lib.agpu_ln_int4_linear_, c, data(x), fp(l[0]), fp(l[1]), real(l[2]), pk, fp(a[2]), fp(a[3]), fp(a[4]), yp, m, n, k, group,
             flags);
    }
    if (out == Py_None) return wrap(std::move(y));
    if (x.dim() <= 2) return same(out);
    std::vector<int64_t> s = x.sizes().vec();
    s.back() = N;
    return wrap(tensor(out).reshape(s));
}

// x, gamma, beta, eps
PyObject *layer_norm(PyObject *const *a) {
    const at::Tensor &x = tensor(a[0]), &g = tensor(a[1]), &b = tensor(a[2]);
    const int64_t d = last(x);
    if (g.numel() != d || b.numel() != d) shape_err("gamma/beta of " + str(d), str(g.numel()) + "/" + str(b.numel()));
    f32(a[0]);
    at::Tensor y = empty(x.sizes(), x);
    call(lib.agpu_layer_norm_, context(x), data(x), data(g), data(b), written(y), i32(d ? x.numel() / d : 0), i32(d), real(a[3]));
    return wrap(std::move(y));
}

// a, b, gamma, beta, eps, want_sum
PyObject *add_layer_norm_dual(PyObject *const *a) {
    const at::Tensor &x = tensor(a[0]), &r = tensor(a[1]);
    if (x.sizes() != r.sizes()) shape_err(str(x.sizes()), str(r.sizes()));
    f32(a[0]);
    f32(a[1]);
    const int64_t d = last(x);
    const int sum = PyObject_IsTrue(a[5]);
    if (sum < 0) throw PyFail();
    at::Tensor s, n = empty(x.sizes(), x);
    if (sum) s = empty(x.sizes(), x);
    call(lib.agpu_add_layer_norm_dual_, context(x), data(x), data(r), fp(a[2]), fp(a[3]), sum ? written(s) : nullptr, written(n),
         i32(d ? x.numel() / d : 0), i32(d), real(a[4]));
    if (!sum) return wrap(std::move(n));
    return Py_BuildValue("(NN)", wrap(std::move(s)), wrap(std::move(n)));
}

// x, mode
PyObject *gelu(PyObject *const *a) {
    const at::Tensor &x = f32(a[0]);
    at::Tensor y = empty(x.sizes(), x);
    call(lib.agpu_gelu_, context(x), data(x), written(y), (size_t)x.numel(), i32(a[1]));
    return wrap(std::move(y));
}

// a, b
PyObject *add_inplace(PyObject *const *a) {
    const at::Tensor &x = tensor(a[0]), &r = tensor(a[1]);
    if (x.numel() != r.numel()) shape_err(str(x.sizes()), str(r.sizes()));
    f32(a[0]);
    f32(a[1]);
    float *xp = written(x);
    call(lib.agpu_add_inplace_, context(x), xp, data(r), (size_t)x.numel());
    return same(a[0]);
}

// data, bias
PyObject *bias_add(PyObject *const *a) {
    const at::Tensor &x = tensor(a[0]), &b = tensor(a[1]);
    const int64_t n = last(x);
    if (b.numel() != n) shape_err("bias of " + str(n), str(b.numel()));
    f32(a[0]);
    float *xp = written(x);
    call(lib.agpu_bias_add_, context(x), xp, data(b), i32(n ? x.numel() / n : 0), i32(n));
    return same(a[0]);
}

// x
PyObject *softmax_rows(PyObject *const *a) {
    const at::Tensor &x = f32(a[0]);
    const int64_t n = last(x);
    at::Tensor y = empty(x.sizes(), x);
    call(lib.agpu_softmax_rows_, context(x), data(x), written(y), i32(n ? x.numel() / n : 0), i32(n));
    return wrap(std::move(y));
}

// tokens, wte, wpe, pos_offset
PyObject *embedding(PyObject *const *a) {
    const at::Tensor &tokens = tensor(a[0]), &wte = tensor(a[1]);
    rank(wte, 2, "wte [vocab, d]");
    const int64_t seq = tokens.numel(), d = wte.size(1);
    at::Tensor out = empty({seq, d}, wte);
    call(lib.agpu_embedding_, context(wte), static_cast<const uint32_t *>(address(a[0])), data(wte), fp(a[2]), written(out), i32(seq), i32(d),
         i32(a[3]));
    return wrap(std::move(out));
}

// x, last_index
PyObject *argmax_rows(PyObject *const *a) {
    const at::Tensor &x = f32(a[0]);
    const int64_t cols = last(x), rows = cols ? x.numel() / cols : 0;
    at::Tensor idx = empty({rows}, x, at::kInt);
    call(lib.agpu_argmax_rows_, context(x), data(x), static_cast<uint32_t *>(idx.data_ptr()), i32(rows), i32(cols), i32(a[1]));
    return wrap(std::move(idx));
}

// qkv, n_heads, d_head
PyObject *split_qkv(PyObject *const *a) {
    const at::Tensor &x = tensor(a[0]);
    const int64_t heads = integer(a[1]), dh = integer(a[2]);
    if (x.dim() != 2 || x.size(1) != 3 * heads * dh) shape_err("[seq, " + str(3 * heads * dh) + "]", str(x.sizes()));
    f32(a[0]);
    const int64_t seq = x.size(0);
    std::array<at::Tensor, 3> t;
    for (at::Tensor &o : t) o = empty({heads, seq, dh}, x);
    call(lib.agpu_split_qkv_, context(x), data(x), written(t[0]), written(t[1]), written(t[2]), i32(seq), i32(heads), i32(dh));
    return Py_BuildValue("(NNN)", wrap(std::move(t[0])), wrap(std::move(t[1])), wrap(std::move(t[2])));
}

// x
PyObject *concat_heads(PyObject *const *a) {
    const at::Tensor &x = f32(a[0]);
    rank(x, 3, "[heads, seq, d_head]");
    const int64_t heads = x.size(0), seq = x.size(1), dh = x.size(2);
    at::Tensor out = empty({seq, heads * dh}, x);
    call(lib.agpu_concat_heads_, context(x), data(x), written(out), i32(seq), i32(heads), i32(dh));
    return wrap(std::move(out));
}

void attend(PyObject *q, PyObject *k, PyObject *v, at::Tensor &o, int64_t heads, int64_t q_len, int64_t kv_len, int64_t q_offset,
            int64_t kv_stride, int64_t dh, int causal) {
    f32(k);
    f32(v);
    const at::Tensor &x = f32(q);
    o = empty(x.sizes(), x);
    call(lib.agpu_attention_, context(x), data(x), data(tensor(k)), data(tensor(v)), written(o), i32(heads), i32(q_len), i32(kv_len),
         i32(q_offset), i32(kv_stride), i32(dh), (int32_t)causal);
}

// q, k, v, kv_len, q_offset, causal
PyObject *attention(PyObject *const *a) {
    const at::Tensor &q = tensor(a[0]), &k = tensor(a[1]);
    rank(q, 3, "q [heads, q_len, d_head]");
    if (k.dim() < 2) shape_err("k [heads, kv_stride, d_head]", str(k.sizes()));
    const int causal = PyObject_IsTrue(a[5]);
    if (causal < 0) throw PyFail();
    at::Tensor o;
    attend(a[0], a[1], a[2], o, q.size(0), q.size(1), a[3] == Py_None ? k.size(1) : integer(a[3]), integer(a[4]), k.size(1), q.size(2), causal);
    return wrap(std::move(o));
}

// q, k, v, seq_len, n_heads, d_head
PyObject *multi_head_flash_attention(PyObject *const *a) {
    const at::Tensor &q = tensor(a[0]), &k = tensor(a[1]), &v = tensor(a[2]);
    const int64_t seq = integer(a[3]), heads = integer(a[4]), dh = integer(a[5]);
    if (q.numel() != heads * seq * dh || k.sizes() != q.sizes() || v.sizes() != q.sizes())
        shape_err("q, k, v of " + str(heads * seq) + " x " + str(dh), str(q.sizes()) + ", " + str(k.sizes()) + ", " + str(v.sizes()));
    at::Tensor o;
    attend(a[0], a[1], a[2], o, heads, seq, seq, 0, seq, dh, 1);
    return wrap(std::move(o));
}

// src, cache, write_pos
PyObject *kv_append(PyObject *const *a) {
    const at::Tensor &src = f32(a[0]), &cache = f32(a[1]);
    rank(src, 3, "src [heads, rows, d_head]");
    if (cache.dim() < 2) shape_err("cache [heads, positions, d_head]", str(cache.sizes()));
    float *cp = written(cache);
    call(lib.agpu_kv_append_, context(src), data(src), cp, i32(src.size(0)), i32(src.size(1)), i32(cache.size(1)), i32(a[2]),
         i32(src.size(2)));
    return same(a[1]);
}

// a, b
PyObject *gemm_f32(PyObject *const *a) {
    const at::Tensor &x = tensor(a[0]), &b = tensor(a[1]);
    rank(x, 2, "A [M, K]");
    if (b.dim() != 2 || b.size(0) != x.size(1)) shape_err("B with " + str(x.size(1)) + " rows", str(b.sizes()));
    f32(a[0]);
    f32(a[1]);
    at::Tensor c = empty({x.size(0), b.size(1)}, x);
    call(lib.agpu_gemm_f32_, context(x), data(x), data(b), written(c), i32(x.size(0)), i32(b.size(1)), i32(x.size(1)));
    return wrap(std::move(c));
}

// ---- several requests over a cache in pages --------------------------------------------------

// A tensor of a given type and rank; sizes of -1 are any.
const at::Tensor &typed(PyObject *o, at::ScalarType type, std::initializer_list<int64_t> sizes, const char *what) {
    const at::Tensor &t = tensor(o);
    bool fits = t.dim() == (int64_t)sizes.size();
    int64_t d = 0;
    for (const int64_t s : sizes) fits = fits && (s < 0 || t.size(d) == s), ++d;
    if (!fits) shape_err(what, str(t.sizes()));
    if (t.scalar_type() != type) shape_err(std::string(what) + " of " + c10::toString(type), c10::toString(t.scalar_type()));
    return t;
}
const at::Tensor &ints(PyObject *o, std::initializer_list<int64_t> sizes, const char *what) {
    const at::Tensor &t = typed(o, at::kInt, sizes, what);
    if (!t.is_contiguous()) shape_err(std::string("contiguous ") + what, "strides " + str(t.strides()));
    return t;
}
// All on one GPU: the one that the operator runs on.
template <class... T>
void together(const at::Tensor &first, const T &...others) {
    if (!first.is_cuda() || !(... && (others.device() == first.device()))) {
        PyErr_SetString(PyExc_AssertionError, "expects device tensors, all on one GPU");
        throw PyFail();
    }
}
const int32_t *ip(const at::Tensor &t) { return static_cast<const int32_t *>(t.const_data_ptr()); }
int32_t *iw(const at::Tensor &t) { return static_cast<int32_t *>(t.mutable_data_ptr()); }

// K or V in pages: [n_pages, n_kv_heads, page_size, 64], a page contiguous, pages anywhere
const at::Tensor &pages(PyObject *o, const char *what) {
    const at::Tensor &t = tensor(o);
    rank(t, 4, what);
    const auto ty = t.scalar_type();
    if (ty != at::kFloat && ty != at::kHalf && ty != at::kBFloat16) shape_err("a cache of float32, float16 or bfloat16", c10::toString(ty));
    const int64_t heads = t.size(1), size = t.size(2), dh = t.size(3);
    if ((dh > 1 && t.stride(3) != 1) || (size > 1 && t.stride(2) != dh) || (heads > 1 && t.stride(1) != size * dh))
        shape_err("contiguous pages [n_kv_heads, page_size, d_head]", "strides " + str(t.strides()));
    return t;
}
int32_t cache_type(const at::Tensor &t) {
    return t.scalar_type() == at::kFloat ? AGPU_CACHE_F32 : t.scalar_type() == at::kHalf ? AGPU_CACHE_F16 : AGPU_CACHE_BF16;
}
void same_cache(const at::Tensor &k, const at::Tensor &v) {
    if (k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type()) shape_err("k_cache and v_cache alike", str(k.sizes()) + ", " + str(v.sizes()));
}
int64_t page_stride(const at::Tensor &t) { return t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2) * t.size(3); }
// Rows [tokens, heads, d_head] at any two strides
const at::Tensor &rows(PyObject *o, int64_t tokens, int64_t heads, int64_t dh, const char *what) {
    const at::Tensor &t = typed(o, at::kFloat, {tokens, heads, dh}, what);
    if (t.size(2) > 1 && t.stride(2) != 1) shape_err(std::string(what) + " with contiguous rows of a head", "strides " + str(t.strides()));
    return t;
}

// Vectors in one allocation, 16 bytes aligned each: an allocation costs the host more than the rest of a small call.
template <size_t N>
std::array<at::Tensor, N> ints_in_one(const int64_t (&sizes)[N], const at::Tensor &like) {
    auto room = [](int64_t n) { return (n + 3) & ~(int64_t)3; };
    int64_t all = 0;
    for (int64_t n : sizes) all += room(n);
    const at::Tensor whole = empty({all}, like, at::kInt);
    std::array<at::Tensor, N> t;
    int64_t at = 0;
    for (size_t i = 0; i < N; at += room(sizes[i++])) {
        auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(), whole.dtype());
        impl->set_storage_offset(at);
        impl->set_sizes_contiguous(at::IntArrayRef(&sizes[i], 1));
        t[i] = at::Tensor(std::move(impl));
    }
    return t;
}

// cached_lens, new_lens, block_tables, free_pages, n_free, page_size, max_tokens
PyObject *paged_plan(PyObject *const *a) {
    const at::Tensor &tables = ints(a[2], {-1, -1}, "block_tables [batch, width]");
    const int64_t batch = tables.size(0);
    const at::Tensor &cached = ints(a[0], {batch}, "cached_lens [batch]"), &fresh = ints(a[1], {batch}, "new_lens [batch]");
    const at::Tensor &stack = ints(a[3], {-1}, "free_pages [stack_size]"), &n_free = ints(a[4], {1}, "n_free [1]");
    const int64_t max_tokens = integer(a[6]);
    if (max_tokens < 0) shape_err("max_tokens >= 0", str(max_tokens));
    together(tables, cached, fresh, stack, n_free);
    std::array<at::Tensor, 5> t = ints_in_one<5>({batch, batch + 1, max_tokens, max_tokens, 1}, tables);
    int32_t *const tp = iw(tables), *const sp = iw(stack);
    call(lib.agpu_paged_plan_, context(tables), ip(cached), ip(fresh), tp, sp, ip(n_free), iw(t[0]), iw(t[1]), iw(t[2]), iw(t[3]), iw(t[4]), i32(batch),
         i32(tables.size(1)), i32(stack.numel()), i32(a[5]), i32(max_tokens));
    return Py_BuildValue("(NNNNN)", wrap(std::move(t[0])), wrap(std::move(t[1])), wrap(std::move(t[2])), wrap(std::move(t[3])), wrap(std::move(t[4])));
}

// k, v, k_cache, v_cache, slots
PyObject *paged_kv_append(PyObject *const *a) {
    const at::Tensor &kc = pages(a[2], "k_cache [n_pages, n_kv_heads, page_size, d_head]"), &vc = pages(a[3], "v_cache [n_pages, n_kv_heads, page_size, d_head]");
    same_cache(kc, vc);
    const at::Tensor &slots = ints(a[4], {-1}, "slots [tokens]");
    const int64_t tokens = slots.size(0), heads = kc.size(1), dh = kc.size(3);
    const at::Tensor &k = rows(a[0], tokens, heads, dh, "k [tokens, n_kv_heads, d_head]"), &v = rows(a[1], tokens, heads, dh, "v [tokens, n_kv_heads, d_head]");
    together(kc, vc, slots, k, v);
    void *const kp = kc.mutable_data_ptr(), *const vp = vc.mutable_data_ptr();
    call(lib.agpu_paged_kv_append_, context(kc), data(k), data(v), k.stride(0), k.stride(1), v.stride(0), v.stride(1), kp, vp, page_stride(kc), page_stride(vc),
         ip(slots), i32(tokens), i32(heads), i32(kc.size(0)), i32(kc.size(2)), i32(dh), cache_type(kc));
    return Py_BuildValue("(OO)", a[2], a[3]);
}

// Whether two tensors have memory in common, and not only the storage they lie in: caches, their weights and rows may be parts of one arena.  (A lazy clone is of another storage.)
paged::Pieces memory(const at::Tensor &t) {
    const int64_t size = t.element_size();
    const void *const at = t.const_data_ptr();
    if (t.numel() == 0) return paged::Pieces::one(at, 0);
    if (t.dim() == 3 && t.scalar_type() == at::kFloat && t.size(2) == 64 && t.stride(2) == 1) return paged::Pieces::rows(static_cast<const float *>(at), t.size(0), t.size(1), t.stride(0), t.stride(1));
    return paged::Pieces::pages(at, t.size(0), t.stride(0) * size, t.numel() / t.size(0) * size);  // (each contiguous)
}
bool share_memory(const at::Tensor &a, const at::Tensor &b) { return a.is_alias_of(b) && paged::share(memory(a), memory(b)); }

// What paged_attention and the operators like it have in common: q, k_cache, v_cache; then block_tables, kv_lens, query_start; out behind them.
struct Attends {
    const at::Tensor &kc, &vc, &q, &tables, &lens, &start;
    const bool ragged, given;
    const int64_t tokens, heads, batch;
    Attends(PyObject *q_, PyObject *k_, PyObject *v_, PyObject *tables_, PyObject *lens_, PyObject *start_, PyObject *out)
        : kc(pages(k_, "k_cache [n_pages, n_kv_heads, page_size, d_head]")), vc(pages(v_, "v_cache [n_pages, n_kv_heads, page_size, d_head]")),
          q(rows(q_, -1, -1, kc.size(3), "q [tokens, n_heads, d_head]")), tables(ints(tables_, {-1, -1}, "block_tables [batch, width]")),
          lens(ints(lens_, {tables.size(0)}, "kv_lens [batch]")), start(start_ != Py_None ? ints(start_, {tables.size(0) + 1}, "query_start [batch + 1]") : lens),
          ragged(start_ != Py_None), given(out != Py_None), tokens(q.size(0)), heads(q.size(1)), batch(tables.size(0)) {
        same_cache(kc, vc);
        if (!ragged && tokens != batch) shape_err("a row for each of " + str(batch) + " requests without query_start", str(tokens));
        if (given) {
            const at::Tensor &o = typed(out, at::kFloat, {tokens, heads, q.size(2)}, "out [tokens, n_heads, d_head]");
            if (!o.is_contiguous()) shape_err("contiguous out", "strides " + str(o.strides()));
            for (const at::Tensor *t : {&q, &kc, &vc})
                if (share_memory(o, *t)) shape_err("out with memory of its own", "that of an input");
        }
    }
    // (after what else there is to check of shapes)
    template <class... T>
    at::Tensor out(PyObject *o, const T &...others) const {
        together(q, kc, vc, tables, lens, start, others...);
        if (given) together(q, tensor(o));
        return given ? tensor(o) : empty(q.sizes(), q);
    }
    const int32_t *starts() const { return ragged ? ip(start) : nullptr; }
};

// q, k_cache, v_cache, block_tables, kv_lens, query_start, window, sinks, out
PyObject *paged_attention(PyObject *const *a) {
    const Attends c(a[0], a[1], a[2], a[3], a[4], a[5], a[8]);
    at::Tensor o = c.out(a[8]);
    float *const op = written(o);
    call(lib.agpu_paged_attention_, context(c.q), data(c.q), c.q.stride(0), c.q.stride(1), c.kc.const_data_ptr(), c.vc.const_data_ptr(), page_stride(c.kc), page_stride(c.vc), ip(c.tables),
         ip(c.lens), c.starts(), op, i32(c.tokens), i32(c.batch), i32(c.heads), i32(c.kc.size(1)), i32(c.kc.size(0)), i32(c.kc.size(2)), i32(c.tables.size(1)), i32(a[6]), i32(a[7]),
         i32(c.q.size(2)), cache_type(c.kc));
    return c.given ? same(a[8]) : wrap(std::move(o));
}

// What each key of a cache was given: [n_pages, n_kv_heads, page_size], a page contiguous, pages anywhere
const at::Tensor &weights_of(PyObject *o, const at::Tensor &cache) {
    const int64_t heads = cache.size(1), size = cache.size(2);
    const at::Tensor &t = typed(o, at::kFloat, {cache.size(0), heads, size}, "weights [n_pages, n_kv_heads, page_size]");
    if ((size > 1 && t.stride(2) != 1) || (heads > 1 && t.stride(1) != size)) shape_err("contiguous pages of weights [n_kv_heads, page_size]", "strides " + str(t.strides()));
    return t;
}
int64_t weights_stride(const at::Tensor &t) { return t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2); }

// q, k_cache, v_cache, prefix_tables, prefix_lens, prefix_of, block_tables, kv_lens, query_start, window, sinks, out
PyObject *paged_attention_shared(PyObject *const *a) {
    const Attends c(a[0], a[1], a[2], a[6], a[7], a[8], a[11]);
    const at::Tensor &prefixes = ints(a[3], {-1, -1}, "prefix_tables [n_prefix, width]");
    const at::Tensor &lens = ints(a[4], {prefixes.size(0)}, "prefix_lens [n_prefix]"), &of = ints(a[5], {c.batch}, "prefix_of [batch]");
    at::Tensor o = c.out(a[11], prefixes, lens, of);
    float *const op = written(o);
    call(lib.agpu_paged_attention_shared_, context(c.q), data(c.q), c.q.stride(0), c.q.stride(1), c.kc.const_data_ptr(), c.vc.const_data_ptr(), page_stride(c.kc), page_stride(c.vc),
         ip(prefixes), ip(lens), ip(of), ip(c.tables), ip(c.lens), c.starts(), op, i32(c.tokens), i32(c.batch), i32(c.heads), i32(c.kc.size(1)), i32(c.kc.size(0)), i32(c.kc.size(2)),
         i32(prefixes.size(0)), i32(prefixes.size(1)), i32(c.tables.size(1)), i32(a[9]), i32(a[10]), i32(c.q.size(2)), cache_type(c.kc));
    return c.given ? same(a[11]) : wrap(std::move(o));
}

// q, k_cache, v_cache, weights, block_tables, kv_lens, query_start, window, sinks, out
PyObject *paged_attention_weights(PyObject *const *a) {
    const Attends c(a[0], a[1], a[2], a[4], a[5], a[6], a[9]);
    const at::Tensor &w = weights_of(a[3], c.kc);
    for (const at::Tensor *t : {&c.q, &c.kc, &c.vc})
        if (share_memory(w, *t)) shape_err("weights with memory of their own", "that of another argument");
    if (c.given && share_memory(w, tensor(a[9]))) shape_err("weights with memory of their own", "that of another argument");
    at::Tensor o = c.out(a[9], w);
    float *const op = written(o), *const wp = written(w);
    call(lib.agpu_paged_attention_weights_, context(c.q), data(c.q), c.q.stride(0), c.q.stride(1), c.kc.const_data_ptr(), c.vc.const_data_ptr(), page_stride(c.kc), page_stride(c.vc), wp,
         weights_stride(w), ip(c.tables), ip(c.lens), c.starts(), op, i32(c.tokens), i32(c.batch), i32(c.heads), i32(c.kc.size(1)), i32(c.kc.size(0)), i32(c.kc.size(2)),
         i32(c.tables.size(1)), i32(a[7]), i32(a[8]), i32(c.q.size(2)), cache_type(c.kc));
    PyObject *const first = c.given ? same(a[9]) : wrap(std::move(o));
    return Py_BuildValue("(NO)", first, a[3]);
}

// k_cache, v_cache, weights, block_tables, kv_lens, limit, keep, recent, sinks
PyObject *paged_evict(PyObject *const *a) {
    const at::Tensor &kc = pages(a[0], "k_cache [n_pages, n_kv_heads, page_size, d_head]"), &vc = pages(a[1], "v_cache [n_pages, n_kv_heads, page_size, d_head]");
    same_cache(kc, vc);
    const at::Tensor &w = weights_of(a[2], kc), &tables = ints(a[3], {-1, -1}, "block_tables [batch, width]"), &lens = ints(a[4], {tables.size(0)}, "kv_lens [batch]");
    for (const at::Tensor *t : {&kc, &vc})
        if (share_memory(w, *t)) shape_err("weights with memory of their own", "that of a cache");
    if (share_memory(kc, vc) && (kc.const_data_ptr() != vc.const_data_ptr() || page_stride(kc) != page_stride(vc))) shape_err("k_cache and v_cache apart, or the same", "caches that share memory");
    together(kc, vc, w, tables, lens);
    const int32_t limit = i32(a[5]), keep = i32(a[6]), recent = i32(a[7]), sinks = i32(a[8]);
    void *const kp = kc.mutable_data_ptr(), *const vp = vc.mutable_data_ptr();
    float *const wp = written(w);
    call(lib.agpu_paged_evict_, context(kc), kp, vp, page_stride(kc), page_stride(vc), wp, weights_stride(w), ip(tables), ip(lens), i32(tables.size(0)), i32(kc.size(1)),
         i32(kc.size(0)), i32(kc.size(2)), i32(tables.size(1)), limit, keep, recent, sinks, i32(kc.size(3)), cache_type(kc));
    return Py_BuildValue("(OOO)", a[0], a[1], a[2]);
}

// kv_lens, block_tables, free_pages, n_free, page_size, limit, keep
PyObject *paged_trim(PyObject *const *a) {
    const at::Tensor &tables = ints(a[1], {-1, -1}, "block_tables [batch, width]"), &lens = ints(a[0], {tables.size(0)}, "kv_lens [batch]");
    const at::Tensor &stack = ints(a[2], {-1}, "free_pages [stack_size]"), &n_free = ints(a[3], {1}, "n_free [1]");
    const int64_t batch = tables.size(0);
    together(tables, lens, stack, n_free);
    const int32_t size = i32(a[4]), limit = i32(a[5]), keep = i32(a[6]);
    std::array<at::Tensor, 3> t = ints_in_one<3>({batch, batch, 1}, tables);
    int32_t *const sp = iw(stack);
    call(lib.agpu_paged_trim_, context(tables), ip(lens), ip(tables), sp, ip(n_free), iw(t[0]), iw(t[1]), iw(t[2]), i32(batch), i32(tables.size(1)), i32(stack.numel()), size, limit, keep);
    return Py_BuildValue("(NNN)", wrap(std::move(t[0])), wrap(std::move(t[1])), wrap(std::move(t[2])));
}

// A setting of sample: a number for all rows, or a tensor with one a row
struct PerRow {
    const at::Tensor *t = nullptr;
    PerRow(PyObject *o, at::ScalarType type, int64_t n, const at::Tensor &like, const char *what) {
        if (!THPVariable_Check(o)) return;
        t = &typed(o, type, {n}, what);
        if (!t->is_contiguous()) shape_err(std::string("contiguous ") + what, "strides " + str(t->strides()));
        if (t->device() != like.device()) {
            PyErr_SetString(PyExc_AssertionError, "expects device tensors, all on one GPU");
            throw PyFail();
        }
    }
    const float *floats() const { return t ? data(*t) : nullptr; }
};

// logits, u, temperature, top_k, top_p, min_p
PyObject *sample(PyObject *const *a) {
    const at::Tensor &x = tensor(a[0]), &u = tensor(a[1]);
    const int64_t n = last(x), count = n ? x.numel() / n : 0;
    if (x.scalar_type() != at::kFloat || u.scalar_type() != at::kFloat) shape_err("logits and u of Float", std::string(c10::toString(x.scalar_type())) + ", " + c10::toString(u.scalar_type()));
    if (n == 0) shape_err("logits of at least one token", str(x.sizes()));
    if (u.numel() != count) shape_err("u with a number for each of " + str(count) + " rows", str(u.sizes()));
    if (!x.is_contiguous() || !u.is_contiguous()) shape_err("contiguous logits and u", "strides " + str(x.strides()) + ", " + str(u.strides()));
    const PerRow temperature(a[2], at::kFloat, count, x, "temperature [rows]"), top_k(a[3], at::kInt, count, x, "top_k [rows]");
    const PerRow top_p(a[4], at::kFloat, count, x, "top_p [rows]"), min_p(a[5], at::kFloat, count, x, "min_p [rows]");
    const float t = temperature.t ? 1.0f : real(a[2]), p = top_p.t ? 1.0f : real(a[4]), m = min_p.t ? 0.0f : real(a[5]);
    const int32_t k = top_k.t ? 0 : i32(a[3]);
    together(x, u);
    at::Tensor out = empty(x.sizes().slice(0, x.dim() - 1), x, at::kInt);
    call(lib.agpu_sample_, context(x), data(x), data(u), iw(out), i32(count), i32(n), t, k, p, m, temperature.floats(), top_k.t ? ip(*top_k.t) : nullptr, top_p.floats(),
         min_p.floats());
    return wrap(std::move(out));
}

// ---- the module ---------------------------------------------------------------------------

template <PyObject *(*OP)(PyObject *const *), int NARGS>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
    if (n != NARGS) return PyErr_Format(PyExc_TypeError, "expects %d arguments, got %zd", NARGS, n);
    if (!g_error) return PyErr_Format(PyExc_RuntimeError, "bind() has not been called");
    try {
        return OP(args);
    } catch (const PyFail &) {
        return nullptr;
    } catch (...) {  // torch's own (out of memory, a bad size): the Python error that torch makes of it
        torch::translate_exception_to_python(std::current_exception());
        return nullptr;
    }
}

// bind(library path, AgpuError, ops.context, _lib.ptr)
PyObject *bind(PyObject *, PyObject *args) {
    const char *path;
    PyObject *error, *context, *ptr;
    if (!PyArg_ParseTuple(args, "sOOO", &path, &error, &context, &ptr)) return nullptr;
    void *so = dlopen(path, RTLD_NOW | RTLD_LOCAL);  // the copy that is loaded already
    if (!so) return PyErr_Format(PyExc_OSError, "%s", dlerror());
#define X(f)                                                  \
    lib.f##_ = reinterpret_cast<decltype(&f)>(dlsym(so, #f)); \
    if (!lib.f##_) return PyErr_Format(PyExc_OSError, "%s lacks " #f, path);
    AGPU_OPS(X)
#undef X
    Py_INCREF(error);
    Py_INCREF(context);
    Py_INCREF(ptr);
    g_error = error, g_context = context, g_ptr = ptr;
    Py_RETURN_NONE;
}

// forget(address of a context that is about to be destroyed)
PyObject *forget(PyObject *, PyObject *handle) {
    const void *h = PyLong_AsVoidPtr(handle);
    if (PyErr_Occurred()) return nullptr;
    for (size_t i = g_ctx.size(); i-- > 0;)
        if (g_ctx[i].handle == h) g_ctx.erase(g_ctx.begin() + (long)i);
    Py_RETURN_NONE;
}

#define OP(name, n) {#name, (PyCFunction)(void (*)(void))entry<name, n>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    OP(int4_linear, 9), OP(layer_norm, 4), OP(add_layer_norm_dual, 6), OP(gelu, 2), OP(add_inplace, 2), OP(bias_add, 2), OP(softmax_rows, 1),
    OP(embedding, 4), OP(argmax_rows, 2), OP(split_qkv, 3), OP(concat_heads, 1), OP(attention, 6), OP(multi_head_flash_attention, 6),
    OP(kv_append, 3), OP(gemm_f32, 2), OP(paged_plan, 7), OP(paged_kv_append, 5), OP(paged_attention, 9),
    OP(paged_attention_shared, 12), OP(paged_attention_weights, 10), OP(paged_evict, 9), OP(paged_trim, 7), OP(sample, 6),
    {"bind", bind, METH_VARARGS, nullptr}, {"forget", forget, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops() { return PyModule_Create(&module); }
