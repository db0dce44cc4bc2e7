// The decode step's operators for Python: tensors in, calls of the C ABI out.
//
// The C ABI cannot see a tensor's device, element type, number of elements and
// inner strides: they are checked here, which in Python (five attributes of up to
// nine tensors, and twenty-odd numbers through ctypes) cost 3 to 5 of the 7.5 us
// of a call whose kernel runs 3.  A function takes what its namesake in decode.py
// does, in order, and returns the library's status; a tensor that does not fit is
// a ValueError.  The library's functions come as addresses (bind), so the one
// that ctypes has loaded is the one called.
#include <torch/csrc/autograd/python_variable.h>

#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>

#include <climits>
#include <cstdint>
#include <exception>

#include "clove/gemm_c.h"

namespace {

struct Refused : std::exception {};  // (a Python error is set)

[[noreturn]] void refuse(PyObject* kind, const char* name, const char* what) {
    PyErr_Format(kind, "%s %s", name, what);
    throw Refused();
}

decltype(&clove_qk_norm_rope) g_rope;
decltype(&clove_paged_attention) g_attend;
decltype(&clove_cache_evict) g_evict;
decltype(&clove_penalize_logits) g_penalize;

constexpr auto kInt = at::kInt, kFloat = at::kFloat;

// What decode.py's KVCache holds: the description and the device of its tensors
struct CacheAt {
    clove_kv_cache_t c;
    int device;
};

struct Args {
    PyObject* const* at;
    mutable int device = -1;  // of the tensors so far
    // One device for all of a call's tensors, whose stream the call goes to
    void on(int index, const char* name) const {
        if (device < 0) device = index;
        if (index == device) return;
        PyErr_Format(PyExc_ValueError, "%s is on cuda:%d, other tensors are on cuda:%d", name, index, device);
        throw Refused();
    }
    const at::Tensor& tensor(int i, const char* name, at::ScalarType type) const {
        if (!THPVariable_Check(at[i])) refuse(PyExc_TypeError, name, "is not a tensor");
        const at::Tensor& x = THPVariable_Unpack(at[i]);
        if (x.scalar_type() != type || !x.is_cuda()) {
            PyErr_Format(PyExc_ValueError, "%s must be %s on the GPU, not %s on %s", name, c10::toString(type),
                         c10::toString(x.scalar_type()), x.device().str().c_str());
            throw Refused();
        }
        on(x.get_device(), name);
        return x;
    }
    at::ScalarType type(int i, const char* name) const {
        if (!THPVariable_Check(at[i])) refuse(PyExc_TypeError, name, "is not a tensor");
        return THPVariable_Unpack(at[i]).scalar_type();
    }
    bool none(int i) const { return at[i] == Py_None; }
    int number(int i, const char* name) const {
        const long v = PyLong_AsLong(at[i]);
        if (v == -1 && PyErr_Occurred()) throw Refused();
        if (v < INT_MIN || v > INT_MAX) refuse(PyExc_OverflowError, name, "has more than 32 bits");
        return (int)v;
    }
    float real(int i) const {
        const double v = PyFloat_AsDouble(at[i]);
        if (v == -1.0 && PyErr_Occurred()) throw Refused();
        return (float)v;
    }
    const clove_kv_cache_t* cache(int i) const {
        const void* p = PyLong_AsVoidPtr(at[i]);
        if (!p && PyErr_Occurred()) throw Refused();
        const CacheAt* x = static_cast<const CacheAt*>(p);
        on(x->device, "the cache");
        return &x->c;
    }
    // None: torch's current one.  (The library works on the current device, so the
    // tensors have to be there.)
    void* stream(int i) const {
        if (const int now = c10::hip::current_device(); device >= 0 && device != now) {
            PyErr_Format(PyExc_ValueError, "the tensors are on cuda:%d, the current device is cuda:%d", device, now);
            throw Refused();
        }
        if (none(i)) return c10::hip::getCurrentHIPStream().stream();
        PyObject* x = PyLong_Check(at[i]) ? (Py_INCREF(at[i]), at[i]) : PyObject_GetAttrString(at[i], "cuda_stream");
        if (!x) throw Refused();
        void* p = PyLong_AsVoidPtr(x);
        Py_DECREF(x);
        if (!p && PyErr_Occurred()) throw Refused();
        return p;
    }
};

// a b, or more than any tensor has
int64_t times(int64_t a, int64_t b) {
    int64_t r;
    return __builtin_mul_overflow(a, b, &r) ? INT64_MAX : r;
}

struct Rows {
    void* at = nullptr;
    int64_t stride = 0;
};

// A tensor read as `rows` rows of `width` adjacent elements; its first dimension is
// the row where it has more than one.
Rows rows(const at::Tensor& x, const char* name, int64_t n, int64_t width) {
    if (x.is_contiguous() && x.numel() == times(n, width)) return {x.data_ptr(), width};
    const auto shape = x.sizes(), strides = x.strides();
    const int dims = (int)shape.size();
    int64_t have = 1, inner = 1, stride = 0;
    for (int d = dims - 1; d >= (dims > 1 ? 1 : 0); --d) {
        if (shape[d] != 1 && strides[d] != inner) {
            inner = -1;
            break;
        }
        inner *= shape[d];
    }
    if (dims > 1) have = shape[0], stride = strides[0];
    if (have < n || inner < width) {
        PyErr_Format(PyExc_ValueError, "%s holds %lld rows of %lld adjacent elements, %lld rows of %lld are wanted", name,
                     (long long)have, (long long)(inner < 0 ? 1 : inner), (long long)n, (long long)width);
        throw Refused();
    }
    return {x.data_ptr(), n > 1 ? stride : width};
}
Rows rows(const Args& a, int i, const char* name, at::ScalarType type, int64_t n, int64_t width) {
    return rows(a.tensor(i, name, type), name, n, width);
}

// Equally long lists one after another: how far apart they lie tells the library how
// long they are, so no part of longer ones is taken.
Rows lists(const Args& a, int i, const char* name, at::ScalarType type, int64_t n) {
    const at::Tensor& x = a.tensor(i, name, type);
    if (x.dim() == 0) refuse(PyExc_ValueError, name, "must have a dimension");
    const Rows r = rows(x, name, n, x.size(-1));
    if (n > 1 && r.stride != x.size(-1)) refuse(PyExc_ValueError, name, "must have its rows one after another");
    return {r.at, x.size(-1)};
}

// At least `n` adjacent elements (None: null)
template <class T>
T* flat(const Args& a, int i, const char* name, at::ScalarType type, int64_t n) {
    if (a.none(i)) return nullptr;
    const at::Tensor& x = a.tensor(i, name, type);
    if (x.numel() < n || !x.is_contiguous()) {
        PyErr_Format(PyExc_ValueError, "%s must be %lld adjacent elements, not %lld%s", name, (long long)n, (long long)x.numel(),
                     x.is_contiguous() ? "" : " apart from another");
        throw Refused();
    }
    return static_cast<T*>(x.data_ptr());
}

int code(at::ScalarType t) {
    if (t == at::kHalf) return CLOVE_DTYPE_FP16;
    if (t == at::kBFloat16) return CLOVE_DTYPE_BF16;
    if (t == at::kFloat) return CLOVE_DTYPE_FP32;
    PyErr_Format(PyExc_ValueError, "element type %s is not fp16, bf16 or fp32", c10::toString(t));
    throw Refused();
}
at::ScalarType type_of(const clove_kv_cache_t* c) {
    return c->dtype == CLOVE_DTYPE_FP16 ? at::kHalf : c->dtype == CLOVE_DTYPE_BF16 ? at::kBFloat16 : at::kFloat;
}
// (pages of nothing are refused by the library)
int64_t pages(const clove_kv_cache_t* c, int keys) { return c->page_size > 0 ? ((int64_t)keys + c->page_size - 1) / c->page_size : 0; }

clove_status_t rope(const Args& a) {
    const int T = a.number(7, "T"), hq = a.number(8, "q_heads"), hk = a.number(9, "kv_heads"), D = a.number(10, "head_dim");
    const int R = a.none(11) ? D : a.number(11, "rot_dim"), turned = PyObject_IsTrue(a.at[13]);
    const float eps = a.real(12);
    if (turned < 0) throw Refused();
    const at::ScalarType t = a.type(0, "qkv");
    const Rows x = rows(a, 0, "qkv", t, T, times((int64_t)hq + 2 * (int64_t)hk, D));
    const Rows q = rows(a, 6, "q_out", t, T, times(hq, D));
    const Rows k = a.none(14) ? Rows{} : rows(a, 14, "k_out", t, T, times(hk, D));
    const float *c = nullptr, *s = nullptr;
    int most = 0;
    if (R) {
        const at::Tensor &xc = a.tensor(3, "cos", kFloat), &xs = a.tensor(4, "sin", kFloat);
        const int64_t half = R / 2, n = xc.dim() ? xc.size(0) : 0;
        if (!xc.is_contiguous() || !xs.is_contiguous() || xc.sizes() != xs.sizes() || xc.numel() != times(n, half) || n > INT_MAX) {
            PyErr_Format(PyExc_ValueError, "cos and sin must be dense, [max_position, %lld]", (long long)half);
            throw Refused();
        }
        most = (int)n, c = static_cast<const float*>(xc.data_ptr()), s = static_cast<const float*>(xs.data_ptr());
    }
    const void *wq = flat<void>(a, 1, "q_weight", t, D), *wk = flat<void>(a, 2, "k_weight", t, D);
    const int32_t* positions = R ? flat<int32_t>(a, 5, "positions", kInt, T) : nullptr;
    const clove_kv_cache_t* cache = a.none(15) ? nullptr : a.cache(15);
    const int32_t* slots = flat<int32_t>(a, 16, "slots", kInt, T);
    const int dt = code(t);
    void* stream = a.stream(17);
    clove_status_t st;
    Py_BEGIN_ALLOW_THREADS
    st = g_rope(x.at, x.stride, wq, wk, eps, c, s, most, positions, q.at, q.stride, k.at, k.stride, cache, slots, T, hq, hk, D, R,
                turned, dt, stream);
    Py_END_ALLOW_THREADS
    return st;
}

clove_status_t attend(const Args& a) {
    const clove_kv_cache_t* cache = a.cache(1);
    const int B = a.number(5, "batch"), hq = a.number(6, "q_heads"), most = a.number(7, "max_context"), window = a.number(10, "window");
    const float scale = a.real(8), cap = a.real(9);
    const at::ScalarType t = type_of(cache);
    const int64_t width = times(hq, cache->head_dim);
    const Rows q = rows(a, 0, "q", t, B, width), o = rows(a, 4, "out", t, B, width);
    const Rows table = rows(a, 2, "block_table", kInt, B, pages(cache, most));
    const Rows w = a.none(11) ? Rows{} : rows(a, 11, "weights", kFloat, B, most);
    const int32_t* lens = flat<int32_t>(a, 3, "context_lens", kInt, B);
    void* stream = a.stream(12);
    clove_status_t st;
    Py_BEGIN_ALLOW_THREADS
    st = g_attend(q.at, q.stride, cache, static_cast<const int32_t*>(table.at), table.stride, lens, o.at, o.stride,
                  static_cast<float*>(w.at), w.stride, B, hq, most, scale, cap, window, stream);
    Py_END_ALLOW_THREADS
    return st;
}

clove_status_t evict(const Args& a) {
    const clove_kv_cache_t* cache = a.cache(0);
    const int B = a.number(8, "batch"), most = a.number(9, "max_context"), budget = a.number(10, "budget");
    const int sinks = a.number(11, "sinks"), recent = a.number(12, "recent");
    const Rows table = rows(a, 1, "block_table", kInt, B, pages(cache, most));
    const Rows w = rows(a, 3, "weights", kFloat, B, most), p = rows(a, 4, "positions", kInt, B, most);
    const Rows wo = rows(a, 5, "weights_out", kFloat, B, most), po = rows(a, 6, "positions_out", kInt, B, most);
    const int32_t* lens = flat<int32_t>(a, 2, "context_lens", kInt, B);
    int32_t* lens_out = flat<int32_t>(a, 7, "lens_out", kInt, B);
    void* stream = a.stream(13);
    clove_status_t st;
    Py_BEGIN_ALLOW_THREADS
    st = g_evict(cache, static_cast<const int32_t*>(table.at), table.stride, lens, static_cast<const float*>(w.at), w.stride,
                 static_cast<const int32_t*>(p.at), p.stride, static_cast<float*>(wo.at), wo.stride, static_cast<int32_t*>(po.at),
                 po.stride, lens_out, B, most, budget, sinks, recent, stream);
    Py_END_ALLOW_THREADS
    return st;
}

clove_status_t penalize(const Args& a) {
    const int B = a.number(2, "batch"), V = a.number(3, "vocab");
    const at::ScalarType t = a.type(0, "logits"), to = a.type(1, "out");
    const Rows x = rows(a, 0, "logits", t, B, V), o = rows(a, 1, "out", to, B, V);
    const Rows h = a.none(4) ? Rows{} : lists(a, 4, "history", kInt, B);
    Rows ids, values;
    if (!a.none(10)) {
        ids = lists(a, 10, "bias_ids", kInt, B), values = lists(a, 11, "bias_values", kFloat, B);
        if (ids.stride != values.stride) refuse(PyExc_ValueError, "bias_ids and bias_values", "must be equally long");
    }
    const Rows m = a.none(13) ? Rows{} : rows(a, 13, "allowed", kInt, B, ((int64_t)V + 31) / 32);
    const int32_t *hn = flat<int32_t>(a, 5, "history_lens", kInt, B), *pn = flat<int32_t>(a, 6, "prompt_lens", kInt, B);
    const float *r = flat<float>(a, 7, "repetition", kFloat, B), *p = flat<float>(a, 8, "presence", kFloat, B),
                *f = flat<float>(a, 9, "frequency", kFloat, B);
    const int32_t* bn = flat<int32_t>(a, 12, "bias_counts", kInt, B);
    const int dt = code(t), dto = code(to);
    void* stream = a.stream(14);
    clove_status_t st;
    Py_BEGIN_ALLOW_THREADS
    st = g_penalize(x.at, x.stride, dt, o.at, o.stride, dto, B, V, static_cast<const int32_t*>(h.at), h.stride, hn, pn, r, p, f,
                    static_cast<const int32_t*>(ids.at), static_cast<const float*>(values.at), ids.stride, bn,
                    static_cast<const uint32_t*>(m.at), m.stride, stream);
    Py_END_ALLOW_THREADS
    return st;
}

// the status as a Python number; no exception leaves
template <clove_status_t (*F)(const Args&), int N>
PyObject* entry(PyObject*, PyObject* const* at, Py_ssize_t n) {
    if (n != N) return PyErr_Format(PyExc_TypeError, "%d arguments are wanted, not %zd", N, n);
    try {
        return PyLong_FromLong((long)F(Args{at}));
    } catch (const Refused&) {
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

PyObject* bind(PyObject*, PyObject* const* at, Py_ssize_t n) {
    void* p[4];
    if (n != 4) return PyErr_Format(PyExc_TypeError, "4 addresses are wanted, not %zd", n);
    for (int i = 0; i < 4; ++i)
        if (!(p[i] = PyLong_AsVoidPtr(at[i])))
            return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "address %d is null", i);
    g_rope = reinterpret_cast<decltype(g_rope)>(p[0]);
    g_attend = reinterpret_cast<decltype(g_attend)>(p[1]);
    g_evict = reinterpret_cast<decltype(g_evict)>(p[2]);
    g_penalize = reinterpret_cast<decltype(g_penalize)>(p[3]);
    Py_RETURN_NONE;
}

template <class F>
PyCFunction fast(F f) {
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}
PyMethodDef methods[] = {{"bind", fast(bind), METH_FASTCALL, nullptr},
                         {"qk_norm_rope", fast(entry<rope, 18>), METH_FASTCALL, nullptr},
                         {"paged_attention", fast(entry<attend, 13>), METH_FASTCALL, nullptr},
                         {"cache_evict", fast(entry<evict, 14>), METH_FASTCALL, nullptr},
                         {"penalize_logits", fast(entry<penalize, 15>), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_decode", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__decode() { return PyModule_Create(&module); }
