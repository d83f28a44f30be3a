// Python binding of the C ABI for torch tensors: `_binding`, a module whose functions are the entry points of
// include/scmx.h, scmx_cache.h and scmx_mx.h that enqueue work (and their queries of sizes), under the same names and with the same arguments except the
// last.  A pointer argument takes a tensor (contiguous, on the GPU), None or an integer address; a format argument an object
// whose buffer is the scmx_format; the stream is the caller's current one and is not passed.  A negative status raises.
//
// A decode step is a few hundred calls of a few microseconds of GPU work each, so the host's share per call decides: through
// ctypes a call cost 8-10 us (argument conversion; pointers, stream and format descriptor made in Python each time).  One
// GEMV call 11.9 -> 5.8 us, a linear layer on 40 rows 16.7 -> 10.3, a decode step of two OLMoE blocks 320 -> 205.  The
// allocation helpers are there for the same reason.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ops/empty.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <exception>
#include <initializer_list>
#include <optional>
#include <tuple>
#include <type_traits>
#include <utility>
#include <vector>

#include "../../include/scmx_cache.h"
#include "../../include/scmx_mx.h"

namespace {

// A Python exception is set.
struct Raised {};

void fail(PyObject* type, const char* text) {
    PyErr_SetString(type, text);
    throw Raised();
}

// In a catch block: the Python exception of what was thrown, torch's own types (out of memory, a Python error) among them.
PyObject* raised() {
    try {
        throw;
    } catch (const Raised&) {
    } catch (...) {
        torch::translate_exception_to_python(std::current_exception());
    }
    return nullptr;
}

int64_t as_int(PyObject* o) {
    const int64_t v = PyLong_Check(o) ? PyLong_AsLongLong(o) : [&] {
        PyObject* i = PyNumber_Index(o);
        if (!i) throw Raised();
        const int64_t r = PyLong_AsLongLong(i);
        Py_DECREF(i);
        return r;
    }();
    if (v == -1 && PyErr_Occurred()) throw Raised();
    return v;
}

void* as_pointer(PyObject* o) {
    if (o == Py_None) return nullptr;
    if (THPVariable_Check(o)) {
        const at::Tensor& t = THPVariable_Unpack(o);
        if (!t.is_cuda()) fail(PyExc_ValueError, "scmx kernels take CUDA (ROCm) tensors; got a CPU tensor");
        if (!t.is_contiguous()) fail(PyExc_ValueError, "scmx kernels take contiguous tensors");
        return t.data_ptr();
    }
    return reinterpret_cast<void*>(as_int(o));
}

template <typename T>
T convert(PyObject* o) {
    if constexpr (std::is_same_v<T, const scmx_format*>) {
        Py_buffer b;
        if (PyObject_GetBuffer(o, &b, PyBUF_SIMPLE)) throw Raised();
        const bool whole = b.len >= Py_ssize_t(sizeof(scmx_format));
        const T p = static_cast<T>(b.buf);   // the caller's reference to the object keeps the memory
        PyBuffer_Release(&b);
        if (!whole) fail(PyExc_ValueError, "the format argument is smaller than a scmx_format");
        return p;
    } else if constexpr (std::is_pointer_v<T>) {
        return static_cast<T>(as_pointer(o));
    } else if constexpr (std::is_floating_point_v<T>) {
        const double v = PyFloat_AsDouble(o);
        if (v == -1.0 && PyErr_Occurred()) throw Raised();
        return T(v);
    } else {
        const int64_t v = as_int(o);
        if (int64_t(T(v)) != v || (std::is_unsigned_v<T> && v < 0)) fail(PyExc_ValueError, "integer argument out of range");
        return T(v);
    }
}

PyObject* status(const char* name, int rc) {
    if (rc == SCMX_OK) Py_RETURN_NONE;
    PyErr_Format(rc == SCMX_ERR_ARG || rc == SCMX_ERR_FORMAT || rc == SCMX_ERR_WORKSPACE ? PyExc_ValueError : PyExc_RuntimeError,
                 "%s failed (%d): %s", name, rc, scmx_last_error());
    return nullptr;
}

// One entry point as a METH_FASTCALL function: its parameters but the last from the arguments, the last the current stream.
template <auto FN, typename Sig = decltype(FN)>
struct Call;
template <auto FN, typename... P>
struct Call<FN, int (*)(P...)> {
    static const char* name;
    template <size_t... I>
    static int run(PyObject* const* args, std::index_sequence<I...>) {
        using Params = std::tuple<P...>;
        std::tuple<std::tuple_element_t<I, Params>...> v{convert<std::tuple_element_t<I, Params>>(args[I])...};
        void* stream = c10::hip::getCurrentHIPStream().stream();
        int rc;
        Py_BEGIN_ALLOW_THREADS;
        rc = FN(std::get<I>(v)..., stream);
        Py_END_ALLOW_THREADS;
        return rc;
    }
    static PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
        constexpr size_t N = sizeof...(P) - 1;
        try {
            if (n != Py_ssize_t(N)) {
                PyErr_Format(PyExc_TypeError, "%s takes %zu arguments (the stream is the current one), got %zd", name, N, n);
                return nullptr;
            }
            return status(name, run(args, std::make_index_sequence<N>()));
        } catch (...) {
            return raised();
        }
    }
};
template <auto FN, typename... P>
const char* Call<FN, int (*)(P...)>::name = "";

// A size or choice the library answers without device work: every argument converted, the value returned.
template <auto FN, typename Sig = decltype(FN)>
struct Query;
template <auto FN, typename R, typename... P>
struct Query<FN, R (*)(P...)> {
    template <size_t... I>
    static PyObject* run(PyObject* const* args, std::index_sequence<I...>) {
        return PyLong_FromLongLong(static_cast<long long>(FN(convert<P>(args[I])...)));
    }
    static PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
        try {
            if (n != Py_ssize_t(sizeof...(P))) fail(PyExc_TypeError, "wrong number of arguments");
            return run(args, std::index_sequence_for<P...>());
        } catch (const Raised&) {
            return nullptr;
        }
    }
};

struct NoGil {
    PyThreadState* const state = PyEval_SaveThread();
    ~NoGil() { PyEval_RestoreThread(state); }
};

// empty_<type>(like, dims...): an uninitialised tensor on the device of `like`.
template <at::ScalarType TYPE>
PyObject* empty(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        if (n < 2 || !THPVariable_Check(args[0])) fail(PyExc_TypeError, "empty_*(tensor, dims...)");
        int64_t dims[4];
        if (n > 5) fail(PyExc_TypeError, "at most four dimensions");
        for (Py_ssize_t i = 1; i < n; ++i) dims[i - 1] = as_int(args[i]);
        const at::Tensor& like = THPVariable_Unpack(args[0]);
        const at::TensorOptions options = at::TensorOptions().dtype(TYPE).device(like.device());
        at::Tensor t;
        {
            const NoGil released;   // the allocator may ask the driver, or wait for the GPU
            t = at::empty(at::IntArrayRef(dims, size_t(n - 1)), options);
        }
        return THPVariable_Wrap(std::move(t));
    } catch (...) {
        return raised();
    }
}

// A contiguous tensor on the GPU, and if `type` is given of that type; NULL: something else.
const at::Tensor* plain(PyObject* o, at::ScalarType type = at::ScalarType::Undefined) {
    if (!THPVariable_Check(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.is_cuda() && t.is_contiguous() && (type == at::ScalarType::Undefined || t.scalar_type() == type) ? &t : nullptr;
}

// gemv(format, xq, xscale, codes, bcodes, wscale, N, epi, res, eidx, xstride, shared, pro, nw, eps): sc_decode.gemv for the operands of
// every decode step -- plain tensors, up to eight rows -- in one call: output (and workspace) allocated, the kernel launched.  None
// where an operand is anything else: the caller's general way converts or refuses it.  With both in Python a call on one row of
// 2048 x 2048 took the host 5.0 us, in its kernel's 4.0.
PyObject* gemv(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        if (n != 15) fail(PyExc_TypeError, "gemv takes 15 arguments");
        for (int i : {6, 7, 10, 12})
            if (!PyLong_Check(args[i])) Py_RETURN_NONE;
        if (args[11] != Py_None && !PyLong_Check(args[11])) Py_RETURN_NONE;
        const int N = convert<int>(args[6]), epi = convert<int>(args[7]), xstride = convert<int>(args[10]), pro = convert<int>(args[12]);
        const at::Tensor* x = plain(args[1], pro == 0 ? at::ScalarType::Char : at::ScalarType::BFloat16);
        const at::Tensor *codes = plain(args[3]), *bcodes = plain(args[4]), *wscale = plain(args[5]);
        const at::Tensor* xscale = pro == 0 ? plain(args[2]) : x;
        const at::Tensor* res = epi == SCMX_EPI_RES ? plain(args[8]) : x;
        const at::Tensor* nw = pro == 2 ? plain(args[13]) : x;
        if (!x || !codes || !bcodes || !wscale || !xscale || !res || !nw || x->dim() < 1 || x->dim() > 2) Py_RETURN_NONE;
        if (pro == 2 && !PyFloat_Check(args[14])) Py_RETURN_NONE;
        const at::Tensor* eidx = args[9] == Py_None ? nullptr : plain(args[9], at::ScalarType::Int);
        const int64_t rows = x->dim() == 2 ? x->size(0) : 1, K64 = x->size(-1), slots64 = eidx ? eidx->numel() : 0;
        if ((args[9] != Py_None && !eidx) || N < 0 || K64 > INT32_MAX || slots64 > INT32_MAX - 1 || (!eidx && rows > 8)) Py_RETURN_NONE;
        const scmx_format* fmt = convert<const scmx_format*>(args[0]);
        const int K = int(K64), shared = args[11] == Py_None ? -1 : convert<int>(args[11]);
        const float eps = pro == 2 ? convert<float>(args[14]) : 0.0f;
        const int batch = !eidx && rows > 1 ? int(rows) : 1, slots = int(slots64) + (args[11] != Py_None);
        const int64_t width = epi == SCMX_EPI_SWIGLU ? N / 2 : N;
        const auto ptr = [](const at::Tensor* t) { return t->data_ptr(); };
        at::Tensor out;
        int rc;
        {
            const NoGil released;   // the allocator may ask the driver, or wait for the GPU
            const at::TensorOptions options = at::TensorOptions().dtype(at::ScalarType::BFloat16).device(x->device());
            out = eidx ? at::empty({slots, width}, options) : batch > 1 ? at::empty({batch, width}, options) : at::empty({width}, options);
            const auto *xs = pro == 0 ? static_cast<const float*>(ptr(xscale)) : nullptr;
            const auto *rs = epi == SCMX_EPI_RES ? static_cast<const uint16_t*>(ptr(res)) : nullptr;
            const auto *w = pro == 2 ? static_cast<const uint16_t*>(ptr(nw)) : nullptr;
            const auto *c = static_cast<const uint32_t*>(ptr(codes));
            const auto *b = static_cast<const uint8_t*>(ptr(bcodes));
            const auto *s = static_cast<const float*>(ptr(wscale));
            auto* o = static_cast<uint16_t*>(out.data_ptr());
            if (eidx) {
                rc = scmx_gemv(fmt, ptr(x), xs, c, b, s, rs, o, epi, pro, w, eps, batch, N, K, static_cast<const int32_t*>(ptr(eidx)),
                               int(slots64), xstride, shared, c10::hip::getCurrentHIPStream().stream());
            } else {
                const size_t need = batch > 1 ? scmx_gemv_rows_workspace(fmt, pro, batch, N, K) : 0;
                const at::Tensor work = need ? at::empty({int64_t(need)}, options.dtype(at::ScalarType::Byte)) : at::Tensor();
                rc = scmx_gemv_rows(fmt, ptr(x), xs, c, b, s, rs, o, epi, pro, w, eps, batch, N, K, need ? work.data_ptr() : nullptr, need,
                                    c10::hip::getCurrentHIPStream().stream());
            }
        }
        if (rc != SCMX_OK) return status(eidx ? "scmx_gemv" : "scmx_gemv_rows", rc);
        return THPVariable_Wrap(std::move(out));
    } catch (...) {
        return raised();
    }
}

// ---- drafted tokens over a cache: sc_cache's and sc_draft's functions for the operands of every step, in one call as above ---------
// (None where an operand is anything else: the caller's general way converts or refuses it.  16 tokens through 28 blocks'
// caches, 29 calls that the host bounds: 313 us with checks and allocations in Python, see sc_cache, 140-157 here.)

// A contiguous tensor of `type` on the current device; NULL: something else.  None is not one.
const at::Tensor* local(PyObject* o, at::ScalarType type) {
    const at::Tensor* t = plain(o, type);
    return t && t->get_device() == c10::hip::current_device() ? t : nullptr;
}

struct CacheTensors {
    const at::Tensor *k, *v, *ks = nullptr, *vs = nullptr;
    int64_t hk, rows, d;
    bool four = false;
    float* scale(const at::Tensor* t) const { return t ? static_cast<float*>(t->data_ptr()) : nullptr; }
    static uint8_t* bytes(const at::Tensor* t) { return static_cast<uint8_t*>(t->data_ptr()); }
};
bool cache_of(PyObject* k, PyObject* v, PyObject* ks, PyObject* vs, CacheTensors& c) {
    const bool eight = ks != Py_None;
    c.four = eight && THPVariable_Check(ks) && THPVariable_Unpack(ks).scalar_type() == at::ScalarType::Byte;
    const at::ScalarType type = c.four ? at::ScalarType::Byte : eight ? at::ScalarType::Char : at::ScalarType::BFloat16;
    c.k = local(k, type);
    c.v = local(v, type);
    if (!c.k || !c.v || c.k->dim() != 3 || c.k->sizes() != c.v->sizes() || eight != (vs != Py_None)) return false;
    c.hk = c.k->size(0);
    c.rows = c.k->size(1);
    c.d = c.k->size(2);
    if (c.four) {
        c.ks = local(ks, at::ScalarType::Byte);
        c.vs = local(vs, at::ScalarType::Byte);
        if (!c.ks || !c.vs || c.d % 16) return false;
        for (const at::Tensor* t : {c.ks, c.vs})
            if (t->dim() != 3 || t->size(0) != c.hk || t->size(1) != c.rows || t->size(2) != c.d / 16) return false;
        c.d *= 2;
    } else if (eight) {
        c.ks = local(ks, at::ScalarType::Float);
        c.vs = local(vs, at::ScalarType::Float);
        if (!c.ks || !c.vs) return false;
        for (const at::Tensor* t : {c.ks, c.vs})
            if (t->dim() != 2 || t->size(0) != c.hk || t->size(1) != c.rows) return false;
    }
    return c.hk <= INT32_MAX && c.rows <= INT32_MAX && c.d <= INT32_MAX;
}
// A position: an integer, or an int64 tensor of one value.
bool position_of(PyObject* o, const int64_t*& dev, int64_t& at) {
    dev = nullptr;
    at = 0;
    if (PyLong_CheckExact(o)) {
        at = as_int(o);
        return true;
    }
    const at::Tensor* t = local(o, at::ScalarType::Long);
    if (!t || t->numel() != 1) return false;
    dev = static_cast<const int64_t*>(t->data_ptr());
    return true;
}
// None, or such a tensor of n values.
template <typename T>
bool optional_of(PyObject* o, at::ScalarType type, int64_t n, const T*& p) {
    p = nullptr;
    if (o == Py_None) return true;
    const at::Tensor* t = local(o, type);
    if (!t || t->numel() != n) return false;
    p = static_cast<const T*>(t->data_ptr());
    return true;
}
bool ints_of(PyObject* const* args, std::initializer_list<int> at) {
    for (int i : at)
        if (!PyLong_CheckExact(args[i])) return false;
    return true;
}
// Outputs straight from torch's GPU allocator (every value is written; at::empty's dispatch takes half a microsecond more), and
// workspaces without a tensor around them.
at::Tensor fresh(const at::Tensor& like, at::ScalarType type, at::IntArrayRef size) {
    return at::Tensor(at::detail::empty_cuda(size, type, like.device(), std::nullopt));
}
c10::DataPtr scratch(size_t bytes) { return c10::hip::HIPCachingAllocator::get()->allocate(bytes); }
void* stream() { return c10::hip::getCurrentHIPStream().stream(); }

// cache_write(y, qn, kn, eps, L, hq, hk, d, kcache, vcache, pos, inv_freq, kscale, vscale, depth)
PyObject* cache_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        if (n != 15) fail(PyExc_TypeError, "cache_write takes 15 arguments");
        CacheTensors c;
        const int64_t* dev;
        int64_t pos;
        const int32_t* depth;
        if (!ints_of(args, {4, 5, 6, 7}) || !PyFloat_Check(args[3]) || !cache_of(args[8], args[9], args[12], args[13], c) ||
            !position_of(args[10], dev, pos))
            Py_RETURN_NONE;
        const int64_t L = as_int(args[4]), hq = as_int(args[5]), hk = as_int(args[6]), d = as_int(args[7]);
        const at::Tensor *y = local(args[0], at::ScalarType::BFloat16), *qn = local(args[1], at::ScalarType::BFloat16),
                         *kn = local(args[2], at::ScalarType::BFloat16), *freq = local(args[11], at::ScalarType::Float);
        if (!y || !qn || !kn || !freq || L < 0 || L > INT32_MAX || hq < 1 || hq > 65535 || hk != c.hk || d != c.d || y->dim() != 2 ||
            y->size(0) < L || y->size(1) != (hq + 2 * hk) * d || qn->numel() != d || kn->numel() != d || freq->numel() != d / 2 ||
            !optional_of(args[14], at::ScalarType::Int, L, depth))
            Py_RETURN_NONE;
        at::Tensor q;
        int rc;
        {
            const NoGil released;
            q = at::Tensor(at::detail::empty_strided_cuda({hq, L, d}, {d, hq * d, 1}, at::ScalarType::BFloat16, y->device()));
            const auto bf = [](const at::Tensor* t) { return static_cast<const uint16_t*>(t->data_ptr()); };
            const float eps = float(PyFloat_AS_DOUBLE(args[3]));
            auto* out = static_cast<uint16_t*>(q.data_ptr());
            const auto* f = static_cast<const float*>(freq->data_ptr());
            rc = c.four ? scmx_cache4_write(nullptr, nullptr, nullptr, bf(y), bf(qn), bf(kn), eps, out, c.bytes(c.k), c.bytes(c.v),
                                            c.bytes(c.ks), c.bytes(c.vs), int(L), int(hq), int(hk), int(d), f, depth, dev, pos,
                                            int(c.rows), stream())
                        : scmx_cache_write(nullptr, nullptr, nullptr, bf(y), bf(qn), bf(kn), eps, out, c.k->data_ptr(), c.v->data_ptr(),
                                           c.scale(c.ks), c.scale(c.vs), int(L), int(hq), int(hk), int(d), f, depth, dev, pos,
                                           int(c.rows), stream());
        }
        if (rc != SCMX_OK) return status(c.four ? "scmx_cache4_write" : "scmx_cache_write", rc);
        return THPVariable_Wrap(std::move(q));
    } catch (...) {
        return raised();
    }
}

// attn_tree(q, kcache, vcache, pos, mask, kscale, vscale, scale, splits)
PyObject* attn_tree(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        if (n != 9) fail(PyExc_TypeError, "attn_tree takes 9 arguments");
        CacheTensors c;
        const int64_t *dev, *mask;
        int64_t pos;
        if (!THPVariable_Check(args[0]) || !cache_of(args[1], args[2], args[5], args[6], c) || !position_of(args[3], dev, pos) ||
            (args[7] != Py_None && !PyFloat_Check(args[7])) || (args[8] != Py_None && !PyLong_CheckExact(args[8])))
            Py_RETURN_NONE;
        const at::Tensor& q = THPVariable_Unpack(args[0]);
        if (!q.is_cuda() || q.get_device() != c10::hip::current_device() || q.scalar_type() != at::ScalarType::BFloat16 || q.dim() != 3)
            Py_RETURN_NONE;
        const int64_t hq = q.size(0), T = q.size(1), d = q.size(2);   // the view of [T, hq, d] storage
        if (T < 1 || T > 64 || hq < 1 || hq > 65535 || d != c.d || c.hk < 1 || hq % c.hk || c.rows < T || q.stride(2) != 1 ||
            (hq > 1 && q.stride(0) != d) || (T > 1 && q.stride(1) != hq * d) ||
            !optional_of(args[4], at::ScalarType::Long, T, mask) || pos < 0 || pos > INT32_MAX - 64)
            Py_RETURN_NONE;
        const int splits = args[8] != Py_None ? convert<int>(args[8])
                                              : (c.four ? scmx_attn_tree4_splits : scmx_attn_tree_splits)(
                                                    int(T), dev ? int(c.rows) : int(pos + T), int(hq), int(c.hk), int(d));
        if (splits < 1 || splits > 64) Py_RETURN_NONE;
        const float scale = args[7] == Py_None ? float(1.0 / std::sqrt(double(d))) : float(PyFloat_AS_DOUBLE(args[7]));
        at::Tensor out;
        int rc;
        {
            const NoGil released;
            out = fresh(q, at::ScalarType::BFloat16, {T, hq * d});
            const c10::DataPtr work = scratch(splits > 1 ? size_t(splits * T * hq * (d + 2)) * sizeof(float) : 0);
            const auto* from = static_cast<const uint16_t*>(q.data_ptr());
            auto* to = static_cast<uint16_t*>(out.data_ptr());
            float* parts = splits > 1 ? static_cast<float*>(work.get()) : nullptr;
            rc = c.four ? scmx_attn_tree4(from, c.bytes(c.k), c.bytes(c.v), c.bytes(c.ks), c.bytes(c.vs), mask, dev, pos, to, int(T), int(hq),
                                          int(c.hk), int(d), int(c.rows), scale, parts, splits, stream())
                        : scmx_attn_tree(from, c.k->data_ptr(), c.v->data_ptr(), c.scale(c.ks), c.scale(c.vs), mask, dev, pos, to, int(T),
                                         int(hq), int(c.hk), int(d), int(c.rows), scale, parts, splits, stream());
        }
        if (rc != SCMX_OK) return status(c.four ? "scmx_attn_tree4" : "scmx_attn_tree", rc);
        return THPVariable_Wrap(std::move(out));
    } catch (...) {
        return raised();
    }
}

// cache_read(kcache, vcache, kscale, vscale, n, row0)
PyObject* cache_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        if (n != 6) fail(PyExc_TypeError, "cache_read takes 6 arguments");
        CacheTensors c;
        if (args[2] == Py_None || !ints_of(args, {4, 5}) || !cache_of(args[0], args[1], args[2], args[3], c)) Py_RETURN_NONE;
        const int64_t rows = as_int(args[4]), row0 = as_int(args[5]);
        if (rows < 0 || row0 < 0 || row0 > INT32_MAX || rows > c.rows) Py_RETURN_NONE;
        at::Tensor k, v;
        int rc;
        {
            const NoGil released;
            k = fresh(*c.k, at::ScalarType::BFloat16, {c.hk, rows, c.d});
            v = fresh(*c.k, at::ScalarType::BFloat16, {c.hk, rows, c.d});
            const auto codes = [](const at::Tensor* t) { return static_cast<const int8_t*>(t->data_ptr()); };
            auto *kp = static_cast<uint16_t*>(k.data_ptr()), *vp = static_cast<uint16_t*>(v.data_ptr());
            rc = c.four ? scmx_cache4_read(c.bytes(c.k), c.bytes(c.v), c.bytes(c.ks), c.bytes(c.vs), kp, vp, int(c.hk), int(c.d), int(c.rows),
                                           int(row0), int(rows), stream())
                        : scmx_cache_read(codes(c.k), codes(c.v), c.scale(c.ks), c.scale(c.vs), kp, vp, int(c.hk), int(c.d), int(c.rows),
                                          int(row0), int(rows), stream());
        }
        if (rc != SCMX_OK) return status(c.four ? "scmx_cache4_read" : "scmx_cache_read", rc);
        PyObject *pk = THPVariable_Wrap(std::move(k)), *pv = THPVariable_Wrap(std::move(v));
        return Py_BuildValue("(NN)", pk, pv);
    } catch (...) {
        return raised();
    }
}

// cache_keep(caches, path, count, pos): True, or None
PyObject* cache_keep(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        if (n != 4) fail(PyExc_TypeError, "cache_keep takes 4 arguments");
        const at::Tensor *path = local(args[1], at::ScalarType::Int), *count = local(args[2], at::ScalarType::Int);
        const int64_t* dev;
        int64_t pos;
        if (!PyList_CheckExact(args[0]) || !path || !count || count->numel() != 1 || path->numel() > 64 || !position_of(args[3], dev, pos))
            Py_RETURN_NONE;
        const Py_ssize_t layers = PyList_GET_SIZE(args[0]);
        std::vector<uint64_t> pointers;
        pointers.reserve(size_t(layers) * 4);
        CacheTensors c, first{};
        for (Py_ssize_t i = 0; i < layers; ++i) {
            PyObject* t = PyList_GET_ITEM(args[0], i);
            if (!PyTuple_CheckExact(t) || PyTuple_GET_SIZE(t) != 4) Py_RETURN_NONE;
            c = CacheTensors();
            if (!cache_of(PyTuple_GET_ITEM(t, 0), PyTuple_GET_ITEM(t, 1), PyTuple_GET_ITEM(t, 2), PyTuple_GET_ITEM(t, 3), c))
                Py_RETURN_NONE;
            if (i == 0) first = c;
            else if (c.hk != first.hk || c.rows != first.rows || c.d != first.d || !c.ks != !first.ks || c.four != first.four) Py_RETURN_NONE;
            for (const at::Tensor* x : {c.k, c.v, c.ks, c.vs})
                if (x) pointers.push_back(reinterpret_cast<uintptr_t>(x->data_ptr()));
        }
        if (layers < 1 || layers > 1024) Py_RETURN_NONE;
        const auto ints = [](const at::Tensor* t) { return static_cast<const int32_t*>(t->data_ptr()); };
        const int rc = first.four ? scmx_cache4_keep(pointers.data(), int(layers), int(first.hk), int(first.d), int(first.rows), ints(path),
                                                     ints(count), int(path->numel()), dev, pos, stream())
                                  : scmx_cache_keep(pointers.data(), int(layers), first.ks != nullptr, int(first.hk), int(first.d),
                                                    int(first.rows), ints(path), ints(count), int(path->numel()), dev, pos, stream());
        if (rc != SCMX_OK) return status(first.four ? "scmx_cache4_keep" : "scmx_cache_keep", rc);
        Py_RETURN_TRUE;
    } catch (...) {
        return raised();
    }
}

// verify_drafts(logits, tokens, parents, temperature, uniforms, draft, levels): what sc_draft.verify_drafts has left of its arguments
PyObject* verify_drafts(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        if (n != 7) fail(PyExc_TypeError, "verify_drafts takes 7 arguments");
        if (!THPVariable_Check(args[0]) || !PyFloat_Check(args[3]) || !PyLong_CheckExact(args[6])) Py_RETURN_NONE;
        const bool f32 = THPVariable_Unpack(args[0]).scalar_type() == at::ScalarType::Float;
        const at::Tensor *logits = local(args[0], f32 ? at::ScalarType::Float : at::ScalarType::BFloat16),
                         *tokens = local(args[1], at::ScalarType::Long), *parents = local(args[2], at::ScalarType::Int);
        if (!logits || !tokens || !parents || logits->dim() != 2) Py_RETURN_NONE;
        const int64_t T = logits->size(0), V = logits->size(1), levels = as_int(args[6]);
        const float *u, *draft;
        if (T < 1 || T > 64 || V < 1 || V > INT32_MAX || levels < 0 || levels > 16 || tokens->numel() != T || parents->numel() != T ||
            !optional_of(args[4], at::ScalarType::Float, T, u) || !optional_of(args[5], at::ScalarType::Float, T * V, draft))
            Py_RETURN_NONE;
        const size_t need = scmx_verify_workspace(int(T), int(V), int(levels));
        at::Tensor path, count, next;
        int rc;
        {
            const NoGil released;
            path = fresh(*logits, at::ScalarType::Int, {T});
            count = fresh(*logits, at::ScalarType::Int, {1});
            next = fresh(*logits, at::ScalarType::Long, {1});
            const c10::DataPtr work = scratch(need);
            rc = scmx_verify_drafts(static_cast<const int64_t*>(tokens->data_ptr()), static_cast<const int32_t*>(parents->data_ptr()),
                                    logits->data_ptr(), f32, draft, PyFloat_AS_DOUBLE(args[3]), u, static_cast<int32_t*>(path.data_ptr()),
                                    static_cast<int32_t*>(count.data_ptr()), static_cast<int64_t*>(next.data_ptr()), int(T),
                                    int(V), int(levels), work.get(), need, stream());
        }
        if (rc != SCMX_OK) return status("scmx_verify_drafts", rc);
        PyObject *a = THPVariable_Wrap(std::move(path)), *b = THPVariable_Wrap(std::move(count)), *c = THPVariable_Wrap(std::move(next));
        return Py_BuildValue("(NNN)", a, b, c);
    } catch (...) {
        return raised();
    }
}

// ---- microscaled 4-bit values: sc_mx's functions for the operands of every step, in one call as above ------------------------------

// Rows [M, K] of `x` on the current device, K contiguous values each, `ld` apart.
bool rows_of(const at::Tensor& x, int64_t& M, int64_t& K, int64_t& ld) {
    if (!x.is_cuda() || x.get_device() != c10::hip::current_device() || x.dim() != 2) return false;
    M = x.size(0);
    K = x.size(1);
    ld = M > 1 ? x.stride(0) : K;
    return M <= INT32_MAX && K >= 32 && K % 32 == 0 && K <= INT32_MAX && x.stride(1) == 1 && ld >= K;
}
// None, or the weight bf16 [K] of a norm of up to 16384 values.
bool norm_of(PyObject* o, PyObject* eps, int64_t K, const uint16_t*& nw, float& e) {
    nw = nullptr;
    e = 0.0f;
    if (o == Py_None) return true;
    const at::Tensor* t = local(o, at::ScalarType::BFloat16);
    if (!t || t->numel() != K || K > 16384 || !PyFloat_Check(eps)) return false;
    nw = static_cast<const uint16_t*>(t->data_ptr());
    e = float(PyFloat_AS_DOUBLE(eps));
    return true;
}
// codes uint8 [rows, K / 2] and scales uint8 [rows, K / 32].
bool pair_of(PyObject* codes, PyObject* scales, const at::Tensor*& c, const at::Tensor*& s) {
    c = local(codes, at::ScalarType::Byte);
    s = local(scales, at::ScalarType::Byte);
    return c && s && c->dim() == 2 && s->dim() == 2 && c->size(0) == s->size(0) && c->size(1) == 16 * s->size(1) && s->size(1) > 0 &&
           c->size(0) <= INT32_MAX && c->size(1) <= INT32_MAX / 2;
}
uint8_t* bytes(const at::Tensor& t) { return static_cast<uint8_t*>(t.data_ptr()); }

// mx_quantize(x, nw, eps)
PyObject* mx_quantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        if (n != 3) fail(PyExc_TypeError, "mx_quantize takes 3 arguments");
        int64_t M, K, ld;
        const uint16_t* nw;
        float eps;
        if (!THPVariable_Check(args[0])) Py_RETURN_NONE;
        const at::Tensor& x = THPVariable_Unpack(args[0]);
        const at::ScalarType t = x.scalar_type();
        const int type = t == at::ScalarType::BFloat16 ? SCMX_MX_BF16 : t == at::ScalarType::Half ? SCMX_MX_F16 : t == at::ScalarType::Float ? SCMX_MX_F32 : -1;
        if (type < 0 || !rows_of(x, M, K, ld) || !norm_of(args[1], args[2], K, nw, eps) || (nw && type != SCMX_MX_BF16)) Py_RETURN_NONE;
        at::Tensor codes, scales;
        int rc;
        {
            const NoGil released;
            codes = fresh(x, at::ScalarType::Byte, {M, K / 2});
            scales = fresh(x, at::ScalarType::Byte, {M, K / 32});
            rc = scmx_mx_quantize(x.data_ptr(), type, ld, nw, eps, bytes(codes), bytes(scales), int(M), int(K), stream());
        }
        if (rc != SCMX_OK) return status("scmx_mx_quantize", rc);
        PyObject *a = THPVariable_Wrap(std::move(codes)), *b = THPVariable_Wrap(std::move(scales));
        return Py_BuildValue("(NN)", a, b);
    } catch (...) {
        return raised();
    }
}

// mx_dequantize(codes, scales, f32)
PyObject* mx_dequantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        if (n != 3) fail(PyExc_TypeError, "mx_dequantize takes 3 arguments");
        const at::Tensor *codes, *scales;
        if (!PyBool_Check(args[2]) || !pair_of(args[0], args[1], codes, scales)) Py_RETURN_NONE;
        const bool f32 = args[2] == Py_True;
        const int64_t M = codes->size(0), K = 2 * codes->size(1);
        at::Tensor out;
        int rc;
        {
            const NoGil released;
            out = fresh(*codes, f32 ? at::ScalarType::Float : at::ScalarType::BFloat16, {M, K});
            rc = scmx_mx_dequantize(bytes(*codes), bytes(*scales), out.data_ptr(), f32 ? SCMX_MX_F32 : SCMX_MX_BF16, int(M), int(K), stream());
        }
        if (rc != SCMX_OK) return status("scmx_mx_dequantize", rc);
        return THPVariable_Wrap(std::move(out));
    } catch (...) {
        return raised();
    }
}

// mx_mm(xcodes, xscales, wcodes, wscales, epi, res)
PyObject* mx_mm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        if (n != 6) fail(PyExc_TypeError, "mx_mm takes 6 arguments");
        const at::Tensor *xc, *xs, *wc, *ws, *res = nullptr;
        if (!PyLong_CheckExact(args[4]) || !pair_of(args[0], args[1], xc, xs) || !pair_of(args[2], args[3], wc, ws) || xc->size(1) != wc->size(1)) Py_RETURN_NONE;
        const int64_t epi = as_int(args[4]), M = xc->size(0), N = wc->size(0), K = 2 * xc->size(1);
        if (epi < 1 || epi > 3 || N < 1 || (epi == 3 && N % 4)) Py_RETURN_NONE;
        if (epi == 2) {
            res = local(args[5], at::ScalarType::BFloat16);
            if (!res || res->dim() != 2 || res->size(0) != M || res->size(1) != N) Py_RETURN_NONE;
        }
        at::Tensor out;
        int rc;
        {
            const NoGil released;
            out = fresh(*xc, at::ScalarType::BFloat16, {M, epi == 3 ? N / 2 : N});
            rc = scmx_mx_mm(bytes(*xc), bytes(*xs), bytes(*wc), bytes(*ws), res ? static_cast<const uint16_t*>(res->data_ptr()) : nullptr,
                            static_cast<uint16_t*>(out.data_ptr()), int(epi), int(M), int(N), int(K), stream());
        }
        if (rc != SCMX_OK) return status("scmx_mx_mm", rc);
        return THPVariable_Wrap(std::move(out));
    } catch (...) {
        return raised();
    }
}

// mx_linear(x, wcodes, wscales, epi, res, nw, eps)
PyObject* mx_linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        if (n != 7) fail(PyExc_TypeError, "mx_linear takes 7 arguments");
        int64_t M, K, ld;
        const uint16_t* nw;
        float eps;
        const at::Tensor *codes, *scales, *res = nullptr;
        if (!THPVariable_Check(args[0]) || !PyLong_CheckExact(args[3])) Py_RETURN_NONE;
        const at::Tensor& x = THPVariable_Unpack(args[0]);
        const int64_t epi = as_int(args[3]);
        if (x.scalar_type() != at::ScalarType::BFloat16 || !rows_of(x, M, K, ld) || !pair_of(args[1], args[2], codes, scales) ||
            2 * codes->size(1) != K || !norm_of(args[5], args[6], K, nw, eps) || epi < 1 || epi > 3)
            Py_RETURN_NONE;
        const int64_t N = codes->size(0);
        if (N < 1 || (epi == 3 && N % 4)) Py_RETURN_NONE;
        if (epi == 2) {
            res = local(args[4], at::ScalarType::BFloat16);
            if (!res || res->dim() != 2 || res->size(0) != M || res->size(1) != N) Py_RETURN_NONE;
        }
        at::Tensor out;
        int rc;
        {
            const NoGil released;
            out = fresh(x, at::ScalarType::BFloat16, {M, epi == 3 ? N / 2 : N});
            const size_t need = scmx_mx_linear_workspace(int(M), int(N), int(K), nw != nullptr);
            const c10::DataPtr work = scratch(need);
            rc = scmx_mx_linear(static_cast<const uint16_t*>(x.data_ptr()), ld, nw, eps, bytes(*codes), bytes(*scales),
                                res ? static_cast<const uint16_t*>(res->data_ptr()) : nullptr, static_cast<uint16_t*>(out.data_ptr()), int(epi),
                                int(M), int(N), int(K), work.get(), need, stream());
        }
        if (rc != SCMX_OK) return status("scmx_mx_linear", rc);
        return THPVariable_Wrap(std::move(out));
    } catch (...) {
        return raised();
    }
}

#define ENTRY(fn) \
    {#fn, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(((Call<&fn>::name = #fn), &Call<&fn>::call))), METH_FASTCALL, nullptr}
#define QUERY(fn) {#fn, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&Query<&fn>::call)), METH_FASTCALL, nullptr}
#define FUNCTION(fn) {#fn, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&fn)), METH_FASTCALL, nullptr}
#define EMPTY(suffix, type) \
    {"empty_" #suffix, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&empty<at::ScalarType::type>)), METH_FASTCALL, nullptr}

PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, nullptr, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() {
    static PyMethodDef methods[] = {
        ENTRY(scmx_unpack_i8), ENTRY(scmx_act_quant), ENTRY(scmx_act_quant_blocked), ENTRY(scmx_mm_i8_i32), ENTRY(scmx_mm_epi),
        ENTRY(scmx_mm_w4a8), ENTRY(scmx_mm_w4a8_blocked), ENTRY(scmx_linear_w4a8), ENTRY(scmx_linear_w4a8_static),
        ENTRY(scmx_rmsnorm_quant), ENTRY(scmx_rmsnorm_quant_blocked), ENTRY(scmx_rmsnorm), ENTRY(scmx_linear_bf16), ENTRY(scmx_res_norm_quant),
        ENTRY(scmx_swiglu_quant), ENTRY(scmx_qkv_headnorm), ENTRY(scmx_qkv_headnorm_rope), ENTRY(scmx_qkv_fullnorm),
        ENTRY(scmx_qkv_fullnorm_rope), ENTRY(scmx_attn_decode), ENTRY(scmx_attn_decode_qkv), ENTRY(scmx_attn_prefill), ENTRY(scmx_attn_prefill_split),
        ENTRY(scmx_gemv), ENTRY(scmx_gemv_rows), ENTRY(scmx_route_topk), ENTRY(scmx_norm_linear), ENTRY(scmx_route_sort), ENTRY(scmx_moe_mm),
        ENTRY(scmx_moe_mm_i8), ENTRY(scmx_moe_mm_blocked), ENTRY(scmx_moe_gather_blocked), ENTRY(scmx_act_quant_sorted),
        ENTRY(scmx_moe_combine), ENTRY(scmx_moe_combine_blocked), ENTRY(scmx_rot_quant), ENTRY(scmx_mxfp4_to_sc),
        ENTRY(scmx_quantize_sc), ENTRY(scmx_quantize_family),
        QUERY(scmx_linear_w4a8_workspace), QUERY(scmx_gemv_rows_workspace), QUERY(scmx_mm_w4a8_prefers_blocked),
        QUERY(scmx_moe_mm_takes_slots),
        ENTRY(scmx_cache_write), ENTRY(scmx_cache_read), ENTRY(scmx_cache_keep), ENTRY(scmx_attn_tree), ENTRY(scmx_verify_drafts),
        QUERY(scmx_verify_workspace), QUERY(scmx_attn_tree_splits),
        FUNCTION(cache_write), FUNCTION(cache_read), FUNCTION(cache_keep), FUNCTION(attn_tree), FUNCTION(verify_drafts),
        ENTRY(scmx_mx_quantize), ENTRY(scmx_mx_dequantize), ENTRY(scmx_mx_mm), ENTRY(scmx_mx_linear), ENTRY(scmx_cache4_write),
        ENTRY(scmx_cache4_read), ENTRY(scmx_cache4_keep), ENTRY(scmx_attn_tree4), QUERY(scmx_mx_linear_workspace), QUERY(scmx_attn_tree4_splits),
        FUNCTION(mx_quantize), FUNCTION(mx_dequantize), FUNCTION(mx_mm), FUNCTION(mx_linear),
        FUNCTION(gemv),
        EMPTY(bf16, BFloat16), EMPTY(i8, Char), EMPTY(u8, Byte), EMPTY(i32, Int), EMPTY(i64, Long), EMPTY(f32, Float),
        {nullptr, nullptr, 0, nullptr}};
    module_def.m_methods = methods;
    return PyModule_Create(&module_def);
}
