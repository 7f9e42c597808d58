// calls.cpp -- the serving calls' way from Python tensors to the C ABI, for
// operands that need no copy, conversion or error message.
//
// A decode step's kernels take 3 to 10 us; the same checks and address
// arithmetic in Python took 4 to 8 us a call on top of the launch.  Each function
// here answers a call whose operands are exactly what the library reads
// (device tensors of one device that is current, int32 offsets, 16-byte rows) and
// returns None for any other: the Python function behind it then converts,
// copies or raises.  Nothing is kept between calls.
//
// The library's entry points come from bind(), so this module links none of it;
// the current device and stream are asked of torch's own functions.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/Functions.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>

namespace {

using at::Tensor;

// Entry points, in the order in which bind() takes them (include/qattn.h).
using PromptWs = int64_t (*)(int32_t, int32_t, int64_t, int32_t, int32_t, int32_t);
using Prompt = int (*)(const void*, const int64_t*, const void*, const int64_t*, const void*, const int64_t*, void*,
                       const int64_t*, float*, const int64_t*, const int32_t*, int32_t, int32_t, int64_t, int32_t,
                       int32_t, int32_t, float, int32_t, void*, int64_t, void*);
using PagedWs = int64_t (*)(int32_t, int32_t, int64_t, int32_t, int32_t, int32_t, int32_t, int32_t);
using Paged = int (*)(const void*, const int64_t*, const void*, const int64_t*, const void*, const int64_t*,
                      const int32_t*, int32_t, int32_t, int32_t, const int32_t*, void*, const int64_t*, float*,
                      const int64_t*, const int32_t*, int32_t, int32_t, int64_t, int32_t, int32_t, int32_t, float,
                      int32_t, void*, int64_t, void*);
using Append = int (*)(const void*, const int64_t*, const void*, const int64_t*, void*, const int64_t*, void*,
                       const int64_t*, const int32_t*, int32_t, int32_t, int32_t, const int32_t*, int32_t*,
                       const int32_t*, int32_t, int32_t, int64_t, int32_t, int32_t, int32_t, void*);
using Compact = int (*)(void*, const int64_t*, void*, const int64_t*, int32_t, const int32_t*, int32_t, int32_t,
                        int32_t, const int32_t*, const int32_t*, int32_t, int32_t*, int32_t, int32_t, int32_t, int32_t,
                        void*);
using Copy = int (*)(void*, const int64_t*, void*, const int64_t*, int32_t, int32_t, int32_t, const int32_t*,
                     const int32_t*, int32_t, int32_t, int32_t, int32_t, void*);

using QuantWs = int64_t (*)(int32_t, int32_t, int64_t, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t);
using Quant = int (*)(const void*, const int64_t*, const void*, const void*, const int64_t*, const void*, const void*,
                      const int64_t*, const int32_t*, int32_t, int32_t, int32_t, const int32_t*, void*, const int64_t*,
                      float*, const int64_t*, const int32_t*, int32_t, int32_t, int64_t, int32_t, int32_t, int32_t,
                      float, int32_t, int32_t, void*, int64_t, void*);
using QuantAppend = int (*)(const void*, const int64_t*, const void*, const int64_t*, void*, void*, const int64_t*,
                            void*, void*, const int64_t*, const int32_t*, int32_t, int32_t, int32_t, const int32_t*,
                            int32_t*, const int32_t*, int32_t, int32_t, int64_t, int32_t, int32_t, int32_t, int32_t,
                            void*);
using QuantRead = int (*)(const void*, const void*, const int64_t*, const void*, const void*, const int64_t*,
                          const int32_t*, int32_t, int32_t, int32_t, const int32_t*, void*, const int64_t*, void*,
                          const int64_t*, const int32_t*, int32_t, int32_t, int64_t, int32_t, int32_t, int32_t, int32_t,
                          void*);

PromptWs prompt_ws;
Prompt prompt_fwd;
PagedWs paged_ws;
Paged paged_fwd;
Append kv_append;
Compact kv_compact;
Copy kv_copy;
QuantWs quant_ws;
Quant quant_fwd;
QuantAppend quant_append_rows;
QuantRead quant_read_rows;
PyObject *current_device, *current_stream;  // torch._C functions
uint64_t ready;                             // bit d: qattn_init ran on device d

constexpr int64_t kInt = INT32_MAX;

// A call's device: that of its first tensor, current and set up.
struct Call {
    int device = -1;
    at::ScalarType type = at::ScalarType::Undefined;
    void* stream = nullptr;

    // A tensor that the call may read as it is.
    bool plain(PyObject* o, const Tensor*& t) {
        if (!THPVariable_CheckExact(o)) return false;
        t = &THPVariable_Unpack(o);
        if (!t->is_cuda() || t->layout() != at::kStrided || t->requires_grad()) return false;
        if (t->_fw_grad(0).defined()) return false;  // (a tangent; there is one level only)
        const int d = t->get_device();
        if (device < 0) device = d;
        return d == device;
    }
    // fp16 or bf16 rows on 16-byte boundaries, of the call's one type.
    bool rows(PyObject* o, int64_t dim, const Tensor*& t) {
        if (!plain(o, t) || t->dim() != dim || !t->numel()) return false;
        if (type == at::ScalarType::Undefined) type = t->scalar_type();
        if (t->scalar_type() != type || (type != at::kHalf && type != at::kBFloat16)) return false;
        return aligned(*t);
    }
    static bool aligned(const Tensor& t) {
        const auto st = t.strides();
        int64_t outer = 0;
        for (size_t i = 0; i + 1 < st.size(); ++i) outer |= st[i];
        return st.back() == 1 && !(outer & 7) && !((uintptr_t)t.data_ptr() & 15);
    }
    // Runs of bytes of a quantised cache.
    bool bytes(PyObject* o, int64_t dim, const Tensor*& t) {
        type = at::kByte;
        return plain(o, t) && t->dim() == dim && t->numel() && t->scalar_type() == at::kByte &&
               t->strides().back() == 1;
    }
    // Caches that are written: of one shape, no stride of 0, not the same memory.
    bool caches(PyObject* ok, PyObject* ov, int64_t dim, const Tensor*& k, const Tensor*& v, bool u8 = false) {
        if (!(u8 ? bytes(ok, dim, k) && bytes(ov, dim, v) : rows(ok, dim, k) && rows(ov, dim, v)) ||
            k->sizes() != v->sizes() || k->data_ptr() == v->data_ptr())
            return false;
        for (const Tensor* t : {k, v})
            for (int64_t s : t->strides())
                if (!s) return false;
        for (int64_t n : k->sizes())
            if (n > kInt) return false;
        return true;
    }
    bool ints(PyObject* o, int64_t dim, const Tensor*& t) {
        return plain(o, t) && t->dim() == dim && t->scalar_type() == at::kInt && t->is_contiguous();
    }
    // The device is the current one and set up; its current stream.
    bool here() {
        if (device < 0 || device > 63 || !(ready >> device & 1)) return false;
        PyObject* d = PyObject_CallNoArgs(current_device);
        if (!d) return PyErr_Clear(), false;
        const long cur = PyLong_AsLong(d);
        if (cur != device) return Py_DECREF(d), false;
        PyObject* s = PyObject_CallOneArg(current_stream, d);
        Py_DECREF(d);
        if (!s) return PyErr_Clear(), false;
        stream = PyLong_AsVoidPtr(s);
        Py_DECREF(s);
        if (PyErr_Occurred()) return PyErr_Clear(), false;
        return true;
    }
    // QATTN_DTYPE_F16, _BF16, _U8
    int32_t code() const { return type == at::kHalf ? 0 : type == at::kByte ? 2 : 1; }
    at::TensorOptions options(at::ScalarType t) const {
        return at::TensorOptions().dtype(t).device(at::Device(at::kCUDA, (at::DeviceIndex)device));
    }
};

int64_t* strides5(const Tensor& t, int64_t (&st)[5]) {
    const auto s = t.strides();
    const bool all = s.size() == 5;
    st[0] = all ? s[0] : 0;
    for (int i = 0; i < 4; ++i) st[i + 1] = s[i + all];
    return st;
}

// A quantised cache (a tuple of K, V, K_scale, V_scale) that the library reads as it is.
struct Quantized {
    const Tensor *K, *V, *Ks, *Vs;
    int32_t pages, page_size, heads, dim, bits;
    int64_t cs[4], ss[4];

    bool take(Call& c, PyObject* o, bool written) {
        if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) return false;
        const Tensor** at[4] = {&K, &V, &Ks, &Vs};
        for (int i = 0; i < 4; ++i) {
            if (!c.plain(PyTuple_GET_ITEM(o, i), *at[i])) return false;
            const Tensor& t = **at[i];
            if (t.scalar_type() != at::kByte || t.dim() != 4 || !t.numel()) return false;
        }
        for (int i = 0; i < 3; ++i)
            if (K->size(i) != Ks->size(i) || K->size(i) > kInt) return false;
        const int64_t D = 32 * Ks->size(3), width = K->size(3);
        if ((D != 32 && D != 64 && D != 128) || (8 * width != 4 * D && 8 * width != 8 * D)) return false;
        if (!pair(*K, *V, 16, written, cs) || !pair(*Ks, *Vs, D / 32, written, ss)) return false;
        pages = (int32_t)K->size(0), page_size = (int32_t)K->size(1), heads = (int32_t)K->size(2), dim = (int32_t)D;
        bits = (int32_t)(8 * width / D);
        return true;
    }

private:
    // Two tensors laid out alike in rows on `unit`-byte boundaries, if written each in
    // memory of its own.
    static bool pair(const Tensor& a, const Tensor& b, int64_t unit, bool written, int64_t (&st)[4]) {
        const auto s = a.strides();
        if (a.sizes() != b.sizes() || s != b.strides() || (s[3] != 1 && a.size(3) > 1)) return false;
        const uintptr_t x = (uintptr_t)a.data_ptr(), y = (uintptr_t)b.data_ptr();
        if ((s[0] | s[1] | s[2]) & (unit - 1) || (x | y) & (uintptr_t)(unit - 1)) return false;
        if (written && (x == y || !s[0] || !s[1] || !s[2])) return false;
        st[0] = s[0], st[1] = s[1], st[2] = s[2], st[3] = 1;
        return true;
    }
};

// An int argument in [0, 2^31); false for anything else.
bool small_int(PyObject* o, int32_t& v) {
    if (!PyLong_CheckExact(o)) return false;
    const long x = PyLong_AsLong(o);
    if (x == -1 && PyErr_Occurred()) return PyErr_Clear(), false;
    if (x < 0 || x > kInt) return false;
    v = (int32_t)x;
    return true;
}

// Offsets of packed rows, or none: row s is sequence s's.
bool offsets(Call& c, PyObject* ocu, PyObject* oms, int64_t T, int64_t B, const int32_t*& cu, int32_t& ms) {
    if (ocu == Py_None) {
        cu = nullptr, ms = 1;
        return T == B;
    }
    const Tensor* t;
    if (!c.ints(ocu, 1, t) || t->size(0) != B + 1 || !small_int(oms, ms)) return false;
    cu = t->data_ptr<int32_t>();
    return true;
}

// O like Q (nothing is returned for a layout that the kernels cannot write), and LSE.
bool outputs(const Call& c, const Tensor& Q, bool want_lse, Tensor& O, Tensor& LSE) {
    O = at::empty_like(Q);
    if (!Call::aligned(O)) return false;
    if (want_lse) LSE = at::empty({Q.size(0), Q.size(1)}, c.options(at::kFloat));
    return true;
}

PyObject* wrap(const Tensor& O, const Tensor& LSE, bool want_lse) {
    PyObject* o = THPVariable_Wrap(O);
    if (!want_lse || !o) return o;
    PyObject* l = THPVariable_Wrap(LSE);
    if (!l) return Py_DECREF(o), nullptr;
    PyObject* both = PyTuple_New(2);
    if (!both) return Py_DECREF(o), Py_DECREF(l), nullptr;
    PyTuple_SET_ITEM(both, 0, o);
    PyTuple_SET_ITEM(both, 1, l);
    return both;
}

// While it lives other Python threads run: a launch waits where the stream's queue is
// full, an allocation where memory has to be freed first.  (Operands are held by the
// caller's frame.)
class Unlocked {
    PyThreadState* state_ = PyEval_SaveThread();

public:
    Unlocked() = default;
    Unlocked(const Unlocked&) = delete;
    Unlocked& operator=(const Unlocked&) = delete;
    ~Unlocked() { PyEval_RestoreThread(state_); }
};

PyObject* none() { Py_RETURN_NONE; }

// C++ exceptions (an allocation that fails) end here: the Python function
// makes the same call and raises.
template <class F>
PyObject* guarded(F f) {
    try {
        return f();
    } catch (...) {
        PyErr_Clear();
        return none();
    }
}

// prompt(Q, K, V, cu_seqlens, max_seqlen, return_lse)
PyObject* prompt(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Call c;
        const Tensor *Q, *K, *V, *cu;
        int32_t ms;
        if (n != 6 || !c.rows(a[0], 3, Q) || !c.rows(a[1], 3, K) || !c.rows(a[2], 3, V) || !c.ints(a[3], 1, cu) ||
            !small_int(a[4], ms) || !PyBool_Check(a[5]) || cu->size(0) < 2)
            return none();
        const int64_t T = Q->size(0), Hq = Q->size(1), D = Q->size(2), Hkv = K->size(1);
        if (K->sizes() != V->sizes() || K->size(0) != T || K->size(2) != D || Hq % Hkv || T > kInt || Hq > kInt ||
            !c.here())
            return none();
        const bool want = a[5] == Py_True;
        const int32_t B = (int32_t)cu->size(0) - 1;
        Tensor O, LSE;
        const int rc = [&] {
            Unlocked others;
            const int64_t bytes = prompt_ws(B, ms, T, (int32_t)Hq, (int32_t)Hkv, (int32_t)D);
            if (!outputs(c, *Q, want, O, LSE)) return -1;
            Tensor ws;
            if (bytes) ws = at::empty({bytes}, c.options(at::kByte));
            return prompt_fwd(Q->data_ptr(), Q->strides().data(), K->data_ptr(), K->strides().data(), V->data_ptr(),
                              V->strides().data(), O.data_ptr(), O.strides().data(),
                              want ? LSE.data_ptr<float>() : nullptr, want ? LSE.strides().data() : nullptr,
                              cu->data_ptr<int32_t>(), B, ms, T, (int32_t)Hq, (int32_t)Hkv, (int32_t)D,
                              (float)(1.0 / std::sqrt((double)D)), c.code(), bytes ? ws.data_ptr() : nullptr, bytes,
                              c.stream);
        }();
        return rc ? none() : wrap(O, LSE, want);
    });
}

// paged(Q, K_cache, V_cache, page_table, context_lens, cu_seqlens, max_seqlen, return_lse)
PyObject* paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Call c;
        const Tensor *Q, *K, *V, *table, *ctx;
        if (n != 8 || !c.rows(a[0], 3, Q) || !c.rows(a[1], 4, K) || !c.rows(a[2], 4, V) || !c.ints(a[3], 2, table) ||
            !c.ints(a[4], 1, ctx) || !PyBool_Check(a[7]))
            return none();
        const int64_t T = Q->size(0), Hq = Q->size(1), D = Q->size(2), Hkv = K->size(2), B = ctx->size(0);
        const int32_t* cu;
        int32_t ms;
        if (K->sizes() != V->sizes() || K->size(3) != D || Hq % Hkv || table->size(0) < B || T > kInt || Hq > kInt ||
            B > kInt || table->size(1) > kInt || K->size(0) > kInt || K->size(1) > kInt ||
            !offsets(c, a[5], a[6], T, B, cu, ms) || !c.here())
            return none();
        const bool want = a[7] == Py_True;
        const int32_t cols = (int32_t)table->size(1), ps = (int32_t)K->size(1);
        Tensor O, LSE;
        const int rc = [&] {
            Unlocked others;
            const int64_t bytes = paged_ws((int32_t)B, ms, T, (int32_t)Hq, (int32_t)Hkv, (int32_t)D, cols, ps);
            if (!outputs(c, *Q, want, O, LSE)) return -1;
            Tensor ws;
            if (bytes) ws = at::empty({bytes}, c.options(at::kByte));
            return paged_fwd(Q->data_ptr(), Q->strides().data(), K->data_ptr(), K->strides().data(), V->data_ptr(),
                             V->strides().data(), table->data_ptr<int32_t>(), cols, (int32_t)K->size(0), ps,
                             ctx->data_ptr<int32_t>(), O.data_ptr(), O.strides().data(),
                             want ? LSE.data_ptr<float>() : nullptr, want ? LSE.strides().data() : nullptr, cu,
                             (int32_t)B, ms, T, (int32_t)Hq, (int32_t)Hkv, (int32_t)D,
                             (float)(1.0 / std::sqrt((double)D)), c.code(), bytes ? ws.data_ptr() : nullptr, bytes,
                             c.stream);
        }();
        return rc ? none() : wrap(O, LSE, want);
    });
}

// append(K, V, K_cache, V_cache, page_table, context_lens, cu_seqlens, max_seqlen)
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Call c;
        const Tensor *K, *V, *Kc, *Vc, *table, *ctx;
        if (n != 8 || !c.rows(a[0], 3, K) || !c.rows(a[1], 3, V) || !c.caches(a[2], a[3], 4, Kc, Vc) ||
            !c.ints(a[4], 2, table) || !c.ints(a[5], 1, ctx))
            return none();
        const int64_t T = K->size(0), B = ctx->size(0);
        const int32_t* cu;
        int32_t ms;
        if (K->sizes() != V->sizes() || K->size(1) != Kc->size(2) || K->size(2) != Kc->size(3) || table->size(0) < B ||
            T > kInt || B > kInt || table->size(1) > kInt || !offsets(c, a[6], a[7], T, B, cu, ms) || !c.here())
            return none();
        int64_t ks[5], vs[5];
        Tensor after;
        const int rc = [&] {
            Unlocked others;
            after = at::empty_like(*ctx);
            return kv_append(K->data_ptr(), K->strides().data(), V->data_ptr(), V->strides().data(), Kc->data_ptr(),
                             strides5(*Kc, ks), Vc->data_ptr(), strides5(*Vc, vs), table->data_ptr<int32_t>(),
                             (int32_t)table->size(1), (int32_t)Kc->size(0), (int32_t)Kc->size(1),
                             ctx->data_ptr<int32_t>(), after.data_ptr<int32_t>(), cu, (int32_t)B, ms, T,
                             (int32_t)Kc->size(2), (int32_t)Kc->size(3), c.code(), c.stream);
        }();
        return rc ? none() : THPVariable_Wrap(after);
    });
}

// compact(K_cache, V_cache, page_table, context_lens, accepted)
PyObject* compact(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Call c;
        const Tensor *Kc, *Vc, *table, *ctx, *path;
        if (n != 5 || !THPVariable_CheckExact(a[0])) return none();
        const int64_t dim = THPVariable_Unpack(a[0]).dim();
        const bool u8 = THPVariable_Unpack(a[0]).scalar_type() == at::kByte;
        if ((dim != 4 && dim != 5) || !c.caches(a[0], a[1], dim, Kc, Vc, u8) || !c.ints(a[2], 2, table) ||
            !c.ints(a[3], 1, ctx) || !c.ints(a[4], 2, path))
            return none();
        const int64_t B = ctx->size(0);
        if (table->size(0) < B || path->size(0) != B || B > kInt || table->size(1) > kInt || path->size(1) > kInt ||
            !c.here())
            return none();
        int64_t ks[5], vs[5];
        const int64_t layers = dim == 5 ? Kc->size(0) : 1, o = dim - 4;
        Tensor after;
        const int rc = [&] {
            Unlocked others;
            after = at::empty_like(*ctx);
            return kv_compact(Kc->data_ptr(), strides5(*Kc, ks), Vc->data_ptr(), strides5(*Vc, vs), (int32_t)layers,
                              table->data_ptr<int32_t>(), (int32_t)table->size(1), (int32_t)Kc->size(o),
                              (int32_t)Kc->size(o + 1), ctx->data_ptr<int32_t>(), path->data_ptr<int32_t>(),
                              (int32_t)path->size(1), after.data_ptr<int32_t>(), (int32_t)B, (int32_t)Kc->size(o + 2),
                              (int32_t)Kc->size(o + 3), c.code(), c.stream);
        }();
        return rc ? none() : THPVariable_Wrap(after);
    });
}

// copy(K_cache, V_cache, src_pages, dst_pages): True where the copies were launched
PyObject* copy(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Call c;
        const Tensor *Kc, *Vc, *src, *dst;
        if (n != 4 || !THPVariable_CheckExact(a[0])) return none();
        const int64_t dim = THPVariable_Unpack(a[0]).dim();
        const bool u8 = THPVariable_Unpack(a[0]).scalar_type() == at::kByte;
        if ((dim != 4 && dim != 5) || !c.caches(a[0], a[1], dim, Kc, Vc, u8) || !c.ints(a[2], 1, src) ||
            !c.ints(a[3], 1, dst) || src->size(0) != dst->size(0) || src->size(0) > kInt || !c.here())
            return none();
        int64_t ks[5], vs[5];
        const int64_t layers = dim == 5 ? Kc->size(0) : 1, o = dim - 4;
        const int rc = [&] {
            Unlocked others;
            return kv_copy(Kc->data_ptr(), strides5(*Kc, ks), Vc->data_ptr(), strides5(*Vc, vs), (int32_t)layers,
                           (int32_t)Kc->size(o), (int32_t)Kc->size(o + 1), src->data_ptr<int32_t>(),
                           dst->data_ptr<int32_t>(), (int32_t)src->size(0), (int32_t)Kc->size(o + 2),
                           (int32_t)Kc->size(o + 3), c.code(), c.stream);
        }();
        if (rc) return none();
        Py_RETURN_TRUE;
    });
}

// quant_append(K, V, cache, page_table, context_lens, cu_seqlens, max_seqlen)
PyObject* quant_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Call c;
        Quantized q;
        const Tensor *K, *V, *table, *ctx;
        if (n != 7 || !quant_fwd || !c.rows(a[0], 3, K) || !c.rows(a[1], 3, V) || !q.take(c, a[2], true) ||
            !c.ints(a[3], 2, table) || !c.ints(a[4], 1, ctx))
            return none();
        const int64_t T = K->size(0), B = ctx->size(0);
        const int32_t* cu;
        int32_t ms;
        if (K->sizes() != V->sizes() || K->size(1) != q.heads || K->size(2) != q.dim || table->size(0) < B ||
            T > kInt || B > kInt || table->size(1) > kInt || !offsets(c, a[5], a[6], T, B, cu, ms) || !c.here())
            return none();
        Tensor after;
        const int rc = [&] {
            Unlocked others;
            after = at::empty_like(*ctx);
            return quant_append_rows(K->data_ptr(), K->strides().data(), V->data_ptr(), V->strides().data(),
                                     q.K->data_ptr(), q.V->data_ptr(), q.cs, q.Ks->data_ptr(), q.Vs->data_ptr(), q.ss,
                                     table->data_ptr<int32_t>(), (int32_t)table->size(1), q.pages, q.page_size,
                                     ctx->data_ptr<int32_t>(), after.data_ptr<int32_t>(), cu, (int32_t)B, ms, T,
                                     q.heads, q.dim, c.code(), q.bits, c.stream);
        }();
        return rc ? none() : THPVariable_Wrap(after);
    });
}

// quant_read(cache, page_table, starts, cu_seqlens, max_seqlen, total_tokens, dtype)
PyObject* quant_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Call c;
        Quantized q;
        const Tensor *table, *start;
        if (n != 7 || !quant_fwd || !q.take(c, a[0], false) || !c.ints(a[1], 2, table) || !c.ints(a[2], 1, start) ||
            !THPDtype_Check(a[6]))
            return none();
        c.type = reinterpret_cast<THPDtype*>(a[6])->scalar_type;
        const int64_t B = start->size(0);
        const int32_t* cu;
        int32_t ms, T = (int32_t)std::min(B, kInt);
        if ((c.type != at::kHalf && c.type != at::kBFloat16) || table->size(0) < B || B > kInt ||
            table->size(1) > kInt || !offsets(c, a[3], a[4], B, B, cu, ms) ||
            !(cu ? small_int(a[5], T) : a[5] == Py_None || (small_int(a[5], T) && T == B)) || !c.here())
            return none();
        Tensor K, V;
        const int rc = [&] {
            Unlocked others;
            K = at::empty({T, q.heads, q.dim}, c.options(c.type));
            V = at::empty({T, q.heads, q.dim}, c.options(c.type));
            return quant_read_rows(q.K->data_ptr(), q.V->data_ptr(), q.cs, q.Ks->data_ptr(), q.Vs->data_ptr(), q.ss,
                                   table->data_ptr<int32_t>(), (int32_t)table->size(1), q.pages, q.page_size,
                                   start->data_ptr<int32_t>(), K.data_ptr(), K.strides().data(), V.data_ptr(),
                                   V.strides().data(), cu, (int32_t)B, ms, T, q.heads, q.dim, c.code(), q.bits,
                                   c.stream);
        }();
        return rc ? none() : wrap(K, V, true);
    });
}

// quant_paged(Q, cache, page_table, context_lens, cu_seqlens, max_seqlen, return_lse)
PyObject* quant_paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Call c;
        Quantized q;
        const Tensor *Q, *table, *ctx;
        if (n != 7 || !quant_fwd || !c.rows(a[0], 3, Q) || !q.take(c, a[1], false) || !c.ints(a[2], 2, table) ||
            !c.ints(a[3], 1, ctx) || !PyBool_Check(a[6]))
            return none();
        const int64_t T = Q->size(0), Hq = Q->size(1), B = ctx->size(0);
        const int32_t* cu;
        int32_t ms;
        if (Q->size(2) != q.dim || Hq % q.heads || table->size(0) < B || T > kInt || Hq > kInt || B > kInt ||
            table->size(1) > kInt || !offsets(c, a[4], a[5], T, B, cu, ms) || !c.here())
            return none();
        const bool want = a[6] == Py_True;
        const int32_t cols = (int32_t)table->size(1);
        Tensor O, LSE;
        const int rc = [&] {
            Unlocked others;
            const int64_t bytes = quant_ws((int32_t)B, ms, T, (int32_t)Hq, q.heads, q.dim, cols, q.page_size, q.bits);
            if (!outputs(c, *Q, want, O, LSE)) return -1;
            Tensor ws;
            if (bytes) ws = at::empty({bytes}, c.options(at::kByte));
            return quant_fwd(Q->data_ptr(), Q->strides().data(), q.K->data_ptr(), q.V->data_ptr(), q.cs,
                             q.Ks->data_ptr(), q.Vs->data_ptr(), q.ss, table->data_ptr<int32_t>(), cols, q.pages,
                             q.page_size, ctx->data_ptr<int32_t>(), O.data_ptr(), O.strides().data(),
                             want ? LSE.data_ptr<float>() : nullptr, want ? LSE.strides().data() : nullptr, cu,
                             (int32_t)B, ms, T, (int32_t)Hq, q.heads, q.dim, (float)(1.0 / std::sqrt((double)q.dim)),
                             c.code(), q.bits, bytes ? ws.data_ptr() : nullptr, bytes, c.stream);
        }();
        return rc ? none() : wrap(O, LSE, want);
    });
}

// n addresses of entry points; false with an error set where one is none.
bool addresses(PyObject* const* a, int n, void** at) {
    for (int i = 0; i < n; ++i) {
        at[i] = PyLong_AsVoidPtr(a[i]);
        if (!at[i]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null entry point");
            return false;
        }
    }
    return true;
}

// bind(addresses of the seven entry points, torch's current-device and
// current-raw-stream functions)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    void* at[7];
    if (n != 9) {
        PyErr_SetString(PyExc_TypeError, "bind takes seven addresses and two functions");
        return nullptr;
    }
    if (!addresses(a, 7, at)) return nullptr;
    prompt_ws = (PromptWs)at[0], prompt_fwd = (Prompt)at[1], paged_ws = (PagedWs)at[2], paged_fwd = (Paged)at[3];
    kv_append = (Append)at[4], kv_compact = (Compact)at[5], kv_copy = (Copy)at[6];
    Py_INCREF(a[7]);
    Py_INCREF(a[8]);
    Py_XDECREF(current_device);
    Py_XDECREF(current_stream);
    current_device = a[7], current_stream = a[8];
    return none();
}

// bind_quantized(addresses of the four entry points over a quantised cache)
PyObject* bind_quantized(PyObject*, PyObject* const* a, Py_ssize_t n) {
    void* at[4];
    if (n != 4) {
        PyErr_SetString(PyExc_TypeError, "bind_quantized takes four addresses");
        return nullptr;
    }
    if (!addresses(a, 4, at)) return nullptr;
    quant_ws = (QuantWs)at[0], quant_fwd = (Quant)at[1], quant_append_rows = (QuantAppend)at[2];
    quant_read_rows = (QuantRead)at[3];
    return none();
}

// set_ready(device): qattn_init has run there
PyObject* set_ready(PyObject*, PyObject* d) {
    const long i = PyLong_AsLong(d);
    if (i == -1 && PyErr_Occurred()) return nullptr;
    if (prompt_fwd && i >= 0 && i < 64) ready |= uint64_t(1) << i;
    return none();
}

#define FAST(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(prompt),       FAST(paged),      FAST(append),      FAST(compact), FAST(copy),
                         FAST(quant_append), FAST(quant_read), FAST(quant_paged), FAST(bind), FAST(bind_quantized),
                         {"set_ready", set_ready, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() { return PyModule_Create(&module); }
