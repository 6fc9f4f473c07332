// The decoder-step calls of docc_b200.ops for torch tensors, without the interpreter between the checks.
//
// On the device these calls take two to twenty microseconds; the Python form spends ten to fifteen on asking tensors for their
// properties, allocating outputs and converting arguments. This module does the same for the ordinary call: every array a plain torch
// tensor on the calling thread's CUDA device, types and shapes as documented. Anything else (host arrays, DeviceArrays, subclasses,
// arguments that have to be refused, a captured call that needs scratch of its own) is answered with None, and ops takes its own path,
// which checks again, names what is wrong and raises. So nothing here decides what is allowed, only what is common. A call that the entry
// refused (invalid argument, unsupported) has launched nothing and may be repeated; any other status raises here, since its kernel may be
// queued already.
//
// The entries are reached through the addresses that ops binds, those of the runtime library it has loaded.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ops/empty.h>
#include <c10/core/impl/VirtualGuardImpl.h>

#include <cmath>

#include "docc_b200/rt.h"

namespace {

decltype(&docc_b200_rmsnorm) f_rmsnorm;
decltype(&docc_b200_rmsnorm_q8) f_rmsnorm_q8;
decltype(&docc_b200_rope) f_rope;
decltype(&docc_b200_rope_append) f_rope_append;
decltype(&docc_b200_paged_attention) f_paged_attention;
decltype(&docc_b200_token_logprobs) f_token_logprobs;

PyObject* check;  // check(status, name) raises

using at::Tensor;

c10::DeviceIndex current_device() {
    static const c10::impl::VirtualGuardImpl guard(c10::DeviceType::CUDA);
    return guard.getDevice().index();
}

// The calling thread's device, if the first argument is a CUDA tensor (a process without one is not asked).
bool device_for(PyObject* first, c10::DeviceIndex& device) {
    if (!THPVariable_CheckExact(first) || !THPVariable_Unpack(first).is_cuda()) return false;
    device = current_device();
    return true;
}
// The tensor behind an argument if the fast path takes it, else nullptr.
const Tensor* plain(PyObject* o, c10::DeviceIndex device) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || t.layout() != c10::kStrided || !t.is_cuda() || t.device().index() != device || t.is_neg() || t.is_conj()) return nullptr;
    return &t;
}
int precision(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return DOCC_B200_PREC_S;
        case at::kHalf: return DOCC_B200_PREC_H;
        case at::kBFloat16: return DOCC_B200_PREC_B;
        default: return 0;
    }
}
bool vector_of(const Tensor& t, at::ScalarType type, int64_t n) {
    return t.scalar_type() == type && t.dim() == 1 && t.size(0) == n && t.is_contiguous();
}
// Rows over the last dimension: contiguous, or a 2-D view whose rows are.
bool rows_of(const Tensor& t, int64_t& rows, int64_t& cols, int64_t& ld) {
    if (t.dim() == 0) return false;
    cols = t.size(-1);
    rows = 1;
    for (int64_t d = 0; d + 1 < t.dim(); d++) rows *= t.size(d);
    ld = cols;
    if (t.is_contiguous()) return true;
    if (t.dim() != 2 || t.stride(1) != 1 || t.stride(0) < cols) return false;
    ld = t.stride(0);
    return true;
}
// Strides of [a, b, D] or [a, b, c, D] with contiguous D; none of them 0, which for a tensor that is written would have to be refused.
struct Strides {
    int64_t s[3];
    const int64_t* of = nullptr;
    bool take(const Tensor& t) {
        if (t.is_contiguous()) return true;
        const int64_t last = t.dim() - 1;
        if (t.stride(last) != 1) return false;
        for (int64_t d = 0; d < last; d++) {
            s[d] = t.stride(d);
            if (s[d] <= 0) return false;
        }
        of = s;
        return true;
    }
};
bool number(PyObject* o, double& v) {
    v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}
bool whole(PyObject* o, int64_t& v) {
    if (!PyLong_Check(o)) return false;
    v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}
PyObject* tuple_of(std::initializer_list<Tensor> ts) {
    PyObject* out = PyTuple_New(Py_ssize_t(ts.size()));
    if (!out) return nullptr;
    Py_ssize_t i = 0;
    for (const Tensor& t : ts) {
        PyObject* w = THPVariable_Wrap(t);
        if (!w) {
            Py_DECREF(out);
            return nullptr;
        }
        PyTuple_SET_ITEM(out, i++, w);
    }
    return out;
}
Tensor empty(c10::IntArrayRef shape, const Tensor& like, at::ScalarType type) { return at::empty(shape, like.options().dtype(type).requires_grad(false)); }
Tensor empty_like(const Tensor& t) { return empty(t.sizes(), t, t.scalar_type()); }

// The memory of a call's arguments, kept while the interpreter's lock is given up: another thread may give a tensor other memory then
// (resize_, set_), and what it had must not be handed out before the kernel that reads it is queued.
class Held {
    c10::SmallVector<c10::Storage, 9> storages;

public:
    Held(std::initializer_list<const Tensor*> tensors) {
        for (const Tensor* t : tensors)
            if (t) storages.push_back(t->storage());
    }
    template <size_t N> Held(const Tensor* const (&tensors)[N], const Tensor* more) {
        for (const Tensor* t : tensors) storages.push_back(t->storage());
        if (more) storages.push_back(more->storage());
    }
};
class Unlocked {
    PyThreadState* const thread = PyEval_SaveThread();

public:
    ~Unlocked() { PyEval_RestoreThread(thread); }
};
// The entry with the interpreter's lock given up: it may wait, for a stream when its scratch grows or for room in a launch queue. Its
// arguments have been taken from the tensors before.
template <typename F, typename... Args> int unlocked(const Held&, F entry, Args... args) {
    const Unlocked lock;
    return entry(args...);
}
// The answer to a status other than OK.
PyObject* refused(int status, const char* name) {
    if (status == DOCC_B200_ERR_INVALID_ARG || status == DOCC_B200_ERR_UNSUPPORTED) Py_RETURN_NONE;
    PyObject* r = PyObject_CallFunction(check, "is", status, name);
    if (r) {
        Py_DECREF(r);
        PyErr_Format(PyExc_RuntimeError, "%s failed with status %d", name, status);
    }
    return nullptr;
}

// rmsnorm(X, gamma, residual, eps) and rmsnorm_quant(X, gamma, residual, eps, group)
PyObject* norm(PyObject* const* args, Py_ssize_t n, bool quant) {
    HANDLE_TH_ERRORS
    c10::DeviceIndex device;
    if (n != (quant ? 5 : 4) || !device_for(args[0], device)) Py_RETURN_NONE;
    const Tensor* x = plain(args[0], device);
    const Tensor* g = args[1] == Py_None ? nullptr : plain(args[1], device);
    const Tensor* r = args[2] == Py_None ? nullptr : plain(args[2], device);
    int64_t rows, cols, ldx, ldr = 0, rr, rc, group = 0;
    double eps;
    if (!x || (!g && args[1] != Py_None) || (!r && args[2] != Py_None) || !precision(*x) || !rows_of(*x, rows, cols, ldx) || !number(args[3], eps))
        Py_RETURN_NONE;
    if (g && !vector_of(*g, at::kFloat, cols)) Py_RETURN_NONE;
    if (r && (r->scalar_type() != x->scalar_type() || r->sizes() != x->sizes() || !rows_of(*r, rr, rc, ldr))) Py_RETURN_NONE;
    if (quant && (!whole(args[4], group) || (group != 0 && group != 128))) Py_RETURN_NONE;
    const Held held{x, g, r};
    Tensor s;
    if (r) s = empty_like(*x);
    void* gp = g ? g->data_ptr() : nullptr;
    void* rp = r ? r->data_ptr() : nullptr;
    void* sp = r ? s.data_ptr() : nullptr;
    if (!quant) {
        const Tensor y = empty_like(*x);
        const int status = unlocked(held, f_rmsnorm, precision(*x), rows, cols, x->data_ptr(), ldx, rp, ldr, gp, eps, sp, y.data_ptr(), 0);
        if (status != DOCC_B200_OK) return refused(status, "docc_b200_rmsnorm");
        return r ? tuple_of({y, s}) : THPVariable_Wrap(y);
    }
    c10::SmallVector<int64_t, 5> shape(x->sizes().begin(), x->sizes().end());
    shape.back() = group ? (cols + group - 1) / group : 1;
    const Tensor q = empty(x->sizes(), *x, at::kFloat8_e4m3fn), scales = empty(shape, *x, at::kFloat);
    const int status = unlocked(held, f_rmsnorm_q8, precision(*x), rows, cols, x->data_ptr(), ldx, rp, ldr, gp, eps, group, sp, q.data_ptr(),
                                scales.data_ptr(), 0);
    if (status != DOCC_B200_OK) return refused(status, "docc_b200_rmsnorm_q8");
    return r ? tuple_of({q, scales, s}) : tuple_of({q, scales});
    END_HANDLE_TH_ERRORS
}
PyObject* rmsnorm(PyObject*, PyObject* const* args, Py_ssize_t n) { return norm(args, n, false); }
PyObject* rmsnorm_quant(PyObject*, PyObject* const* args, Py_ssize_t n) { return norm(args, n, true); }

bool frequencies(const Tensor& f, int64_t D) { return f.scalar_type() == at::kDouble && f.dim() == 1 && f.is_contiguous() && 2 * f.size(0) <= D; }

// rope(X, positions, inv_freq, interleaved, mscale, inverse, out)
PyObject* rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    c10::DeviceIndex device;
    if (n != 7 || !device_for(args[0], device)) Py_RETURN_NONE;
    const Tensor *x = plain(args[0], device), *p = plain(args[1], device), *f = plain(args[2], device);
    const Tensor* given = args[6] == Py_None ? nullptr : plain(args[6], device);
    const int interleaved = PyObject_IsTrue(args[3]), inverse = PyObject_IsTrue(args[5]);
    double mscale;
    if (!x || !p || !f || (!given && args[6] != Py_None) || interleaved < 0 || inverse < 0 || x->dim() != 3 || !precision(*x) || !number(args[4], mscale)) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    if (!vector_of(*p, at::kLong, x->size(0)) || !frequencies(*f, x->size(2))) Py_RETURN_NONE;
    if (given && (given->sizes() != x->sizes() || given->scalar_type() != x->scalar_type())) Py_RETURN_NONE;
    const Tensor out = given ? *given : empty_like(*x);
    Strides xs, ys;
    if (!xs.take(*x) || !ys.take(out)) Py_RETURN_NONE;
    const int status = unlocked(Held{x, p, f, given}, f_rope, precision(*x), x->size(0), x->size(1), x->size(2), 2 * f->size(0), interleaved, inverse,
                                x->data_ptr(), xs.of, static_cast<const int64_t*>(p->data_ptr()), static_cast<const double*>(f->data_ptr()),
                                float(mscale), out.data_ptr(), ys.of, 0);
    if (status != DOCC_B200_OK) return refused(status, "docc_b200_rope");
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

bool cache_of(const Tensor& c, const Tensor& q, int64_t kv) {
    return c.dim() == 4 && c.size(1) == kv && c.size(3) == q.size(2) && c.scalar_type() == q.scalar_type();
}

// rope_append(q, k, v, positions, inv_freq, k_cache, v_cache, slots, interleaved, mscale, out)
PyObject* rope_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    c10::DeviceIndex device;
    if (n != 11 || !device_for(args[0], device)) Py_RETURN_NONE;
    const Tensor* t[8];
    for (int i = 0; i < 8; i++)
        if (!(t[i] = plain(args[i], device))) Py_RETURN_NONE;
    const Tensor &q = *t[0], &k = *t[1], &v = *t[2], &p = *t[3], &f = *t[4], &kc = *t[5], &vc = *t[6], &slots = *t[7];
    const Tensor* given = args[10] == Py_None ? nullptr : plain(args[10], device);
    const int interleaved = PyObject_IsTrue(args[8]);
    double mscale;
    if ((!given && args[10] != Py_None) || interleaved < 0 || !number(args[9], mscale)) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    if (q.dim() != 3 || k.dim() != 3 || k.sizes() != v.sizes() || k.size(0) != q.size(0) || k.size(2) != q.size(2) || !precision(q) ||
        k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
        Py_RETURN_NONE;
    const int64_t T = q.size(0), kv = k.size(1), D = q.size(2);
    if (!vector_of(p, at::kLong, T) || !vector_of(slots, at::kLong, T) || !frequencies(f, D)) Py_RETURN_NONE;
    if (kc.sizes() != vc.sizes() || !cache_of(kc, q, kv) || !cache_of(vc, q, kv)) Py_RETURN_NONE;
    if (given && (given->sizes() != q.sizes() || given->scalar_type() != q.scalar_type())) Py_RETURN_NONE;
    const Tensor out = given ? *given : empty_like(q);
    Strides qs, ks, vs, os, kcs, vcs;
    if (!qs.take(q) || !ks.take(k) || !vs.take(v) || !os.take(out) || !kcs.take(kc) || !vcs.take(vc)) Py_RETURN_NONE;
    const int status = unlocked(Held(t, given), f_rope_append, precision(q), T, q.size(1), kv, D, 2 * f.size(0), interleaved, q.data_ptr(), qs.of,
                                k.data_ptr(), ks.of, v.data_ptr(), vs.of, static_cast<const int64_t*>(p.data_ptr()),
                                static_cast<const double*>(f.data_ptr()), float(mscale), out.data_ptr(), os.of, kc.data_ptr(), kcs.of, vc.data_ptr(),
                                vcs.of, kc.size(0), kc.size(2), static_cast<const int64_t*>(slots.data_ptr()), 0);
    if (status != DOCC_B200_OK) return refused(status, "docc_b200_rope_append");
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// paged_attention(q, k_cache, v_cache, page_table, lengths, scale, softcap, window, return_lse, out)
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    c10::DeviceIndex device;
    if (n != 10 || !device_for(args[0], device)) Py_RETURN_NONE;
    const Tensor* t[5];
    for (int i = 0; i < 5; i++)
        if (!(t[i] = plain(args[i], device))) Py_RETURN_NONE;
    const Tensor &q = *t[0], &kc = *t[1], &vc = *t[2], &table = *t[3], &lengths = *t[4];
    const Tensor* given = args[9] == Py_None ? nullptr : plain(args[9], device);
    const int want_lse = PyObject_IsTrue(args[8]);
    double scale = 0, softcap;
    int64_t window;
    if ((!given && args[9] != Py_None) || want_lse < 0 || (args[5] != Py_None && !number(args[5], scale)) || !number(args[6], softcap) ||
        !whole(args[7], window)) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    if (q.dim() != 3 || kc.dim() != 4 || !precision(q)) Py_RETURN_NONE;
    const int64_t B = q.size(0), Hq = q.size(1), D = q.size(2), kv = kc.size(1);
    if (kc.sizes() != vc.sizes() || !cache_of(kc, q, kv) || !cache_of(vc, q, kv) || kv == 0 || Hq % kv != 0) Py_RETURN_NONE;
    if (!vector_of(lengths, at::kInt, B) || table.scalar_type() != at::kInt || table.dim() != 2 || table.size(0) != B || !table.is_contiguous())
        Py_RETURN_NONE;
    if (given && (given->sizes() != q.sizes() || given->scalar_type() != q.scalar_type())) Py_RETURN_NONE;
    const Tensor out = given ? *given : empty_like(q);
    Strides qs, os, kcs, vcs;
    if (!qs.take(q) || !os.take(out) || !kcs.take(kc) || !vcs.take(vc)) Py_RETURN_NONE;
    Tensor lse;
    if (want_lse) lse = empty({B, Hq}, q, at::kFloat);
    if (args[5] == Py_None) scale = 1.0 / std::sqrt(double(D > 1 ? D : 1));
    const int status = unlocked(Held(t, given), f_paged_attention, precision(q), B, Hq, kv, D, float(scale), float(softcap), window, q.data_ptr(),
                                qs.of, kc.data_ptr(), kcs.of, vc.data_ptr(), vcs.of, kc.size(0), kc.size(2),
                                static_cast<const int32_t*>(table.data_ptr()), table.size(1), table.size(1),
                                static_cast<const int32_t*>(lengths.data_ptr()), out.data_ptr(), os.of, want_lse ? lse.data_ptr() : nullptr, nullptr,
                                0, 0);
    if (status != DOCC_B200_OK) return refused(status, "docc_b200_paged_attention");
    return want_lse ? tuple_of({out, lse}) : THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// token_logprobs(logits, ids, k, scale)
PyObject* token_logprobs(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    c10::DeviceIndex device;
    if (n != 4 || !device_for(args[0], device)) Py_RETURN_NONE;
    const Tensor *x = plain(args[0], device), *ids = plain(args[1], device);
    int64_t rows, vocab, ld, k;
    double scale;
    if (!x || !ids || x->dim() != 2 || !precision(*x) || !rows_of(*x, rows, vocab, ld) || !vector_of(*ids, at::kLong, rows) || !whole(args[2], k) ||
        k < 0 || k > 32 || !number(args[3], scale))
        Py_RETURN_NONE;
    const Tensor logp = empty({rows}, *x, at::kFloat), entropy = empty({rows}, *x, at::kFloat);
    const Tensor top_ids = empty({rows, k}, *x, at::kLong), top_logp = empty({rows, k}, *x, at::kFloat);
    const int status = unlocked(Held{x, ids}, f_token_logprobs, precision(*x), rows, vocab, x->data_ptr(), ld, float(scale),
                                static_cast<const int64_t*>(ids->data_ptr()), logp.data_ptr(), entropy.data_ptr(), k,
                                static_cast<int64_t*>(top_ids.data_ptr()), top_logp.data_ptr(), 0);
    if (status != DOCC_B200_OK) return refused(status, "docc_b200_token_logprobs");
    return tuple_of({logp, entropy, top_ids, top_logp});
    END_HANDLE_TH_ERRORS
}

// bind(addresses of the six entries, in the order below, check)
PyObject* bind(PyObject*, PyObject* args) {
    unsigned long long a[6];
    PyObject* raise;
    if (!PyArg_ParseTuple(args, "KKKKKKO", &a[0], &a[1], &a[2], &a[3], &a[4], &a[5], &raise)) return nullptr;
    Py_INCREF(raise);
    Py_XDECREF(check);
    check = raise;
    f_rmsnorm = reinterpret_cast<decltype(f_rmsnorm)>(a[0]);
    f_rmsnorm_q8 = reinterpret_cast<decltype(f_rmsnorm_q8)>(a[1]);
    f_rope = reinterpret_cast<decltype(f_rope)>(a[2]);
    f_rope_append = reinterpret_cast<decltype(f_rope_append)>(a[3]);
    f_paged_attention = reinterpret_cast<decltype(f_paged_attention)>(a[4]);
    f_token_logprobs = reinterpret_cast<decltype(f_token_logprobs)>(a[5]);
    Py_RETURN_NONE;
}

template <typename F> PyCFunction as_method(F f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)); }

PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, nullptr},
                         {"rmsnorm", as_method(rmsnorm), METH_FASTCALL, nullptr},
                         {"rmsnorm_quant", as_method(rmsnorm_quant), METH_FASTCALL, nullptr},
                         {"rope", as_method(rope), METH_FASTCALL, nullptr},
                         {"rope_append", as_method(rope_append), METH_FASTCALL, nullptr},
                         {"paged_attention", as_method(paged_attention), METH_FASTCALL, nullptr},
                         {"token_logprobs", as_method(token_logprobs), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "docc_b200_decode_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_docc_b200_decode_calls() { return PyModule_Create(&module); }
