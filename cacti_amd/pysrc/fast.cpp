// The operators of ops.py as CPython functions.  A small operator is host work: of the 6 to 7 us that a call took in Python
// over the C ABI some 2 were the launch (which the device needs as well, 2.3 us from one small kernel to the next); the
// rest went into allocating the results (torch.empty: 1.5 us each from Python, a third of it here), a Python call for
// every property of a tensor that is looked at, and the conversion of arguments.  us per call from Python, before ->
// here: gemm 6.3 -> 4.0, rms_norm 4.8 -> 3.7, its adjoint (two kernels) 10.6 -> 8.0, silu_gate 4.8 -> 3.7.
//
// Tensors come as torch hands them over; what an operator wants of them is checked as before (AssertionError), a status of
// the C ABI that is not 0 is raised by ffi.check.  The other entry points (FN) take pointers as integers or None and
// return the status.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <stdint.h>

#include <initializer_list>
#include <tuple>
#include <type_traits>
#include <utility>
#include <vector>

#include "../../include/cacti_gpu_hip_ffi.h"

namespace {

template <class T>
bool convert(PyObject *o, T *out)
{
    if constexpr (std::is_pointer_v<T>) {
        *out = o == Py_None ? nullptr : (T)PyLong_AsVoidPtr(o);
        return *out || o == Py_None || !PyErr_Occurred();
    } else if constexpr (std::is_floating_point_v<T>) {
        *out = (T)PyFloat_AsDouble(o);
        return !PyErr_Occurred();
    } else {
        const long long v = PyLong_AsLongLong(o);
        if (v == -1 && PyErr_Occurred()) return false;
        *out = (T)v;
        if ((long long)*out != v) {
            PyErr_SetString(PyExc_OverflowError, "argument does not fit the C type");
            return false;
        }
        return true;
    }
}

// f with the arguments of a function of type R (*)(A...)
template <class F, class R, class... A, size_t... I>
PyObject *apply(const F &f, R (*)(A...), PyObject *const *args, Py_ssize_t n, std::index_sequence<I...>)
{
    if (n != (Py_ssize_t)sizeof...(A)) {
        PyErr_Format(PyExc_TypeError, "%d arguments expected, %d given", (int)sizeof...(A), (int)n);
        return nullptr;
    }
    std::tuple<A...> v;
    if (!(convert(args[I], &std::get<I>(v)) && ...)) return nullptr;
    R r;
    Py_BEGIN_ALLOW_THREADS
    r = f(std::get<I>(v)...);
    Py_END_ALLOW_THREADS
    if constexpr (std::is_signed_v<R>) return PyLong_FromLongLong((long long)r);
    else return PyLong_FromUnsignedLongLong((unsigned long long)r);
}

template <class R, class... A>
PyObject *apply(R (*fn)(A...), PyObject *const *args, Py_ssize_t n)
{
    return apply(fn, fn, args, n, std::index_sequence_for<A...>{});
}

// ---------------------------------------------------------------- operators on tensors
PyObject *g_check = nullptr;                   // ffi.check

struct PyFailed {};                            // a Python exception is set
[[noreturn]] void fail(PyObject *type, const char *what)
{
    PyErr_SetString(type, what);
    throw PyFailed();
}
void require(bool ok, const char *what)
{
    if (!ok) fail(PyExc_AssertionError, what);
}

const at::Tensor &tensor(PyObject *o)
{
    if (!THPVariable_Check(o)) fail(PyExc_TypeError, "a tensor expected");
    return THPVariable_Unpack(o);
}
const at::Tensor &checked(const at::Tensor &t, at::ScalarType dtype)
{
    if (!(t.is_cuda() && t.is_contiguous() && t.scalar_type() == dtype)) {
        PyErr_Format(PyExc_AssertionError, "contiguous %s tensor on the GPU expected, got %s on %s%s", c10::toString(dtype),
                     c10::toString(t.scalar_type()), t.device().str().c_str(), t.is_contiguous() ? "" : ", strided");
        throw PyFailed();
    }
    return t;
}
const at::Tensor &f16(PyObject *o) { return checked(tensor(o), at::kHalf); }
const at::Tensor &f32(PyObject *o) { return checked(tensor(o), at::kFloat); }

at::Tensor empty(at::IntArrayRef sizes, const at::Tensor &like, at::ScalarType dtype)
{
    return at::empty(sizes, at::TensorOptions().dtype(dtype).device(like.device()));
}
at::Tensor new_like(const at::Tensor &t) { return empty(t.sizes(), t, t.scalar_type()); }

void *stream() { return c10::hip::getCurrentHIPStream().stream(); }

template <class T>
T number(PyObject *o)
{
    T v;
    if (!convert(o, &v)) throw PyFailed();
    return v;
}
int truth(PyObject *o)
{
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw PyFailed();
    return v;
}

// the call itself runs without the interpreter lock (taken again also where it throws: a tensor without storage does); a
// status that is not 0 becomes the exception ffi.check raises
struct Unlocked {
    PyThreadState *st = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(st); }
};
template <class F>
auto unlocked(F f)
{
    const Unlocked u;
    return f();
}
void raise_status(int rc)
{
    PyObject *r = PyObject_CallFunction(g_check, "i", rc);
    Py_XDECREF(r);
    if (r) PyErr_SetString(PyExc_RuntimeError, "status of an entry point");
    throw PyFailed();
}
template <class F>
void run(F f)
{
    const int rc = unlocked(f);
    if (rc) raise_status(rc);
}

PyObject *wrap(at::Tensor t)
{
    PyObject *o = THPVariable_Wrap(std::move(t));
    if (!o) throw PyFailed();
    return o;
}
// a result tensor: the argument it accumulates into (the same object is returned) or a new one
struct Result {
    at::Tensor t;
    PyObject *arg;
    int acc() const { return arg != nullptr; }
    void *ptr() const { return t.data_ptr(); }
    PyObject *take() const
    {
        if (!arg) return wrap(t);
        Py_INCREF(arg);
        return arg;
    }
};
Result result(PyObject *acc, const at::Tensor &like)
{
    if (acc == Py_None) return {new_like(like), nullptr};
    return {f16(acc), acc};
}
PyObject *take2(const Result &a, const Result &b)
{
    PyObject *x = a.take(), *y = b.take(), *r = PyTuple_New(2);
    PyTuple_SET_ITEM(r, 0, x);
    PyTuple_SET_ITEM(r, 1, y);
    return r;
}

// The tensors of a list or tuple, held: another thread may change the list while a call runs without the interpreter lock.
struct Tensors {
    std::vector<at::Tensor> t;
    explicit Tensors(PyObject *o)
    {
        PyObject *seq = PySequence_Fast(o, "a sequence of tensors expected");
        if (!seq) throw PyFailed();
        const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
        t.reserve(n);
        for (Py_ssize_t i = 0; i < n; i++) {
            PyObject *e = PySequence_Fast_GET_ITEM(seq, i);
            if (!THPVariable_Check(e)) {
                Py_DECREF(seq);
                fail(PyExc_TypeError, "a tensor expected");
            }
            t.push_back(THPVariable_Unpack(e));
        }
        Py_DECREF(seq);
    }
    size_t size() const { return t.size(); }
    const at::Tensor &operator[](size_t i) const { return t[i]; }
    std::vector<void *> pointers() const
    {
        std::vector<void *> p(t.size());
        for (size_t i = 0; i < t.size(); i++) p[i] = t[i].data_ptr();
        return p;
    }
};

void gemm_into(int ta, int tb, int64_t M, int64_t N, int64_t K, float alpha, const at::Tensor &a, const at::Tensor &b, float beta,
               const at::Tensor &out)
{
    void *st = stream();
    size_t need = 0;
    auto call = [&](void *ws, size_t bytes) {
        return cacti_hip_gemm_f16_ws(ta, tb, M, N, K, alpha, a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), beta, out.data_ptr(),
                                     out.stride(0), ws, bytes, &need, st);
    };
    run([&] { return call(nullptr, 0); });
    if (need > 0) {                              // not launched: the product wants a workspace
        const at::Tensor ws = empty({(int64_t)need}, a, at::kByte);
        const size_t bytes = need;
        run([&] { return call(ws.data_ptr(), bytes); });
    }
}

struct Shape {
    int64_t M, N, K;
};
Shape product_shape(const at::Tensor &a, const at::Tensor &b, int ta, int tb)
{
    require(a.dim() == 2 && b.dim() == 2 && a.stride(1) == 1 && b.stride(1) == 1, "gemm: matrices with contiguous rows expected");
    const Shape s = {a.size(ta ? 1 : 0), b.size(tb ? 0 : 1), a.size(ta ? 0 : 1)};
    require(s.K == b.size(tb ? 1 : 0), "gemm: inner dimensions differ");
    return s;
}

// (a, b, ta, tb, alpha, beta, out)
PyObject *gemm(PyObject *const *v)
{
    const at::Tensor &a = tensor(v[0]), &b = tensor(v[1]);
    const int ta = truth(v[2]), tb = truth(v[3]);
    const float alpha = number<float>(v[4]), beta = number<float>(v[5]);
    const Shape s = product_shape(a, b, ta, tb);
    if (v[6] == Py_None) {
        require(beta == 0.f, "gemm: beta without out");
        at::Tensor out = empty({s.M, s.N}, a, at::kHalf);
        gemm_into(ta, tb, s.M, s.N, s.K, alpha, a, b, beta, out);
        return wrap(std::move(out));
    }
    const at::Tensor &out = tensor(v[6]);
    require(out.dim() == 2 && out.size(0) == s.M && out.size(1) == s.N && out.stride(1) == 1, "gemm: shape of out");
    gemm_into(ta, tb, s.M, s.N, s.K, alpha, a, b, beta, out);
    Py_INCREF(v[6]);
    return v[6];
}

// (As, Bs, outs, ta, tb, alpha, beta)
PyObject *gemm_batched(PyObject *const *v)
{
    const Tensors as(v[0]), bs(v[1]), outs(v[2]);
    const int ta = truth(v[3]), tb = truth(v[4]);
    const float alpha = number<float>(v[5]), beta = number<float>(v[6]);
    const size_t n = as.size();
    require(n > 0 && bs.size() == n && outs.size() == n, "gemm_batched: lists of one length expected");
    const at::Tensor &a = as[0], &b = bs[0], &o = outs[0];
    const Shape s = product_shape(a, b, ta, tb);
    const std::vector<void *> pa = as.pointers(), pb = bs.pointers(), po = outs.pointers();
    bool aligned = true;
    for (int64_t x : {a.size(1), b.size(1), s.N, a.stride(0), b.stride(0), o.stride(0)}) aligned = aligned && x % 8 == 0;
    for (const std::vector<void *> *v : {&pa, &pb, &po})
        for (void *p : *v) aligned = aligned && reinterpret_cast<uintptr_t>(p) % 16 == 0;
    if (!aligned) {
        // operands whose rows are not all 16-byte aligned run one after another; each may want a workspace
        for (size_t z = 0; z < n; z++) gemm_into(ta, tb, s.M, s.N, s.K, alpha, as[z], bs[z], beta, outs[z]);
        Py_RETURN_NONE;
    }
    void *st = stream();
    run([&] {
        return cacti_hip_gemm_f16_batched(ta, tb, (int64_t)n, s.M, s.N, s.K, alpha, pa.data(), a.stride(0), pb.data(), b.stride(0), beta,
                                          po.data(), o.stride(0), st);
    });
    Py_RETURN_NONE;
}

// (q, k, v, alpha)
PyObject *attention_fwd(PyObject *const *v)
{
    const at::Tensor &q = f16(v[0]), &k = f16(v[1]), &w = f16(v[2]);
    const float alpha = number<float>(v[3]);
    require(q.dim() == 3, "attention: [S, H, Dh] expected");
    const int64_t S = q.size(0), H = q.size(1), Dh = q.size(2);
    const Result o = {new_like(q), nullptr};
    const Result stats = {empty({(int64_t)(cacti_hip_attention_stats_bytes(S, H) / 4)}, q, at::kFloat), nullptr};
    void *st = stream();
    run([&] { return cacti_hip_attention_fwd(S, H, Dh, alpha, q.data_ptr(), k.data_ptr(), w.data_ptr(), H * Dh, o.ptr(), stats.ptr(), st); });
    return take2(o, stats);
}

// (q, k, v, dO, stats, alpha, acc, o)
PyObject *attention_bwd(PyObject *const *v)
{
    const at::Tensor &q = f16(v[0]), &k = f16(v[1]), &w = f16(v[2]), &dO = f16(v[3]), &stats = tensor(v[4]);
    const float alpha = number<float>(v[5]);
    const void *o = v[7] == Py_None ? nullptr : f16(v[7]).data_ptr();
    require(q.dim() == 3, "attention: [S, H, Dh] expected");
    const int64_t S = q.size(0), H = q.size(1), Dh = q.size(2);
    const bool into = v[6] != Py_None;
    auto given = [&]() {
        const Tensors acc(v[6]);
        require(acc.size() == 3, "attention_bwd: acc = (dq, dk, dv)");
        return acc.t;
    };
    const std::vector<at::Tensor> d = into ? given() : std::vector<at::Tensor>{new_like(q), new_like(q), new_like(q)};
    const size_t bytes = cacti_hip_attention_bwd_workspace_used(S, H, Dh, H * Dh);
    const at::Tensor ws = empty({(int64_t)bytes}, q, at::kByte);
    void *st = stream();
    run([&] {
        return cacti_hip_attention_bwd(S, H, Dh, alpha, q.data_ptr(), k.data_ptr(), w.data_ptr(), o, dO.data_ptr(), H * Dh, stats.data_ptr(),
                                       d[0].data_ptr(), into, d[1].data_ptr(), into, d[2].data_ptr(), into, ws.data_ptr(), bytes, st);
    });
    PyObject *r = PyTuple_New(3);
    if (!r) throw PyFailed();
    for (int i = 0; i < 3; i++) PyTuple_SET_ITEM(r, i, THPVariable_Wrap(d[i]));     // (a tensor that was given: its own object)
    return r;
}

// (x, w, eps)
PyObject *rms_norm_fwd(PyObject *const *v)
{
    const at::Tensor &x = f16(v[0]), &w = f16(v[1]);
    const float eps = number<float>(v[2]);
    require(x.dim() == 2, "rms_norm: [N, D] expected");
    at::Tensor y = new_like(x);
    void *st = stream();
    run([&] { return cacti_hip_rms_norm_fwd(x.size(0), x.size(1), x.data_ptr(), w.data_ptr(), eps, y.data_ptr(), st); });
    return wrap(std::move(y));
}

// (a, b, w, eps)
PyObject *add_rms_norm_fwd(PyObject *const *v)
{
    const at::Tensor &a = f16(v[0]), &b = f16(v[1]), &w = f16(v[2]);
    const float eps = number<float>(v[3]);
    require(a.dim() == 2, "add_rms_norm: [N, D] expected");
    const Result s = {new_like(a), nullptr}, y = {new_like(a), nullptr};
    void *st = stream();
    run([&] {
        return cacti_hip_add_rms_norm_fwd(a.size(0), a.size(1), a.data_ptr(), b.data_ptr(), w.data_ptr(), eps, s.ptr(), y.ptr(), st);
    });
    return take2(s, y);
}

// (x, w, eps, dy, dx_acc, dw_acc)
PyObject *rms_norm_bwd(PyObject *const *v)
{
    const at::Tensor &x = f16(v[0]), &w = f16(v[1]), &dy = f16(v[3]);
    const float eps = number<float>(v[2]);
    require(x.dim() == 2, "rms_norm: [N, D] expected");
    const Result dx = result(v[4], x), dw = result(v[5], w);
    const size_t bytes = cacti_hip_rms_norm_bwd_workspace(x.size(0), x.size(1));
    const at::Tensor ws = empty({(int64_t)bytes}, x, at::kByte);
    void *st = stream();
    run([&] {
        return cacti_hip_rms_norm_bwd(x.size(0), x.size(1), x.data_ptr(), w.data_ptr(), eps, dy.data_ptr(), dx.ptr(), dx.acc(), dw.ptr(),
                                      dw.acc(), ws.data_ptr(), bytes, st);
    });
    return take2(dx, dw);
}

// (x, cos, sin)
PyObject *rope_fwd(PyObject *const *v)
{
    const at::Tensor &x = f16(v[0]), &c = f16(v[1]), &s = f16(v[2]);
    require(x.dim() == 3, "rope: [S, H, Dh] expected");
    at::Tensor y = new_like(x);
    void *st = stream();
    run([&] {
        return cacti_hip_rope_fwd(x.size(0), x.size(1), x.size(2), x.data_ptr(), c.data_ptr(), s.data_ptr(), y.data_ptr(), st);
    });
    return wrap(std::move(y));
}

// (dy, cos, sin, dx_acc)
PyObject *rope_bwd(PyObject *const *v)
{
    const at::Tensor &dy = f16(v[0]), &c = f16(v[1]), &s = f16(v[2]);
    require(dy.dim() == 3, "rope: [S, H, Dh] expected");
    const Result dx = result(v[3], dy);
    void *st = stream();
    run([&] {
        return cacti_hip_rope_bwd(dy.size(0), dy.size(1), dy.size(2), dy.data_ptr(), c.data_ptr(), s.data_ptr(), dx.ptr(), dx.acc(), st);
    });
    return dx.take();
}

// (g, u)
PyObject *silu_gate_fwd(PyObject *const *v)
{
    const at::Tensor &g = f16(v[0]), &u = f16(v[1]);
    at::Tensor h = new_like(g);
    void *st = stream();
    run([&] { return cacti_hip_silu_gate_fwd(g.numel(), g.data_ptr(), u.data_ptr(), h.data_ptr(), st); });
    return wrap(std::move(h));
}

// (g, u, dh, dg_acc, du_acc)
PyObject *silu_gate_bwd(PyObject *const *v)
{
    const at::Tensor &g = f16(v[0]), &u = f16(v[1]), &dh = f16(v[2]);
    const Result dg = result(v[3], g), du = result(v[4], u);
    void *st = stream();
    run([&] {
        return cacti_hip_silu_gate_bwd(g.numel(), g.data_ptr(), u.data_ptr(), dh.data_ptr(), dg.ptr(), dg.acc(), du.ptr(), du.acc(), st);
    });
    return take2(dg, du);
}

// (a, b, out)
PyObject *add_f16(PyObject *const *v)
{
    const at::Tensor &a = tensor(v[0]), &b = tensor(v[1]);
    // (element for element in memory order: the result has a's strides, whatever they are)
    const Result out = v[2] == Py_None ? Result{at::empty_like(a), nullptr} : Result{tensor(v[2]), v[2]};
    void *st = stream();
    run([&] { return cacti_hip_add_f16(a.numel(), a.data_ptr(), b.data_ptr(), out.ptr(), st); });
    return out.take();
}

// (logit, tok, scale, acc)
PyObject *softmax_ce_bwd(PyObject *const *v)
{
    const at::Tensor &logit = f16(v[0]), &tok = tensor(v[1]), &scale = f32(v[2]);
    require(logit.dim() == 2, "softmax_ce: [N, V] expected");
    const Result d = result(v[3], logit);
    void *st = stream();
    run([&] {
        return cacti_hip_softmax_ce_bwd(logit.size(0), logit.size(1), logit.data_ptr(), tok.data_ptr(), scale.data_ptr(), d.ptr(), d.acc(), st);
    });
    return d.take();
}

// ---------------------------------------------------------------- paged cache, drafted tokens, distillation
// The device of a call's tensors for its duration, and the stream that is current there
struct OnDevice {
    c10::DeviceGuard guard;
    c10::Device dev;
    explicit OnDevice(const at::Tensor &t) : guard(t.device()), dev(t.device()) {}
    void *stream() const { return c10::hip::getCurrentHIPStream(dev.index()).stream(); }
    const at::Tensor &here(const at::Tensor &t) const
    {
        require(t.device() == dev, "tensors of one device expected");
        return t;
    }
    const at::Tensor &here(PyObject *o, at::ScalarType dtype) const { return here(checked(tensor(o), dtype)); }
    void *pointer(PyObject *o, at::ScalarType dtype, int64_t numel) const     // or null for None
    {
        if (o == Py_None) return nullptr;
        const at::Tensor &t = here(o, dtype);
        require(t.numel() == numel, "a tensor has another number of elements");
        return t.data_ptr();
    }
};
const at::Tensor &on_gpu(const at::Tensor &t)
{
    require(t.is_cuda(), "tensor on the GPU expected");
    return t;
}

// [T, H, Dh] f16 whose rows may be strided
struct Rows {
    const at::Tensor &t;
    int64_t T, H, Dh, ld;
    Rows(PyObject *o, const OnDevice &on, const char *what) : t(on.here(on_gpu(tensor(o))))
    {
        require(t.scalar_type() == at::kHalf && t.dim() == 3, what);
        T = t.size(0), H = t.size(1), Dh = t.size(2);
        require((Dh <= 1 || t.stride(2) == 1) && (H <= 1 || t.stride(1) == Dh), what);
        ld = T > 1 ? t.stride(0) : H * Dh;
    }
};
// [N, V] f16 whose rows may be strided
struct Logits {
    const at::Tensor &t;
    int64_t N, V, ld;
    Logits(PyObject *o, const OnDevice &on, const char *what) : t(on.here(on_gpu(tensor(o))))
    {
        require(t.scalar_type() == at::kHalf && t.dim() == 2, what);
        N = t.size(0), V = t.size(1);
        require(N == 0 || V <= 1 || t.stride(1) == 1, what);
        ld = N > 1 ? t.stride(0) : V;
    }
};

// (k_pages, v_pages, k_scale, v_scale, table, starts, lens), what an append and an attention call have in common
struct Paged {
    const at::Tensor &k, &v, &table;
    void *ks, *vs, *starts, *lens;
    int bits;
    int64_t P, Hkv, page, B, W, ldt;
    Paged(PyObject *const *o, const OnDevice &on)
        : k(on.here(on_gpu(tensor(o[0])))), v(on.here(on_gpu(tensor(o[1])))), table(on.here(on_gpu(tensor(o[4]))))
    {
        bits = k.scalar_type() == at::kHalf ? 16 : 8;
        require(k.dim() == 4 && k.is_contiguous() && v.is_contiguous() && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() &&
                    (bits == 16 || k.scalar_type() == at::kFloat8_e4m3fn),
                "paged cache: two contiguous tensors [pages, heads, page, Dp] of f16 or float8_e4m3fn expected");
        P = k.size(0), Hkv = k.size(1), page = k.size(2);
        ks = on.pointer(o[2], at::kFloat, P * Hkv), vs = on.pointer(o[3], at::kFloat, P * Hkv);
        require(table.scalar_type() == at::kInt && table.dim() == 2 && (table.size(1) <= 1 || table.stride(1) == 1),
                "paged cache: table [sequences, pages] of int32 expected");
        B = table.size(0), W = table.size(1), ldt = B > 1 ? table.stride(0) : W;
        require(o[5] != Py_None && o[6] != Py_None, "paged cache: starts [sequences + 1] and lens [sequences] of int32 expected");
        starts = on.pointer(o[5], at::kInt, B + 1), lens = on.pointer(o[6], at::kInt, B);
    }
    void bounds(int64_t max_new, int64_t T) const
    {
        require(max_new > 0 || (max_new == 0 && (T == 0 || B == 0)), "paged cache: max_new is at least 1 where there are rows and sequences");
    }
    void holds(int64_t Dh) const { require(k.size(3) == (Dh + 15) / 16 * 16, "paged cache: pages of another head dimension"); }
};

// (k, v, k_pages, v_pages, k_scale, v_scale, table, starts, lens, cos, sin, q, q_out, max_new, status)
PyObject *paged_append(PyObject *const *o)
{
    const OnDevice on(on_gpu(tensor(o[0])));
    const Rows k(o[0], on, "paged_append: k [T, heads, Dh] f16 expected"), v(o[1], on, "paged_append: v [T, heads, Dh] f16 expected");
    const Paged c(o + 2, on);
    const at::Tensor &cos = on.here(o[9], at::kHalf), &sin = on.here(o[10], at::kHalf);
    c.holds(k.Dh);
    require(v.t.sizes() == k.t.sizes() && k.H == c.Hkv, "paged_append: k, v and the pages have other shapes than each other");
    require(cos.dim() == 2 && cos.size(1) == k.Dh && sin.sizes() == cos.sizes(), "paged_append: cos and sin [positions, Dh] expected");
    int64_t H = k.H, ldq = 0, ldqo = 0;
    void *q = nullptr, *qo = nullptr;
    Result out = {at::Tensor(), nullptr};
    if (o[11] != Py_None) {
        const Rows r(o[11], on, "paged_append: q [T, heads, Dh] f16 expected");
        require(r.T == k.T && r.Dh == k.Dh, "paged_append: q has other rows than k");
        H = r.H, ldq = r.ld, q = r.t.data_ptr();
        if (o[12] == Py_None) out.t = empty({r.T, r.H, r.Dh}, r.t, at::kHalf), ldqo = H * k.Dh;
        else {
            const Rows w(o[12], on, "paged_append: out [T, heads, Dh] f16 expected");
            require(w.t.sizes() == r.t.sizes(), "paged_append: shape of out");
            out = {w.t, o[12]}, ldqo = w.ld;
        }
        qo = out.t.data_ptr();
    } else require(o[12] == Py_None, "paged_append: out without q");
    const int64_t max_new = o[13] == Py_None ? k.T : number<int64_t>(o[13]);
    c.bounds(max_new, k.T);
    void *status = on.pointer(o[14], at::kInt, 1), *st = on.stream();
    if (k.T > 0 && c.B > 0)
        run([&] {
            return cacti_hip_paged_append(k.T, c.B, H, k.H, k.Dh, max_new, q, ldq, k.t.data_ptr(), k.ld, v.t.data_ptr(), v.ld, cos.data_ptr(),
                                          sin.data_ptr(), cos.size(0), qo, ldqo, c.k.data_ptr(), c.v.data_ptr(), c.ks, c.vs, c.bits, c.P,
                                          c.page, c.table.data_ptr(), c.ldt, c.W, c.starts, c.lens, status, st);
        });
    if (!out.t.defined()) Py_RETURN_NONE;
    return out.take();
}

// (q, k_pages, v_pages, k_scale, v_scale, table, starts, lens, alpha, max_new, out, status)
PyObject *paged_attention(PyObject *const *o)
{
    const OnDevice on(on_gpu(tensor(o[0])));
    const Rows q(o[0], on, "paged_attention: q [T, heads, Dh] f16 expected");
    const Paged c(o + 1, on);
    c.holds(q.Dh);
    const float alpha = number<float>(o[8]);
    const int64_t max_new = o[9] == Py_None ? q.T : number<int64_t>(o[9]);
    c.bounds(max_new, q.T);
    Result out = {at::Tensor(), nullptr};
    int64_t ldo = q.H * q.Dh;
    if (o[10] == Py_None) out.t = empty({q.T, q.H, q.Dh}, q.t, at::kHalf);
    else {
        const Rows w(o[10], on, "paged_attention: out [T, heads, Dh] f16 expected");
        require(w.t.sizes() == q.t.sizes(), "paged_attention: shape of out");
        out = {w.t, o[10]}, ldo = w.ld;
    }
    void *status = on.pointer(o[11], at::kInt, 1), *st = on.stream();
    if (q.T > 0 && c.B > 0) {
        const size_t bytes = cacti_hip_paged_attention_workspace(q.T, c.B, q.H, c.Hkv, q.Dh, max_new);
        const at::Tensor ws = empty({(int64_t)bytes}, q.t, at::kByte);
        run([&] {
            return cacti_hip_paged_attention_f16(q.T, c.B, q.H, c.Hkv, q.Dh, max_new, alpha, q.t.data_ptr(), q.ld, c.k.data_ptr(),
                                                 c.v.data_ptr(), c.ks, c.vs, c.bits, c.P, c.page, c.table.data_ptr(), c.ldt, c.W, c.starts,
                                                 c.lens, out.ptr(), ldo, ws.data_ptr(), bytes, status, st);
        });
    }
    return out.take();
}

// (target, draft, tok, starts, u, r, temperature, status): (accepted, next)
PyObject *verify_draft(PyObject *const *o)
{
    const OnDevice on(on_gpu(tensor(o[0])));
    const Logits t(o[0], on, "verify_draft: target [T, V] f16 expected");
    const void *draft = nullptr;
    int64_t ldd = 0;
    if (o[1] != Py_None) {
        const Logits d(o[1], on, "verify_draft: draft [T, V] f16 expected");
        require(d.t.sizes() == t.t.sizes(), "verify_draft: draft has another shape than target");
        draft = d.t.data_ptr(), ldd = d.ld;
    }
    const at::Tensor &starts = on.here(o[3], at::kInt);
    const int64_t B = starts.numel() - 1;
    require(B >= 0, "verify_draft: starts [sequences + 1] expected");
    void *tok = on.pointer(o[2], at::kShort, t.N), *u = on.pointer(o[4], at::kFloat, t.N), *r = on.pointer(o[5], at::kFloat, B);
    const double temperature = number<double>(o[6]);
    void *status = on.pointer(o[7], at::kInt, 1), *st = on.stream();
    const Result accepted = {empty({B}, t.t, at::kInt), nullptr}, next = {empty({t.N}, t.t, at::kShort), nullptr};
    if (t.N > 0 && B > 0) {
        const size_t bytes = cacti_hip_verify_draft_workspace(t.N, B, t.V);
        const at::Tensor ws = empty({(int64_t)bytes}, t.t, at::kByte);
        run([&] {
            return cacti_hip_verify_draft_f16(t.N, B, t.V, t.t.data_ptr(), t.ld, draft, ldd, tok, starts.data_ptr(), u, r, temperature,
                                              accepted.ptr(), next.ptr(), ws.data_ptr(), bytes, status, st);
        });
    } else if (B > 0) accepted.t.zero_();
    return take2(accepted, next);
}

// (logit, idx, val, temperature, status): (loss, stats)
PyObject *distill_topk_fwd(PyObject *const *o)
{
    const OnDevice on(on_gpu(tensor(o[0])));
    const Logits z(o[0], on, "distill_topk: logits [N, V] f16 expected");
    const at::Tensor &idx = on.here(o[1], at::kShort), &val = on.here(o[2], at::kHalf);
    require(idx.dim() == 2 && idx.size(0) == z.N && val.sizes() == idx.sizes(), "distill_topk: idx and val [N, K] expected");
    const double temperature = number<double>(o[3]);
    void *status = on.pointer(o[4], at::kInt, 1), *st = on.stream();
    const Result loss = {empty({z.N}, z.t, at::kFloat), nullptr}, stats = {empty({z.N, 2}, z.t, at::kFloat), nullptr};
    if (z.N > 0)
        run([&] {
            return cacti_hip_distill_topk_fwd(z.N, z.V, idx.size(1), z.t.data_ptr(), z.ld, idx.data_ptr(), val.data_ptr(), temperature,
                                              loss.ptr(), stats.ptr(), status, st);
        });
    return take2(loss, stats);
}

// (logit, idx, val, stats, scale, temperature, acc)
PyObject *distill_topk_bwd(PyObject *const *o)
{
    const OnDevice on(on_gpu(tensor(o[0])));
    const Logits z(o[0], on, "distill_topk: logits [N, V] f16 expected");
    const at::Tensor &idx = on.here(o[1], at::kShort), &val = on.here(o[2], at::kHalf);
    require(idx.dim() == 2 && idx.size(0) == z.N && val.sizes() == idx.sizes(), "distill_topk: idx and val [N, K] expected");
    const void *stats = on.pointer(o[3], at::kFloat, 2 * z.N), *scale = on.pointer(o[4], at::kFloat, z.N);
    const double temperature = number<double>(o[5]);
    Result d = {at::Tensor(), nullptr};
    int64_t ldd = z.V;
    if (o[6] == Py_None) d.t = empty({z.N, z.V}, z.t, at::kHalf);
    else {
        const Logits w(o[6], on, "distill_topk: acc [N, V] f16 expected");
        require(w.t.sizes() == z.t.sizes(), "distill_topk: shape of acc");
        d = {w.t, o[6]}, ldd = w.ld;
    }
    void *st = on.stream();
    if (z.N > 0)
        run([&] {
            return cacti_hip_distill_topk_bwd(z.N, z.V, idx.size(1), z.t.data_ptr(), z.ld, idx.data_ptr(), val.data_ptr(), stats, scale,
                                              temperature, d.ptr(), ldd, d.acc(), st);
        });
    return d.take();
}

// ---------------------------------------------------------------- drawn tokens, adapters, several answers in one cache
PyObject *tuple_of(std::initializer_list<Result> rs)
{
    PyObject *r = PyTuple_New((Py_ssize_t)rs.size());
    if (!r) throw PyFailed();
    Py_ssize_t i = 0;
    for (const Result &x : rs) PyTuple_SET_ITEM(r, i++, x.take());
    return r;
}
// a gradient of the logits' shape: the argument that is added to, or a new one
struct LogitGradient {
    Result r = {at::Tensor(), nullptr};
    int64_t ld;
    LogitGradient(PyObject *acc, const Logits &z, const OnDevice &on, const char *what) : ld(z.V)
    {
        if (acc == Py_None) r.t = empty({z.N, z.V}, z.t, at::kHalf);
        else {
            const Logits w(acc, on, what);
            require(w.t.sizes() == z.t.sizes(), what);
            r = {w.t, acc}, ld = w.ld;
        }
    }
};
Result new_f32(at::IntArrayRef sizes, const at::Tensor &like) { return {empty(sizes, like, at::kFloat), nullptr}; }
Result new_i32(at::IntArrayRef sizes, const at::Tensor &like) { return {empty(sizes, like, at::kInt), nullptr}; }
void given(PyObject *o, const char *what) { require(o != Py_None, what); }

// (logit, tok, temperature, mask, status): (logp, stats)
PyObject *token_logp_fwd(PyObject *const *o)
{
    const OnDevice on(on_gpu(tensor(o[0])));
    const Logits z(o[0], on, "token_logp: logits [N, V] f16 expected");
    given(o[1], "token_logp: tok [N] expected");
    const void *tok = on.pointer(o[1], at::kShort, z.N), *mask = on.pointer(o[3], at::kBool, z.N);
    const double temperature = number<double>(o[2]);
    void *status = on.pointer(o[4], at::kInt, 1), *st = on.stream();
    const Result logp = new_f32({z.N}, z.t), stats = new_f32({z.N, 2}, z.t);
    if (z.N > 0)
        run([&] {
            return cacti_hip_token_logp_fwd(z.N, z.V, z.t.data_ptr(), z.ld, tok, mask, temperature, logp.ptr(), stats.ptr(), status, st);
        });
    return take2(logp, stats);
}

// (logit, tok, stats, dlogp, temperature, acc)
PyObject *token_logp_bwd(PyObject *const *o)
{
    const OnDevice on(on_gpu(tensor(o[0])));
    const Logits z(o[0], on, "token_logp: logits [N, V] f16 expected");
    given(o[1], "token_logp: tok [N] expected"), given(o[2], "token_logp: stats [N, 2] expected"), given(o[3], "token_logp: dlogp [N] expected");
    const void *tok = on.pointer(o[1], at::kShort, z.N), *stats = on.pointer(o[2], at::kFloat, 2 * z.N), *dlogp = on.pointer(o[3], at::kFloat, z.N);
    const double temperature = number<double>(o[4]);
    const LogitGradient d(o[5], z, on, "token_logp: acc [N, V] f16 expected");
    void *st = on.stream();
    if (z.N > 0)
        run([&] {
            return cacti_hip_token_logp_bwd(z.N, z.V, z.t.data_ptr(), z.ld, tok, stats, dlogp, temperature, d.r.ptr(), d.ld, d.r.acc(), st);
        });
    return d.r.take();
}

// (logit, tok, old, adv, scale, ref, mask, clip_lo, clip_hi, beta, temperature, acc, status): (loss, logp, dlogit)
PyObject *policy_loss(PyObject *const *o)
{
    const OnDevice on(on_gpu(tensor(o[0])));
    const Logits z(o[0], on, "policy_loss: logits [N, V] f16 expected");
    for (int i = 1; i <= 4; i++) given(o[i], "policy_loss: tok, old, adv and scale [N] expected");
    const void *tok = on.pointer(o[1], at::kShort, z.N), *old = on.pointer(o[2], at::kFloat, z.N), *adv = on.pointer(o[3], at::kFloat, z.N),
               *scale = on.pointer(o[4], at::kFloat, z.N), *ref = on.pointer(o[5], at::kFloat, z.N), *mask = on.pointer(o[6], at::kBool, z.N);
    const double lo = number<double>(o[7]), hi = number<double>(o[8]), beta = number<double>(o[9]), temperature = number<double>(o[10]);
    const LogitGradient d(o[11], z, on, "policy_loss: acc [N, V] f16 expected");
    void *status = on.pointer(o[12], at::kInt, 1), *st = on.stream();
    const Result loss = new_f32({z.N}, z.t), logp = new_f32({z.N}, z.t);
    if (z.N > 0)
        run([&] {
            return cacti_hip_policy_loss(z.N, z.V, z.t.data_ptr(), z.ld, tok, mask, old, adv, ref, scale, lo, hi, beta, temperature, loss.ptr(),
                                         logp.ptr(), d.r.ptr(), d.ld, d.r.acc(), status, st);
        });
    return tuple_of({loss, logp, d.r});
}

// (logp, ref, starts, scale, beta, smoothing, mask, mean, status): (loss, reward, dlogp)
PyObject *preference_loss(PyObject *const *o)
{
    const OnDevice on(on_gpu(tensor(o[0])));
    const at::Tensor &logp = on.here(o[0], at::kFloat), &starts = on.here(o[2], at::kInt);
    const int64_t N = logp.numel(), pairs = (starts.numel() - 1) / 2;
    require(starts.numel() % 2 == 1, "preference_loss: starts [2 pairs + 1] expected");
    given(o[3], "preference_loss: scale [pairs] expected");
    const void *ref = on.pointer(o[1], at::kFloat, N), *scale = on.pointer(o[3], at::kFloat, pairs), *mask = on.pointer(o[6], at::kBool, N);
    const double beta = number<double>(o[4]), smoothing = number<double>(o[5]);
    const int mean = truth(o[7]);
    void *status = on.pointer(o[8], at::kInt, 1), *st = on.stream();
    const Result loss = new_f32({pairs}, logp), reward = new_f32({2 * pairs}, logp), dlogp = new_f32({N}, logp);
    if (N > 0 && pairs > 0)
        run([&] {
            return cacti_hip_preference_loss(N, pairs, logp.data_ptr(), ref, mask, starts.data_ptr(), scale, beta, smoothing, mean, loss.ptr(),
                                             reward.ptr(), dlogp.ptr(), status, st);
        });
    else {
        // no pairs, or texts of no rows: their rewards are 0
        dlogp.t.zero_();
        reward.t.zero_();
        loss.t.fill_(0.69314718055994530942);
    }
    return tuple_of({loss, reward, dlogp});
}

// x, A, B, starts, ids, scale of a call over adapters
struct Adapters {
    const Logits x;
    const at::Tensor &A, &B, &starts;
    const void *ids, *scale;
    int64_t n, R, K, N, S, max_new;
    Adapters(PyObject *const *o, PyObject *most, const OnDevice &on)
        : x(o[0], on, "adapter: x [T, K] f16 expected"), A(on.here(o[1], at::kHalf)), B(on.here(o[2], at::kHalf)), starts(on.here(o[3], at::kInt))
    {
        require(A.dim() == 3 && B.dim() == 3 && A.size(0) == B.size(0) && A.size(1) == B.size(2), "adapter: A [n, R, K] and B [n, N, R] expected");
        n = A.size(0), R = A.size(1), K = A.size(2), N = B.size(1), S = starts.numel() - 1;
        require(x.V == K, "adapter: x has rows of another length than A");
        require(S >= 0, "adapter: starts [sequences + 1] expected");
        given(o[4], "adapter: ids [sequences] expected"), given(o[5], "adapter: scale [adapters] expected");
        ids = on.pointer(o[4], at::kInt, S), scale = on.pointer(o[5], at::kFloat, n);
        max_new = most == Py_None ? x.N : number<int64_t>(most);
        require(max_new > 0 || (max_new == 0 && (x.N == 0 || S == 0)), "adapter: max_new is at least 1 where there are rows and sequences");
    }
    bool some() const { return x.N > 0 && S > 0; }
};

// (x, A, B, starts, ids, scale, base, out, max_new, status): (y, h)
PyObject *adapter_fwd(PyObject *const *o)
{
    const OnDevice on(on_gpu(tensor(o[0])));
    const Adapters g(o, o[8], on);
    const int64_t T = g.x.N;
    const void *base = nullptr;
    int64_t ldb = 0, ldy = g.N;
    auto rows = [&](PyObject *p, const char *what) {
        Logits r(p, on, what);
        require(r.N == T && r.V == g.N, what);
        return r;
    };
    if (o[6] != Py_None) {
        const Logits b = rows(o[6], "adapter_fwd: base [T, N] f16 expected");
        base = b.t.data_ptr(), ldb = b.ld;
    }
    Result y = {at::Tensor(), nullptr};
    if (o[7] == Py_None) y.t = empty({T, g.N}, g.x.t, at::kHalf);
    else {
        const Logits w = rows(o[7], "adapter_fwd: out [T, N] f16 expected");
        y = {w.t, o[7]}, ldy = w.ld;
    }
    const Result h = new_f32({T, g.R}, g.x.t);
    void *status = on.pointer(o[9], at::kInt, 1), *st = on.stream();
    if (g.some()) {
        const size_t bytes = cacti_hip_adapter_fwd_workspace(T, g.S, g.K, g.N, g.R, g.max_new);
        at::Tensor ws;
        if (bytes) ws = empty({(int64_t)bytes}, g.x.t, at::kByte);
        run([&] {
            return cacti_hip_adapter_fwd(T, g.S, g.K, g.N, g.R, g.n, g.max_new, g.x.t.data_ptr(), g.x.ld, g.A.data_ptr(), g.B.data_ptr(),
                                         g.starts.data_ptr(), g.ids, g.scale, base, ldb, y.ptr(), ldy, h.ptr(), bytes ? ws.data_ptr() : nullptr, bytes, status, st);
        });
    }
    return take2(y, h);
}

// (x, A, B, starts, ids, scale, h, dy, dx_acc, dA_acc, dB_acc, max_new, status): (dx, dA, dB)
PyObject *adapter_bwd(PyObject *const *o)
{
    const OnDevice on(on_gpu(tensor(o[0])));
    const Adapters g(o, o[11], on);
    const int64_t T = g.x.N;
    const at::Tensor &h = on.here(o[6], at::kFloat);
    require(h.dim() == 2 && h.size(0) == T && h.size(1) == g.R, "adapter_bwd: h [T, R] f32 expected");
    const Logits dy(o[7], on, "adapter_bwd: dy [T, N] f16 expected");
    require(dy.N == T && dy.V == g.N, "adapter_bwd: dy [T, N] f16 expected");
    Result dx = {at::Tensor(), nullptr};
    int64_t lddx = g.K;
    if (o[8] == Py_None) dx.t = empty({T, g.K}, g.x.t, at::kHalf);
    else {
        const Logits w(o[8], on, "adapter_bwd: dx_acc [T, K] f16 expected");
        require(w.N == T && w.V == g.K, "adapter_bwd: dx_acc [T, K] f16 expected");
        dx = {w.t, o[8]}, lddx = w.ld;
    }
    auto weights = [&](PyObject *acc, const at::Tensor &like) {
        const Result r = result(acc, like);
        require(r.t.sizes() == like.sizes(), "adapter_bwd: a gradient of another shape than its adapter");
        on.here(r.t);
        return r;
    };
    const Result dA = weights(o[9], g.A), dB = weights(o[10], g.B);
    void *status = on.pointer(o[12], at::kInt, 1), *st = on.stream();
    if (g.some()) {
        const size_t bytes = cacti_hip_adapter_bwd_workspace(T, g.K, g.N, g.R, g.n);
        const at::Tensor ws = empty({(int64_t)bytes}, g.x.t, at::kByte);
        run([&] {
            return cacti_hip_adapter_bwd(T, g.S, g.K, g.N, g.R, g.n, g.max_new, g.x.t.data_ptr(), g.x.ld, g.A.data_ptr(), g.B.data_ptr(),
                                         g.starts.data_ptr(), g.ids, g.scale, h.data_ptr(), dy.t.data_ptr(), dy.ld, dx.ptr(), lddx, dx.acc(),
                                         dA.ptr(), dA.acc(), dB.ptr(), dB.acc(), ws.data_ptr(), bytes, status, st);
        });
    } else {
        if (!dA.acc()) dA.t.zero_();
        if (!dB.acc()) dB.t.zero_();
    }
    return tuple_of({dx, dA, dB});
}

// refs and table of a call that hands pages out
struct Book {
    const at::Tensor &refs, &table;
    int64_t P, B, W, ldt;
    Book(PyObject *r, PyObject *t, const OnDevice &on) : refs(on.here(r, at::kInt)), table(on.here(on_gpu(tensor(t))))
    {
        require(table.scalar_type() == at::kInt && table.dim() == 2 && (table.size(1) <= 1 || table.stride(1) == 1),
                "paged cache: table [sequences, pages] of int32 expected");
        P = refs.numel(), B = table.size(0), W = table.size(1), ldt = B > 1 ? table.stride(0) : W;
    }
    bool some() const { return P > 0 && B > 0 && W > 0; }
};

// (refs, table, lens, parent, page, out, status): (table, lens)
PyObject *paged_fork(PyObject *const *o)
{
    const OnDevice on(on_gpu(tensor(o[0])));
    const Book k(o[0], o[1], on);
    given(o[2], "paged_fork: lens [sequences] expected"), given(o[3], "paged_fork: parent [sequences] expected");
    const void *lens = on.pointer(o[2], at::kInt, k.B), *parent = on.pointer(o[3], at::kInt, k.B);
    const int64_t page = number<int64_t>(o[4]);
    Result table = {at::Tensor(), nullptr}, now = {at::Tensor(), nullptr};
    int64_t ldn = k.W;
    if (o[5] == Py_None) table = new_i32({k.B, k.W}, k.refs), now = new_i32({k.B}, k.refs);
    else {
        require(PyTuple_Check(o[5]) && PyTuple_GET_SIZE(o[5]) == 2, "paged_fork: out = (table, lens) expected");
        PyObject *t = PyTuple_GET_ITEM(o[5], 0), *l = PyTuple_GET_ITEM(o[5], 1);
        const Book w(o[0], t, on);
        require(w.table.sizes() == k.table.sizes() && on.here(l, at::kInt).numel() == k.B, "paged_fork: shapes of out");
        table = {w.table, t}, now = {tensor(l), l}, ldn = w.ldt;
    }
    void *status = on.pointer(o[6], at::kInt, 1), *st = on.stream();
    if (k.some())
        run([&] {
            return cacti_hip_paged_fork(k.P, k.B, k.W, page, k.refs.data_ptr(), k.table.data_ptr(), k.ldt, lens, parent, table.ptr(), ldn, now.ptr(),
                                        status, st);
        });
    else require(k.B == 0, "paged_fork: a cache or a table without pages");
    return take2(table, now);
}

// (refs, table, first, lens, page, status): (src, dst, slots)
PyObject *paged_fit(PyObject *const *o)
{
    const OnDevice on(on_gpu(tensor(o[0])));
    const Book k(o[0], o[1], on);
    given(o[2], "paged_fit: first [sequences] expected"), given(o[3], "paged_fit: lens [sequences] expected");
    const void *first = on.pointer(o[2], at::kInt, k.B), *lens = on.pointer(o[3], at::kInt, k.B);
    const int64_t page = number<int64_t>(o[4]);
    void *status = on.pointer(o[5], at::kInt, 1), *st = on.stream();
    const Result src = new_i32({k.B}, k.refs), dst = new_i32({k.B}, k.refs), slots = new_i32({k.B}, k.refs);
    if (k.some()) {
        const size_t bytes = cacti_hip_paged_fit_workspace(k.P, k.B);
        const at::Tensor ws = empty({(int64_t)bytes}, k.refs, at::kByte);
        run([&] {
            return cacti_hip_paged_fit(k.P, k.B, k.W, page, k.refs.data_ptr(), k.table.data_ptr(), k.ldt, first, lens, src.ptr(), dst.ptr(),
                                       slots.ptr(), ws.data_ptr(), bytes, status, st);
        });
    } else require(k.B == 0, "paged_fit: a cache or a table without pages");
    return tuple_of({src, dst, slots});
}

// (refs, table): (src, dst, used)
PyObject *paged_compact(PyObject *const *o)
{
    const OnDevice on(on_gpu(tensor(o[0])));
    const Book k(o[0], o[1], on);
    void *st = on.stream();
    const Result src = new_i32({k.P / 2}, k.refs), dst = new_i32({k.P / 2}, k.refs), used = new_i32({1}, k.refs);
    require(k.some(), "paged_compact: a cache or a table without pages");
    const size_t bytes = cacti_hip_paged_compact_workspace(k.P);
    const at::Tensor ws = empty({(int64_t)bytes}, k.refs, at::kByte);
    run([&] {
        return cacti_hip_paged_compact(k.P, k.B, k.W, k.refs.data_ptr(), k.table.data_ptr(), k.ldt, src.ptr(), dst.ptr(), used.ptr(), ws.data_ptr(),
                                       bytes, st);
    });
    return tuple_of({src, dst, used});
}

// (caches, src, dst, slots)
PyObject *paged_copy(PyObject *const *o)
{
    const OnDevice on(on_gpu(tensor(o[1])));
    const at::Tensor &src = on.here(o[1], at::kInt);
    const int64_t n = src.numel();
    given(o[2], "paged_copy: dst, as many as src, expected");
    const void *dst = on.pointer(o[2], at::kInt, n), *slots = on.pointer(o[3], at::kInt, n);
    PyObject *seq = PySequence_Fast(o[0], "paged_copy: a list of caches expected");
    if (!seq) throw PyFailed();
    struct Held {
        PyObject *o;
        ~Held() { Py_DECREF(o); }
    } hold{seq};
    const int64_t layers = PySequence_Fast_GET_SIZE(seq);
    std::vector<at::Tensor> held;
    std::vector<void *> k, v, ks, vs;
    for (int64_t l = 0; l < layers; l++) {
        PyObject *c = PySequence_Fast_GET_ITEM(seq, l);
        require(PyTuple_Check(c) && PyTuple_GET_SIZE(c) == 4, "paged_copy: a cache is (k_pages, v_pages, k_scale, v_scale)");
        const at::Tensor &kt = on.here(on_gpu(tensor(PyTuple_GET_ITEM(c, 0)))), &vt = on.here(on_gpu(tensor(PyTuple_GET_ITEM(c, 1))));
        require(kt.dim() == 4 && kt.is_contiguous() && vt.is_contiguous() && vt.sizes() == kt.sizes() && vt.scalar_type() == kt.scalar_type() &&
                    (kt.scalar_type() == at::kHalf || kt.scalar_type() == at::kFloat8_e4m3fn) && kt.size(3) % 16 == 0,
                "paged cache: two contiguous tensors [pages, heads, page, Dp] of f16 or float8_e4m3fn expected");
        require(held.empty() || (held[0].sizes() == kt.sizes() && held[0].scalar_type() == kt.scalar_type()), "paged_copy: caches of one shape and type expected");
        const bool scaled = kt.scalar_type() != at::kHalf;
        for (int i = 2; i < 4; i++) require((PyTuple_GET_ITEM(c, i) != Py_None) == scaled, "paged cache: pages of 8 bits have scales, pages of 16 bits none");
        k.push_back(kt.data_ptr()), v.push_back(vt.data_ptr());
        ks.push_back(on.pointer(PyTuple_GET_ITEM(c, 2), at::kFloat, kt.size(0) * kt.size(1)));
        vs.push_back(on.pointer(PyTuple_GET_ITEM(c, 3), at::kFloat, kt.size(0) * kt.size(1)));
        // (held: another thread may change the list while the call runs)
        held.push_back(kt), held.push_back(vt);
        for (int i = 2; i < 4 && scaled; i++) held.push_back(tensor(PyTuple_GET_ITEM(c, i)));
    }
    void *st = on.stream();
    if (layers > 0 && n > 0 && held[0].numel() > 0) {
        const at::Tensor &t = held[0];
        run([&] {
            return cacti_hip_paged_copy(layers, k.data(), v.data(), ks.data(), vs.data(), t.scalar_type() == at::kHalf ? 16 : 8, t.size(0), t.size(1),
                                        t.size(2), t.size(3), n, src.data_ptr(), dst, slots, st);
        });
    }
    Py_RETURN_NONE;
}

// (xs)
PyObject *digests(PyObject *const *v)
{
    const Tensors xs(v[0]);
    std::vector<int64_t> ns(xs.size());
    for (size_t i = 0; i < xs.size(); i++) ns[i] = checked(xs[i], at::kHalf).numel();
    require(xs.size() > 0, "digests: no tensors");
    const at::Tensor out = empty({(int64_t)xs.size(), 257}, xs[0], at::kLong);
    const std::vector<void *> p = xs.pointers();
    void *st = stream();
    run([&] { return cacti_hip_digests_f16_batch((int)p.size(), p.data(), ns.data(), out.data_ptr(), nullptr, st); });
    return take2({out.narrow(1, 0, 256), nullptr}, {out.select(1, 256), nullptr});
}

// (grads, avgs, avg2s, masters, params, scalars)
PyObject *adamw32_step(PyObject *const *v)
{
    const Tensors g(v[0]), a(v[1]), b(v[2]), w(v[3]), p(v[4]);
    const size_t n = g.size();
    require(a.size() == n && b.size() == n && w.size() == n && p.size() == n, "adamw32_step: lists of one length expected");
    float sc[7];
    PyObject *seq = PySequence_Fast(v[5], "adamw32_step: seven scalars expected");
    if (!seq) throw PyFailed();
    bool ok = PySequence_Fast_GET_SIZE(seq) == 7;
    for (int i = 0; ok && i < 7; i++) ok = convert(PySequence_Fast_GET_ITEM(seq, i), &sc[i]);
    Py_DECREF(seq);
    if (PyErr_Occurred()) throw PyFailed();
    require(ok, "adamw32_step: seven scalars expected");
    std::vector<int64_t> ns(n);
    for (size_t i = 0; i < n; i++) {
        ns[i] = checked(g[i], at::kHalf).numel();
        require(checked(a[i], at::kFloat).numel() == ns[i] && checked(b[i], at::kFloat).numel() == ns[i] &&
                    checked(w[i], at::kFloat).numel() == ns[i] && checked(p[i], at::kHalf).numel() == ns[i],
                "adamw32_step: tensors of one size expected");
    }
    if (n == 0) Py_RETURN_NONE;
    const std::vector<void *> pg = g.pointers(), pa = a.pointers(), pb = b.pointers(), pw = w.pointers(), pp = p.pointers();
    void *st = stream();
    run([&] {
        return cacti_hip_adamw32_step_f16_batch((int)n, pg.data(), pa.data(), pb.data(), pw.data(), pp.data(), ns.data(), sc, nullptr, st);
    });
    Py_RETURN_NONE;
}

// (iter_nr, grad_scale, lr, wd, a1, a2, eps)
PyObject *adamw32_scalars(PyObject *const *v)
{
    float out[7];
    const int iter_nr = number<int>(v[0]);
    float in[6];
    for (int i = 0; i < 6; i++) in[i] = number<float>(v[1 + i]);
    const int rc = cacti_adamw32_scalars(iter_nr, in[0], in[1], in[2], in[3], in[4], in[5], out);
    if (rc) raise_status(rc);
    PyObject *r = PyList_New(7);
    for (int i = 0; i < 7; i++) PyList_SET_ITEM(r, i, PyFloat_FromDouble(out[i]));
    return r;
}

// an operator of N arguments as a CPython function
template <PyObject *(*F)(PyObject *const *), int N>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "%d arguments expected, %d given", N, (int)n);
        return nullptr;
    }
    try {
        return F(args);
    } catch (const PyFailed &) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

PyObject *set_check(PyObject *, PyObject *f)
{
    Py_INCREF(f);
    Py_XSETREF(g_check, f);
    Py_RETURN_NONE;
}

// cacti_hip_read_i32 (device pointer, stream): (status, value)
PyObject *read_i32(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    const void *p = nullptr;
    void *st = nullptr;
    if (n != 2 || !convert(args[0], &p) || !convert(args[1], &st)) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "2 arguments expected");
        return nullptr;
    }
    int32_t v = 0;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = cacti_hip_read_i32(p, &v, st);
    Py_END_ALLOW_THREADS
    return Py_BuildValue("(ii)", rc, (int)v);
}

#define FN(name)                                                                                      \
    {#name, (PyCFunction)(void (*)(void))(+[](PyObject *, PyObject *const *args, Py_ssize_t n) {       \
         return apply(&cacti_hip_##name, args, n);                                                    \
     }),                                                                                              \
     METH_FASTCALL, nullptr}

#define OP(name, n) {#name, (PyCFunction)(void (*)(void))(&entry<name, n>), METH_FASTCALL, nullptr}

PyMethodDef methods[] = {
    {"set_check", set_check, METH_O, nullptr},
    OP(gemm, 7),
    OP(gemm_batched, 7),
    OP(attention_fwd, 4),
    OP(attention_bwd, 8),
    OP(rms_norm_fwd, 3),
    OP(add_rms_norm_fwd, 4),
    OP(rms_norm_bwd, 6),
    OP(rope_fwd, 3),
    OP(rope_bwd, 4),
    OP(silu_gate_fwd, 2),
    OP(silu_gate_bwd, 5),
    OP(add_f16, 3),
    OP(softmax_ce_bwd, 4),
    OP(paged_append, 15),
    OP(paged_attention, 12),
    OP(verify_draft, 8),
    OP(distill_topk_fwd, 5),
    OP(distill_topk_bwd, 7),
    OP(token_logp_fwd, 5),
    OP(token_logp_bwd, 6),
    OP(policy_loss, 13),
    OP(preference_loss, 9),
    OP(adapter_fwd, 10),
    OP(adapter_bwd, 13),
    OP(paged_fork, 7),
    OP(paged_fit, 6),
    OP(paged_compact, 2),
    OP(paged_copy, 4),
    OP(digests, 1),
    OP(adamw32_step, 6),
    OP(adamw32_scalars, 7),
    FN(gemm_f16_strided_batched_tri),
    FN(accumulate_1d_f32),
    FN(accumulate_1d_f16),
    FN(accumulate_1d_u16),
    FN(rope_tables),
    FN(causal_softmax_fwd),
    FN(causal_softmax_bwd),
    FN(softmax_ce_fwd),
    FN(embed_fwd),
    FN(embed_bwd),
    FN(nan_count_f16),
    FN(abs_log2_hist8_f16),
    FN(online_average_scale_f16_f32),
    FN(online_average_square_scale_f16_f32),
    FN(online_adamw_update_f32),
    FN(cast_f32_f16),
    FN(cast_f16_f32),
    FN(raw_cast_bf16_f16),
    FN(raw_cast_bf16_f32),
    FN(raw_cast_f32_bf16),
    FN(raw_cast_f16_bf16),
    {"read_i32", (PyCFunction)(void (*)(void))read_i32, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fast(void) { return PyModule_Create(&module); }
