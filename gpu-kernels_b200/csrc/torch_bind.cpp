// torch_bind.cpp — the torch side of the 16-bit linear and mixture-of-experts operators:
// argument checks, output tensors and the call of the C ABI, as a CPython extension.
//
// A decode step's operators take a few microseconds on the GPU, less than their checks,
// allocations and argument conversions take in Python (a 16-token router: 15 us of host time
// a call from Python, about 6 from here).  It holds no computation: every function is one or
// more calls of the C ABI, through addresses that the package passes in once (bind), so that
// it follows whichever build of the library is loaded.
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/empty_like.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "../../include/nvfp4_b200.h"

namespace {

struct Entries {
    decltype(&nvfp4_linear) linear;
    decltype(&nvfp4_linear_dgrad) dgrad;
    decltype(&nvfp4_linear_wgrad) wgrad;
    decltype(&nvfp4_activation_backward) act_backward;
    decltype(&nvfp4_activation_backward_workspace_size) act_backward_ws;
    decltype(&nvfp4_moe_route) route;
    decltype(&nvfp4_moe_route_workspace_size) route_ws;
    decltype(&nvfp4_moe_route_backward) route_backward;
    decltype(&nvfp4_moe_dispatch) dispatch;
    decltype(&nvfp4_moe_combine) combine;
    decltype(&nvfp4_moe_combine_backward) combine_backward;
} L;
PyObject *on_status = nullptr;  // called with (status, entry point) where a status is not OK

struct Refused {};  // a Python exception has been set

[[noreturn]] void refuse(const std::string &what) {
    PyErr_SetString(PyExc_ValueError, what.c_str());
    throw Refused();
}

void check(int status, const char *where) {
    if (status == NVFP4_OK) return;
    PyObject *r = PyObject_CallFunction(on_status, "is", status, where);
    Py_XDECREF(r);
    if (r) PyErr_SetString(PyExc_RuntimeError, where);
    throw Refused();
}

// ------------------------------------------------------------------------- arguments
const at::Tensor &tensor(PyObject *o, const char *name) {
    if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
    return THPVariable_Unpack(o);
}

const at::Tensor *maybe(PyObject *o, const char *name) { return o == Py_None ? nullptr : &tensor(o, name); }

void *ptr(const at::Tensor *t) { return t ? t->data_ptr() : nullptr; }

int64_t integer(PyObject *o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Refused();
    return v;
}

int small(int64_t v, const char *what) {
    if (v < 0 || v > INT32_MAX) refuse(std::string(what) + " is out of range");
    return (int)v;
}

bool truth(PyObject *o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Refused();
    return v != 0;
}

double number(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Refused();
    return v;
}

int dtype16(const at::Tensor &t) {
    return t.scalar_type() == at::kBFloat16 ? NVFP4_BF16 : t.scalar_type() == at::kHalf ? NVFP4_F16 : -1;
}

std::string shape_text(at::IntArrayRef s) {
    std::string r = "(";
    for (size_t i = 0; i < s.size(); i++) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + ")";
}

// A contiguous tensor of this shape and type, on `like`'s device.
const at::Tensor &expect(const at::Tensor &t, const char *name, at::IntArrayRef shape, at::ScalarType type,
                         const at::Tensor &like) {
    if (t.scalar_type() != type || t.device() != like.device() || t.sizes() != shape || !t.is_contiguous())
        refuse(std::string(name) + " must be a contiguous " + c10::toString(type) + " tensor " + shape_text(shape) +
               " on " + like.device().str());
    return t;
}

struct Rows {
    int M, K, dtype;
    int64_t pitch;
};

// A 2-D 16-bit CUDA tensor whose rows are contiguous.
Rows rows_of(const at::Tensor &x, const char *name) {
    Rows r;
    r.dtype = dtype16(x);
    if (!x.is_cuda() || x.dim() != 2 || r.dtype < 0)
        refuse(std::string(name) + " must be a 2-D bf16 or fp16 CUDA tensor");
    r.M = small(x.size(0), "the number of rows");
    r.K = small(x.size(1), "the number of columns");
    r.pitch = r.M > 1 ? x.stride(0) : r.K;  // a single row's stride says nothing
    if ((r.K > 1 && x.stride(1) != 1) || r.pitch < r.K) refuse(std::string(name) + " must have contiguous rows");
    if (r.K % 8 || r.pitch % 8 || !r.K)
        refuse(std::string(name) + " must have a multiple of 8 columns, rows 16 bytes aligned");
    return r;
}

int groups_of(const at::Tensor *offs, const at::Tensor &x) {
    if (!offs) return 1;
    if (offs->scalar_type() != at::kInt || offs->dim() != 1 || offs->numel() < 2 || offs->device() != x.device() ||
        !offs->is_contiguous())
        refuse("m_offsets must be a contiguous 1-D int32 tensor of groups + 1 entries on the device");
    if (offs->numel() > 257) refuse("at most 256 groups");
    return (int)offs->numel() - 1;
}

// Rows N of one group's weight.
int weight_rows(const at::Tensor &w, int groups, const Rows &x, const at::Tensor &like) {
    if (w.dim() != 2 || w.size(1) != x.K || w.size(0) % groups)
        refuse(std::string("w must be [") + (groups > 1 ? "groups * N, " : "N, ") + std::to_string(x.K) + "]");
    expect(w, "w", w.sizes(), like.scalar_type(), like);
    const int N = small(w.size(0) / groups, "N");
    if (N % 8 || !N) refuse("N must be a multiple of 8");
    return N;
}

int out_columns(int act, int N) {
    if (act != NVFP4_ACT_SWIGLU) return N;
    if (N % 32) refuse("swiglu: N must be a multiple of 32 (gate and up rows in blocks of 16)");
    return N / 2;
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, const at::Tensor &like) {
    return at::detail::empty_cuda(shape, type, like.device(), std::nullopt);
}

// `out` may not share memory with an input of the call: tiles are stored while others are
// still being read.
void apart(const at::Tensor &out, const at::Tensor *in, const char *name) {
    if (!in || !out.numel() || !in->numel()) return;
    const auto end = [](const at::Tensor &t) {
        int64_t last = 0;
        for (int64_t d = 0; d < t.dim(); d++) last += (t.size(d) - 1) * t.stride(d);
        return static_cast<const char *>(t.data_ptr()) + (last + 1) * t.element_size();
    };
    if (static_cast<const char *>(out.data_ptr()) < end(*in) && static_cast<const char *>(in->data_ptr()) < end(out))
        refuse(std::string("out must not share memory with ") + name);
}

// Runs f (allocations and calls of the C ABI) without the GIL: a launch waits where the
// stream's queue is full, and what it waits for may be a host callback that needs the GIL.
template <typename F>
int unlocked(F f) {
    struct Unlock {
        PyThreadState *state = PyEval_SaveThread();
        ~Unlock() { PyEval_RestoreThread(state); }
    } unlock;
    return f();
}

// The current stream of the tensors' device, made current for the call.
struct Stream {
    explicit Stream(const at::Tensor &t)
        : guard(t.device()), handle(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
    c10::cuda::CUDAGuard guard;
    void *handle;
};

PyObject *wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }

PyObject *none() { Py_RETURN_NONE; }

template <size_t N>
PyObject *tuple_of(PyObject *const (&items)[N]) {
    PyObject *t = PyTuple_New(N);
    if (!t) throw Refused();
    for (size_t i = 0; i < N; i++) PyTuple_SET_ITEM(t, i, items[i]);
    return t;
}

// ------------------------------------------------------------------------- operators
// linear(x, w, m_offsets, bias, activation, residual, out, return_preact)
PyObject *linear(PyObject *const *a) {
    const at::Tensor &x = tensor(a[0], "x"), &w = tensor(a[1], "w");
    const at::Tensor *offs = maybe(a[2], "m_offsets"), *bias = maybe(a[3], "bias"), *res = maybe(a[5], "residual");
    const int act = (int)integer(a[4]);
    const Rows r = rows_of(x, "x");
    const int G = groups_of(offs, x), N = weight_rows(w, G, r, x), No = out_columns(act, N);
    const auto type = x.scalar_type();
    if (bias) {
        if (!offs && bias->dim() == 1) expect(*bias, "bias", {N}, type, x);
        else expect(*bias, "bias", {G, N}, type, x);
    }
    if (res) expect(*res, "residual", {r.M, No}, type, x);
    at::Tensor y, z;
    if (a[6] != Py_None) {
        y = expect(tensor(a[6], "out"), "out", {r.M, No}, type, x);
        apart(y, &x, "x");
        apart(y, &w, "w");
        apart(y, bias, "bias");
        apart(y, offs, "m_offsets");
        // the residual itself is fine: each element is read where it is then written
        if (res && res->data_ptr() != y.data_ptr()) apart(y, res, "residual");
    }
    const bool preact = truth(a[7]);
    check(unlocked([&] {
              if (!y.defined()) y = empty({r.M, No}, type, x);
              if (preact) z = empty({r.M, N}, type, x);
              const Stream s(x);
              return L.linear(x.data_ptr(), r.pitch, w.data_ptr(), ptr(bias), ptr(res), y.data_ptr(),
                              preact ? z.data_ptr() : nullptr, static_cast<const int32_t *>(ptr(offs)), G, r.M, N, r.K,
                              act, r.dtype, s.handle);
          }),
          "nvfp4_linear");
    if (!preact) return wrap(std::move(y));
    return tuple_of<2>({wrap(std::move(y)), wrap(std::move(z))});
}

// linear_backward(dy, x, w, m_offsets, preact, activation, bias_grad, input_grad, weight_grad)
PyObject *linear_backward(PyObject *const *a) {
    const at::Tensor &dy = tensor(a[0], "dy"), &x = tensor(a[1], "x"), &w = tensor(a[2], "w");
    const at::Tensor *offs = maybe(a[3], "m_offsets"), *z = maybe(a[4], "preact");
    const int act = (int)integer(a[5]);
    const bool bias_grad = truth(a[6]), input_grad = truth(a[7]), weight_grad = truth(a[8]);
    const Rows r = rows_of(x, "x");
    const int G = groups_of(offs, x), N = weight_rows(w, G, r, x), No = out_columns(act, N);
    const auto type = x.scalar_type();
    expect(dy, "dy", {r.M, No}, type, x);
    if (act) {
        if (!z) refuse("an activation's gradient needs preact");
        expect(*z, "preact", {r.M, N}, type, x);
    }
    const int32_t *o = static_cast<const int32_t *>(ptr(offs));
    at::Tensor dx, dw, db;
    const char *where = "nvfp4_activation_backward";
    const int status = unlocked([&] {
        at::Tensor dz = dy, ws;
        const Stream s(x);
        int st = NVFP4_OK;
        if (bias_grad || (act && (input_grad || weight_grad))) {
            if (act) dz = empty({r.M, N}, type, x);
            size_t bytes = 0;
            if (bias_grad) {
                db = offs ? empty({G, N}, type, x) : empty({N}, type, x);
                bytes = L.act_backward_ws(G, r.M, N);
                ws = empty({(int64_t)(bytes / 4)}, at::kFloat, x);
            }
            st = L.act_backward(dy.data_ptr(), act ? z->data_ptr() : nullptr, act ? dz.data_ptr() : nullptr,
                                bias_grad ? db.data_ptr() : nullptr, o, G, r.M, N, act, r.dtype,
                                bias_grad ? ws.data_ptr() : nullptr, bytes, s.handle);
        }
        if (!st && input_grad) {
            where = "nvfp4_linear_dgrad";
            dx = empty({r.M, r.K}, type, x);
            st = L.dgrad(dz.data_ptr(), w.data_ptr(), dx.data_ptr(), o, G, r.M, N, r.K, r.dtype, s.handle);
        }
        if (!st && weight_grad) {
            where = "nvfp4_linear_wgrad";
            dw = empty(w.sizes(), type, x);
            st = L.wgrad(dz.data_ptr(), x.data_ptr(), r.pitch, dw.data_ptr(), o, G, r.M, N, r.K, r.dtype,
                         s.handle);
        }
        return st;
    });
    check(status, where);
    return tuple_of<3>({input_grad ? wrap(std::move(dx)) : none(), weight_grad ? wrap(std::move(dw)) : none(),
                        bias_grad ? wrap(std::move(db)) : none()});
}

struct Logits {
    int T, E, dtype;
};

Logits logits_of(const at::Tensor &l) {
    Logits r;
    r.dtype = l.scalar_type() == at::kFloat ? NVFP4_F32 : dtype16(l);
    if (!l.is_cuda() || l.dim() != 2 || r.dtype < 0 || !l.is_contiguous())
        refuse("logits must be a contiguous 2-D bf16, fp16 or fp32 CUDA tensor");
    r.T = small(l.size(0), "the number of tokens");
    r.E = small(l.size(1), "the number of experts");
    return r;
}

// moe_route(logits, top_k, scoring, bias, renormalize, scale)
PyObject *moe_route(PyObject *const *a) {
    const at::Tensor &l = tensor(a[0], "logits");
    const int k = small(integer(a[1]), "top_k"), scoring = (int)integer(a[2]);
    const at::Tensor *bias = maybe(a[3], "bias");
    const bool renormalize = truth(a[4]);
    const float scale = (float)number(a[5]);
    const Logits r = logits_of(l);
    if (bias) {
        if (scoring != NVFP4_SCORE_SIGMOID) refuse("a selection bias needs sigmoid scoring");
        expect(*bias, "bias", {r.E}, at::kFloat, l);
    }
    at::Tensor weights, experts, rows, offs;
    check(unlocked([&] {
              weights = empty({r.T, k}, at::kFloat, l);
              experts = empty({r.T, k}, at::kInt, l);
              rows = empty({r.T, k}, at::kInt, l);
              offs = empty({r.E + 1}, at::kInt, l);
              at::Tensor ws;
              size_t bytes = 0;
              if (r.T > 64) {  // fewer tokens need none
                  bytes = L.route_ws(r.T, r.E);
                  ws = empty({(int64_t)(bytes / 4)}, at::kInt, l);
              }
              const Stream s(l);
              return L.route(l.data_ptr(), r.dtype, static_cast<const float *>(ptr(bias)), r.T, r.E, k, scoring,
                             renormalize, scale, weights.data_ptr<float>(), experts.data_ptr<int>(),
                             rows.data_ptr<int>(), offs.data_ptr<int>(), bytes ? ws.data_ptr() : nullptr, bytes,
                             s.handle);
          }),
          "nvfp4_moe_route");
    return tuple_of<4>({wrap(std::move(weights)), wrap(std::move(experts)), wrap(std::move(rows)),
                        wrap(std::move(offs))});
}

// moe_route_backward(dweights, logits, experts, scoring, renormalize, scale)
PyObject *moe_route_backward(PyObject *const *a) {
    const at::Tensor &dw = tensor(a[0], "dweights"), &l = tensor(a[1], "logits"), &e = tensor(a[2], "experts");
    const int scoring = (int)integer(a[3]);
    const bool renormalize = truth(a[4]);
    const float scale = (float)number(a[5]);
    const Logits r = logits_of(l);
    if (e.dim() != 2) refuse("experts must be 2-D");
    const int k = small(e.size(1), "top_k");
    expect(e, "experts", {r.T, k}, at::kInt, l);
    expect(dw, "dweights", {r.T, k}, at::kFloat, l);
    at::Tensor dl;
    check(unlocked([&] {
              dl = empty({r.T, r.E}, l.scalar_type(), l);
              const Stream s(l);
              return L.route_backward(dw.data_ptr<float>(), l.data_ptr(), r.dtype, e.data_ptr<int>(), r.T, r.E, k,
                                      scoring, renormalize, scale, dl.data_ptr(), s.handle);
          }),
          "nvfp4_moe_route_backward");
    return wrap(std::move(dl));
}

// A Routing (weights, experts, rows, m_offsets) on `like`'s device.
struct Routed {
    int T, k, E;
    const float *weights;
    const int *rows, *offs;
};

Routed routed(PyObject *o, const at::Tensor &like) {
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) refuse("routing must be a Routing");
    const at::Tensor &w = tensor(PyTuple_GET_ITEM(o, 0), "routing.weights");
    const at::Tensor &rows = tensor(PyTuple_GET_ITEM(o, 2), "routing.rows");
    const at::Tensor &offs = tensor(PyTuple_GET_ITEM(o, 3), "routing.m_offsets");
    if (rows.dim() != 2 || offs.dim() != 1 || offs.numel() < 2)
        refuse("routing.rows must be 2-D and routing.m_offsets 1-D");
    expect(rows, "routing.rows", rows.sizes(), at::kInt, like);
    expect(offs, "routing.m_offsets", offs.sizes(), at::kInt, like);
    expect(w, "routing.weights", rows.sizes(), at::kFloat, like);
    return {small(rows.size(0), "the number of tokens"), small(rows.size(1), "top_k"),
            small(offs.numel() - 1, "the number of experts"), w.data_ptr<float>(), rows.data_ptr<int>(),
            offs.data_ptr<int>()};
}

int columns(const at::Tensor &t, const char *name, int64_t rows) {
    if (t.size(0) != rows || !t.is_contiguous())
        refuse(std::string(name) + " must be a contiguous 2-D bf16 or fp16 CUDA tensor of " + std::to_string(rows) +
               " rows");
    const int K = small(t.size(1), "the number of columns");
    if (K % 8 || !K) refuse(std::string(name) + " must have a multiple of 8 columns");
    return K;
}

const at::Tensor &matrix16(PyObject *o, const char *name) {
    const at::Tensor &t = tensor(o, name);
    if (!t.is_cuda() || t.dim() != 2 || dtype16(t) < 0)
        refuse(std::string(name) + " must be a contiguous 2-D bf16 or fp16 CUDA tensor");
    return t;
}

// moe_dispatch(x, routing)
PyObject *moe_dispatch(PyObject *const *a) {
    const at::Tensor &x = matrix16(a[0], "x");
    const Routed r = routed(a[1], x);
    const int K = columns(x, "x", r.T);
    at::Tensor out;
    check(unlocked([&] {
              out = empty({(int64_t)r.T * r.k, K}, x.scalar_type(), x);
              const Stream s(x);
              return L.dispatch(x.data_ptr(), r.rows, r.offs, r.T, r.E, r.k, K, out.data_ptr(), s.handle);
          }),
          "nvfp4_moe_dispatch");
    return wrap(std::move(out));
}

// moe_combine(x_rows, routing, residual, weighted)
PyObject *moe_combine(PyObject *const *a) {
    const at::Tensor &x = matrix16(a[0], "x_rows");
    const Routed r = routed(a[1], x);
    const int K = columns(x, "x_rows", (int64_t)r.T * r.k);
    const at::Tensor *res = maybe(a[2], "residual");
    if (res) expect(*res, "residual", {r.T, K}, x.scalar_type(), x);
    const float *weights = truth(a[3]) ? r.weights : nullptr;
    at::Tensor y;
    check(unlocked([&] {
              y = empty({r.T, K}, x.scalar_type(), x);
              const Stream s(x);
              return L.combine(x.data_ptr(), dtype16(x), r.rows, weights, ptr(res), r.T, r.k, K, y.data_ptr(), s.handle);
          }),
          "nvfp4_moe_combine");
    return wrap(std::move(y));
}

// moe_combine_backward(dy, x_rows, routing)
PyObject *moe_combine_backward(PyObject *const *a) {
    const at::Tensor &dy = tensor(a[0], "dy"), &x = matrix16(a[1], "x_rows");
    const Routed r = routed(a[2], x);
    const int K = columns(x, "x_rows", (int64_t)r.T * r.k);
    expect(dy, "dy", {r.T, K}, x.scalar_type(), x);
    at::Tensor dx, dw;
    check(unlocked([&] {
              dx = empty({(int64_t)r.T * r.k, K}, x.scalar_type(), x);
              dw = empty({r.T, r.k}, at::kFloat, x);
              const Stream s(x);
              return L.combine_backward(dy.data_ptr(), x.data_ptr(), dtype16(x), r.rows, r.weights, r.offs, r.T, r.E,
                                        r.k, K, dx.data_ptr(), dw.data_ptr<float>(), s.handle);
          }),
          "nvfp4_moe_combine_backward");
    return tuple_of<2>({wrap(std::move(dx)), wrap(std::move(dw))});
}

// bind(on_status, addresses of the entry points in the order of Entries)
PyObject *bind(PyObject *const *a) {
    static_assert(sizeof(Entries) == 11 * sizeof(void *), "one address each");
    void *at[11];
    for (int i = 0; i < 11; i++) at[i] = reinterpret_cast<void *>((uintptr_t)PyLong_AsUnsignedLongLong(a[1 + i]));
    if (PyErr_Occurred()) throw Refused();
    memcpy(&L, at, sizeof(L));
    Py_INCREF(a[0]);
    Py_XSETREF(on_status, a[0]);
    return none();
}

// Every function takes exactly N positional arguments; C++ exceptions (torch's own, out of
// memory) become Python ones here.
template <PyObject *(*F)(PyObject *const *), int N>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, n);
        return nullptr;
    }
    try {
        return F(args);
    } catch (const Refused &) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

#define METHOD(name, n) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(&entry<name, n>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind, 12),           METHOD(linear, 8),          METHOD(linear_backward, 9),
                         METHOD(moe_route, 6),       METHOD(moe_route_backward, 6), METHOD(moe_dispatch, 2),
                         METHOD(moe_combine, 4),     METHOD(moe_combine_backward, 3), {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_bind() { return PyModule_Create(&module); }
