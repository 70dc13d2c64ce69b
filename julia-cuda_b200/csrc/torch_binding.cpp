// The fine-tuning operators on torch tensors, from Python: argument checks, the current stream, scratch
// from torch's allocator, and the call into the C ABI (include/julia_cuda.h). Written against CPython and
// ATen rather than ctypes because these calls are short: checked in Python, a backward linear layer of 64
// rows spent 15 us in the host of which the C entry was 7.
//
// training.py holds the documented functions; each passes its arguments here in order.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "../../include/julia_cuda.h"

namespace {

PyObject *g_error = nullptr;  // JuliaCudaError

// Thrown with a Python error set.
struct Raised {};

[[noreturn]] void fail(const std::string &msg) {
    PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, msg.c_str());
    throw Raised();
}

// What an argument is called in messages.
struct Name {
    const char *op, *arg;
    std::string str() const { return std::string(op) + ": " + arg; }
};

// A tensor argument, or nullptr for None.
const at::Tensor *tensor(const Name &n, PyObject *o, bool needed = true) {
    if (o == Py_None) {
        if (needed) fail(n.str() + " must be a tensor, not None");
        return nullptr;
    }
    if (!THPVariable_Check(o)) fail(n.str() + " must be a tensor");
    return &THPVariable_Unpack(o);
}

struct Matrix {
    void *p = nullptr;
    size_t ld = 0;
};

std::string shape_of(const at::Tensor &t) {
    std::string s = "[";
    for (int64_t i = 0; i < t.dim(); i++) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + "] of " + c10::toString(t.scalar_type());
}

// A [rows, cols] tensor of `type` on device `dev` with contiguous rows that do not overlap.
Matrix matrix(const Name &n, const at::Tensor *t, int64_t rows, int64_t cols, at::ScalarType type, int dev) {
    if (!t) return {};
    if (t->scalar_type() != type || t->dim() != 2 || t->size(0) != rows || t->size(1) != cols || !t->is_cuda() ||
        t->get_device() != dev)
        fail(n.str() + " must be a [" + std::to_string(rows) + ", " + std::to_string(cols) +
             "] tensor on the current device of " + c10::toString(type) + ", not " + shape_of(*t));
    const int64_t sr = t->stride(0), sc = t->stride(1);
    if ((cols > 1 && sc != 1) || (rows > 1 && sr < cols))
        fail(n.str() + " must have contiguous rows that do not overlap");
    return {t->data_ptr(), (size_t)(rows > 1 ? sr : cols)};
}

void *vector(const Name &n, const at::Tensor *t, int64_t count, at::ScalarType type, int dev) {
    if (!t) return nullptr;
    if (t->scalar_type() != type || t->numel() != count || !t->is_cuda() || t->get_device() != dev || !t->is_contiguous())
        fail(n.str() + " must be a contiguous tensor on the current device of " + std::to_string(count) + " elements of " +
             c10::toString(type) + ", not " + shape_of(*t));
    return t->data_ptr();
}
float *floats(const Name &n, PyObject *o, int64_t count, int dev, bool needed = false) {
    return static_cast<float *>(vector(n, tensor(n, o, needed), count, at::kFloat, dev));
}

// The device of an operator's first tensor, which must be the current one.
int device_of(const char *op, const at::Tensor &t) {
    const int dev = t.is_cuda() ? (int)t.get_device() : -1;
    if (dev < 0 || dev != (int)c10::cuda::current_device()) fail(std::string(op) + ": the tensors are not on the current device");
    return dev;
}

void check_sizes(const char *op, const at::Tensor &t) {
    for (const int64_t n : t.sizes())
        if (n > 0x7FFFFFFFll) fail(std::string(op) + ": at most 2^31 - 1 rows and columns");
}

uint32_t type_of(const char *op, const at::Tensor &x, bool halves) {
    if (x.dim() != 2) fail(std::string(op) + ": x must be a matrix");
    check_sizes(op, x);
    switch (x.scalar_type()) {
        case at::kHalf: return JC_F16;
        case at::kBFloat16: return JC_BF16;
        case at::kFloat:
            if (!halves) return JC_F32;
            [[fallthrough]];
        default: fail(std::string(op) + ": x must be a matrix of float16" + (halves ? " or bfloat16" : ", bfloat16 or float32"));
    }
}

uint32_t act_of(const char *op, PyObject *o) {
    const char *s = PyUnicode_Check(o) ? PyUnicode_AsUTF8(o) : nullptr;
    if (s && !strcmp(s, "none")) return 0;
    if (s && !strcmp(s, "relu")) return JC_EPI_RELU;
    if (s && !strcmp(s, "gelu")) return JC_EPI_GELU;
    PyErr_Clear();
    fail(std::string(op) + ": act must be one of none, relu, gelu");
}

// The stream argument: None (the current one), a torch stream, or a cudaStream_t as a number.
struct Queue {
    void *handle;
    bool current;
};
Queue queue_of(PyObject *o, int dev) {
    if (o == Py_None) return {c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(), true};
    PyObject *h = PyLong_Check(o) ? Py_NewRef(o) : PyObject_GetAttrString(o, "cuda_stream");
    if (!h) throw Raised();
    void *p = PyLong_AsVoidPtr(h);
    Py_DECREF(h);
    if (!p && PyErr_Occurred()) throw Raised();
    return {p, false};
}

// Scratch of `bytes`: the caller's `ws`, or torch's, from the pool of the stream that will use it: a block
// of another stream's pool may still be in use by what that stream has queued.
void *scratch(const Name &n, PyObject *ws, size_t bytes, const at::Tensor &like, const Queue &q, int dev, at::Tensor *keep) {
    if (bytes == 0) return nullptr;
    if (const at::Tensor *t = tensor(n, ws, false)) {
        if (!t->is_cuda() || t->get_device() != dev || !t->is_contiguous() || (size_t)t->nbytes() < bytes)
            fail(n.str() + " needs " + std::to_string(bytes) + " contiguous bytes on the current device");
        return t->data_ptr();
    }
    c10::cuda::OptionalCUDAStreamGuard on;
    if (!q.current)
        on.reset_stream(c10::cuda::getStreamFromExternal(static_cast<cudaStream_t>(q.handle), (c10::DeviceIndex)dev));
    *keep = at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
    return keep->data_ptr();
}

PyObject *done(int rc, const char *entry) {
    if (rc != 0) fail(std::string(entry) + ": " + jc_last_error());
    Py_RETURN_NONE;
}

double number(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised();
    return v;
}

// Runs f with its arguments counted, torch's exceptions turned into Python's.
template <class F>
PyObject *call(Py_ssize_t got, Py_ssize_t want, F &&f) {
    try {
        if (got != want) {
            PyErr_Format(PyExc_TypeError, "%zd arguments expected", want);
            return nullptr;
        }
        return f();
    } catch (const Raised &) {
        return nullptr;
    } catch (const std::exception &e) {
        PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

PyObject *set_error(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return call(n, 1, [&]() -> PyObject * {
        Py_XSETREF(g_error, Py_NewRef(a[0]));
        Py_RETURN_NONE;
    });
}

// (x, gamma, beta, y, stats, eps, stream)
PyObject *layer_norm(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return call(n, 7, [&] {
        const char *op = "layer_norm";
        const at::Tensor &x = *tensor({op, "x"}, a[0]);
        const uint32_t type = type_of(op, x, false);
        const int dev = device_of(op, x);
        const int64_t rows = x.size(0), d = x.size(1);
        const at::ScalarType st = x.scalar_type();
        const Matrix mx = matrix({op, "x"}, &x, rows, d, st, dev), my = matrix({op, "y"}, tensor({op, "y"}, a[3]), rows, d, st, dev);
        return done(jc_layer_norm(type, mx.p, mx.ld, floats({op, "gamma"}, a[1], d, dev, true), floats({op, "beta"}, a[2], d, dev),
                                  (float)number(a[5]), (uint32_t)rows, (uint32_t)d, my.p, my.ld,
                                  floats({op, "stats"}, a[4], 2 * rows, dev), queue_of(a[6], dev).handle),
                    "jc_layer_norm");
    });
}

// (dy, x, gamma, stats, dx, dgamma, dbeta, add, ws, stream)
PyObject *layer_norm_backward(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return call(n, 10, [&] {
        const char *op = "layer_norm_backward";
        const at::Tensor &x = *tensor({op, "x"}, a[1]);
        const uint32_t type = type_of(op, x, false);
        const int dev = device_of(op, x);
        const int64_t rows = x.size(0), d = x.size(1);
        const at::ScalarType st = x.scalar_type();
        const Matrix mdy = matrix({op, "dy"}, tensor({op, "dy"}, a[0]), rows, d, st, dev), mx = matrix({op, "x"}, &x, rows, d, st, dev),
                     mdx = matrix({op, "dx"}, tensor({op, "dx"}, a[4]), rows, d, st, dev),
                     madd = matrix({op, "add"}, tensor({op, "add"}, a[7], false), rows, d, st, dev);
        const float *gamma = floats({op, "gamma"}, a[2], d, dev, true), *stats = floats({op, "stats"}, a[3], 2 * rows, dev, true);
        float *dgamma = floats({op, "dgamma"}, a[5], d, dev), *dbeta = floats({op, "dbeta"}, a[6], d, dev);
        const Queue q = queue_of(a[9], dev);
        at::Tensor keep;
        const size_t need = dgamma || dbeta ? 4 * jc_layer_norm_ws_floats((uint32_t)rows, (uint32_t)d) : 0;
        float *ws = static_cast<float *>(scratch({op, "ws"}, a[8], need, x, q, dev, &keep));
        return done(jc_layer_norm_backward(type, mdy.p, mdy.ld, mx.p, mx.ld, gamma, stats, madd.p, madd.ld, (uint32_t)rows,
                                           (uint32_t)d, mdx.p, mdx.ld, dgamma, dbeta, ws, q.handle),
                    "jc_layer_norm_backward");
    });
}

// (x, w, y, bias, act, res, z, ws, stream)
PyObject *linear(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return call(n, 9, [&] {
        const char *op = "linear";
        const at::Tensor &x = *tensor({op, "x"}, a[0]), &w = *tensor({op, "w"}, a[1]);
        const uint32_t type = type_of(op, x, true);
        check_sizes(op, w);
        const int dev = device_of(op, x);
        const int64_t m = x.size(0), k = x.size(1), c = w.dim() == 2 ? w.size(0) : 0;
        const at::ScalarType st = x.scalar_type();
        const Matrix mx = matrix({op, "x"}, &x, m, k, st, dev), mw = matrix({op, "w"}, &w, c, k, st, dev),
                     my = matrix({op, "y"}, tensor({op, "y"}, a[2]), m, c, st, dev),
                     mr = matrix({op, "res"}, tensor({op, "res"}, a[5], false), m, c, st, dev),
                     mz = matrix({op, "z"}, tensor({op, "z"}, a[6], false), m, c, st, dev);
        const Queue q = queue_of(a[8], dev);
        at::Tensor keep;
        const size_t need = jc_linear_ws_bytes(mx.p, mx.ld, mw.p, mw.ld, (uint32_t)m, (uint32_t)c, (uint32_t)k);
        void *ws = scratch({op, "ws"}, a[7], need, x, q, dev, &keep);
        return done(jc_linear(type, act_of(op, a[4]), mx.p, mx.ld, mw.p, mw.ld, floats({op, "bias"}, a[3], c, dev), mr.p, mr.ld,
                              my.p, my.ld, mz.p, mz.ld, (uint32_t)m, (uint32_t)c, (uint32_t)k, ws, q.handle),
                    "jc_linear");
    });
}

// (dy, x, w, z, act, dx, dw, dbias, ws, stream)
PyObject *linear_backward(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return call(n, 10, [&] {
        const char *op = "linear_backward";
        const at::Tensor &x = *tensor({op, "x"}, a[1]), &w = *tensor({op, "w"}, a[2]);
        const uint32_t type = type_of(op, x, true), act = act_of(op, a[4]);
        check_sizes(op, w);
        const int dev = device_of(op, x);
        const int64_t m = x.size(0), k = x.size(1), c = w.dim() == 2 ? w.size(0) : 0;
        const at::ScalarType st = x.scalar_type();
        const Matrix mdy = matrix({op, "dy"}, tensor({op, "dy"}, a[0]), m, c, st, dev), mx = matrix({op, "x"}, &x, m, k, st, dev),
                     mw = matrix({op, "w"}, &w, c, k, st, dev), mz = matrix({op, "z"}, tensor({op, "z"}, a[3], false), m, c, st, dev),
                     mdx = matrix({op, "dx"}, tensor({op, "dx"}, a[5], false), m, k, st, dev),
                     mdw = matrix({op, "dw"}, tensor({op, "dw"}, a[6], false), c, k, st, dev);
        float *dbias = floats({op, "dbias"}, a[7], c, dev);
        const Queue q = queue_of(a[9], dev);
        at::Tensor keep;
        const size_t need = jc_linear_backward_ws_bytes(mx.p, mx.ld, mw.p, mw.ld, (uint32_t)m, (uint32_t)c, (uint32_t)k);
        void *ws = scratch({op, "ws"}, a[8], need, x, q, dev, &keep);
        return done(jc_linear_backward(type, act, mdy.p, mdy.ld, mx.p, mx.ld, mw.p, mw.ld, mz.p, mz.ld, (uint32_t)m, (uint32_t)c,
                                       (uint32_t)k, mdx.p, mdx.ld, mdw.p, mdw.ld, dbias, ws, q.handle),
                    "jc_linear_backward");
    });
}

// (logits, offsets, gold, loss, dlogits, weight, stream)
PyObject *choice_loss(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return call(n, 7, [&] {
        const char *op = "choice_loss";
        const at::Tensor &l = *tensor({op, "logits"}, a[0]), &g = *tensor({op, "gold"}, a[2]);
        const int dev = device_of(op, l);
        const int64_t all = l.numel(), r = g.numel();
        if (all > 0x7FFFFFFFll || r > 0x7FFFFFFFll) fail("choice_loss: at most 2^31 - 1 logits and requests");
        auto ints = [&](const char *arg, PyObject *o, int64_t count) {
            return static_cast<const int32_t *>(vector({op, arg}, tensor({op, arg}, o), count, at::kInt, dev));
        };
        return done(jc_choice_loss(floats({op, "logits"}, a[0], all, dev, true), (uint32_t)all, ints("offsets", a[1], r + 1),
                                   ints("gold", a[2], r), floats({op, "weight"}, a[5], r, dev), (uint32_t)r,
                                   floats({op, "loss"}, a[3], r, dev, true), floats({op, "dlogits"}, a[4], all, dev),
                                   queue_of(a[6], dev).handle),
                    "jc_choice_loss");
    });
}

// (handle, device, t, lr, beta1, beta2, eps, grad_scale, stream)
PyObject *adamw_step(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return call(n, 9, [&] {
        void *h = PyLong_AsVoidPtr(a[0]);
        const int dev = (int)PyLong_AsLong(a[1]);
        const unsigned long long t = PyLong_AsUnsignedLongLong(a[2]);
        if (PyErr_Occurred()) throw Raised();
        return done(jc_adamw_step(static_cast<JcAdamW *>(h), t, (float)number(a[3]), number(a[4]), number(a[5]),
                                  (float)number(a[6]), floats({"AdamW", "grad_scale"}, a[7], 1, dev), queue_of(a[8], dev).handle),
                    "jc_adamw_step");
    });
}

#define JC_METHOD(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {JC_METHOD(set_error), JC_METHOD(layer_norm), JC_METHOD(layer_norm_backward), JC_METHOD(linear),
                           JC_METHOD(linear_backward), JC_METHOD(choice_loss), JC_METHOD(adamw_step), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_binding", "The fine-tuning operators on torch tensors.", -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) { return PyModule_Create(&g_module); }
