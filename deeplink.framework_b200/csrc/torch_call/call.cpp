// Calls a DIOPI function from Python without a ctypes conversion per argument: the tensor handles are plain structs on the stack,
// filled from the at::Tensor behind each argument, the way DIPU's generated wrappers pass their tensors. About 2 us a call with
// nine tensors against 11 us through ctypes, which is what a decode step's small operators cost on the host.
//
//   f = bind(address, signature, dtype_error)      f(context pointer, *arguments) -> diopiError_t
//
// Signature letters as in diopi.py: T tensor, t tensor or None, s scalar by pointer, i int64, r enum, d double, b bool.
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstring>
#include <exception>

#include "minihost/minihost_structs.h"

#if !defined(__x86_64__)
#error "the argument order used by invoke() is the x86-64 System V one"
#endif

namespace {

constexpr int kMaxArgs = 16;

struct Bound {
    void* fn;
    char sig[kMaxArgs + 1];
    PyObject* error;   // raised for a dtype without a DIOPI counterpart
};

bool dtype_of(at::ScalarType t, diopiDtype_t* out) {
    switch (t) {
        case at::kChar: *out = diopi_dtype_int8; return true;
        case at::kByte: *out = diopi_dtype_uint8; return true;
        case at::kShort: *out = diopi_dtype_int16; return true;
        case at::kInt: *out = diopi_dtype_int32; return true;
        case at::kLong: *out = diopi_dtype_int64; return true;
        case at::kHalf: *out = diopi_dtype_float16; return true;
        case at::kFloat: *out = diopi_dtype_float32; return true;
        case at::kDouble: *out = diopi_dtype_float64; return true;
        case at::kBool: *out = diopi_dtype_bool; return true;
        case at::kBFloat16: *out = diopi_dtype_bfloat16; return true;
        default: return false;
    }
}

bool describe(const Bound* f, const at::Tensor& t, diopiTensor* d) {
    if (!dtype_of(t.scalar_type(), &d->dtype)) {
        PyErr_Format(f->error, "dtype %s has no diopi counterpart", c10::toString(t.scalar_type()));
        return false;
    }
    if (t.dim() > 8) {
        PyErr_SetString(f->error, "could not create a tensor handle");
        return false;
    }
    d->data = t.data_ptr();
    d->device = t.is_cuda() ? diopi_device : diopi_host;
    d->device_index = t.is_cuda() ? t.get_device() : 0;
    d->ndim = t.dim();
    d->numel = t.numel();
    d->itemsize = static_cast<int64_t>(t.element_size());
    int64_t span = d->numel > 0 ? 1 : 0;
    for (int64_t i = 0; i < d->ndim; ++i) {
        d->shape[i] = t.size(i);
        d->stride[i] = t.stride(i);
        if (d->numel > 0) span += (d->shape[i] - 1) * (d->stride[i] < 0 ? 0 : d->stride[i]);
    }
    d->storage_nbytes = static_cast<size_t>(span * d->itemsize);
    return true;
}

// Integer-class arguments (pointers, int64, enum, bool) and doubles travel in separate register files, and integer-class arguments
// beyond the sixth in order on the stack; a callee does not look at arguments it does not have. So one call shape serves every signature.
int invoke(void* fn, const uint64_t* a, const double* d) {
    using U = uint64_t;
    using F = int (*)(U, U, U, U, U, U, U, U, U, U, U, U, U, U, U, U, U, double, double, double, double);
    return reinterpret_cast<F>(fn)(a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7], a[8], a[9], a[10], a[11], a[12], a[13], a[14], a[15], a[16], d[0], d[1], d[2], d[3]);
}

PyObject* call(PyObject* self, PyObject* const* args, Py_ssize_t n) {
    const Bound* f = static_cast<const Bound*>(PyCapsule_GetPointer(self, "dipu_b200.bound"));
    if (f == nullptr) return nullptr;
    const Py_ssize_t want = static_cast<Py_ssize_t>(std::strlen(f->sig));
    if (n != want + 1) return PyErr_Format(PyExc_TypeError, "expects %zd arguments after ctx, got %zd", want, n - 1);
    diopiTensor tensors[kMaxArgs];
    diopiScalar_t scalars[kMaxArgs];
    uint64_t a[kMaxArgs + 1] = {0};
    double d[4] = {0.0, 0.0, 0.0, 0.0};
    int na = 0, nd = 0;
    a[na++] = PyLong_AsUnsignedLongLong(args[0]);
    for (Py_ssize_t i = 0; i < want; ++i) {
        PyObject* x = args[i + 1];
        switch (f->sig[i]) {
            case 'T':
            case 't':
                if (x == Py_None) {
                    a[na++] = 0;
                } else if (THPVariable_Check(x)) {
                    try {
                        if (!describe(f, THPVariable_Unpack(x), &tensors[i])) return nullptr;
                    } catch (const std::exception& e) {   // a tensor without plain storage or strides
                        PyErr_SetString(f->error, e.what());
                        return nullptr;
                    }
                    a[na++] = reinterpret_cast<uint64_t>(&tensors[i]);
                } else {   // a handle made by the caller
                    PyObject* p = PyObject_GetAttrString(x, "ptr");
                    if (p == nullptr) return nullptr;
                    a[na++] = PyLong_AsUnsignedLongLong(p);
                    Py_DECREF(p);
                }
                break;
            case 's':
                if (x == Py_None) {
                    a[na++] = 0;
                } else {
                    if (PyLong_Check(x)) {
                        scalars[i].stype = diopi_dtype_int64;
                        scalars[i].ival = PyLong_AsLongLong(x);
                    } else {
                        scalars[i].stype = diopi_dtype_float64;
                        scalars[i].fval = PyFloat_AsDouble(x);
                    }
                    a[na++] = reinterpret_cast<uint64_t>(&scalars[i]);
                }
                break;
            case 'd': d[nd++] = PyFloat_AsDouble(x); break;
            case 'b': {
                const int v = PyObject_IsTrue(x);
                if (v < 0) return nullptr;
                a[na++] = static_cast<uint64_t>(v);
                break;
            }
            default: {
                PyObject* v = PyNumber_Index(x);   // an integer of any kind; a fraction or a text is an error
                if (v == nullptr) return nullptr;
                a[na++] = static_cast<uint64_t>(PyLong_AsLongLong(v));
                Py_DECREF(v);
            }
        }
        if (PyErr_Occurred()) return nullptr;
    }
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = invoke(f->fn, a, d);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

PyMethodDef call_def = {"call", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(call)), METH_FASTCALL, nullptr};

PyObject* bind(PyObject*, PyObject* args) {
    unsigned long long address;
    const char* sig;
    PyObject* error;
    if (!PyArg_ParseTuple(args, "KsO", &address, &sig, &error)) return nullptr;
    int doubles = 0;
    for (const char* c = sig; *c; ++c) {
        if (std::strchr("Ttsirdb", *c) == nullptr) return PyErr_Format(PyExc_ValueError, "signature letter %c", *c);
        doubles += *c == 'd';
    }
    if (std::strlen(sig) > kMaxArgs || doubles > 4) return PyErr_Format(PyExc_ValueError, "too many arguments: %s", sig);
    Bound* f = new Bound();
    f->fn = reinterpret_cast<void*>(address);
    std::strcpy(f->sig, sig);
    Py_INCREF(error);
    f->error = error;
    PyObject* capsule = PyCapsule_New(f, "dipu_b200.bound", nullptr);   // bound once per function, for the life of the process
    if (capsule == nullptr) return nullptr;
    PyObject* r = PyCFunction_New(&call_def, capsule);
    Py_DECREF(capsule);
    return r;
}

PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, "bind(address, signature, dtype_error)"}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "dipu_b200_call", "DIOPI calls with stack-allocated tensor handles", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_dipu_b200_call() { return PyModule_Create(&module); }
