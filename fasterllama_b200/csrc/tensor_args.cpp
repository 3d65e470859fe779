// tensor_args.cpp — the argument checks of the Python binding for torch tensors, in C++: shape, type, device and layout of a tensor and its
// address in about a tenth of a microsecond.  From Python every attribute of a tensor costs that much, and a decode call names a
// dozen tensors: its host time would be that of three kernel launches.  Python module `_tensor_args`.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

namespace {

// t, name, shape (tuple), dtype or None, device index or None -> tensor, or nullptr with the exception set
const at::Tensor *checked(PyObject *const *a, Py_ssize_t n, const char *what) {
    if (n != 5) {
        PyErr_SetString(PyExc_TypeError, "expected (tensor, name, shape, dtype, device)");
        return nullptr;
    }
    if (!THPVariable_Check(a[0])) {
        PyErr_Format(PyExc_ValueError, "%U must be a torch tensor", a[1]);
        return nullptr;
    }
    const at::Tensor &t = THPVariable_Unpack(a[0]);
    if (a[4] != Py_None) {
        const long dev = PyLong_AsLong(a[4]);
        if (dev == -1 && PyErr_Occurred()) return nullptr;
        if (t.get_device() != dev) {
            PyErr_Format(PyExc_ValueError, "%U is on another device (%d) than the cache (%ld)", a[1], (int)t.get_device(), dev);
            return nullptr;
        }
    }
    bool ok = t.layout() == at::kStrided && (a[3] == Py_None || (THPDtype_Check(a[3]) && t.scalar_type() == reinterpret_cast<THPDtype *>(a[3])->scalar_type));
    if (ok && PyTuple_Check(a[2])) {
        ok = t.dim() == PyTuple_GET_SIZE(a[2]);
        for (int64_t i = 0; ok && i < t.dim(); ++i) {
            const long long want = PyLong_AsLongLong(PyTuple_GET_ITEM(a[2], i));
            if (want == -1 && PyErr_Occurred()) return nullptr;
            ok = t.size(i) == want;
        }
    } else {
        ok = false;
    }
    if (!ok) {
        PyErr_Format(PyExc_ValueError, "%U must be a %s %S tensor of shape %S", a[1], what, a[3], a[2]);
        return nullptr;
    }
    return &t;
}

// Address of a dense tensor.
PyObject *dense(PyObject *, PyObject *const *a, Py_ssize_t n) {
    const at::Tensor *t = checked(a, n, "dense");
    if (!t) return nullptr;
    if (!t->is_contiguous()) return PyErr_Format(PyExc_ValueError, "%U must be a dense tensor", a[1]);
    return PyLong_FromVoidPtr(t->data_ptr());
}

// The same, 0 for None.
PyObject *opt(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    if (n > 0 && a[0] == Py_None) return PyLong_FromLong(0);
    return dense(self, a, n);
}

// (address, elements between two tokens' rows) of q, k or v [B,S,heads,d]: dense heads, one stride between tokens.
PyObject *rows(PyObject *, PyObject *const *a, Py_ssize_t n) {
    const at::Tensor *t = checked(a, n, "token-row");
    if (!t) return nullptr;
    if (t->dim() != 4) return PyErr_Format(PyExc_ValueError, "%U must be [B,S,heads,d]", a[1]);
    const int64_t B = t->size(0), S = t->size(1), H = t->size(2), d = t->size(3);
    int64_t row = H * d;
    if (!t->is_contiguous()) {
        row = S > 1 ? t->stride(1) : (B > 1 ? t->stride(0) : H * d);
        if (t->stride(3) != 1 || (H > 1 && t->stride(2) != d) || (S > 1 && t->stride(1) != row) || (B > 1 && t->stride(0) != S * row) || row < H * d)
            return PyErr_Format(PyExc_ValueError, "%U must be [B,S,heads,d] with unit element stride, head stride d and one stride between tokens", a[1]);
    }
    return Py_BuildValue("(NL)", PyLong_FromVoidPtr(t->data_ptr()), (long long)row);
}

PyMethodDef methods[] = {
    {"dense", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(dense)), METH_FASTCALL, "address of a dense tensor"},
    {"opt", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(opt)), METH_FASTCALL, "the same, 0 for None"},
    {"rows", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rows)), METH_FASTCALL, "address and token-row stride"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_args", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

} // namespace

PyMODINIT_FUNC PyInit__tensor_args(void) { return PyModule_Create(&module); }
