// Python module mcv_b200._tensors: the per-call checks of tensors in the
// token-mixing binding.  A decode step's kernel takes 2 to 5 us on the GPU; checking and
// packing the nine tensors of a gated delta step took 4.7 us with each attribute asked for
// from Python, 2.0 with them looked at here.
#include <Python.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <exception>

namespace {

const at::Tensor* tensor(PyObject* o, const char* what) {
    if (THPVariable_Check(o)) return &THPVariable_Unpack(o);
    PyErr_Format(PyExc_TypeError, "mcv_b200: %s must be a tensor", what);
    return nullptr;
}

// Runs f, an exception of torch's becoming a RuntimeError.
template <class F>
PyObject* guarded(F f) {
    try {
        return f();
    } catch (const std::exception& e) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

bool arguments(Py_ssize_t n, Py_ssize_t want, const char* who) {
    if (n == want) return true;
    PyErr_Format(PyExc_TypeError, "%s takes %zd arguments", who, want);
    return false;
}

PyObject* address(const at::Tensor& t) { return PyLong_FromVoidPtr(t.data_ptr()); }

PyObject* dense_address(const at::Tensor& t, at::ScalarType type, const char* type_name, const int64_t* shape, int64_t dims,
                        const char* what, long dev) {
    if (t.scalar_type() == type && t.dim() == dims && t.get_device() == dev && t.is_contiguous() &&
        t.sizes() == at::IntArrayRef(shape, dims))
        return address(t);
    std::string s;
    for (int64_t i = 0; i < dims; ++i) s += (i ? ", " : "") + std::to_string(shape[i]);
    PyErr_Format(PyExc_RuntimeError, "mcv_b200: %s must be a contiguous %s tensor [%s] on cuda:%ld", what, type_name,
                 s.c_str(), dev);
    return nullptr;
}

// rows(t, what, dev): address, token and head stride (0 where there is one) of [tokens, heads, dim] fp16 with contiguous rows.
PyObject* rows(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!arguments(n, 3, "rows")) return nullptr;
    return guarded([&]() -> PyObject* {
        const char* what = PyUnicode_AsUTF8(args[1]);
        if (!what) return nullptr;
        const long dev = PyLong_AsLong(args[2]);
        if (dev == -1 && PyErr_Occurred()) return nullptr;
        const at::Tensor* t = tensor(args[0], what);
        if (!t) return nullptr;
        if (t->scalar_type() != at::kHalf || t->dim() != 3 || t->get_device() != dev) {
            PyErr_Format(PyExc_RuntimeError, "mcv_b200: %s must be float16 [tokens, heads, dim] on cuda:%ld", what, dev);
            return nullptr;
        }
        const auto stride = t->strides(), size = t->sizes();
        if (stride[2] != 1 && size[2] != 1) {
            PyErr_Format(PyExc_RuntimeError, "mcv_b200: rows of %s must be contiguous", what);
            return nullptr;
        }
        // a dimension of size 1 is never stepped along, and may have any stride
        return Py_BuildValue("(NLL)", address(*t), size[0] == 1 ? 0ll : static_cast<long long>(stride[0]),
                             size[1] == 1 ? 0ll : static_cast<long long>(stride[1]));
    });
}

// dense(t, dtype, shape, what, dev): address of a contiguous tensor of this type and shape, None for None.
PyObject* dense(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!arguments(n, 5, "dense")) return nullptr;
    if (args[0] == Py_None) Py_RETURN_NONE;
    return guarded([&]() -> PyObject* {
        const char* what = PyUnicode_AsUTF8(args[3]);
        if (!what) return nullptr;
        const long dev = PyLong_AsLong(args[4]);
        if (dev == -1 && PyErr_Occurred()) return nullptr;
        const at::Tensor* t = tensor(args[0], what);
        if (!t) return nullptr;
        if (!THPDtype_Check(args[1]) || !PyTuple_Check(args[2]) || PyTuple_GET_SIZE(args[2]) > 8) {
            PyErr_SetString(PyExc_TypeError, "dense: a dtype and a shape of up to 8 dimensions");
            return nullptr;
        }
        const THPDtype* type = reinterpret_cast<THPDtype*>(args[1]);
        int64_t shape[8];
        const int64_t dims = PyTuple_GET_SIZE(args[2]);
        for (int64_t i = 0; i < dims; ++i) {
            shape[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(args[2], i));
            if (shape[i] == -1 && PyErr_Occurred()) return nullptr;
        }
        return dense_address(*t, type->scalar_type, type->name, shape, dims, what, dev);
    });
}

// rows_out(x, out, what, dev): address of a dense output of x's type and shape, or of x itself (in place).
PyObject* rows_out(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!arguments(n, 4, "rows_out")) return nullptr;
    return guarded([&]() -> PyObject* {
        const char* what = PyUnicode_AsUTF8(args[2]);
        if (!what) return nullptr;
        const long dev = PyLong_AsLong(args[3]);
        if (dev == -1 && PyErr_Occurred()) return nullptr;
        const at::Tensor *x = tensor(args[0], "x"), *out = x ? tensor(args[1], what) : nullptr;
        if (!out) return nullptr;
        if (out->data_ptr() == x->data_ptr() && x->numel() > 0) {
            if (out->scalar_type() == x->scalar_type() && out->sizes() == x->sizes() && out->strides() == x->strides())
                return address(*x);
            // the call takes an output at x's address to have x's strides
            PyErr_Format(PyExc_RuntimeError, "mcv_b200: %s begins where its input does but is laid out differently", what);
            return nullptr;
        }
        return dense_address(*out, at::kHalf, "float16", x->sizes().data(), x->dim(), what, dev);
    });
}

PyMethodDef methods[] = {
    {"rows", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rows)), METH_FASTCALL,
     "rows(t, what, dev): address, token and head stride of fp16 [tokens, heads, dim]"},
    {"dense", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(dense)), METH_FASTCALL,
     "dense(t, dtype, shape, what, dev): address of a contiguous tensor, None for None"},
    {"rows_out", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rows_out)), METH_FASTCALL,
     "rows_out(x, out, what, dev): address of a dense output like x, or of x in place"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", "Per-call checks of tensors.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__tensors() { return PyModule_Create(&module); }
