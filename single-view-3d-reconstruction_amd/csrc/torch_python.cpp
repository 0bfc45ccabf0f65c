// Python's direct way to the operators that are called with long lists or for little work (torch_train_ops.cpp): the module
// sv3d._call.  Its functions take the operators' arguments by position, turn them into C++ values (an optimizer step on five
// lists of 72 shape-only tensors took 71 us this way, 96 us through the generic arguments of torch.ops) and call the operator
// through the dispatcher, so that everything that works on operators (autograd, shape-only tensors, tracing modes) still
// sees them.  Arguments that are not plain tensors (subclasses with their own __torch_function__, or an active mode of that
// kind) are answered with NotImplemented: the caller then goes through torch.ops.
#include <Python.h>

#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <pybind11/pybind11.h>

#include "torch_util.h"

namespace {

struct NotPlain {};

Tensor tensor_of(PyObject *o)
{
    if (!THPVariable_CheckExact(o)) throw NotPlain();
    return THPVariable_Unpack(o);
}

optional<Tensor> maybe_tensor_of(PyObject *o)
{
    if (o == Py_None) return c10::nullopt;
    return tensor_of(o);
}

PyObject *item(PyObject *seq, Py_ssize_t i) { return PyList_Check(seq) ? PyList_GET_ITEM(seq, i) : PyTuple_GET_ITEM(seq, i); }

Py_ssize_t length(PyObject *seq)
{
    if (PyList_Check(seq)) return PyList_GET_SIZE(seq);
    if (PyTuple_Check(seq)) return PyTuple_GET_SIZE(seq);
    throw NotPlain();
}

std::vector<Tensor> tensors_of(PyObject *seq)
{
    const Py_ssize_t n = length(seq);
    std::vector<Tensor> out;
    out.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) out.push_back(tensor_of(item(seq, i)));
    return out;
}

int64_t int_of(PyObject *o)
{
    if (!PyLong_Check(o)) throw NotPlain();
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        throw NotPlain();
    }
    return v;
}

double double_of(PyObject *o)
{
    if (PyFloat_CheckExact(o)) return PyFloat_AS_DOUBLE(o);
    return (double)int_of(o);
}

bool bool_of(PyObject *o)
{
    if (!PyBool_Check(o)) throw NotPlain();
    return o == Py_True;
}

// Runs f with the arguments taken apart by it; what cannot be taken apart goes back to Python.
template <class F>
PyObject *call(Py_ssize_t got, Py_ssize_t want, F f)
{
    HANDLE_TH_ERRORS
    if (got != want || at::impl::torch_function_mode_enabled()) Py_RETURN_NOTIMPLEMENTED;
    try {
        return THPVariable_Wrap(f());
    } catch (const NotPlain &) {
        Py_RETURN_NOTIMPLEMENTED;
    }
    END_HANDLE_TH_ERRORS
}

PyObject *layer_norm(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return call(n, 6, [&] {
        const Tensor x = tensor_of(a[0]);
        std::vector<int64_t> shape;
        for (Py_ssize_t i = 0, k = length(a[1]); i < k; ++i) shape.push_back(int_of(item(a[1], i)));
        const auto weight = maybe_tensor_of(a[2]), bias = maybe_tensor_of(a[3]);
        const double eps = double_of(a[4]);
        const bool f32_out = bool_of(a[5]);
        static auto op = find_op<Tensor(const Tensor &, IntList, const optional<Tensor> &, const optional<Tensor> &, double,
                                        bool)>("sv3d::layer_norm");
        pybind11::gil_scoped_release release;
        return op.call(x, shape, weight, bias, eps, f32_out);
    });
}

PyObject *grad_square_sums(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return call(n, 1, [&] {
        const auto grads = tensors_of(a[0]);
        static auto op = find_op<Tensor(at::TensorList)>("sv3d::grad_square_sums");
        pybind11::gil_scoped_release release;
        return op.call(grads);
    });
}

PyObject *adamw_step(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return call(n, 18, [&] {
        std::vector<Tensor> list[6];
        for (int i = 0; i < 6; ++i) list[i] = tensors_of(a[i]);
        const auto lr_tensor = maybe_tensor_of(a[6]), grad_scale = maybe_tensor_of(a[7]), found_inf = maybe_tensor_of(a[8]),
                   sums = maybe_tensor_of(a[9]);
        double d[6];
        for (int i = 0; i < 6; ++i) d[i] = double_of(a[10 + i]);
        const bool maximize = bool_of(a[16]);
        const int64_t seed = int_of(a[17]);
        using L = at::TensorList;
        using O = const optional<Tensor> &;
        static auto op = find_op<Tensor(L, L, L, L, L, L, O, O, O, O, double, double, double, double, double, double, bool,
                                        int64_t)>("sv3d::adamw_step");
        pybind11::gil_scoped_release release;
        return op.call(list[0], list[1], list[2], list[3], list[4], list[5], lr_tensor, grad_scale, found_inf, sums, d[0], d[1],
                       d[2], d[3], d[4], d[5], maximize, seed);
    });
}

PyMethodDef methods[] = {
    {"layer_norm", (PyCFunction)(void (*)(void))layer_norm, METH_FASTCALL, "sv3d::layer_norm by position"},
    {"grad_square_sums", (PyCFunction)(void (*)(void))grad_square_sums, METH_FASTCALL, "sv3d::grad_square_sums by position"},
    {"adamw_step", (PyCFunction)(void (*)(void))adamw_step, METH_FASTCALL, "sv3d::adamw_step by position"},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_call", "Direct calls of sv3d operators", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__call(void) { return PyModule_Create(&module); }
