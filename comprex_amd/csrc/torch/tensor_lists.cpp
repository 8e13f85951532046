// The addresses of a list of torch tensors, checked, for the calls over many tensors (comprex_amd/device.py).
// Asking 161 tensors for five properties each takes Python 34 us, property by property, where the GPU takes 20 us
// for what is done with them; this takes 1.7.  It answers the ordinary case only: anything else is -1, and the
// caller looks for itself what is wrong.
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>

namespace {

// cx_dtype of parameters and gradients (include/comprex_gfx950.h), and the types of 8-bit moments
int type_code(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return 0;
        case at::kBFloat16: return 3;
        case at::kHalf: return 4;
        case at::kFloat8_e4m3fn: return 100;
        case at::kByte: return 101;
        default: return -1;
    }
}

int addresses_of(PyObject* list, const int64_t* sizes, uint64_t* out, int64_t device) {
    int code = 0;
    bool any = false;
    const Py_ssize_t n = PyList_GET_SIZE(list);
    for (Py_ssize_t k = 0; k < n; ++k) {
        PyObject* item = PyList_GET_ITEM(list, k);
        out[k] = 0;
        if (item == Py_None) continue;
        if (!THPVariable_Check(item)) return -1;
        const at::Tensor& t = THPVariable_Unpack(item);
        if (!t.defined() || t.layout() != at::kStrided || !t.is_cuda() || t.get_device() != device || t.numel() != sizes[k] ||
            !t.is_contiguous())
            return -1;
        const int c = type_code(t.scalar_type());
        if (c < 0 || (any && c != code)) return -1;
        code = c;
        any = true;
        out[k] = reinterpret_cast<uint64_t>(t.const_data_ptr());
    }
    return code;
}

// addresses(tensors, count, sizes, out, device): `sizes` the address of the `count` int64 element counts they have to
// have, `out` that of as many uint64 (0 for None), `device` the GPU they have to be on.  Their type (type_code; 0 of
// nothing but None), or -1.
PyObject* addresses(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 5) {
        PyErr_SetString(PyExc_TypeError, "addresses(tensors, count, sizes, out, device)");
        return nullptr;
    }
    const long long count = PyLong_AsLongLong(args[1]);
    const unsigned long long sizes = PyLong_AsUnsignedLongLong(args[2]), out = PyLong_AsUnsignedLongLong(args[3]);
    const long long device = PyLong_AsLongLong(args[4]);
    if (PyErr_Occurred()) return nullptr;
    if (!PyList_Check(args[0]) || PyList_GET_SIZE(args[0]) != count) return PyLong_FromLong(-1);
    int code = -1;
    try {
        code = addresses_of(args[0], reinterpret_cast<const int64_t*>(sizes), reinterpret_cast<uint64_t*>(out), device);
    } catch (const std::exception&) {  // a tensor without storage of its own, for instance
    }
    return PyLong_FromLong(code);
}

// unmoved(tensors, count, at, sizes, type): whether `tensors` are `count` tensors at the addresses that the uint64 at `at`
// say, contiguous, with the element counts that the int64 at `sizes` say and of that type (type_code); without the last
// two the addresses alone count.  (Memory that was let go of may come back as another tensor's at the same address.)
PyObject* unmoved(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 3 && n != 5) {
        PyErr_SetString(PyExc_TypeError, "unmoved(tensors, count, at[, sizes, type])");
        return nullptr;
    }
    const long long count = PyLong_AsLongLong(args[1]);
    const unsigned long long at = PyLong_AsUnsignedLongLong(args[2]);
    const unsigned long long counts = n == 5 ? PyLong_AsUnsignedLongLong(args[3]) : 0;
    const long long type = n == 5 ? PyLong_AsLongLong(args[4]) : 0;
    if (PyErr_Occurred()) return nullptr;
    const int64_t* sizes = reinterpret_cast<const int64_t*>(counts);
    const uint64_t* want = reinterpret_cast<const uint64_t*>(at);
    if (!PyList_Check(args[0]) || PyList_GET_SIZE(args[0]) != count) Py_RETURN_FALSE;
    try {
        for (Py_ssize_t k = 0; k < count; ++k) {
            PyObject* item = PyList_GET_ITEM(args[0], k);
            if (!THPVariable_Check(item)) Py_RETURN_FALSE;
            const at::Tensor& t = THPVariable_Unpack(item);
            if (reinterpret_cast<uint64_t>(t.const_data_ptr()) != want[k]) Py_RETURN_FALSE;
            if (sizes && (t.numel() != sizes[k] || type_code(t.scalar_type()) != type || !t.is_contiguous())) Py_RETURN_FALSE;
        }
    } catch (const std::exception&) {
        Py_RETURN_FALSE;
    }
    Py_RETURN_TRUE;
}

PyMethodDef methods[] = {{"addresses", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(addresses)), METH_FASTCALL,
                          "addresses(tensors, count, sizes, out, device) -> type or -1"},
                         {"unmoved", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(unmoved)), METH_FASTCALL,
                          "unmoved(tensors, count, at[, sizes, type]) -> bool"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_lists", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_lists() { return PyModule_Create(&module); }
