// oneccl_amd._tensors: what the ctypes binding asks of its tensors before a call, one C++ pass instead of an attribute access per
// property and tensor (400 tensors: 4 us, 145 in Python).  Every function answers None where a condition does not hold, or where it
// cannot tell; the binding then goes through the same conditions in Python, which names the one that failed.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

namespace {

// The tensor behind an object: dense memory of `dtype` on GPU `device` (-1: in host memory); NULL otherwise.
const at::Tensor* dense(PyObject* o, PyObject* dtype, long device) {
    if (!THPVariable_Check(o) || !THPDtype_Check(dtype)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.layout() != at::kStrided || !(device < 0 ? t.is_cpu() : t.is_cuda()) || t.get_device() != device || t.scalar_type() != ((THPDtype*)dtype)->scalar_type) return nullptr;
    return &t;
}

PyObject* none() {
    PyErr_Clear();
    Py_RETURN_NONE;
}

// memory(tensor, dtype, least, device): the address of a contiguous tensor of `least` elements or more
PyObject* memory(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 4) return none();
    const long long least = PyLong_AsLongLong(a[2]);
    const long device = PyLong_AsLong(a[3]);
    if (PyErr_Occurred()) return none();
    try {
        const at::Tensor* t = dense(a[0], a[1], device);
        if (t && t->numel() >= least && t->is_contiguous()) return PyLong_FromVoidPtr(t->data_ptr());
    }
    catch (...) {
    }
    return none();
}

// rows(tensor, hidden, dtype, device): (rows, elements from row to row, address) of a matrix whose rows are contiguous and do not
// overlap; `hidden` for the distance where there is one row, or none
PyObject* rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 4) return none();
    const long long hidden = PyLong_AsLongLong(a[1]);
    const long device = PyLong_AsLong(a[3]);
    if (PyErr_Occurred()) return none();
    try {
        const at::Tensor* t = dense(a[0], a[2], device);
        if (t && t->dim() == 2 && t->size(1) == hidden && (hidden <= 1 || t->stride(1) == 1) && (t->size(0) <= 1 || t->stride(0) >= hidden))
            return Py_BuildValue("LLN", (long long)t->size(0), t->size(0) > 1 ? (long long)t->stride(0) : hidden, PyLong_FromVoidPtr(t->data_ptr()));
    }
    catch (...) {
    }
    return none();
}

// addresses(tensors, dtype, least, device): the addresses of a list or tuple of contiguous tensors as the bytes of a table of
// pointers; least: a buffer of as many 64-bit numbers of elements
PyObject* addresses(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 4 || !(PyList_Check(a[0]) || PyTuple_Check(a[0]))) return none();
    const long device = PyLong_AsLong(a[3]);
    Py_buffer least;
    if (PyErr_Occurred() || PyObject_GetBuffer(a[2], &least, PyBUF_SIMPLE) != 0) return none();
    const Py_ssize_t k = PySequence_Fast_GET_SIZE(a[0]);
    PyObject* table = least.len == k * 8 ? PyBytes_FromStringAndSize(nullptr, k * 8) : nullptr;
    bool all = table != nullptr;
    try {
        for (Py_ssize_t i = 0; all && i < k; i++) {
            const at::Tensor* t = dense(PySequence_Fast_GET_ITEM(a[0], i), a[1], device);
            all = t && t->numel() >= ((const int64_t*)least.buf)[i] && t->is_contiguous();
            if (all) ((uint64_t*)PyBytes_AS_STRING(table))[i] = (uint64_t)(uintptr_t)t->data_ptr();
        }
    }
    catch (...) {
        all = false;
    }
    PyBuffer_Release(&least);
    if (all) return table;
    Py_XDECREF(table);
    return none();
}

PyMethodDef kMethods[] = {
    { "memory", (PyCFunction)(void (*)(void))memory, METH_FASTCALL, "memory(tensor, dtype, least, device) -> address or None" },
    { "rows", (PyCFunction)(void (*)(void))rows, METH_FASTCALL, "rows(tensor, hidden, dtype, device) -> (rows, distance, address) or None" },
    { "addresses", (PyCFunction)(void (*)(void))addresses, METH_FASTCALL, "addresses(tensors, dtype, least, device) -> bytes or None" },
    { nullptr, nullptr, 0, nullptr },
};
PyModuleDef kModule = { PyModuleDef_HEAD_INIT, "_tensors", "Properties and addresses of tensors.", -1, kMethods, nullptr, nullptr, nullptr, nullptr };

}  // namespace

PyMODINIT_FUNC PyInit__tensors(void) {
    return PyModule_Create(&kModule);
}
