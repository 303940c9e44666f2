/* describe_py.c -- the Python binding's tensor descriptors (openasr_b200/_describe.so).
 *
 * describe(tensor, types) -> bytes of one oasr_tensor: ne = reversed shape, nb = reversed
 * byte strides.  `types` maps torch dtypes to (tensor type, element size).  An operator of
 * twelve tensors spends longer describing them in Python (0.9 us each) than its kernel
 * runs; through the tensor's own data_ptr / shape / stride it is a third of that. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "oasr_b200.h"

static PyObject *s_data_ptr, *s_shape, *s_stride, *s_dtype;

static PyObject *describe(PyObject *self, PyObject *const *args, Py_ssize_t n) {
    (void)self;
    if (n != 2 || !PyDict_Check(args[1])) {
        PyErr_SetString(PyExc_TypeError, "describe(tensor, types)");
        return NULL;
    }
    oasr_tensor d = {0, 0, NULL, {1, 1, 1, 1}, {0, 0, 0, 0}};
    PyObject *dtype = PyObject_GetAttr(args[0], s_dtype);
    if (!dtype) return NULL;
    PyObject *type = PyDict_GetItemWithError(args[1], dtype); /* borrowed */
    if (!type) {
        if (!PyErr_Occurred()) PyErr_Format(PyExc_KeyError, "unsupported tensor dtype %S", dtype);
        Py_DECREF(dtype);
        return NULL;
    }
    Py_DECREF(dtype);
    if (!PyTuple_Check(type) || PyTuple_GET_SIZE(type) != 2) {
        PyErr_SetString(PyExc_TypeError, "types maps to (type, element size)");
        return NULL;
    }
    d.type = (int32_t)PyLong_AsLong(PyTuple_GET_ITEM(type, 0));
    const int64_t es = PyLong_AsLongLong(PyTuple_GET_ITEM(type, 1));
    PyObject *ptr = PyObject_CallMethodNoArgs(args[0], s_data_ptr);
    if (!ptr) return NULL;
    d.data = (void *)(uintptr_t)PyLong_AsUnsignedLongLong(ptr);
    Py_DECREF(ptr);
    PyObject *shape = PyObject_GetAttr(args[0], s_shape);
    if (!shape) return NULL;
    PyObject *stride = PyObject_CallMethodNoArgs(args[0], s_stride);
    if (!stride || !PyTuple_Check(shape) || !PyTuple_Check(stride) || PyTuple_GET_SIZE(shape) != PyTuple_GET_SIZE(stride)) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "shape and stride must be tuples of one length");
        Py_DECREF(shape);
        Py_XDECREF(stride);
        return NULL;
    }
    const Py_ssize_t dims = PyTuple_GET_SIZE(shape);
    for (Py_ssize_t i = 0; i < 4; ++i) {
        if (i < dims) {
            d.ne[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, dims - 1 - i));
            d.nb[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(stride, dims - 1 - i)) * es;
        } else {
            d.nb[i] = i ? d.nb[i - 1] * d.ne[i - 1] : es;
        }
    }
    Py_DECREF(shape);
    Py_DECREF(stride);
    if (PyErr_Occurred()) return NULL;
    return PyBytes_FromStringAndSize((const char *)&d, sizeof d);
}

static PyMethodDef methods[] = {
    {"describe", (PyCFunction)(void (*)(void))describe, METH_FASTCALL, "bytes of one oasr_tensor"}, {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_describe", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__describe(void) {
    s_data_ptr = PyUnicode_InternFromString("data_ptr");
    s_shape = PyUnicode_InternFromString("shape");
    s_stride = PyUnicode_InternFromString("stride");
    s_dtype = PyUnicode_InternFromString("dtype");
    if (!s_data_ptr || !s_shape || !s_stride || !s_dtype) return NULL;
    return PyModule_Create(&module);
}
