/*
 * Tensor records for the Python binding, packed in C.
 *
 * Reading pointer, type, sizes and strides of a tensor and packing them takes the interpreter about 1.3 us per tensor,
 * which for the seven tensors of a decoding step is as long as its kernels; from here it is a fifth of that.  The module is
 * optional: without it (no Python headers at build time) native.py packs the same records itself.
 *
 *   set_dtypes((float16, bfloat16, float32, bool, int32, uint8))    the objects whose position is the record's type code
 *   records(t0, t1, ...) -> (buffer, [address or None, ...])        kfa_tensor records; None stays None
 *   addressable(t0, ...) -> bool     unit channel stride, 16-byte aligned base, other strides positive multiples of 8
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "../../include/kfa.h"

#define MAX_DTYPES 8

static PyObject *name_data_ptr, *name_dtype, *name_shape, *name_stride;
static PyObject* dtypes[MAX_DTYPES];
static int dtype_count = 0;

/* Fills `out` from a tuple of at most six integers; returns its length or -1. */
static int integers(PyObject* tuple, int64_t* out) {
    if (!tuple) return -1;
    int n = -1;
    if (PyTuple_Check(tuple) && PyTuple_GET_SIZE(tuple) <= 6) {
        n = (int)PyTuple_GET_SIZE(tuple);
        for (int i = 0; i < n; ++i) {
            out[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(tuple, i));
            if (out[i] == -1 && PyErr_Occurred()) n = -1;
            if (n < 0) break;
        }
    } else {
        PyErr_SetString(PyExc_ValueError, "a tensor with at most six axes is required");
    }
    Py_DECREF(tuple);
    return n;
}

static int pointer_of(PyObject* t, uint64_t* out) {
    PyObject* p = PyObject_CallMethodNoArgs(t, name_data_ptr);
    if (!p) return -1;
    *out = PyLong_AsUnsignedLongLong(p);
    Py_DECREF(p);
    return PyErr_Occurred() ? -1 : 0;
}

static int describe(PyObject* t, kfa_tensor* r) {
    uint64_t address;
    if (pointer_of(t, &address) < 0) return -1;
    r->data = (void*)(uintptr_t)address;
    PyObject* dtype = PyObject_GetAttr(t, name_dtype);
    if (!dtype) return -1;
    r->dtype = -1;
    for (int i = 0; i < dtype_count; ++i)
        if (dtypes[i] == dtype) r->dtype = i;
    Py_DECREF(dtype);
    r->ndim = integers(PyObject_GetAttr(t, name_shape), r->sizes);
    if (r->ndim < 0) return -1;
    return integers(PyObject_CallMethodNoArgs(t, name_stride), r->strides) == r->ndim ? 0 : -1;
}

static PyObject* records(PyObject* self, PyObject* const* args, Py_ssize_t n) {
    (void)self;
    PyObject* buffer = PyByteArray_FromStringAndSize(NULL, n * (Py_ssize_t)sizeof(kfa_tensor));
    PyObject* addresses = PyList_New(n);
    if (!buffer || !addresses) goto fail;
    kfa_tensor* base = (kfa_tensor*)PyByteArray_AS_STRING(buffer);
    memset(base, 0, (size_t)n * sizeof(kfa_tensor));
    for (Py_ssize_t i = 0; i < n; ++i) {
        if (args[i] == Py_None) {
            PyList_SET_ITEM(addresses, i, Py_NewRef(Py_None));
            continue;
        }
        if (describe(args[i], base + i) < 0) goto fail;
        PyObject* address = PyLong_FromVoidPtr(base + i);
        if (!address) goto fail;
        PyList_SET_ITEM(addresses, i, address);
    }
    PyObject* result = PyTuple_Pack(2, buffer, addresses);
    Py_DECREF(buffer);
    Py_DECREF(addresses);
    return result;
fail:
    Py_XDECREF(buffer);
    Py_XDECREF(addresses);
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "tensor record");
    return NULL;
}

static PyObject* addressable(PyObject* self, PyObject* const* args, Py_ssize_t n) {
    (void)self;
    for (Py_ssize_t i = 0; i < n; ++i) {
        int64_t sizes[6], strides[6];
        uint64_t address;
        if (pointer_of(args[i], &address) < 0) return NULL;
        const int axes = integers(PyObject_GetAttr(args[i], name_shape), sizes);
        if (axes < 0 || integers(PyObject_CallMethodNoArgs(args[i], name_stride), strides) != axes) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "tensor strides");
            return NULL;
        }
        int ok = axes > 0 && strides[axes - 1] == 1 && address % 16 == 0;
        for (int a = 0; ok && a < axes - 1; ++a) ok = sizes[a] == 1 || (strides[a] > 0 && strides[a] % 8 == 0);
        if (!ok) Py_RETURN_FALSE;
    }
    Py_RETURN_TRUE;
}

static PyObject* set_dtypes(PyObject* self, PyObject* tuple) {
    (void)self;
    if (!PyTuple_Check(tuple) || PyTuple_GET_SIZE(tuple) > MAX_DTYPES) {
        PyErr_SetString(PyExc_TypeError, "set_dtypes takes a tuple of at most eight types");
        return NULL;
    }
    for (int i = 0; i < dtype_count; ++i) Py_CLEAR(dtypes[i]);
    dtype_count = (int)PyTuple_GET_SIZE(tuple);
    for (int i = 0; i < dtype_count; ++i) dtypes[i] = Py_NewRef(PyTuple_GET_ITEM(tuple, i));
    Py_RETURN_NONE;
}

static PyMethodDef methods[] = {
    {"records", (PyCFunction)(void (*)(void))records, METH_FASTCALL, "kfa_tensor records of tensors"},
    {"addressable", (PyCFunction)(void (*)(void))addressable, METH_FASTCALL, "16-byte addressable rows"},
    {"set_dtypes", set_dtypes, METH_O, "types by record code"},
    {NULL, NULL, 0, NULL}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast_records", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__fast_records(void) {
    name_data_ptr = PyUnicode_InternFromString("data_ptr");
    name_dtype = PyUnicode_InternFromString("dtype");
    name_shape = PyUnicode_InternFromString("shape");
    name_stride = PyUnicode_InternFromString("stride");
    if (!name_data_ptr || !name_dtype || !name_shape || !name_stride) return NULL;
    return PyModule_Create(&module);
}
