/* pycall.c -- the Python mirror's short call path (module _xm_call).
 *
 * A decode step calls the single-token operators for every layer, and describing
 * a tensor to the C ABI takes several Python operations each through ctypes.
 * call() does that in C with the CPython API alone: it reads every tensor's
 * device, contiguity, shape, type and address, fills the xm_tensor descriptors,
 * and calls the operator's entry point.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>

#include "../../include/xm_ops.h"

#define MAX_IN 16
#define MAX_TYPES 8

typedef xm_status (*fwd_fn)(const void *, const xm_tensor *, int32_t, xm_tensor *, void *, size_t, void *);
typedef xm_status (*size_fn)(const void *, const xm_tensor *, int32_t, size_t *);

static PyObject *tensor_type, *types[MAX_TYPES];
static int32_t codes[MAX_TYPES];
static int n_types;
static PyObject *s_device, *s_contiguous, *s_make, *s_ptr, *s_shape, *s_dtype;

/* setup(Tensor, ((dtype, code), ...)) */
static PyObject *setup(PyObject *self, PyObject *args) {
    (void)self;
    PyObject *tensor, *pairs;
    if (!PyArg_ParseTuple(args, "OO!", &tensor, &PyTuple_Type, &pairs)) return NULL;
    Py_INCREF(tensor);
    Py_XSETREF(tensor_type, tensor);
    n_types = 0;
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(pairs) && i < MAX_TYPES; ++i) {
        PyObject *t;
        int code;
        if (!PyArg_ParseTuple(PyTuple_GET_ITEM(pairs, i), "Oi", &t, &code)) return NULL;
        Py_INCREF(t);
        types[n_types] = t;
        codes[n_types++] = code;
    }
    Py_RETURN_NONE;
}

static PyObject *method(PyObject *t, PyObject *name) {
    PyObject *a[1] = {t};
    return PyObject_VectorcallMethod(name, a, 1 | PY_VECTORCALL_ARGUMENTS_OFFSET, NULL);
}

static int64_t int_method(PyObject *t, PyObject *name) {
    PyObject *r = method(t, name);
    if (r == NULL) return -1;
    const unsigned long long v = PyLong_AsUnsignedLongLongMask(r);
    Py_DECREF(r);
    return (int64_t)v;
}

/* 1: a tensor on device `index`; 0: not; -1: error */
static int on_device(PyObject *t, long index) {
    const int is = PyObject_IsInstance(t, tensor_type);
    if (is <= 0) return is;
    const int64_t d = int_method(t, s_device);
    if (d == -1 && PyErr_Occurred()) return -1;
    return d == index;
}

static int is_contiguous(PyObject *t) {
    PyObject *r = method(t, s_contiguous);
    if (r == NULL) return -1;
    const int v = PyObject_IsTrue(r);
    Py_DECREF(r);
    return v;
}

static int describe(PyObject *t, xm_tensor *d) {
    const int64_t ptr = int_method(t, s_ptr);
    if (ptr == -1 && PyErr_Occurred()) return -1;
    PyObject *shape = PyObject_GetAttr(t, s_shape);
    if (shape == NULL) return -1;
    const Py_ssize_t rank = PyTuple_Check(shape) ? PyTuple_GET_SIZE(shape) : -1;
    if (rank < 0 || rank > XM_MAX_RANK) {
        Py_DECREF(shape);
        PyErr_SetString(PyExc_ValueError, "tensor rank above 8 is not supported");
        return -1;
    }
    d->data = (void *)(uintptr_t)ptr;
    d->rank = (int32_t)rank;
    for (Py_ssize_t i = 0; i < rank; ++i) {
        d->shape[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, i));
        if (d->shape[i] == -1 && PyErr_Occurred()) {
            Py_DECREF(shape);
            return -1;
        }
    }
    Py_DECREF(shape);
    PyObject *type = PyObject_GetAttr(t, s_dtype);
    if (type == NULL) return -1;
    d->dtype = 0;
    for (int i = 0; i < n_types; ++i)
        if (types[i] == type) d->dtype = codes[i];
    Py_DECREF(type);
    return 0;
}

/* call(fwd, size, attrs, inputs, blank, outputs, device, inplace, alloc, stream) -> (status, which)
 *   fwd, size   entry points as integers (size 0: the operator takes no workspace)
 *   attrs       address of the attribute struct
 *   inputs      tuple of tensors or None; blank: the descriptors of absent inputs, as bytes
 *   outputs     tuple of contiguous tensors
 *   inplace     index of an input that must not be copied, or -1
 *   alloc       alloc(bytes) -> a uint8 tensor
 * status is the entry point's; or -1: input `which` is not a tensor on the device,
 * -2: input `which` would have to be copied, -3: output `which` is not a contiguous
 * tensor on the device. */
static PyObject *call(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    (void)self;
    if (n != 10 || !PyTuple_Check(a[3]) || !PyBytes_Check(a[4]) || !PyTuple_Check(a[5])) {
        PyErr_SetString(PyExc_TypeError, "call: wrong arguments");
        return NULL;
    }
    const fwd_fn fwd = (fwd_fn)(uintptr_t)PyLong_AsUnsignedLongLongMask(a[0]);
    const size_fn size = (size_fn)(uintptr_t)PyLong_AsUnsignedLongLongMask(a[1]);
    const void *attrs = (const void *)(uintptr_t)PyLong_AsUnsignedLongLongMask(a[2]);
    const Py_ssize_t n_in = PyTuple_GET_SIZE(a[3]), n_out = PyTuple_GET_SIZE(a[5]);
    const long index = PyLong_AsLong(a[6]), inplace = PyLong_AsLong(a[7]);
    void *stream = (void *)(uintptr_t)PyLong_AsUnsignedLongLongMask(a[9]);
    if (PyErr_Occurred()) return NULL;
    xm_tensor in[MAX_IN], out[MAX_IN];
    if (n_in > MAX_IN || n_out > MAX_IN || PyBytes_GET_SIZE(a[4]) != (Py_ssize_t)(n_in * sizeof(xm_tensor))) {
        PyErr_SetString(PyExc_TypeError, "call: wrong number of tensors");
        return NULL;
    }
    memcpy(in, PyBytes_AS_STRING(a[4]), (size_t)n_in * sizeof(xm_tensor));
    PyObject *copies[MAX_IN + 1];
    int n_copies = 0;
    PyObject *result = NULL;
    long status = 0, which = 0;
    for (Py_ssize_t i = 0; i < n_in; ++i) {
        PyObject *t = PyTuple_GET_ITEM(a[3], i);
        if (t == Py_None) continue;
        const int here = on_device(t, index);
        if (here < 0) goto done;
        if (here == 0) {
            status = -1, which = (long)i;
            goto answer;
        }
        const int dense = is_contiguous(t);
        if (dense < 0) goto done;
        if (dense == 0) {
            if (i == inplace) {
                status = -2, which = (long)i;
                goto answer;
            }
            t = method(t, s_make);
            if (t == NULL) goto done;
            copies[n_copies++] = t;
        }
        if (describe(t, &in[i]) < 0) goto done;
    }
    for (Py_ssize_t i = 0; i < n_out; ++i) {
        PyObject *t = PyTuple_GET_ITEM(a[5], i);
        const int here = on_device(t, index);
        if (here < 0) goto done;
        const int dense = here ? is_contiguous(t) : 0;
        if (dense < 0) goto done;
        if (!dense) {
            status = -3, which = (long)i;
            goto answer;
        }
        if (describe(t, &out[i]) < 0) goto done;
    }
    {
        size_t bytes = 0;
        void *ws = NULL;
        if (size != NULL) {
            status = size(attrs, in, (int32_t)n_in, &bytes);
            if (status != 0) goto answer;
            if (bytes > 0) {
                PyObject *count = PyLong_FromSize_t(bytes);
                if (count == NULL) goto done;
                PyObject *t = PyObject_CallOneArg(a[8], count);
                Py_DECREF(count);
                if (t == NULL) goto done;
                copies[n_copies++] = t;
                const int64_t ptr = int_method(t, s_ptr);
                if (ptr == -1 && PyErr_Occurred()) goto done;
                ws = (void *)(uintptr_t)ptr;
            }
        }
        /* a launch may wait for room in its queue: other threads run meanwhile (the caller's tuples hold the tensors) */
        PyThreadState *const thread = PyEval_SaveThread();
        status = fwd(attrs, in, (int32_t)n_in, out, ws, bytes, stream);
        PyEval_RestoreThread(thread);
    }
answer:
    result = Py_BuildValue("(ll)", status, which);
done:
    for (int i = 0; i < n_copies; ++i) Py_DECREF(copies[i]);
    return result;
}

static PyMethodDef methods[] = {
    {"setup", setup, METH_VARARGS, "setup(Tensor, ((dtype, code), ...))"},
    {"call", (PyCFunction)(void (*)(void))call, METH_FASTCALL,
     "call(fwd, size, attrs, inputs, blank, outputs, device, inplace, alloc, stream) -> (status, which)"},
    {NULL, NULL, 0, NULL},
};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_xm_call", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__xm_call(void) {
    s_device = PyUnicode_InternFromString("get_device");
    s_contiguous = PyUnicode_InternFromString("is_contiguous");
    s_make = PyUnicode_InternFromString("contiguous");
    s_ptr = PyUnicode_InternFromString("data_ptr");
    s_shape = PyUnicode_InternFromString("shape");
    s_dtype = PyUnicode_InternFromString("dtype");
    if (!s_device || !s_contiguous || !s_make || !s_ptr || !s_shape || !s_dtype) return NULL;
    return PyModule_Create(&module);
}
