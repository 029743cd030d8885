// pycall.cpp -- the Python mirror's short call path (module _xm_call).
//
// A decode step calls the single-token operators for every layer, and describing
// a tensor to the C ABI takes several Python operations each through ctypes, or
// method calls through the CPython API (half a microsecond a tensor). Here the
// tensors are read through torch's C++ API, which also allocates the outputs and
// the workspace, and the operator's entry point is called with the interpreter
// lock free. What torch throws is raised as torch's own functions raise it. Built
// against the headers of the Python and the torch that run it.
#include <Python.h>

#include <cstdint>
#include <cstring>
#include <vector>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include "../../include/xm_ops.h"

namespace {

constexpr int kMaxTensors = 16;

using FwdFn = xm_status (*)(const void *, const xm_tensor *, int32_t, xm_tensor *, void *, size_t, void *);
using SizeFn = xm_status (*)(const void *, const xm_tensor *, int32_t, size_t *);

int32_t code_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return XM_DTYPE_FLOAT;
        case at::kBFloat16: return XM_DTYPE_BFLOAT16;
        case at::kHalf: return XM_DTYPE_FLOAT16;
        case at::kInt: return XM_DTYPE_INT32;
        case at::kLong: return XM_DTYPE_INT64;
        default: return 0;
    }
}

void describe(const at::Tensor &t, xm_tensor *d) {
    const auto sizes = t.sizes();
    TORCH_CHECK_VALUE(sizes.size() <= XM_MAX_RANK, "tensor rank above 8 is not supported");
    d->data = t.data_ptr();
    d->rank = static_cast<int32_t>(sizes.size());
    for (size_t i = 0; i < sizes.size(); ++i) d->shape[i] = sizes[i];
    d->dtype = code_of(t.scalar_type());
}

bool on_device(PyObject *o, int64_t index) {
    if (!THPVariable_Check(o)) return false;
    const at::Tensor &t = THPVariable_Unpack(o);
    return t.is_cuda() && t.get_device() == index;
}

// status is the entry point's; or -1: input `which` is not a tensor on the device, -2: input `which` would have to be
// copied, -3: output `which` is not a contiguous tensor on the device.
struct Answer {
    long status, which;
};

// Describes the inputs over the descriptors of absent ones; copies of those that are not contiguous go to `keep`.
Answer describe_inputs(PyObject *tensors, int64_t index, long inplace, xm_tensor *in, std::vector<at::Tensor> &keep) {
    const Py_ssize_t n = PyTuple_GET_SIZE(tensors);
    for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject *o = PyTuple_GET_ITEM(tensors, i);
        if (o == Py_None) continue;
        if (!on_device(o, index)) return Answer{-1, static_cast<long>(i)};
        const at::Tensor &t = THPVariable_Unpack(o);
        if (t.is_contiguous()) {
            describe(t, &in[i]);
        } else {
            if (i == inplace) return Answer{-2, static_cast<long>(i)};
            keep.push_back(t.contiguous());
            describe(keep.back(), &in[i]);
        }
    }
    return Answer{0, 0};
}

// Asks for the workspace, allocates it on the current stream and calls the entry point.
long run(FwdFn fwd, SizeFn size, const void *attrs, const xm_tensor *in, Py_ssize_t n_in, xm_tensor *out, int64_t index,
         void *stream, std::vector<at::Tensor> &keep) {
    size_t bytes = 0;
    void *ws = nullptr;
    if (size != nullptr) {
        const xm_status s = size(attrs, in, static_cast<int32_t>(n_in), &bytes);
        if (s != XM_OK) return s;
        if (bytes > 0) {
            keep.push_back(at::empty({static_cast<int64_t>(bytes)},
                                     at::TensorOptions(at::kByte).device(at::kCUDA, static_cast<c10::DeviceIndex>(index))));
            ws = keep.back().data_ptr();
        }
    }
    // a launch may wait for room in its queue: other threads run meanwhile (the caller's tuples hold the tensors)
    PyThreadState *const thread = PyEval_SaveThread();
    const xm_status s = fwd(attrs, in, static_cast<int32_t>(n_in), out, ws, bytes, stream);
    PyEval_RestoreThread(thread);
    return s;
}

void *pointer(PyObject *o) { return reinterpret_cast<void *>(static_cast<uintptr_t>(PyLong_AsUnsignedLongLongMask(o))); }

// call(fwd, size, attrs, inputs, blank, outputs, device, inplace, alloc, stream) -> (status, which)
//   fwd, size   entry points as integers (size 0: the operator takes no workspace)
//   attrs       address of the attribute struct
//   inputs      tuple of tensors or None; blank: the descriptors of absent inputs, as bytes
//   outputs     tuple of contiguous tensors
//   inplace     index of an input that must not be copied, or -1
//   alloc       not used: the workspace is allocated here
PyObject *call(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 10 || !PyTuple_Check(a[3]) || !PyBytes_Check(a[4]) || !PyTuple_Check(a[5])) {
        PyErr_SetString(PyExc_TypeError, "call: wrong arguments");
        return nullptr;
    }
    const Py_ssize_t n_in = PyTuple_GET_SIZE(a[3]), n_out = PyTuple_GET_SIZE(a[5]);
    const long index = PyLong_AsLong(a[6]), inplace = PyLong_AsLong(a[7]);
    const auto fwd = reinterpret_cast<FwdFn>(pointer(a[0]));
    const auto size = reinterpret_cast<SizeFn>(pointer(a[1]));
    const void *attrs = pointer(a[2]);
    void *stream = pointer(a[9]);
    if (PyErr_Occurred()) return nullptr;
    if (n_in > kMaxTensors || n_out > kMaxTensors ||
        PyBytes_GET_SIZE(a[4]) != static_cast<Py_ssize_t>(n_in * sizeof(xm_tensor))) {
        PyErr_SetString(PyExc_TypeError, "call: wrong number of tensors");
        return nullptr;
    }
    xm_tensor in[kMaxTensors], out[kMaxTensors];
    std::memcpy(in, PyBytes_AS_STRING(a[4]), static_cast<size_t>(n_in) * sizeof(xm_tensor));
    std::vector<at::Tensor> keep;
    Answer answer = describe_inputs(a[3], index, inplace, in, keep);
    for (Py_ssize_t i = 0; answer.status == 0 && i < n_out; ++i) {
        PyObject *o = PyTuple_GET_ITEM(a[5], i);
        if (!on_device(o, index) || !THPVariable_Unpack(o).is_contiguous()) answer = Answer{-3, static_cast<long>(i)};
        else describe(THPVariable_Unpack(o), &out[i]);
    }
    if (answer.status == 0) answer.status = run(fwd, size, attrs, in, n_in, out, index, stream, keep);
    return Py_BuildValue("(ll)", answer.status, answer.which);
    END_HANDLE_TH_ERRORS
}

// serve(fwd, size, attrs, inputs, blanks, outputs, shapes, inplace) -> outputs, or (status, which) as integers
// The same on input 0's device and the stream that is current there, with outputs that are None allocated:
//   blanks      bytes of the absent inputs' descriptors for input 0 in float32, bfloat16, float16 and any other type
//   shapes      per output None (the shape and type of input 0) or (own, sizes...): float32, or with own 1 input 0's type
// Further statuses: -4: input 0 is not a CUDA tensor, -5: it is not on the current device.
PyObject *serve(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 8 || !PyTuple_Check(a[3]) || !PyTuple_Check(a[4]) || PyTuple_GET_SIZE(a[4]) != 4 || !PyTuple_Check(a[5]) ||
        !PyTuple_Check(a[6]) || PyTuple_GET_SIZE(a[5]) != PyTuple_GET_SIZE(a[6])) {
        PyErr_SetString(PyExc_TypeError, "serve: wrong arguments");
        return nullptr;
    }
    const Py_ssize_t n_in = PyTuple_GET_SIZE(a[3]), n_out = PyTuple_GET_SIZE(a[5]);
    const long inplace = PyLong_AsLong(a[7]);
    const auto fwd = reinterpret_cast<FwdFn>(pointer(a[0]));
    const auto size = reinterpret_cast<SizeFn>(pointer(a[1]));
    const void *attrs = pointer(a[2]);
    if (PyErr_Occurred()) return nullptr;
    if (n_in < 1 || n_in > kMaxTensors || n_out > kMaxTensors) {
        PyErr_SetString(PyExc_TypeError, "serve: wrong number of tensors");
        return nullptr;
    }
    PyObject *first = PyTuple_GET_ITEM(a[3], 0);
    if (!THPVariable_Check(first) || !THPVariable_Unpack(first).is_cuda()) return Py_BuildValue("(ll)", -4L, 0L);
    const at::Tensor &x = THPVariable_Unpack(first);
    const int64_t index = x.get_device();
    if (index != c10::cuda::current_device()) return Py_BuildValue("(ll)", -5L, 0L);
    const int32_t code = code_of(x.scalar_type());
    PyObject *blank = PyTuple_GET_ITEM(
        a[4], code == XM_DTYPE_FLOAT ? 0 : code == XM_DTYPE_BFLOAT16 ? 1 : code == XM_DTYPE_FLOAT16 ? 2 : 3);
    if (!PyBytes_Check(blank) || PyBytes_GET_SIZE(blank) != static_cast<Py_ssize_t>(n_in * sizeof(xm_tensor)))
        TORCH_CHECK(false, "serve: wrong descriptors");
    xm_tensor in[kMaxTensors], out[kMaxTensors];
    std::memcpy(in, PyBytes_AS_STRING(blank), static_cast<size_t>(n_in) * sizeof(xm_tensor));
    std::vector<at::Tensor> keep;
    Answer answer = describe_inputs(a[3], index, inplace, in, keep);
    if (answer.status != 0) return Py_BuildValue("(ll)", answer.status, answer.which);
    at::Tensor made[kMaxTensors];
    for (Py_ssize_t i = 0; i < n_out; ++i) {
        PyObject *o = PyTuple_GET_ITEM(a[5], i), *shape = PyTuple_GET_ITEM(a[6], i);
        if (o != Py_None) {
            if (!on_device(o, index) || !THPVariable_Unpack(o).is_contiguous())
                return Py_BuildValue("(ll)", -3L, static_cast<long>(i));
            made[i] = THPVariable_Unpack(o);
        } else if (shape == Py_None) {
            made[i] = at::empty(x.sizes(), x.options());
        } else {
            int64_t sizes[XM_MAX_RANK];
            const Py_ssize_t rank = PyTuple_Check(shape) ? PyTuple_GET_SIZE(shape) - 1 : -1;
            if (rank < 0 || rank > XM_MAX_RANK) TORCH_CHECK(false, "serve: wrong shape");
            for (Py_ssize_t k = 0; k < rank; ++k) sizes[k] = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, k + 1));
            const long own = PyLong_AsLong(PyTuple_GET_ITEM(shape, 0));
            if (PyErr_Occurred()) return nullptr;
            made[i] = at::empty(at::IntArrayRef(sizes, static_cast<size_t>(rank)),
                                x.options().dtype(own != 0 ? x.scalar_type() : at::kFloat));
        }
        describe(made[i], &out[i]);
    }
    void *stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index)).stream();
    answer.status = run(fwd, size, attrs, in, n_in, out, index, stream, keep);
    if (answer.status != 0) return Py_BuildValue("(ll)", answer.status, answer.which);
    PyObject *result = PyTuple_New(n_out);
    if (result == nullptr) return nullptr;
    for (Py_ssize_t i = 0; i < n_out; ++i) {
        PyObject *o = PyTuple_GET_ITEM(a[5], i);
        if (o != Py_None) Py_INCREF(o);
        else o = THPVariable_Wrap(std::move(made[i]));
        if (o == nullptr) {
            Py_DECREF(result);
            return nullptr;
        }
        PyTuple_SET_ITEM(result, i, o);
    }
    return result;
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"call", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(call)), METH_FASTCALL,
     "call(fwd, size, attrs, inputs, blank, outputs, device, inplace, alloc, stream) -> (status, which)"},
    {"serve", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(serve)), METH_FASTCALL,
     "serve(fwd, size, attrs, inputs, blanks, outputs, shapes, inplace) -> outputs or (status, which)"},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_xm_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__xm_call(void) {
    PyObject *m = PyModule_Create(&module);
    if (m != nullptr && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) != 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
