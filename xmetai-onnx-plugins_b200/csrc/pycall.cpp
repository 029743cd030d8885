// pycall.cpp -- the Python mirror's short call path (module _xm_call).
//
// A decode step calls the single-token operators for every layer, and describing
// a tensor to the C ABI takes several Python operations each through ctypes, or
// method calls through the CPython API (half a microsecond a tensor). Here the
// tensors are read through torch's C++ API, which also allocates the outputs and
// the workspace and calls the operator's entry point, all with the interpreter
// lock free. What torch throws is raised as torch's own functions raise it. Built
// against the headers of the Python and the torch that run it.
#include <Python.h>

#include <algorithm>
#include <cstdint>
#include <cstring>
#include <utility>
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

constexpr const char *kRank = "tensor rank above 8 is not supported";

void describe(const at::Tensor &t, xm_tensor *d) {
    const auto sizes = t.sizes();
    TORCH_CHECK_VALUE(sizes.size() <= XM_MAX_RANK, kRank);
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

// Other threads run while one of these is there.
struct Unlocked {
    PyThreadState *const thread = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(thread); }
};

// A call in two steps: what the tuples hold is read under the interpreter lock; copies, allocations and the entry point,
// each of which may wait for the device or for room in its queue, come without it (the caller's tuples hold the tensors).
struct Call {
    xm_tensor in[kMaxTensors], out[kMaxTensors];
    Py_ssize_t n_in = 0, n_out = 0;
    struct Copy {
        Py_ssize_t at;
        at::Tensor t;
    };
    std::vector<Copy> copies;  // inputs that are not contiguous
    enum Make : char { kGiven, kOwn, kFloat } make[kMaxTensors] = {};  // outputs to allocate: in input 0's type, in float32
    at::TensorOptions options;  // of input 0
    at::Tensor made[kMaxTensors], workspace;

    // Describes the inputs over the descriptors of absent ones.
    Answer inputs(PyObject *tensors, PyObject *blank, int64_t index, long inplace) {
        n_in = PyTuple_GET_SIZE(tensors);
        std::memcpy(in, PyBytes_AS_STRING(blank), static_cast<size_t>(n_in) * sizeof(xm_tensor));
        for (Py_ssize_t i = 0; i < n_in; ++i) {
            PyObject *o = PyTuple_GET_ITEM(tensors, i);
            if (o == Py_None) continue;
            if (!on_device(o, index)) return Answer{-1, static_cast<long>(i)};
            const at::Tensor &t = THPVariable_Unpack(o);
            if (t.is_contiguous()) {
                describe(t, &in[i]);
            } else {
                if (i == inplace) return Answer{-2, static_cast<long>(i)};
                copies.push_back(Copy{i, t});
            }
        }
        return Answer{0, 0};
    }
    // Describes an output that is given.
    bool output(Py_ssize_t i, PyObject *o, int64_t index) {
        if (!on_device(o, index) || !THPVariable_Unpack(o).is_contiguous()) return false;
        describe(THPVariable_Unpack(o), &out[i]);
        return true;
    }
    // The rest, on the current stream's allocations. stream: what the entry point is given.
    long run(FwdFn fwd, SizeFn size, const void *attrs, int64_t index, void *stream) {
        const Unlocked unlocked;
        for (Copy &c : copies) {
            c.t = c.t.contiguous();
            describe(c.t, &in[c.at]);
        }
        for (Py_ssize_t i = 0; i < n_out; ++i) {
            if (make[i] == kGiven) continue;
            made[i] = at::empty(at::IntArrayRef(out[i].shape, static_cast<size_t>(out[i].rank)),
                                make[i] == kOwn ? options : options.dtype(at::kFloat));
            describe(made[i], &out[i]);
        }
        size_t bytes = 0;
        void *ws = nullptr;
        if (size != nullptr) {
            const xm_status s = size(attrs, in, static_cast<int32_t>(n_in), &bytes);
            if (s != XM_OK) return s;
            if (bytes > 0) {
                workspace = at::empty({static_cast<int64_t>(bytes)},
                                      at::TensorOptions(at::kByte).device(at::kCUDA, static_cast<c10::DeviceIndex>(index)));
                ws = workspace.data_ptr();
            }
        }
        return fwd(attrs, in, static_cast<int32_t>(n_in), out, ws, bytes, stream);
    }
};

void *pointer(PyObject *o) { return reinterpret_cast<void *>(static_cast<uintptr_t>(PyLong_AsUnsignedLongLongMask(o))); }

// call(fwd, size, attrs, inputs, blank, outputs, device, inplace, alloc, stream) -> (status, which)
// A call with outputs, device and stream of the caller's choosing; the operators go through serve.
//   fwd, size   entry points as integers (size 0: the operator takes no workspace)
//   attrs       address of the attribute struct
//   inputs      tuple of tensors or None; blank: the descriptors of absent inputs, as bytes
//   outputs     tuple of contiguous tensors
//   inplace     index of an input that must not be copied, or -1
//   alloc       ignored (the workspace is allocated here)
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
    Call c;
    Answer answer = c.inputs(a[3], a[4], index, inplace);
    c.n_out = n_out;
    for (Py_ssize_t i = 0; answer.status == 0 && i < n_out; ++i)
        if (!c.output(i, PyTuple_GET_ITEM(a[5], i), index)) answer = Answer{-3, static_cast<long>(i)};
    if (answer.status == 0) answer.status = c.run(fwd, size, attrs, index, stream);
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
    Call c;
    Answer answer = c.inputs(a[3], blank, index, inplace);
    c.n_out = n_out;
    c.options = x.options();
    for (Py_ssize_t i = 0; answer.status == 0 && i < n_out; ++i) {
        PyObject *o = PyTuple_GET_ITEM(a[5], i), *shape = PyTuple_GET_ITEM(a[6], i);
        if (o != Py_None) {
            if (!c.output(i, o, index)) answer = Answer{-3, static_cast<long>(i)};
            continue;
        }
        xm_tensor &d = c.out[i];  // (its data once it is there)
        c.make[i] = Call::kOwn;
        const Py_ssize_t rank = shape == Py_None ? x.dim() : PyTuple_Check(shape) ? PyTuple_GET_SIZE(shape) - 1 : -1;
        TORCH_CHECK(rank >= 0, "serve: wrong shape");
        TORCH_CHECK_VALUE(rank <= XM_MAX_RANK, kRank);
        d.rank = static_cast<int32_t>(rank);
        if (shape == Py_None) {
            std::copy(x.sizes().begin(), x.sizes().end(), d.shape);
            continue;
        }
        for (Py_ssize_t k = 0; k < rank; ++k) d.shape[k] = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, k + 1));
        if (PyLong_AsLong(PyTuple_GET_ITEM(shape, 0)) == 0) c.make[i] = Call::kFloat;
        if (PyErr_Occurred()) return nullptr;
    }
    if (answer.status == 0)
        answer.status = c.run(fwd, size, attrs, index,
                              c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index)).stream());
    if (answer.status != 0) return Py_BuildValue("(ll)", answer.status, answer.which);
    PyObject *result = PyTuple_New(n_out);
    if (result == nullptr) return nullptr;
    for (Py_ssize_t i = 0; i < n_out; ++i) {
        PyObject *o = PyTuple_GET_ITEM(a[5], i);
        if (o != Py_None) Py_INCREF(o);
        else o = THPVariable_Wrap(std::move(c.made[i]));
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
