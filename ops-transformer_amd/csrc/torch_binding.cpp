// The Python module opapi_torch: an operator's tensors packed for opapiRunPacked (opapi_descriptor.h) from torch's own objects.
//
// A call on a few rows is bound by the host.  Asking a tensor for its device, type, address, extents and strides costs Python half a microsecond, one
// foreign call another half; read here they take a few tens of nanoseconds.  libcust_opapi.so knows nothing of torch: the function to call comes as an
// address from whoever has loaded the library.
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstring>

#include "acl/acl.h"
#include "opapi_descriptor.h"

namespace {

using RunPacked = decltype(&opapiRunPacked);

constexpr Py_ssize_t kMaxScalars = 16, kMaxTensors = 16;
constexpr int64_t kMaxDims = 8;

// -1: a type the operators do not know.
int64_t CodeOf(c10::ScalarType type) {
    switch (type) {
        case c10::kFloat: return ACL_FLOAT;
        case c10::kHalf: return ACL_FLOAT16;
        case c10::kBFloat16: return ACL_BF16;
        case c10::kChar: return ACL_INT8;
        case c10::kInt: return ACL_INT32;
        case c10::kLong: return ACL_INT64;
        case c10::kBool: return ACL_BOOL;
        default: return -1;
    }
}

// run(function, device, stream, workspace, size, scalars, tensors): both phases on tensors that are all on `device` (the first is not None), scalars starting
// with the operator's number, doubles as they are.  Returns the bytes of workspace that the operator asks for (more than `size`: nothing is enqueued), a
// status of its own below zero, or a tensor that is somewhere else.
PyObject* Run(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 7 || !PyTuple_Check(args[5]) || !PyTuple_Check(args[6]) || PyTuple_GET_SIZE(args[5]) > kMaxScalars ||
        PyTuple_GET_SIZE(args[6]) > kMaxTensors) {
        PyErr_SetString(PyExc_TypeError, "run(function, device, stream, workspace, size, scalars, tensors)");
        return nullptr;
    }
    const auto function = reinterpret_cast<RunPacked>(PyLong_AsSize_t(args[0]));
    const long device = PyLong_AsLong(args[1]);
    void* const stream = PyLong_AsVoidPtr(args[2]);
    void* const workspace = PyLong_AsVoidPtr(args[3]);
    const uint64_t size = PyLong_AsUnsignedLongLong(args[4]);
    if (PyErr_Occurred() != nullptr) return nullptr;

    int64_t packed[kMaxScalars + kMaxTensors * (3 + 2 * kMaxDims)];
    uint64_t length = 0;
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(args[5]); ++i) {
        PyObject* const scalar = PyTuple_GET_ITEM(args[5], i);
        if (PyFloat_Check(scalar)) {
            const double value = PyFloat_AS_DOUBLE(scalar);
            std::memcpy(&packed[length++], &value, sizeof(value));
        } else {
            PyObject* const whole = PyNumber_Index(scalar);
            if (whole == nullptr) return nullptr;
            packed[length++] = PyLong_AsLongLong(whole);
            Py_DECREF(whole);
            if (PyErr_Occurred() != nullptr) return nullptr;
        }
    }
    try {
        for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(args[6]); ++i) {
            PyObject* const object = PyTuple_GET_ITEM(args[6], i);
            if (object == Py_None) {
                for (int j = 0; j < 3; ++j) packed[length++] = 0;
                continue;
            }
            if (!THPVariable_Check(object)) {
                PyErr_Format(PyExc_TypeError, "a tensor is needed, not %s", Py_TYPE(object)->tp_name);
                return nullptr;
            }
            const at::Tensor& t = THPVariable_Unpack(object);
            if (!t.is_cuda() || t.get_device() != device) {
                Py_INCREF(object);
                return object;
            }
            const int64_t code = CodeOf(t.scalar_type());
            if (code < 0 || t.dim() > kMaxDims) {
                PyErr_Format(PyExc_TypeError, "a tensor of %s and %d dimensions is not one the operators know", c10::toString(t.scalar_type()),
                             static_cast<int>(t.dim()));
                return nullptr;
            }
            packed[length++] = t.dim();
            packed[length++] = code;
            packed[length++] = static_cast<int64_t>(reinterpret_cast<uintptr_t>(t.data_ptr()));
            for (const int64_t extent : t.sizes()) packed[length++] = extent;
            for (const int64_t stride : t.strides()) packed[length++] = stride;
        }
    } catch (const std::exception& e) {  // of a tensor without memory, or without strides
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
    uint64_t needed = 0;
    aclnnStatus status;
    Py_BEGIN_ALLOW_THREADS
    status = function(packed, length, workspace, size, stream, &needed);
    Py_END_ALLOW_THREADS
    return status == 0 ? PyLong_FromUnsignedLongLong(needed) : PyLong_FromLongLong(-static_cast<int64_t>(status));
}

PyMethodDef kMethods[] = {{"run", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(Run)), METH_FASTCALL, "Both phases of an operator."},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "opapi_torch", "Operators of libcust_opapi.so on torch tensors.", -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_opapi_torch() { return PyModule_Create(&kModule); }
