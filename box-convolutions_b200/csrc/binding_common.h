// What the binding's sources share: checks, allocation, arguments of CPython calls.  Everything has internal linkage.
#pragma once
#include <ATen/TracerMode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <array>
#include <memory>
#include <mutex>
#include <stdexcept>
#include <string>

#include "../../include/boxconv_b200.h"

namespace {

using at::Tensor;
using Four = std::array<Tensor, 4>;      // x_min, x_max, y_min, y_max
const char *const kParamNames[4] = {"x_min", "x_max", "y_min", "y_max"};

[[noreturn]] void fail(const std::string &text) { throw std::runtime_error(text); }

std::string dtype_name(at::ScalarType t)
{
    switch (t) {
        case at::kFloat: return "torch.float32";
        case at::kDouble: return "torch.float64";
        case at::kHalf: return "torch.float16";
        case at::kBFloat16: return "torch.bfloat16";
        default: return c10::toString(t);
    }
}

bool is_narrow(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }
int io_kind(at::ScalarType t) { return t == at::kHalf ? BC_IO_F16 : (t == at::kBFloat16 ? BC_IO_BF16 : BC_IO_F32); }

void check_status(int status, const char *what)
{
    if (status == BC_OK) return;
    std::string text = std::string(what) + " failed: " + bc_status_string(status);
    if (status == BC_ERR_CUDA && bc_last_cuda_error()[0]) text += std::string(" (") + bc_last_cuda_error() + ")";
    fail(text);
}

// CUDA tensor of float32 or float64, or of exactly `dtype` when that is given.
void require_cuda_float(const Tensor &t, const char *name, at::ScalarType dtype = at::ScalarType::Undefined,
                        bool narrow_too = false)
{
    if (!t.is_cuda())
        fail(std::string("box_convolution: ") + name + " is not a CUDA tensor; this build has no CPU implementation");
    const at::ScalarType have = t.scalar_type();
    if (have != at::kFloat && have != at::kDouble && !(narrow_too && is_narrow(have)))
        fail(std::string("box_convolution: ") + name + " must be float32 or float64, got " + dtype_name(have));
    if (dtype != at::ScalarType::Undefined && have != dtype)
        fail(std::string("box_convolution: ") + name + " is " + dtype_name(have) + " but the call's other tensors are " +
             dtype_name(dtype));
}

Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType dtype, const Tensor &like)
{
    return Tensor(at::detail::empty_cuda(sizes, dtype, like.device(), std::nullopt));
}

// (the caching allocator hands out blocks aligned to 512 bytes)
Tensor new_workspace(size_t bytes, const Tensor &like)
{
    return new_tensor({(int64_t)(bytes ? bytes : 1)}, at::kByte, like);
}

bc_stream_t current_stream(const Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

int to_int(int64_t v)
{
    if (v < 0 || v > 0x7fffffffLL) fail("box_convolution: a size does not fit the library");
    return (int)v;
}

struct Args {
    PyObject *const *v;
    Py_ssize_t n, at = 0;
    Args(PyObject *const *v_, Py_ssize_t n_, Py_ssize_t wanted) : v(v_), n(n_)
    {
        TORCH_CHECK_TYPE(n == wanted, "wrong number of arguments");
    }
    Tensor tensor(const char *name)
    {
        PyObject *o = v[at++];
        TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor");
        return THPVariable_Unpack(o);
    }
    Tensor optional_tensor(const char *name)
    {
        if (v[at] == Py_None) {
            ++at;
            return Tensor();
        }
        return tensor(name);
    }
    Four params()
    {
        Four p;
        for (int i = 0; i < 4; ++i) p[i] = tensor(kParamNames[i]);
        return p;
    }
    double number()
    {
        const double d = PyFloat_AsDouble(v[at++]);
        if (d == -1.0 && PyErr_Occurred()) throw py::error_already_set();
        return d;
    }
    int64_t integer()
    {
        const long long i = PyLong_AsLongLong(v[at++]);
        if (i == -1 && PyErr_Occurred()) throw py::error_already_set();
        return i;
    }
    bool flag()
    {
        const int b = PyObject_IsTrue(v[at++]);
        if (b < 0) throw py::error_already_set();
        return b != 0;
    }
};

PyObject *wrap(const Tensor &t)
{
    if (!t.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(t);
}

}  // namespace

// layers_binding.cpp: the layers around a box convolution, entries of the module's table
extern PyMethodDef layer_methods[];
