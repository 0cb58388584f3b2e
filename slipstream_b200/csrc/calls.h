// What the native calls from Python share: checks of the arguments, allocation of the results, the device and its error word, the
// launch's result, errors.  An extension module includes it once; each has its own copy of what is kept here.
#pragma once

#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <map>
#include <string>

namespace {

struct Refused {
    std::string text;
};
[[noreturn]] void refuse(const std::string& text) { throw Refused{text}; }

// What a module is told before its first call: the error's class, and a function (device index) -> address of the device's error word.
PyObject *error_class, *device_function;
std::map<int64_t, int*> error_words;  // by device

std::string say(at::IntArrayRef v) {
    std::string s = "(";
    for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
    return s + ")";
}

const at::Tensor& tensor_of(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) refuse(std::string(what) + " must be a tensor, not " + Py_TYPE(o)->tp_name);
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda()) refuse(std::string(what) + " must be a CUDA tensor");
    if (t.layout() != at::kStrided) refuse(std::string(what) + " must be a strided tensor");
    return t;
}
const at::Tensor& contiguous_of(PyObject* o, const char* what) {
    const at::Tensor& t = tensor_of(o, what);
    if (!t.is_contiguous()) refuse(std::string(what) + " must be contiguous");
    return t;
}
void same_device(const at::Tensor& a, const at::Tensor& b, const char* what) {
    if (a.get_device() != b.get_device()) refuse(std::string(what) + " is on " + b.device().str() + ", not on " + a.device().str());
}
// 0 float32, 1 bfloat16: the kernels' codes
int64_t code_of(at::ScalarType t) {
    if (t == at::kBFloat16) return 1;
    if (t != at::kFloat) refuse(std::string("kernels take float32 or bfloat16 tensors, not ") + c10::toString(t));
    return 0;
}
at::ScalarType dtype_of(PyObject* o) {
    if (!THPDtype_Check(o)) refuse("dtype must be torch.float32 or torch.bfloat16");
    return reinterpret_cast<THPDtype*>(o)->scalar_type;
}

at::Tensor empty(int64_t rows, int64_t width, at::ScalarType type, const at::Tensor& beside) {
    return at::Tensor(at::detail::empty_strided_cuda({rows, width}, {width, 1}, type, beside.device()));
}

int* error_word(int64_t device) {
    auto found = error_words.find(device);
    if (found != error_words.end()) return found->second;
    PyObject* address = PyObject_CallFunction(device_function, "L", (long long)device);
    if (!address) throw python_error();
    int* word = (int*)PyLong_AsVoidPtr(address);
    Py_DECREF(address);
    if (PyErr_Occurred()) throw python_error();
    return error_words[device] = word;
}

int64_t launches;  // kernels launched here so far
void check(int code, const char* what) {
    if (code) refuse(std::string(what) + ": CUDA error " + std::to_string(code) + " at launch");
    ++launches;
}

// The device of a call's tensors is made the current one for the launch where it is not.
struct OnDevice {
    c10::cuda::OptionalCUDAGuard guard;
    explicit OnDevice(const at::Tensor& t) {
        if (t.get_device() != c10::cuda::current_device()) guard.set_device(t.device());
    }
};

PyObject* pair(at::Tensor a, at::Tensor b) {
    PyObject* out = PyTuple_New(2);
    if (!out) throw python_error();
    PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(a)));
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(b)));
    return out;
}

}  // namespace

#define CALL_BEGIN HANDLE_TH_ERRORS try {
#define CALL_END                                                  \
    } catch (const Refused& r) {                                  \
        PyErr_SetString(error_class, r.text.c_str());             \
        return nullptr;                                           \
    }                                                             \
    END_HANDLE_TH_ERRORS

#define METHOD(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
