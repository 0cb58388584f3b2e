// The 8-bit operators' calls from Python: checks of the arguments, allocation of the results, the current stream, the launch.
//
// These calls are short (a decoded token's norm is 2 us on the device), so what the host does around a launch is most of what an
// eager call takes: with the checks and allocations in Python and the launch through ctypes 6.9 us for a rounding and 7.8 us for a
// product, 4.0 to 4.4 and 3.5 to 4.5 us so, of which the launch itself is 1.6 to 2.5.  Results are as if allocated by torch.empty on the inputs'
// device; an error is the package's KernelError.

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
#include <tuple>

#include "int8_calls.h"

namespace {

constexpr int64_t RUN = 64, MAX_K = 131071;  // as ops/int8.py says them

struct Refused {
    std::string text;
};
[[noreturn]] void refuse(const std::string& text) { throw Refused{text}; }

// What ops/int8.py hands over: the error's class, the entry points, and two functions, (device index) -> address of the device's
// error word, (tokens, features, K, gated, device index) -> plan.
PyObject *error_class, *device_function, *plan_function;
int (*quantize_entry)(const Int8RowsCall*);
int (*dequantize_entry)(const Int8RowsCall*);
int (*norm_entry)(const Int8RowsCall*);
int (*product_entry)(const Int8Call*);

using Plan = std::array<int64_t, 5>;
std::map<int64_t, int*> error_words;                                                      // by device
std::map<std::tuple<int64_t, int64_t, int64_t, int64_t, int64_t>, Plan> plans;           // by (device, features, K, gated, tokens)

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
struct NewRows {
    at::Tensor values, scales;
};
// Int8 rows in one allocation, the scales behind the values: a second one and its release would take 0.4 us more of a call.
NewRows empty_rows(int64_t rows, int64_t width, int64_t stride, const at::Tensor& beside) {
    at::Tensor values(at::detail::empty_strided_cuda({rows * (stride + 4)}, {1}, at::kChar, beside.device()));
    at::Tensor scales = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(values.storage()), values.key_set(), caffe2::TypeMeta::Make<float>());
    scales.unsafeGetTensorImpl()->set_storage_offset(rows * stride / 4);
    scales.unsafeGetTensorImpl()->set_sizes_and_strides(c10::IntArrayRef({rows}), c10::IntArrayRef({1}));
    values.unsafeGetTensorImpl()->set_sizes_and_strides(c10::IntArrayRef({rows, width}), c10::IntArrayRef({stride, 1}));
    return {std::move(values), std::move(scales)};
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

Plan plan_of(PyObject* given, int64_t tokens, int64_t features, int64_t k, int64_t gated, int64_t device) {
    PyObject* made = nullptr;
    // (what a plan depends on: ops/int8.py, int8_plan)
    const int64_t step = tokens <= 640 ? 16 : 256;
    const std::tuple<int64_t, int64_t, int64_t, int64_t, int64_t> key{device, features, k, gated, (tokens + step - 1) / step * step};
    if (given == Py_None) {
        auto found = plans.find(key);
        if (found != plans.end()) return found->second;
        made = given = PyObject_CallFunction(plan_function, "LLLLL", (long long)tokens, (long long)features, (long long)k, (long long)gated, (long long)device);
        if (!given) throw python_error();
    }
    Plan plan{};
    bool ok = PyTuple_Check(given) && PyTuple_GET_SIZE(given) == (Py_ssize_t)plan.size();
    for (size_t i = 0; ok && i < plan.size(); ++i) {
        PyObject* v = PyTuple_GET_ITEM(given, i);
        int past = 0;
        if ((ok = PyLong_Check(v))) plan[i] = PyLong_AsLongLongAndOverflow(v, &past);
        ok = ok && !past && plan[i] >= 0 && plan[i] <= INT32_MAX;
    }
    Py_XDECREF(made);
    if (!ok) refuse("a plan is a tuple of five whole numbers (ops.int8_plan)");
    if (made) plans[key] = plan;
    return plan;
}

int64_t launches;  // kernels launched here so far
void check(int code, const char* what) {
    if (code) refuse(std::string(what) + ": CUDA error " + std::to_string(code) + " at launch");
    ++launches;
}

void check_size(int64_t rows, int64_t width) {
    if (width > INT8_MAX_WIDTH || rows > INT32_MAX)
        refuse("int8 rows are formed " + std::to_string(INT32_MAX) + " at most, of " + std::to_string(INT8_MAX_WIDTH) + " elements at most, not " + std::to_string(rows) + " of " + std::to_string(width));
}

struct Rows {
    int64_t rows, width, stride;
    const at::Tensor *values, *scales;
};
Rows rows_of(PyObject* values, PyObject* scales, const char* what) {
    const at::Tensor &v = tensor_of(values, what), &s = tensor_of(scales, what);
    if (v.dim() != 2 || v.scalar_type() != at::kChar)
        refuse(std::string(what) + ": the values must be a two-dimensional int8 tensor, got " + c10::toString(v.scalar_type()) + " " + say(v.sizes()));
    const int64_t n = v.size(0), k = v.size(1);
    if (s.scalar_type() != at::kFloat || s.numel() != n || !s.is_contiguous() || s.get_device() != v.get_device())
        refuse(std::string(what) + ": the scales must be " + std::to_string(n) + " contiguous float32 numbers beside the values");
    const int64_t stride = n < 2 ? (k + 15) & -16 : v.stride(0);
    if (n && k && ((k > 1 && v.stride(1) != 1) || stride % 16 || stride < k || (uintptr_t)v.data_ptr() % 16))
        refuse(std::string(what) + ": rows must be contiguous and start on 16 bytes (a stride that is a multiple of 16), got strides " + say(v.strides()));
    return {n, k, stride, &v, &s};
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

#define CALL_BEGIN HANDLE_TH_ERRORS try {
#define CALL_END                                                  \
    } catch (const Refused& r) {                                  \
        PyErr_SetString(error_class, r.text.c_str());             \
        return nullptr;                                           \
    }                                                             \
    END_HANDLE_TH_ERRORS

// (x, early) -> values, scales
PyObject* quantize(PyObject*, PyObject* const* args, Py_ssize_t) {
    CALL_BEGIN
    const at::Tensor& x = tensor_of(args[0], "x");
    if (x.dim() != 2) refuse("x must be two-dimensional, got " + say(x.sizes()));
    const int64_t n = x.size(0), k = x.size(1), q_stride = (k + 15) & -16, code = code_of(x.scalar_type());
    if (k < 1) refuse("rows without elements have no scale");
    check_size(n, k);
    if (k > 1 && x.stride(1) != 1) refuse("the rows of x must be contiguous, got strides " + say(x.strides()));
    OnDevice here(x);
    auto [values, scales] = empty_rows(n, k, q_stride, x);
    if (n) {
        Int8RowsCall c = {};
        c.x = x.data_ptr(); c.stride = x.stride(0); c.q = (int8_t*)values.data_ptr(); c.q_stride = q_stride; c.scales = (float*)scales.data_ptr();
        c.rows = n; c.width = k; c.dtype = code; c.early = args[1] == Py_True;
        c.err = error_word(x.get_device()); c.stream = c10::cuda::getCurrentCUDAStream().stream();
        check(quantize_entry(&c), "quantize_rows_int8");
    }
    return pair(std::move(values), std::move(scales));
    CALL_END
}

// (values, scales, dtype, early) -> tensor
PyObject* dequantize(PyObject*, PyObject* const* args, Py_ssize_t) {
    CALL_BEGIN
    const Rows r = rows_of(args[0], args[1], "rows");
    const at::ScalarType type = dtype_of(args[2]);
    const int64_t code = code_of(type);
    check_size(r.rows, r.width);
    OnDevice here(*r.values);
    at::Tensor out = empty(r.rows, r.width, type, *r.values);
    if (r.rows && r.width) {
        Int8RowsCall c = {};
        c.q = (int8_t*)r.values->data_ptr(); c.q_stride = r.stride; c.scales = (float*)r.scales->data_ptr();
        c.rows = r.rows; c.width = r.width; c.dtype = code; c.y = out.data_ptr(); c.early = args[3] == Py_True;
        c.stream = c10::cuda::getCurrentCUDAStream().stream();
        check(dequantize_entry(&c), "dequantize_rows_int8");
    }
    return THPVariable_Wrap(std::move(out));
    CALL_END
}

// (residual, delta or None, weight, eps, residual_out or None) -> values, scales
PyObject* norm(PyObject*, PyObject* const* args, Py_ssize_t) {
    CALL_BEGIN
    const at::Tensor& residual = contiguous_of(args[0], "residual");
    if (residual.scalar_type() != at::kFloat) refuse(std::string("residual must be float32, got ") + c10::toString(residual.scalar_type()));
    if (residual.dim() != 2 || residual.size(1) < 1) refuse("residual must be [tokens, features], got " + say(residual.sizes()));
    const int64_t n = residual.size(0), h = residual.size(1), q_stride = (h + 15) & -16;
    check_size(n, h);
    Int8RowsCall c = {};
    c.x = residual.data_ptr(); c.stride = h; c.rows = n; c.width = h; c.dtype = 1;
    if (args[1] != Py_None) {
        const at::Tensor& delta = contiguous_of(args[1], "delta");
        c.dtype = code_of(delta.scalar_type());
        if (delta.sizes() != residual.sizes()) refuse("delta " + say(delta.sizes()) + " does not match residual " + say(residual.sizes()));
        same_device(residual, delta, "delta");
        c.delta = delta.data_ptr();
        c.y = residual.data_ptr();
    }
    const at::Tensor& weight = contiguous_of(args[2], "norm weight");
    if (weight.numel() != h || (weight.scalar_type() != at::kFloat && weight.scalar_type() != at::kBFloat16))
        refuse("norm weight has the wrong size or dtype");
    same_device(residual, weight, "norm weight");
    c.weight = weight.data_ptr(); c.w_f32 = weight.scalar_type() == at::kFloat;
    c.eps = PyFloat_AsDouble(args[3]);
    if (c.eps == -1.0 && PyErr_Occurred()) throw python_error();
    if (args[4] != Py_None) {
        const at::Tensor& to = contiguous_of(args[4], "residual_out");
        if (to.scalar_type() != at::kFloat || to.sizes() != residual.sizes())
            refuse("residual_out must be float32 " + say(residual.sizes()) + ", got " + c10::toString(to.scalar_type()) + " " + say(to.sizes()));
        same_device(residual, to, "residual_out");
        c.y = to.data_ptr();
    }
    OnDevice here(residual);
    auto [values, scales] = empty_rows(n, h, q_stride, residual);
    if (n) {
        c.q = (int8_t*)values.data_ptr(); c.q_stride = q_stride; c.scales = (float*)scales.data_ptr();
        c.err = error_word(residual.get_device()); c.stream = c10::cuda::getCurrentCUDAStream().stream();
        check(norm_entry(&c), "add_rmsnorm_int8");
    }
    return pair(std::move(values), std::move(scales));
    CALL_END
}

// (x values, x scales, weight values, weight scales, bias or None, dtype, gated, columns or None, plan or None) -> tensor
PyObject* product(PyObject*, PyObject* const* args, Py_ssize_t) {
    CALL_BEGIN
    const Rows x = rows_of(args[0], args[1], "x"), w = rows_of(args[2], args[3], "weight");
    const bool gated = args[6] == Py_True;
    const char* what = gated ? "gate_up_swiglu_int8" : "linear_int8";
    const int64_t tokens = x.rows, features = w.rows, k = x.width;
    if (w.width != k) refuse("weight " + say(w.values->sizes()) + " does not match x " + say(x.values->sizes()));
    if (k < 1 || k > MAX_K) refuse("an int8 product takes 1 to " + std::to_string(MAX_K) + " elements of K, not " + std::to_string(k));
    same_device(*x.values, *w.values, "weight");
    int64_t columns = features;
    if (gated) {
        if (features % (2 * RUN))
            refuse("gate and up rows alternate in runs of " + std::to_string(RUN) + ": " + std::to_string(features) + " rows are no multiple of " + std::to_string(2 * RUN));
        columns = features / 2;
        if (args[7] != Py_None) {
            const int64_t asked = PyLong_AsLongLong(args[7]);
            if (asked == -1 && PyErr_Occurred()) throw python_error();
            if (asked < 0 || asked > columns) refuse(std::to_string(asked) + " features asked of " + std::to_string(columns));
            columns = asked;
        }
    }
    const at::ScalarType type = dtype_of(args[5]);
    Int8Call c = {};
    c.out_f32 = 1 - code_of(type);
    if (args[4] != Py_None) {
        const at::Tensor& bias = contiguous_of(args[4], "bias");
        if (bias.numel() != features || (bias.scalar_type() != at::kFloat && bias.scalar_type() != at::kBFloat16))
            refuse("bias has the wrong size or dtype");
        same_device(*x.values, bias, "bias");
        c.bias = bias.data_ptr(); c.bias_f32 = bias.scalar_type() == at::kFloat;
    }
    OnDevice here(*x.values);
    at::Tensor out = empty(tokens, columns, type, *x.values);
    if (tokens && columns) {
        const int64_t device = x.values->get_device();
        const Plan plan = plan_of(args[8], tokens, features, k, gated, device);
        c.x = x.values->data_ptr(); c.ldx = x.stride; c.x_scale = (const float*)x.scales->data_ptr();
        c.w = w.values->data_ptr(); c.ldw = w.stride; c.w_scale = (const float*)w.scales->data_ptr();
        c.out = out.data_ptr(); c.ldc = columns; c.tokens = tokens; c.features = features; c.K = k; c.gated = gated; c.out_features = columns;
        c.many = plan[0]; c.bn = plan[1]; c.slices = plan[2]; c.per_sm = plan[3]; c.steps = plan[4];
        c.err = error_word(device); c.stream = c10::cuda::getCurrentCUDAStream().stream();
        check(product_entry(&c), what);
    }
    return THPVariable_Wrap(std::move(out));
    CALL_END
}

// (error class, addresses of the four entry points, device function, plan function)
PyObject* use(PyObject*, PyObject* const* args, Py_ssize_t) {
    error_class = Py_NewRef(args[0]);
    quantize_entry = (int (*)(const Int8RowsCall*))PyLong_AsVoidPtr(args[1]);
    dequantize_entry = (int (*)(const Int8RowsCall*))PyLong_AsVoidPtr(args[2]);
    norm_entry = (int (*)(const Int8RowsCall*))PyLong_AsVoidPtr(args[3]);
    product_entry = (int (*)(const Int8Call*))PyLong_AsVoidPtr(args[4]);
    device_function = Py_NewRef(args[5]);
    plan_function = Py_NewRef(args[6]);
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
}

// () -> how many kernels these calls have launched
PyObject* launched(PyObject*, PyObject* const*, Py_ssize_t) { return PyLong_FromLongLong(launches); }

#define METHOD(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(use), METHOD(quantize), METHOD(dequantize), METHOD(norm), METHOD(product), METHOD(launched), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "slipstream_int8_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_slipstream_int8_calls() { return PyModule_Create(&module); }
