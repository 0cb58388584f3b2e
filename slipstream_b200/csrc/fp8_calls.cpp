// The 8-bit float operators' calls from Python: checks of the arguments, allocation of the results, the current stream, the launch.
// Native for the reason that int8_calls.cpp gives.  Results are as if allocated by torch.empty on the inputs' device; an error is the
// package's KernelError.

#include <tuple>

#include "calls.h"
#include "fp8_calls.h"

namespace {

constexpr int64_t BLOCK = FP8_BLOCK, MAX_K = INT32_MAX - 256;
constexpr int64_t NORM_MAX_WIDTH = 48 * 1024 / 8 * BLOCK;  // the norm keeps two words a block of a row in shared memory

// What ops/fp8.py hands over beside the rest: the entry points, and a function (tokens, features, K, gated, device index) -> plan.
PyObject* plan_function;
int (*quantize_entry)(const Fp8RowsCall*);
int (*dequantize_entry)(const Fp8RowsCall*);
int (*norm_entry)(const Fp8RowsCall*);
int (*product_entry)(const Fp8Call*);

using Plan = std::array<int64_t, 4>;
std::map<std::tuple<int64_t, int64_t, int64_t, int64_t, int64_t>, Plan> plans;  // by (device, features, K, gated, tokens)

int64_t blocks_of(int64_t n) { return (n + BLOCK - 1) / BLOCK; }

// values [rows, width] with rows that start on 16 bytes, and scales, in one allocation: of rows [rows, blocks of a row], where the rows of a
// block stand side by side (a product's threads read those of neighbouring tokens); of blocks of 128 rows [blocks of rows, blocks of a row].
struct New {
    at::Tensor values, scales;
    int64_t stride, scale_row, scale_block;
};
New empty_fp8(int64_t rows, int64_t width, bool blocks, const at::Tensor& beside) {
    New r;
    r.stride = (width + 15) & -16;
    const int64_t across = blocks_of(width), down = blocks ? blocks_of(rows) : rows;
    r.scale_row = blocks ? across : 1;
    r.scale_block = blocks ? 1 : rows;
    r.values = at::Tensor(at::detail::empty_strided_cuda({rows * r.stride + 4 * down * across}, {1}, at::kFloat8_e4m3fn, beside.device()));
    r.scales = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(r.values.storage()), r.values.key_set(), caffe2::TypeMeta::Make<float>());
    r.scales.unsafeGetTensorImpl()->set_storage_offset(rows * r.stride / 4);
    r.scales.unsafeGetTensorImpl()->set_sizes_and_strides(c10::IntArrayRef({down, across}), c10::IntArrayRef({r.scale_row, r.scale_block}));
    r.values.unsafeGetTensorImpl()->set_sizes_and_strides(c10::IntArrayRef({rows, width}), c10::IntArrayRef({r.stride, 1}));
    return r;
}

Plan plan_of(PyObject* given, int64_t tokens, int64_t features, int64_t k, int64_t gated, int64_t device) {
    PyObject* made = nullptr;
    // (what a plan depends on: ops/fp8.py, fp8_plan)
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
    if (!ok) refuse("a plan is a tuple of four whole numbers (ops.fp8_plan)");
    if (made) plans[key] = plan;
    return plan;
}

void check_size(int64_t rows, int64_t width) {
    if (width > FP8_MAX_WIDTH || rows > INT32_MAX)
        refuse("fp8 rows are formed " + std::to_string(INT32_MAX) + " at most, of " + std::to_string(FP8_MAX_WIDTH) + " elements at most, not " + std::to_string(rows) + " of " + std::to_string(width));
}

struct Scaled {
    int64_t rows, width, stride, scale_row, scale_block;
    const at::Tensor *values, *scales;
};
Scaled scaled_of(PyObject* values, PyObject* scales, bool blocks, const char* what) {
    const at::Tensor &v = tensor_of(values, what), &s = tensor_of(scales, what);
    if (v.dim() != 2 || v.scalar_type() != at::kFloat8_e4m3fn)
        refuse(std::string(what) + ": the values must be a two-dimensional float8_e4m3fn tensor, got " + c10::toString(v.scalar_type()) + " " + say(v.sizes()));
    const int64_t n = v.size(0), k = v.size(1), down = blocks ? blocks_of(n) : n, across = blocks_of(k);
    if (s.scalar_type() != at::kFloat || s.dim() != 2 || s.size(0) != down || s.size(1) != across || s.get_device() != v.get_device())
        refuse(std::string(what) + ": the scales must be float32 " + say({down, across}) + " beside the values, got " + c10::toString(s.scalar_type()) + " " + say(s.sizes()));
    const int64_t stride = n < 2 ? (k + 15) & -16 : v.stride(0);
    if (n && k && ((k > 1 && v.stride(1) != 1) || stride % 16 || stride < k || (uintptr_t)v.data_ptr() % 16))
        refuse(std::string(what) + ": rows must be contiguous and start on 16 bytes (a stride that is a multiple of 16), got strides " + say(v.strides()));
    return {n, k, stride, s.stride(0), s.stride(1), &v, &s};
}

// (x, blocks, early) -> values, scales
PyObject* quantize(PyObject*, PyObject* const* args, Py_ssize_t) {
    CALL_BEGIN
    const at::Tensor& x = tensor_of(args[0], "x");
    if (x.dim() != 2) refuse("x must be two-dimensional, got " + say(x.sizes()));
    const int64_t n = x.size(0), k = x.size(1), code = code_of(x.scalar_type());
    const bool blocks = args[1] == Py_True;
    if (k < 1) refuse("rows without elements have no scale");
    check_size(n, k);
    if (k > 1 && x.stride(1) != 1) refuse("the rows of x must be contiguous, got strides " + say(x.strides()));
    OnDevice here(x);
    New r = empty_fp8(n, k, blocks, x);
    if (n) {
        Fp8RowsCall c = {};
        c.x = x.data_ptr(); c.stride = x.stride(0); c.q = (uint8_t*)r.values.data_ptr(); c.q_stride = r.stride;
        c.scales = (float*)r.scales.data_ptr(); c.scale_row = r.scale_row; c.scale_block = r.scale_block;
        c.rows = n; c.width = k; c.dtype = code; c.blocks = blocks; c.early = args[2] == Py_True;
        c.err = error_word(x.get_device()); c.stream = c10::cuda::getCurrentCUDAStream().stream();
        check(quantize_entry(&c), blocks ? "quantize_blocks_fp8" : "quantize_rows_fp8");
    }
    return pair(std::move(r.values), std::move(r.scales));
    CALL_END
}

// (values, scales, blocks, dtype, early) -> tensor
PyObject* dequantize(PyObject*, PyObject* const* args, Py_ssize_t) {
    CALL_BEGIN
    const bool blocks = args[2] == Py_True;
    const Scaled r = scaled_of(args[0], args[1], blocks, blocks ? "blocks" : "rows");
    const at::ScalarType type = dtype_of(args[3]);
    const int64_t code = code_of(type);
    check_size(r.rows, r.width);
    OnDevice here(*r.values);
    at::Tensor out = empty(r.rows, r.width, type, *r.values);
    if (r.rows && r.width) {
        Fp8RowsCall c = {};
        c.q = (uint8_t*)r.values->data_ptr(); c.q_stride = r.stride;
        c.scales = (float*)r.scales->data_ptr(); c.scale_row = r.scale_row; c.scale_block = r.scale_block;
        c.rows = r.rows; c.width = r.width; c.dtype = code; c.blocks = blocks; c.y = out.data_ptr(); c.early = args[4] == Py_True;
        c.stream = c10::cuda::getCurrentCUDAStream().stream();
        check(dequantize_entry(&c), "dequantize_fp8");
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
    const int64_t n = residual.size(0), h = residual.size(1);
    check_size(n, h);
    if (h > NORM_MAX_WIDTH) refuse("the norm takes up to " + std::to_string(NORM_MAX_WIDTH) + " features, not " + std::to_string(h));
    Fp8RowsCall c = {};
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
    New r = empty_fp8(n, h, false, residual);
    if (n) {
        c.q = (uint8_t*)r.values.data_ptr(); c.q_stride = r.stride;
        c.scales = (float*)r.scales.data_ptr(); c.scale_row = r.scale_row; c.scale_block = r.scale_block;
        c.err = error_word(residual.get_device()); c.stream = c10::cuda::getCurrentCUDAStream().stream();
        check(norm_entry(&c), "add_rmsnorm_fp8");
    }
    return pair(std::move(r.values), std::move(r.scales));
    CALL_END
}

// (x values, x scales, weight values, weight scales, bias or None, dtype, gated, columns or None, plan or None) -> tensor, or values and scales
PyObject* product(PyObject*, PyObject* const* args, Py_ssize_t) {
    CALL_BEGIN
    const Scaled x = scaled_of(args[0], args[1], false, "x"), w = scaled_of(args[2], args[3], true, "weight");
    const bool gated = args[6] == Py_True;
    const char* what = gated ? "gate_up_swiglu_fp8" : "linear_fp8";
    const int64_t tokens = x.rows, features = w.rows, k = x.width;
    if (w.width != k) refuse("weight " + say(w.values->sizes()) + " does not match x " + say(x.values->sizes()));
    if (k < 1 || k > MAX_K) refuse("an fp8 product takes 1 to " + std::to_string(MAX_K) + " elements of K, not " + std::to_string(k));
    if (tokens > INT32_MAX - 256 || features > INT32_MAX - 256) refuse("an fp8 product takes fewer than " + std::to_string(INT32_MAX - 255) + " tokens and features, not " + say({tokens, features}));
    same_device(*x.values, *w.values, "weight");
    int64_t columns = features;
    if (gated) {
        if (features % (2 * BLOCK))
            refuse("gate and up rows alternate in runs of " + std::to_string(BLOCK) + ": " + std::to_string(features) + " rows are no multiple of " + std::to_string(2 * BLOCK));
        columns = features / 2;
        if (args[7] != Py_None) {
            const int64_t asked = PyLong_AsLongLong(args[7]);
            if (asked == -1 && PyErr_Occurred()) throw python_error();
            if (asked < 0 || asked > columns) refuse(std::to_string(asked) + " features asked of " + std::to_string(columns));
            columns = asked;
        }
    }
    const at::ScalarType type = dtype_of(args[5]);
    const bool to_fp8 = gated && type == at::kFloat8_e4m3fn;
    if (!to_fp8) code_of(type);
    Fp8Call c = {};
    c.out_type = to_fp8 ? 2 : code_of(type);
    if (args[4] != Py_None) {
        const at::Tensor& bias = contiguous_of(args[4], "bias");
        if (bias.numel() != features || (bias.scalar_type() != at::kFloat && bias.scalar_type() != at::kBFloat16))
            refuse("bias has the wrong size or dtype");
        same_device(*x.values, bias, "bias");
        c.bias = bias.data_ptr(); c.bias_f32 = bias.scalar_type() == at::kFloat;
    }
    OnDevice here(*x.values);
    New rows;
    at::Tensor out;
    if (to_fp8) {
        rows = empty_fp8(tokens, columns, false, *x.values);
        c.out = rows.values.data_ptr(); c.ldc = rows.stride; c.out_scale = (float*)rows.scales.data_ptr();
    } else {
        out = empty(tokens, columns, type, *x.values);
        c.out = out.data_ptr(); c.ldc = columns;
    }
    if (tokens && columns) {
        const int64_t device = x.values->get_device();
        const Plan plan = plan_of(args[8], tokens, features, k, gated, device);
        c.x = x.values->data_ptr(); c.ldx = x.stride; c.x_scale = (const float*)x.scales->data_ptr(); c.x_row = x.scale_row; c.x_block = x.scale_block;
        c.w = w.values->data_ptr(); c.ldw = w.stride; c.w_scale = (const float*)w.scales->data_ptr(); c.w_row = w.scale_row; c.w_block = w.scale_block;
        c.tokens = tokens; c.features = features; c.K = k; c.gated = gated; c.out_features = columns;
        c.many = plan[0]; c.bn = plan[1]; c.slices = plan[2]; c.per_sm = plan[3];
        c.err = error_word(device); c.stream = c10::cuda::getCurrentCUDAStream().stream();
        at::Tensor parts;  // (a kernel of the same stream that gets this memory next writes behind those that read it here)
        if (c.many == 1 && c.slices > 1 && c.slices <= 8 && !gated) {
            parts = empty(c.slices * tokens, (features + 3) & -4, at::kFloat, *x.values);
            c.parts = (float*)parts.data_ptr();
        }
        check(product_entry(&c), what);
        if (c.parts) ++launches;  // (the kernel that puts the parts together)
    }
    return to_fp8 ? pair(std::move(rows.values), std::move(rows.scales)) : THPVariable_Wrap(std::move(out));
    CALL_END
}

// (error class, addresses of the four entry points, device function, plan function)
PyObject* use(PyObject*, PyObject* const* args, Py_ssize_t) {
    error_class = Py_NewRef(args[0]);
    quantize_entry = (int (*)(const Fp8RowsCall*))PyLong_AsVoidPtr(args[1]);
    dequantize_entry = (int (*)(const Fp8RowsCall*))PyLong_AsVoidPtr(args[2]);
    norm_entry = (int (*)(const Fp8RowsCall*))PyLong_AsVoidPtr(args[3]);
    product_entry = (int (*)(const Fp8Call*))PyLong_AsVoidPtr(args[4]);
    device_function = Py_NewRef(args[5]);
    plan_function = Py_NewRef(args[6]);
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
}

// () -> how many kernels these calls have launched
PyObject* launched(PyObject*, PyObject* const*, Py_ssize_t) { return PyLong_FromLongLong(launches); }

PyMethodDef methods[] = {METHOD(use), METHOD(quantize), METHOD(dequantize), METHOD(norm), METHOD(product), METHOD(launched), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "slipstream_fp8_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_slipstream_fp8_calls() { return PyModule_Create(&module); }
