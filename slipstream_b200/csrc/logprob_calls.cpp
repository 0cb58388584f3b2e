// The log probabilities' call from Python: checks of the arguments, allocation of the result, the current stream, the launch.
// Native for the reason that int8_calls.cpp gives.  The result is as if allocated by torch.empty on the inputs' device; an error is the
// package's KernelError.

#include "calls.h"
#include "logprob_calls.h"

namespace {

int (*logprobs_entry)(const LogprobCall*);

// A view of `packed` (float32, contiguous) from element `first` on.
at::Tensor view(const at::Tensor& packed, at::ScalarType type, int64_t first, at::IntArrayRef sizes, at::IntArrayRef strides) {
    at::Tensor v = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(packed.storage()), packed.key_set(), c10::scalarTypeToTypeMeta(type));
    v.unsafeGetTensorImpl()->set_storage_offset(first);
    v.unsafeGetTensorImpl()->set_sizes_and_strides(sizes, strides);
    return v;
}

// (logits, tokens, top) -> packed, log probabilities, entropy, ranks, largest log probabilities, their tokens
PyObject* token_logprobs(PyObject*, PyObject* const* args, Py_ssize_t) {
    CALL_BEGIN
    const at::Tensor& logits = tensor_of(args[0], "logits");
    if (logits.dim() != 2) refuse("logits must be two-dimensional, got " + say(logits.sizes()));
    const int64_t n = logits.size(0), v = logits.size(1), code = code_of(logits.scalar_type());
    if (v < 1 || v > INT32_MAX - 65536) refuse("rows have 1 to " + std::to_string(INT32_MAX - 65536) + " logits, not " + std::to_string(v));
    if (n > INT32_MAX / 8) refuse("up to " + std::to_string(INT32_MAX / 8) + " rows, not " + std::to_string(n));
    if (v > 1 && logits.stride(1) != 1) refuse("the rows of the logits must be contiguous, got strides " + say(logits.strides()));
    const at::Tensor& tokens = contiguous_of(args[1], "tokens");
    if (tokens.dim() != 1 || tokens.size(0) != n || (tokens.scalar_type() != at::kInt && tokens.scalar_type() != at::kLong))
        refuse("tokens must be " + std::to_string(n) + " int32 or int64 numbers, got " + c10::toString(tokens.scalar_type()) + " " + say(tokens.sizes()));
    same_device(logits, tokens, "tokens");
    const int64_t top = PyLong_AsLongLong(args[2]);
    if (top == -1 && PyErr_Occurred()) throw python_error();
    if (top < 0 || top > LOGPROBS_MAX_TOP || top > v)
        refuse("0 to " + std::to_string(v < LOGPROBS_MAX_TOP ? v : LOGPROBS_MAX_TOP) + " alternatives of " + std::to_string(v) + ", not " + std::to_string(top));
    OnDevice here(logits);
    const int64_t width = 3 + 2 * top;
    at::Tensor packed = empty(n, width, at::kFloat, logits);
    if (n) {
        LogprobCall c = {};
        c.logits = logits.data_ptr(); c.stride = n > 1 ? logits.stride(0) : v; c.rows = n; c.vocabulary = v; c.dtype = code;
        c.tokens = tokens.data_ptr(); c.wide = tokens.scalar_type() == at::kLong; c.top = top; c.out = (float*)packed.data_ptr();
        c.err = error_word(logits.get_device()); c.stream = c10::cuda::getCurrentCUDAStream().stream();
        check(logprobs_entry(&c), "token_logprobs");
    }
    PyObject* out = PyTuple_New(6);
    if (!out) throw python_error();
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(view(packed, at::kFloat, 0, {n}, {width})));
    PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(view(packed, at::kFloat, 1, {n}, {width})));
    PyTuple_SET_ITEM(out, 3, THPVariable_Wrap(view(packed, at::kInt, 2, {n}, {width})));
    PyTuple_SET_ITEM(out, 4, THPVariable_Wrap(view(packed, at::kFloat, 3, {n, top}, {width, 1})));
    PyTuple_SET_ITEM(out, 5, THPVariable_Wrap(view(packed, at::kInt, 3 + top, {n, top}, {width, 1})));
    PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(packed)));
    return out;
    CALL_END
}

// (error class, address of the entry point, device function)
PyObject* use(PyObject*, PyObject* const* args, Py_ssize_t) {
    error_class = Py_NewRef(args[0]);
    logprobs_entry = (int (*)(const LogprobCall*))PyLong_AsVoidPtr(args[1]);
    device_function = Py_NewRef(args[2]);
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
}

// () -> how many kernels these calls have launched
PyObject* launched(PyObject*, PyObject* const*, Py_ssize_t) { return PyLong_FromLongLong(launches); }

PyMethodDef methods[] = {METHOD(use), METHOD(token_logprobs), METHOD(launched), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "slipstream_logprob_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_slipstream_logprob_calls() { return PyModule_Create(&module); }
