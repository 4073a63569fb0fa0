// Host side of the 8-bit operators' ordinary calls (Python module _fp8_call): checks the tensors, allocates the results and makes
// the library call.  Where anything is out of the ordinary (a wrong type or shape, other strides, another device than the current
// one, a tensor subclass, no rows) a function returns None, and the Python form in ops.py does the same with the messages.
// rms_norm with a residual and an 8-bit result takes 14 us of host time through Python, linear_fp8 12; their kernels for a few
// rows take less.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>

#include "convnn_b200.h"

namespace {

constexpr int64_t BLOCK = 128;

// The C entry points, and the class of a pair of values and scales: given by bind().
decltype(&convnn_b200_rms_norm) norm_fn = nullptr;
decltype(&convnn_b200_rms_norm_fp8) norm_fp8_fn = nullptr;
decltype(&convnn_b200_quantize_fp8) quantize_fn = nullptr;
decltype(&convnn_b200_linear_fp8) linear_fn = nullptr;
PyObject *blocks_class = nullptr, *check_fn = nullptr;

PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 6) {
        PyErr_SetString(PyExc_TypeError, "bind takes four addresses, the class of 8-bit blocks and the status check");
        return nullptr;
    }
    void* at[4];
    for (int i = 0; i < 4; ++i) {
        at[i] = PyLong_AsVoidPtr(args[i]);
        if (PyErr_Occurred()) return nullptr;
    }
    norm_fn = reinterpret_cast<decltype(norm_fn)>(at[0]);
    norm_fp8_fn = reinterpret_cast<decltype(norm_fp8_fn)>(at[1]);
    quantize_fn = reinterpret_cast<decltype(quantize_fn)>(at[2]);
    linear_fn = reinterpret_cast<decltype(linear_fn)>(at[3]);
    Py_INCREF(args[4]);
    Py_INCREF(args[5]);
    blocks_class = args[4];
    check_fn = args[5];
    Py_RETURN_NONE;
}

// A plain tensor on `device` (-1: on any CUDA device, which is then the one); no gradient wanted.
const at::Tensor* plain(PyObject* o, int& device, bool grad) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.layout() != at::kStrided || (grad && t.requires_grad())) return nullptr;
    if (device < 0) device = t.get_device();
    return t.get_device() == device ? &t : nullptr;
}
int dtype_code(at::ScalarType t) { return t == at::kBFloat16 ? CONVNN_BF16 : t == at::kFloat ? CONVNN_F32 : -1; }

// Rows of the last dimension with one stride between them.
bool rows_of(const at::Tensor& t, int64_t& rows, int64_t& ld) {
    const int64_t dim = t.dim();
    if (dim < 1) return false;
    const int64_t D = t.size(dim - 1);
    if (D < 1 || D > (1 << 30)) return false;
    rows = t.numel() / D;
    if (rows < 1) return false;
    ld = D;
    if (dim == 2 && t.stride(1) == 1 && t.stride(0) >= D) {
        ld = t.stride(0);
        return true;
    }
    return t.is_contiguous();
}
// 8-bit rows on 16-byte boundaries, and the scales of one block of channels side by side.
void empty_fp8(at::IntArrayRef shape, int64_t rows, c10::Device device, at::Tensor& values, int64_t& ld, at::Tensor& scales) {
    const int64_t D = shape.back(), blocks = (D + BLOCK - 1) / BLOCK;
    ld = (D + 15) / 16 * 16;
    c10::SmallVector<int64_t, 5> vs(shape.size()), ss(shape.size()), size(shape.begin(), shape.end());
    int64_t lead = 1;
    vs.back() = 1;
    ss.back() = rows;
    for (int64_t i = (int64_t)shape.size() - 2; i >= 0; --i) {
        vs[i] = lead * ld;
        ss[i] = lead;
        lead *= shape[i];
    }
    const auto options = at::TensorOptions().device(device);
    values = at::empty_strided(size, vs, options.dtype(at::kFloat8_e4m3fn));
    size.back() = blocks;
    scales = at::empty_strided(size, ss, options.dtype(at::kFloat));
}
// Steals nothing; new reference.
PyObject* blocks_object(const at::Tensor& values, const at::Tensor& scales) {
    PyObject* v = THPVariable_Wrap(values);
    PyObject* s = v ? THPVariable_Wrap(scales) : nullptr;
    PyObject* both = s ? PyObject_CallFunctionObjArgs(blocks_class, v, s, nullptr) : nullptr;
    Py_XDECREF(v);
    Py_XDECREF(s);
    return both;
}
// Raises what the status stands for.
bool ok(int status) {
    if (status == 0) return true;
    PyObject* r = PyObject_CallFunction(check_fn, "i", status);
    if (r) {
        Py_DECREF(r);
        PyErr_Format(PyExc_RuntimeError, "status %d", status);
    }
    return false;
}
#define OR_NONE(c) \
    if (!(c)) Py_RETURN_NONE

// rms_norm(x, weight, eps, residual, quantize)
PyObject* rms_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    OR_NONE(n == 5 && norm_fn && PyFloat_CheckExact(args[2]) && PyBool_Check(args[4]));
    const bool grad = c10::GradMode::is_enabled(), quantize = args[4] == Py_True, with_residual = args[3] != Py_None;
    int device = -1;
    const at::Tensor *x = plain(args[0], device, grad), *w = x ? plain(args[1], device, grad) : nullptr;
    const at::Tensor* res = w && with_residual ? plain(args[3], device, grad) : nullptr;
    int64_t rows, ldx, ldr = 0, res_rows;
    OR_NONE(w && (res || !with_residual) && device == c10::cuda::current_device());
    const auto type = x->scalar_type();
    const int dt = dtype_code(type);
    OR_NONE(dt >= 0 && w->scalar_type() == type && rows_of(*x, rows, ldx));
    const int64_t D = x->size(-1);
    OR_NONE(w->dim() == 1 && w->size(0) == D && w->is_contiguous());
    at::Tensor sum, y, scales;
    if (res) {
        OR_NONE(res->scalar_type() == type && res->sizes() == x->sizes() && rows_of(*res, res_rows, ldr));
        sum = at::empty(x->sizes(), x->options());
    }
    void* stream = c10::cuda::getCurrentCUDAStream(device).stream();
    const float eps = (float)PyFloat_AS_DOUBLE(args[2]);
    int status;
    if (quantize) {
        int64_t ld;
        empty_fp8(x->sizes(), rows, x->device(), y, ld, scales);
        status = norm_fp8_fn(dt, x->data_ptr(), ldx, res ? res->data_ptr() : nullptr, ldr, w->data_ptr(), eps, res ? sum.data_ptr() : nullptr,
                             D, y.data_ptr(), ld, scales.data_ptr<float>(), 1, rows, rows, (int32_t)D, stream);
    } else {
        y = at::empty(x->sizes(), x->options());
        status = norm_fn(dt, x->data_ptr(), ldx, res ? res->data_ptr() : nullptr, ldr, w->data_ptr(), eps, res ? sum.data_ptr() : nullptr, D,
                         y.data_ptr(), D, rows, (int32_t)D, stream);
    }
    if (!ok(status)) return nullptr;
    PyObject* first = quantize ? blocks_object(y, scales) : THPVariable_Wrap(y);
    if (!first || !res) return first;
    PyObject* second = THPVariable_Wrap(sum);
    PyObject* both = second ? PyTuple_Pack(2, first, second) : nullptr;
    Py_DECREF(first);
    Py_XDECREF(second);
    return both;
    END_HANDLE_TH_ERRORS
}

// quantize_fp8(x, block_rows)
PyObject* quantize_fp8(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    OR_NONE(n == 2 && quantize_fn && PyLong_CheckExact(args[1]));
    const long block_rows = PyLong_AsLong(args[1]);
    if (block_rows == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    int device = -1;
    const at::Tensor* x = plain(args[0], device, c10::GradMode::is_enabled());
    int64_t rows, ldx, ld, row, block;
    OR_NONE(x && device == c10::cuda::current_device() && (block_rows == 1 || (block_rows == BLOCK && x->dim() == 2)));
    const int dt = dtype_code(x->scalar_type());
    OR_NONE(dt >= 0 && rows_of(*x, rows, ldx));
    const int64_t D = x->size(-1);
    at::Tensor values, scales;
    if (block_rows == 1) {
        empty_fp8(x->sizes(), rows, x->device(), values, ld, scales);
        row = 1; block = rows;
    } else {
        ld = (D + 15) / 16 * 16;
        row = (D + BLOCK - 1) / BLOCK; block = 1;
        const auto options = at::TensorOptions().device(x->device());
        values = at::empty_strided({rows, D}, {ld, 1}, options.dtype(at::kFloat8_e4m3fn));
        scales = at::empty({(rows + BLOCK - 1) / BLOCK, row}, options.dtype(at::kFloat));
    }
    if (!ok(quantize_fn(dt, x->data_ptr(), ldx, (int32_t)block_rows, values.data_ptr(), ld, scales.data_ptr<float>(), row, block, rows,
                        (int32_t)D, c10::cuda::getCurrentCUDAStream(device).stream())))
        return nullptr;
    return blocks_object(values, scales);
    END_HANDLE_TH_ERRORS
}

// linear_fp8(a, w, bias, gelu, residual, 0: float32 / 1: bfloat16, quantize)
PyObject* linear_fp8(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    OR_NONE(n == 7 && linear_fn && PyTuple_Check(args[0]) && PyTuple_GET_SIZE(args[0]) == 2 && PyTuple_Check(args[1]) &&
            PyTuple_GET_SIZE(args[1]) == 2 && PyBool_Check(args[3]) && PyLong_CheckExact(args[5]) && PyBool_Check(args[6]));
    const bool grad = c10::GradMode::is_enabled(), gelu = args[3] == Py_True, quantize = args[6] == Py_True;
    const bool with_bias = args[2] != Py_None, with_residual = args[4] != Py_None;
    const int io = (int)PyLong_AsLong(args[5]);
    int device = -1;
    const at::Tensor* a = plain(PyTuple_GET_ITEM(args[0], 0), device, grad);
    const at::Tensor* sa = a ? plain(PyTuple_GET_ITEM(args[0], 1), device, grad) : nullptr;
    const at::Tensor* w = sa ? plain(PyTuple_GET_ITEM(args[1], 0), device, grad) : nullptr;
    const at::Tensor* sw = w ? plain(PyTuple_GET_ITEM(args[1], 1), device, grad) : nullptr;
    OR_NONE(sw && device == c10::cuda::current_device());
    const at::Tensor* bias = with_bias ? plain(args[2], device, grad) : nullptr;
    const at::Tensor* res = with_residual ? plain(args[4], device, grad) : nullptr;
    OR_NONE((bias || !with_bias) && (res || !with_residual));
    const auto type = io == CONVNN_BF16 ? at::kBFloat16 : at::kFloat;
    // (values of more dimensions go through Python, which looks at how their scales are strided)
    OR_NONE((io == CONVNN_F32 || io == CONVNN_BF16) && a->scalar_type() == at::kFloat8_e4m3fn &&
            w->scalar_type() == at::kFloat8_e4m3fn && sa->scalar_type() == at::kFloat && sw->scalar_type() == at::kFloat &&
            a->dim() == 2 && w->dim() == 2 && sa->dim() == 2 && sw->dim() == 2);
    int64_t M, N, lda, ldw, ldr = 0, res_rows;
    OR_NONE(rows_of(*a, M, lda) && rows_of(*w, N, ldw));
    const int64_t K = a->size(1), blocks = (K + BLOCK - 1) / BLOCK;
    OR_NONE(w->size(1) == K && lda % 16 == 0 && ldw % 16 == 0 && N <= (1 << 30) && reinterpret_cast<uintptr_t>(a->data_ptr()) % 16 == 0 &&
            reinterpret_cast<uintptr_t>(w->data_ptr()) % 16 == 0 && sa->size(0) == M && sa->size(1) == blocks &&
            sw->size(0) == (N + BLOCK - 1) / BLOCK && sw->size(1) == blocks);
    if (bias) OR_NONE(bias->scalar_type() == type && bias->dim() == 1 && bias->size(0) == N && bias->is_contiguous());
    if (res)
        OR_NONE(res->scalar_type() == type && res->dim() == 2 && res->size(0) == M && res->size(1) == N && rows_of(*res, res_rows, ldr));
    at::Tensor out, scales;
    int64_t ldo = N;
    const int64_t shape[2] = {M, N};
    if (quantize) empty_fp8(at::IntArrayRef(shape, 2), M, a->device(), out, ldo, scales);
    else out = at::empty(at::IntArrayRef(shape, 2), at::TensorOptions().device(a->device()).dtype(type));
    if (!ok(linear_fn(a->data_ptr(), lda, sa->data_ptr<float>(), sa->stride(0), sa->stride(1), w->data_ptr(), ldw, sw->data_ptr<float>(),
                      sw->stride(0), sw->stride(1), io, bias ? bias->data_ptr() : nullptr, res ? res->data_ptr() : nullptr, ldr,
                      out.data_ptr(), ldo, quantize ? scales.data_ptr<float>() : nullptr, 1, M, M, (int32_t)N, (int32_t)K, gelu,
                      c10::cuda::getCurrentCUDAStream(device).stream())))
        return nullptr;
    return quantize ? blocks_object(out, scales) : THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"bind", FAST(bind)}, {"rms_norm", FAST(rms_norm)}, {"quantize_fp8", FAST(quantize_fp8)},
                         {"linear_fp8", FAST(linear_fp8)}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fp8_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fp8_call() { return PyModule_Create(&module); }
