// Host side of the ordinary calls of the 8-bit operators and of those around a paged cache (Python module _fp8_call): checks the
// tensors, allocates the results and makes the library call.  Where anything is out of the ordinary (a wrong type or shape, other strides, another device than the current
// one, a tensor subclass, no rows) a function returns None, and the Python form in ops.py does the same with the messages.
// rms_norm with a residual and an 8-bit result takes 14 us of host time through Python, linear_fp8 12, qk_norm_rope 20, append_kv 32 and
// tree_attention 30; their kernels for a few rows take less.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>

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

decltype(&convnn_b200_qk_norm_rope) heads_fn = nullptr;
decltype(&convnn_b200_append_kv) append_fn = nullptr;
decltype(&convnn_b200_tree_attention) attention_fn = nullptr;
decltype(&convnn_b200_tree_attention_workspace_bytes) attention_room_fn = nullptr;

PyObject* bind_heads(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 4) {
        PyErr_SetString(PyExc_TypeError, "bind_heads takes four addresses");
        return nullptr;
    }
    void* at[4];
    for (int i = 0; i < 4; ++i) {
        at[i] = PyLong_AsVoidPtr(args[i]);
        if (PyErr_Occurred()) return nullptr;
    }
    heads_fn = reinterpret_cast<decltype(heads_fn)>(at[0]);
    append_fn = reinterpret_cast<decltype(append_fn)>(at[1]);
    attention_fn = reinterpret_cast<decltype(attention_fn)>(at[2]);
    attention_room_fn = reinterpret_cast<decltype(attention_room_fn)>(at[3]);
    Py_RETURN_NONE;
}

// What autograd watches for at this call: gradients that are wanted, tangents (where a level of forward mode is open; there is but one).
struct Watch {
    bool grad, tangents;
};
Watch watching() {
    return {c10::GradMode::is_enabled(),
            c10::AutogradState::get_tls_state().get_fw_grad_mode() && torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr};
}
// A plain tensor on `device` (-1: on any CUDA device, which is then the one); no gradient wanted, and no tangent with it.
const at::Tensor* plain(PyObject* o, int& device, const Watch& watch) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.layout() != at::kStrided || (watch.grad && t.requires_grad()) ||
        (watch.tangents && t._fw_grad(0).defined()))
        return nullptr;
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
    const Watch watch = watching();
    const bool quantize = args[4] == Py_True, with_residual = args[3] != Py_None;
    int device = -1;
    const at::Tensor *x = plain(args[0], device, watch), *w = x ? plain(args[1], device, watch) : nullptr;
    const at::Tensor* res = w && with_residual ? plain(args[3], device, watch) : nullptr;
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
    const at::Tensor* x = plain(args[0], device, watching());
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
    const Watch watch = watching();
    const bool gelu = args[3] == Py_True, quantize = args[6] == Py_True;
    const bool with_bias = args[2] != Py_None, with_residual = args[4] != Py_None;
    const int io = (int)PyLong_AsLong(args[5]);
    int device = -1;
    const at::Tensor* a = plain(PyTuple_GET_ITEM(args[0], 0), device, watch);
    const at::Tensor* sa = a ? plain(PyTuple_GET_ITEM(args[0], 1), device, watch) : nullptr;
    const at::Tensor* w = sa ? plain(PyTuple_GET_ITEM(args[1], 0), device, watch) : nullptr;
    const at::Tensor* sw = w ? plain(PyTuple_GET_ITEM(args[1], 1), device, watch) : nullptr;
    OR_NONE(sw && device == c10::cuda::current_device());
    const at::Tensor* bias = with_bias ? plain(args[2], device, watch) : nullptr;
    const at::Tensor* res = with_residual ? plain(args[4], device, watch) : nullptr;
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

// ---- heads, a paged cache, and attention over it ------------------------------------------------------------------

constexpr int64_t MOST_CHANNELS = 256, MOST_DRAFTED = 64, MOST = 1 << 30;

// Room on the current device, in order of its current stream: as at::empty, of whose 0.9 us the way there is the half.
at::Tensor room_for(at::IntArrayRef shape, at::ScalarType type) {
    return at::detail::empty_generic(shape, c10::cuda::CUDACachingAllocator::get(), c10::DispatchKeySet(c10::DispatchKey::CUDA), type,
                                     std::nullopt);
}
// None, or a plain tensor.
bool maybe(PyObject* o, const at::Tensor*& t, int& device, const Watch& watch) {
    t = o == Py_None ? nullptr : plain(o, device, watch);
    return t || o == Py_None;
}
// (B, T, H, D) or (T, H, D), channels side by side.
bool heads_of(const at::Tensor& t, int64_t B, int64_t T, int64_t D, at::ScalarType type, int32_t& H, int64_t (&stride)[3]) {
    const int64_t dim = t.dim(), f = dim - 3;
    if ((dim != 3 && dim != 4) || t.scalar_type() != type || (f && t.size(0) != B) || (!f && B != 1) || t.size(f) != T || t.size(f + 2) != D ||
        t.size(f + 1) < 1 || t.size(f + 1) > (1 << 20) || (t.stride(f + 2) != 1 && D > 1))
        return false;
    H = (int32_t)t.size(f + 1);
    stride[0] = f ? t.stride(0) : 0;
    stride[1] = t.stride(f);
    stride[2] = t.stride(f + 1);
    return true;
}
bool weight_of(const at::Tensor* w, int64_t D, at::ScalarType type) {
    return !w || (w->scalar_type() == type && w->dim() == 1 && w->size(0) == D && w->is_contiguous());
}
bool rope_of(const at::Tensor* rope, int64_t D, convnn_heads& a) {
    if (!rope) return true;
    if (rope->scalar_type() != at::kFloat || rope->dim() != 2 || rope->size(1) < 2 || rope->size(1) % 2 || rope->size(1) > D ||
        rope->size(0) > MOST || rope->stride(1) != 1 || rope->stride(0) < rope->size(1))
        return false;
    // (a table without rows has no address in torch, and none is no rotation: one that is not followed)
    a.rope = rope->size(0) ? static_cast<const float*>(rope->data_ptr()) : reinterpret_cast<const float*>(16);
    a.rope_stride = rope->stride(0);
    a.rope_rows = (int32_t)rope->size(0);
    a.rotary = (int32_t)rope->size(1);
    return true;
}
bool ints_of(const at::Tensor* t, int64_t n) {
    return !t || (t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == n && (t->stride(0) == 1 || n == 1));
}
bool cache_of(PyObject* o, int& device, const Watch& watch, int64_t B, int64_t H, int64_t D, at::ScalarType type, bool written, convnn_cache& c) {
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 3) return false;
    const at::Tensor* k = plain(PyTuple_GET_ITEM(o, 0), device, watch);
    const at::Tensor* v = k ? plain(PyTuple_GET_ITEM(o, 1), device, watch) : nullptr;
    const at::Tensor* table = v ? plain(PyTuple_GET_ITEM(o, 2), device, watch) : nullptr;
    if (!table || k->scalar_type() != type || v->scalar_type() != type || table->scalar_type() != at::kInt || k->dim() != 4 ||
        v->sizes() != k->sizes() || k->size(1) != H || k->size(3) != D || k->size(0) < 1 || k->size(2) < 1 || k->size(0) > MOST ||
        k->size(2) > MOST || table->dim() != 2 || table->size(0) != B || table->size(1) > MOST || table->size(1) * k->size(2) > MOST ||
        !table->is_contiguous())
        return false;
    // (pages that were strided otherwise may overlap, which Python looks at)
    if (written ? !k->is_contiguous() || !v->is_contiguous() : (k->stride(3) != 1 || v->stride(3) != 1) && D > 1) return false;
    c.k = k->data_ptr();
    c.v = v->data_ptr();
    for (int i = 0; i < 3; ++i) {
        c.k_stride[i] = k->stride(i);
        c.v_stride[i] = v->stride(i);
    }
    c.table = static_cast<const int32_t*>(table->data_ptr());
    c.table_stride = table->size(1);
    c.pages = (int32_t)k->size(0);
    c.page_size = (int32_t)k->size(2);
    c.width = (int32_t)table->size(1);
    return true;
}
bool positions_of(const at::Tensor* t, int64_t B, int64_t T, int64_t dims, convnn_heads& a) {
    if (!t) return true;
    if (t->scalar_type() != at::kInt || t->dim() != dims || t->size(dims - 1) != T || (dims == 2 && t->size(0) != B)) return false;
    a.positions = static_cast<const int32_t*>(t->data_ptr());
    a.position_stride[0] = dims == 2 ? t->stride(0) : 0;
    a.position_stride[1] = t->stride(dims - 1);
    return true;
}
void dense_strides(int64_t (&stride)[3], int64_t T, int64_t H, int64_t D) {
    stride[0] = T * H * D;
    stride[1] = H * D;
    stride[2] = D;
}

// qk_norm_rope(q, k, q_weight, k_weight, rope, positions, eps, interleaved, out)
PyObject* qk_norm_rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    OR_NONE(n == 9 && heads_fn && PyFloat_CheckExact(args[6]) && PyBool_Check(args[7]) && args[8] == Py_None);
    const Watch watch = watching();
    int device = -1;
    const at::Tensor *q = plain(args[0], device, watch), *k, *wq, *wk, *rope, *at_;
    OR_NONE(q && maybe(args[1], k, device, watch) && maybe(args[2], wq, device, watch) && maybe(args[3], wk, device, watch) &&
            maybe(args[4], rope, device, watch) && maybe(args[5], at_, device, watch) && device == c10::cuda::current_device());
    convnn_heads a{};
    const auto type = q->scalar_type();
    const int64_t dim = q->dim();
    OR_NONE((dim == 3 || dim == 4) && dtype_code(type) >= 0);
    const int64_t D = q->size(dim - 1), T = q->size(dim - 3), B = dim == 4 ? q->size(0) : 1;
    OR_NONE(B >= 1 && T >= 1 && B <= MOST && T <= MOST && D >= 1 && D <= MOST_CHANNELS);
    a.dtype = dtype_code(type); a.B = (int32_t)B; a.T = (int32_t)T; a.D = (int32_t)D;
    a.eps = (float)PyFloat_AS_DOUBLE(args[6]);
    a.interleaved = args[7] == Py_True;
    OR_NONE(heads_of(*q, B, T, D, type, a.Hq, a.q_stride) && (!k || (k->dim() == dim && heads_of(*k, B, T, D, type, a.Hk, a.k_stride))) &&
            weight_of(wq, D, type) && weight_of(wk, D, type) && rope_of(rope, D, a) && positions_of(at_, B, T, dim - 2, a));
    a.q = q->data_ptr();
    a.q_weight = wq ? wq->data_ptr() : nullptr;
    a.k_weight = wk ? wk->data_ptr() : nullptr;
    at::Tensor yq = room_for(q->sizes(), type), yk;
    a.q_out = yq.data_ptr();
    dense_strides(a.q_out_stride, T, a.Hq, D);
    if (k) {
        yk = room_for(k->sizes(), type);
        a.k = k->data_ptr();
        a.k_out = yk.data_ptr();
        dense_strides(a.k_out_stride, T, a.Hk, D);
    }
    if (!ok(heads_fn(&a, c10::cuda::getCurrentCUDAStream(device).stream()))) return nullptr;
    PyObject* first = THPVariable_Wrap(yq);
    PyObject* second = first ? (k ? THPVariable_Wrap(yk) : Py_NewRef(Py_None)) : nullptr;
    PyObject* both = second ? PyTuple_Pack(2, first, second) : nullptr;
    Py_XDECREF(first);
    Py_XDECREF(second);
    return both;
    END_HANDLE_TH_ERRORS
}

// append_kv(cache, k, v, lengths, q, q_weight, k_weight, rope, positions, counts, eps, interleaved); False: done, and no queries
PyObject* append_kv(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    OR_NONE(n == 12 && append_fn && PyFloat_CheckExact(args[10]) && PyBool_Check(args[11]));
    const Watch watch = watching();
    int device = -1;
    const at::Tensor *k = plain(args[1], device, watch), *v = k ? plain(args[2], device, watch) : nullptr;
    const at::Tensor *lengths = v ? plain(args[3], device, watch) : nullptr, *q, *wq, *wk, *rope, *at_, *counts;
    OR_NONE(lengths && maybe(args[4], q, device, watch) && maybe(args[5], wq, device, watch) && maybe(args[6], wk, device, watch) &&
            maybe(args[7], rope, device, watch) && maybe(args[8], at_, device, watch) && maybe(args[9], counts, device, watch) &&
            device == c10::cuda::current_device());
    convnn_heads a{};
    convnn_cache c{};
    const auto type = k->scalar_type();
    OR_NONE(k->dim() == 4 && v->dim() == 4 && (!q || q->dim() == 4) && dtype_code(type) >= 0);
    const int64_t D = k->size(3), T = k->size(1), B = k->size(0);
    OR_NONE(B >= 1 && T >= 1 && B <= MOST && T <= MOST && D >= 1 && D <= MOST_CHANNELS);
    a.dtype = dtype_code(type); a.B = (int32_t)B; a.T = (int32_t)T; a.D = (int32_t)D;
    a.eps = (float)PyFloat_AS_DOUBLE(args[10]);
    a.interleaved = args[11] == Py_True;
    int32_t Hv = 0;
    OR_NONE(heads_of(*k, B, T, D, type, a.Hk, a.k_stride) && heads_of(*v, B, T, D, type, Hv, a.v_stride) && Hv == a.Hk &&
            (!q || heads_of(*q, B, T, D, type, a.Hq, a.q_stride)) && weight_of(wq, D, type) && weight_of(wk, D, type) &&
            rope_of(rope, D, a) && positions_of(at_, B, T, 2, a) && ints_of(lengths, B) && ints_of(counts, B) &&
            cache_of(args[0], device, watch, B, a.Hk, D, type, true, c));
    a.k = k->data_ptr();
    a.v = v->data_ptr();
    a.q_weight = wq ? wq->data_ptr() : nullptr;
    a.k_weight = wk ? wk->data_ptr() : nullptr;
    at::Tensor y;
    if (q) {
        y = room_for(q->sizes(), type);
        a.q = q->data_ptr();
        a.q_out = y.data_ptr();
        dense_strides(a.q_out_stride, T, a.Hq, D);
    }
    if (!ok(append_fn(&a, &c, static_cast<const int32_t*>(lengths->data_ptr()),
                      counts ? static_cast<const int32_t*>(counts->data_ptr()) : nullptr, c10::cuda::getCurrentCUDAStream(device).stream())))
        return nullptr;
    // (as in-place operations do, so that autograd notices if it has kept them)
    for (int i = 0; i < 2; ++i) {
        const at::Tensor& pages = THPVariable_Unpack(PyTuple_GET_ITEM(args[0], i));
        if (!pages.is_inference()) pages.unsafeGetTensorImpl()->bump_version();
    }
    if (!q) Py_RETURN_FALSE;
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// tree_attention(q, cache, lengths, tree, counts, scale, out)
PyObject* tree_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    OR_NONE(n == 7 && attention_fn && (args[5] == Py_None || PyFloat_CheckExact(args[5])) && args[6] == Py_None);
    const Watch watch = watching();
    int device = -1;
    const at::Tensor *q = plain(args[0], device, watch), *lengths = q ? plain(args[2], device, watch) : nullptr, *tree, *counts;
    OR_NONE(lengths && maybe(args[3], tree, device, watch) && maybe(args[4], counts, device, watch) && device == c10::cuda::current_device());
    convnn_tree_attention a{};
    convnn_cache c{};
    const auto type = q->scalar_type();
    const int dt = dtype_code(type);
    OR_NONE(q->dim() == 4 && dt >= 0 && PyTuple_Check(args[1]) && PyTuple_GET_SIZE(args[1]) == 3);
    const at::Tensor* pages = plain(PyTuple_GET_ITEM(args[1], 0), device, watch);
    OR_NONE(pages && pages->dim() == 4);
    const int64_t B = q->size(0), T = q->size(1), D = q->size(3), H = pages->size(1), unit = dt == CONVNN_F32 ? 4 : 8;
    OR_NONE(B >= 1 && T >= 1 && T <= MOST_DRAFTED && B <= MOST / T && D >= 1 && D <= MOST_CHANNELS && D % unit == 0 && H >= 1 && H <= (1 << 20));
    a.dtype = dt; a.B = (int32_t)B; a.T = (int32_t)T; a.D = (int32_t)D; a.Hk = (int32_t)H;
    OR_NONE(heads_of(*q, B, T, D, type, a.Hq, a.q_stride) && a.Hq % H == 0 && ints_of(lengths, B) && ints_of(counts, B) &&
            cache_of(args[1], device, watch, B, H, D, type, false, c));
    if (tree) {
        OR_NONE(tree->scalar_type() == at::kLong && tree->dim() == 2 && tree->size(0) == B && tree->size(1) == T);
        a.tree = static_cast<const int64_t*>(tree->data_ptr());
        a.tree_stride[0] = tree->stride(0);
        a.tree_stride[1] = tree->stride(1);
    }
    bool rows = (reinterpret_cast<uintptr_t>(q->data_ptr()) | reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v)) % 16 == 0;
    for (int i = 0; i < 3; ++i) rows = rows && a.q_stride[i] % unit == 0 && c.k_stride[i] % unit == 0 && c.v_stride[i] % unit == 0;
    OR_NONE(rows);
    a.scale = args[5] == Py_None ? (float)std::pow((double)D, -0.5) : (float)PyFloat_AS_DOUBLE(args[5]);
    a.q = q->data_ptr();
    a.lengths = static_cast<const int32_t*>(lengths->data_ptr());
    a.counts = counts ? static_cast<const int32_t*>(counts->data_ptr()) : nullptr;
    at::Tensor out = room_for(q->sizes(), type);
    a.out = out.data_ptr();
    dense_strides(a.out_stride, T, a.Hq, D);
    const size_t need = attention_room_fn(dt, a.T, a.Hq, a.Hk, a.D);
    const c10::DataPtr room = c10::cuda::CUDACachingAllocator::get()->allocate(need);
    if (!ok(attention_fn(&a, &c, room.get(), need, c10::cuda::getCurrentCUDAStream(device).stream()))) return nullptr;
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"bind", FAST(bind)}, {"rms_norm", FAST(rms_norm)}, {"quantize_fp8", FAST(quantize_fp8)},
                         {"linear_fp8", FAST(linear_fp8)}, {"bind_heads", FAST(bind_heads)}, {"qk_norm_rope", FAST(qk_norm_rope)},
                         {"append_kv", FAST(append_kv)}, {"tree_attention", FAST(tree_attention)}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fp8_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fp8_call() { return PyModule_Create(&module); }
