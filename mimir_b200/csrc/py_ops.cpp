// The operators of mimir_b200/tensor.py for the calls that programs are made of: contiguous CUDA tensors of the right shapes and
// element types. A call is taken from the Python arguments to the C ABI here, about 3 us of host time instead of 9 through ctypes.
//
// Every function returns the result, or None for any call it is not made for (another type or subclass, layout, device or shape, a dispatch mode
// or a transform that is active, a status that is not OK): the caller then takes the general path, which makes copies and raises errors.
// tensor.py alone says what an operator means; nothing is accepted here that it would refuse.
#include <Python.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "mimk.h"

namespace {

using at::Tensor;

// No transform or mode wants to see the operations (functorch, tracing, fake tensors ...), nor __torch_function__. Inference mode,
// which takes one key from the default set, does not: what is allocated in it becomes an inference tensor by itself.
bool nothing_watches() {
    const auto tls = c10::impl::tls_local_dispatch_key_set();
    return tls.included_.add(c10::DispatchKey::ADInplaceOrView) == c10::default_included_set && !c10::impl::TorchDispatchModeTLS::any_modes_set() && !at::impl::torch_function_mode_enabled();
}

int dtype_of(at::ScalarType t) { return t == at::kFloat ? MIMK_F32 : t == at::kBFloat16 ? MIMK_BF16 : -1; }

PyTypeObject* parameter_type;  // torch.nn.Parameter, for the life of the module

// A torch.Tensor or torch.nn.Parameter proper, dense and row-major on a CUDA device, of F32 or BF16 elements; null if not.
const Tensor* dense(PyObject* o, bool any_strides = false) {
    if (Py_TYPE(o) != reinterpret_cast<PyTypeObject*>(THPVariableClass) && Py_TYPE(o) != parameter_type) return nullptr;
    const Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.has_storage() || t.is_neg() || dtype_of(t.scalar_type()) < 0) return nullptr;
    if (t.key_set().has_any(c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                                                 c10::DispatchKey::Functionalize, c10::DispatchKey::ZeroTensor})))
        return nullptr;
    if (t.numel() == 0 || (!any_strides && !t.is_contiguous())) return nullptr;
    return &t;
}

bool is_int(PyObject* o, int64_t& v) {
    if (!PyLong_CheckExact(o)) return false;
    v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}
// None: `plain`; a dtype of F32 or BF16: that one
bool out_type(PyObject* o, at::ScalarType plain, at::ScalarType& t) {
    if (o == Py_None) {
        t = plain;
        return true;
    }
    if (!THPDtype_Check(o)) return false;
    t = reinterpret_cast<THPDtype*>(o)->scalar_type;
    return dtype_of(t) >= 0;
}

Tensor empty(at::IntArrayRef shape, at::ScalarType t, const Tensor& like) { return at::detail::empty_cuda(shape, t, like.device(), std::nullopt); }
// The call into the library, f(stream), without the interpreter's lock: it may wait, for the device where a cached buffer grows, or for room
// in a launch queue, and what it waits for may be another Python thread's to issue.
template <class F>
int unlocked(F&& f) {
    void* stream         = c10::cuda::getCurrentCUDAStream().stream();
    PyThreadState* state = PyEval_SaveThread();
    const int status     = f(stream);
    PyEval_RestoreThread(state);
    return status;
}
PyObject* result(int status, Tensor&& out) {
    if (status != MIMK_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
}

// B of a product, [..., k, n]: row-major, or a transposed view of a row-major [..., n, k].
int b_layout(const Tensor& b) {
    if (b.is_contiguous()) return MIMK_B_KN;
    const int64_t r = b.dim(), k = b.size(r - 2), n = b.size(r - 1);
    if ((k != 1 && b.stride(r - 2) != 1) || (n != 1 && b.stride(r - 1) != k)) return -1;
    if (r == 3 && b.size(0) != 1 && b.stride(0) != k * n) return -1;
    return MIMK_B_NK;
}

struct View3 {  // the axes before, at and behind `ax`
    int64_t outer = 1, len = 1, inner = 1;
    int64_t ax;
    View3(const Tensor& x, int64_t axis) : ax(axis < 0 ? axis + x.dim() : axis) {
        for (int64_t i = 0; i < x.dim(); ++i) (i < ax ? outer : i == ax ? len : inner) *= x.size(i);
    }
    bool good(const Tensor& x) const { return ax >= 0 && ax < x.dim(); }
};
std::vector<int64_t> without(const Tensor& x, int64_t ax) {
    std::vector<int64_t> s(x.sizes().begin(), x.sizes().end());
    s.erase(s.begin() + ax);
    return s;
}

#define OP(NAME, N)                                                                   \
    PyObject* NAME(PyObject*, PyObject* const* a, Py_ssize_t n) {                     \
        HANDLE_TH_ERRORS                                                              \
        if (n != N || !nothing_watches()) Py_RETURN_NONE;
#define END_OP          \
    Py_RETURN_NONE;     \
    END_HANDLE_TH_ERRORS \
    }

// a, b, post id, bias, out dtype
OP(product_2d, 5)
    const Tensor *x = dense(a[0]), *w = dense(a[1], true), *bias = a[3] == Py_None ? nullptr : dense(a[3]);
    int64_t post;
    at::ScalarType t;
    if (!x || !w || (!bias && a[3] != Py_None) || !is_int(a[2], post) || x->dim() != 2 || w->dim() != 2 || x->scalar_type() != w->scalar_type()) Py_RETURN_NONE;
    const int64_t m = x->size(0), k = x->size(1), cols = w->size(1);
    const int layout = b_layout(*w);
    if (k != w->size(0) || layout < 0 || !out_type(a[4], x->scalar_type(), t)) Py_RETURN_NONE;
    if (bias && (bias->scalar_type() != at::kFloat || bias->numel() != cols)) Py_RETURN_NONE;
    Tensor out = empty({m, cols}, t, *x);
    mimk_gemm_desc d = {};
    d.batch = 1, d.m = m, d.n = cols, d.k = k, d.stride_c = m * cols;
    d.a = x->data_ptr(), d.b = w->data_ptr(), d.c = out.data_ptr();
    d.in_dtype = dtype_of(x->scalar_type()), d.out_dtype = dtype_of(t), d.b_layout = layout, d.post = int(post);
    d.post_row = bias ? bias->data_ptr() : nullptr;
    return result(unlocked([&](void* stream) { return mimk_gemm(&d, stream); }), std::move(out));
END_OP

// a, b, out dtype
OP(bmm, 3)
    const Tensor *x = dense(a[0]), *w = dense(a[1], true);
    at::ScalarType t;
    if (!x || !w || x->dim() != 3 || w->dim() != 3 || x->scalar_type() != w->scalar_type()) Py_RETURN_NONE;
    const int64_t batch = x->size(0), m = x->size(1), k = x->size(2), cols = w->size(2);
    const int layout = b_layout(*w);
    if (batch != w->size(0) || k != w->size(1) || layout < 0 || !out_type(a[2], x->scalar_type(), t)) Py_RETURN_NONE;
    Tensor out = empty({batch, m, cols}, t, *x);
    mimk_gemm_desc d = {};
    d.batch = batch, d.m = m, d.n = cols, d.k = k, d.stride_a = m * k, d.stride_b = k * cols, d.stride_c = m * cols;
    d.a = x->data_ptr(), d.b = w->data_ptr(), d.c = out.data_ptr();
    d.in_dtype = dtype_of(x->scalar_type()), d.out_dtype = dtype_of(t), d.b_layout = layout, d.post = MIMK_POST_ID;
    return result(unlocked([&](void* stream) { return mimk_gemm(&d, stream); }), std::move(out));
END_OP

// monoid id, axis, x
OP(reduce, 3)
    const Tensor* x = dense(a[2]);
    int64_t monoid, ax;
    if (!x || !is_int(a[0], monoid) || !is_int(a[1], ax)) Py_RETURN_NONE;
    const View3 v(*x, ax);
    if (!v.good(*x)) Py_RETURN_NONE;
    Tensor out = empty(without(*x, v.ax), x->scalar_type(), *x);
    return result(unlocked([&](void* stream) { return mimk_reduce(x->data_ptr(), out.data_ptr(), dtype_of(x->scalar_type()), v.outer, v.len, v.inner, int(monoid), stream); }), std::move(out));
END_OP

// monoid id, axis, x, unary inner id, unary outer id
OP(reduce_of_unary, 5)
    const Tensor* x = dense(a[2]);
    int64_t monoid, ax, inner, outer;
    if (!x || !is_int(a[0], monoid) || !is_int(a[1], ax) || !is_int(a[3], inner) || !is_int(a[4], outer)) Py_RETURN_NONE;
    const View3 v(*x, ax);
    if (!v.good(*x)) Py_RETURN_NONE;
    mimk_producer pre = {};
    pre.inner_op = int32_t(inner), pre.outer_op = int32_t(outer), pre.y_mode = 3;
    Tensor out = empty(without(*x, v.ax), x->scalar_type(), *x);
    return result(unlocked([&](void* stream) { return mimk_reduce_fused(x->data_ptr(), &pre, out.data_ptr(), dtype_of(x->scalar_type()), v.outer, v.len, v.inner, int(monoid), stream); }),
                  std::move(out));
END_OP

// axis, x, out dtype
OP(softmax, 3)
    const Tensor* x = dense(a[1]);
    int64_t ax;
    at::ScalarType t;
    if (!x || !is_int(a[0], ax) || !out_type(a[2], x->scalar_type(), t)) Py_RETURN_NONE;
    const View3 v(*x, ax);
    if (!v.good(*x)) Py_RETURN_NONE;
    Tensor out = empty(x->sizes(), t, *x);
    return result(unlocked([&](void* stream) { return mimk_softmax(x->data_ptr(), out.data_ptr(), dtype_of(x->scalar_type()), dtype_of(t), v.outer, v.len, v.inner, stream); }), std::move(out));
END_OP

// x, gamma, eps, out dtype
OP(rmsnorm, 4)
    const Tensor *x = dense(a[0]), *gamma = dense(a[1]);
    at::ScalarType t;
    if (!x || !gamma || x->dim() < 1 || gamma->scalar_type() != at::kFloat || !PyFloat_CheckExact(a[2]) || !out_type(a[3], x->scalar_type(), t)) Py_RETURN_NONE;
    const int64_t cols = x->size(x->dim() - 1);
    if (gamma->numel() != cols) Py_RETURN_NONE;
    Tensor out = empty(x->sizes(), t, *x);
    return result(unlocked([&](void* stream) { return mimk_rmsnorm(x->data_ptr(), gamma->data_ptr(), out.data_ptr(), dtype_of(x->scalar_type()), dtype_of(t), x->numel() / cols, cols,
                               float(PyFloat_AS_DOUBLE(a[2])), stream); }),
                  std::move(out));
END_OP

// op id, x, out dtype
OP(unary, 3)
    const Tensor* x = dense(a[1]);
    int64_t op;
    at::ScalarType t;
    if (!x || !is_int(a[0], op) || !out_type(a[2], x->scalar_type(), t)) Py_RETURN_NONE;
    Tensor out = empty(x->sizes(), t, *x);
    return result(unlocked([&](void* stream) { return mimk_map_t(int(op), x->data_ptr(), nullptr, out.data_ptr(), dtype_of(x->scalar_type()), dtype_of(t), 1, x->numel(), 1, 3, stream); }),
                  std::move(out));
END_OP

// op id, x, y, out dtype
OP(binary, 4)
    const Tensor *x = dense(a[1]), *y = dense(a[2]);
    int64_t op;
    at::ScalarType t;
    if (!x || !y || !is_int(a[0], op) || x->scalar_type() != y->scalar_type() || x->sizes() != y->sizes() || !out_type(a[3], x->scalar_type(), t)) Py_RETURN_NONE;
    Tensor out = empty(x->sizes(), t, *x);
    return result(unlocked([&](void* stream) { return mimk_map_t(int(op), x->data_ptr(), y->data_ptr(), out.data_ptr(), dtype_of(x->scalar_type()), dtype_of(t), 1, x->numel(), 1, 0, stream); }),
                  std::move(out));
END_OP

// op id, axis, x, y, out dtype
OP(binary_ax, 5)
    const Tensor *x = dense(a[2]), *y = dense(a[3]);
    int64_t op, ax;
    at::ScalarType t;
    if (!x || !y || !is_int(a[0], op) || !is_int(a[1], ax) || x->scalar_type() != y->scalar_type() || !out_type(a[4], x->scalar_type(), t)) Py_RETURN_NONE;
    const View3 v(*x, ax);
    if (!v.good(*x) || y->sizes() != at::IntArrayRef(without(*x, v.ax))) Py_RETURN_NONE;
    Tensor out = empty(x->sizes(), t, *x);
    return result(unlocked([&](void* stream) { return mimk_map_t(int(op), x->data_ptr(), y->data_ptr(), out.data_ptr(), dtype_of(x->scalar_type()), dtype_of(t), v.outer, v.len, v.inner, 1, stream); }),
                  std::move(out));
END_OP

// q, k, v, scale, causal
OP(attention, 5)
    const Tensor *q = dense(a[0]), *k = dense(a[1]), *v = dense(a[2]);
    if (!q || !k || !v || !PyFloat_CheckExact(a[3]) || !PyBool_Check(a[4])) Py_RETURN_NONE;
    const int64_t r = q->dim();
    if (r < 2 || k->dim() != r || k->sizes() != v->sizes() || q->size(r - 1) != k->size(r - 1)) Py_RETURN_NONE;
    if (q->scalar_type() != k->scalar_type() || q->scalar_type() != v->scalar_type()) Py_RETURN_NONE;
    mimk_attn_desc d = {};
    d.batch_heads = 1;
    for (int64_t i = 0; i < r - 2; ++i) {
        if (q->size(i) != k->size(i)) Py_RETURN_NONE;
        d.batch_heads *= q->size(i);
    }
    Tensor out = empty(q->sizes(), q->scalar_type(), *q);
    d.seq_q = q->size(r - 2), d.seq_k = k->size(r - 2), d.head_dim = q->size(r - 1);
    d.q = q->data_ptr(), d.k = k->data_ptr(), d.v = v->data_ptr(), d.o = out.data_ptr();
    d.scale = float(PyFloat_AS_DOUBLE(a[3])), d.causal = a[4] == Py_True, d.dtype = dtype_of(q->scalar_type());
    return result(unlocked([&](void* stream) { return mimk_attn_fwd(&d, stream); }), std::move(out));
END_OP

// x, w1, w3, w2
OP(mlp_gated, 4)
    const Tensor *x = dense(a[0]), *w1 = dense(a[1], true), *w3 = dense(a[2], true), *w2 = dense(a[3], true);
    if (!x || !w1 || !w3 || !w2 || x->dim() != 2 || w1->dim() != 2 || w2->dim() != 2 || w1->sizes() != w3->sizes()) Py_RETURN_NONE;
    const at::ScalarType t = x->scalar_type();
    if (w1->scalar_type() != t || w3->scalar_type() != t || w2->scalar_type() != t) Py_RETURN_NONE;
    const int layout = b_layout(*w1);
    if (layout < 0 || b_layout(*w3) != layout || b_layout(*w2) != layout || x->size(1) != w1->size(0) || w1->size(1) != w2->size(0)) Py_RETURN_NONE;
    mimk_mlp_desc d = {};
    d.m = x->size(0), d.k = x->size(1), d.f = w1->size(1), d.n = w2->size(1);
    Tensor out = empty({d.m, d.n}, t, *x);
    d.x = x->data_ptr(), d.w1 = w1->data_ptr(), d.w3 = w3->data_ptr(), d.w2 = w2->data_ptr(), d.y = out.data_ptr();
    d.dtype = dtype_of(t), d.b_layout = layout;
    return result(unlocked([&](void* stream) { return mimk_mlp_gated(&d, stream); }), std::move(out));
END_OP

// Results as a tuple, or None for a status that is not OK.
PyObject* results(int status, std::vector<Tensor>&& out) {
    if (status != MIMK_OK) Py_RETURN_NONE;
    PyObject* all = PyTuple_New(Py_ssize_t(out.size()));
    if (!all) return nullptr;
    for (size_t i = 0; i < out.size(); ++i) {
        PyObject* o = THPVariable_Wrap(std::move(out[i]));
        if (!o) {
            Py_DECREF(all);
            return nullptr;
        }
        PyTuple_SET_ITEM(all, Py_ssize_t(i), o);
    }
    return all;
}
// A gradient of w's shape, in w's storage layout.
Tensor like_weight(const Tensor& w, int layout) {
    return layout == MIMK_B_KN ? empty({w.size(0), w.size(1)}, w.scalar_type(), w) : empty({w.size(1), w.size(0)}, w.scalar_type(), w).t();
}
bool mlp_train_desc(PyObject* const* a, mimk_mlp_train_desc& d, const Tensor* (&t)[4]) {
    t[0] = dense(a[0]);
    for (int i = 1; i < 4; ++i) t[i] = dense(a[i], true);
    for (const Tensor* x : t)
        if (!x || x->dim() != 2 || x->scalar_type() != t[0]->scalar_type()) return false;
    const int layout = b_layout(*t[1]);
    if (layout < 0 || b_layout(*t[2]) != layout || b_layout(*t[3]) != layout) return false;
    if (t[1]->sizes() != t[2]->sizes() || t[0]->size(1) != t[1]->size(0) || t[1]->size(1) != t[3]->size(0)) return false;
    d = {};
    d.m = t[0]->size(0), d.k = t[0]->size(1), d.f = t[1]->size(1), d.n = t[3]->size(1);
    d.x = t[0]->data_ptr(), d.w1 = t[1]->data_ptr(), d.w3 = t[2]->data_ptr(), d.w2 = t[3]->data_ptr();
    d.dtype = dtype_of(t[0]->scalar_type()), d.b_layout = layout;
    return true;
}

// x, w1, w3, w2 -> y, kept
OP(mlp_gated_fwd, 4)
    mimk_mlp_train_desc d;
    const Tensor* t[4];
    if (!mlp_train_desc(a, d, t)) Py_RETURN_NONE;
    Tensor y = empty({d.m, d.n}, t[0]->scalar_type(), *t[0]);
    d.y = y.data_ptr();
    uint64_t kept = 0;
    if (mimk_mlp_gated_train_sizes(&d, &kept, &d.workspace_bytes, nullptr) != MIMK_OK) Py_RETURN_NONE;
    Tensor buffer = empty({int64_t(kept)}, at::kByte, y), scratch = empty({int64_t(d.workspace_bytes)}, at::kByte, y);
    d.kept = buffer.data_ptr(), d.workspace = scratch.data_ptr();
    const int status = unlocked([&](void* stream) { return mimk_mlp_gated_fwd(&d, stream); });
    return results(status, {std::move(y), std::move(buffer)});
END_OP

// x, w1, w3, w2, dy, the kept buffer, the extents it is for -> dx, dw1, dw3, dw2
OP(mlp_gated_bwd, 7)
    mimk_mlp_train_desc d;
    const Tensor *t[4], *dy = dense(a[4]);
    if (!mlp_train_desc(a, d, t) || !dy || dy->dim() != 2 || dy->size(0) != d.m || dy->size(1) != d.n || dy->scalar_type() != t[0]->scalar_type()) Py_RETURN_NONE;
    if (!THPVariable_Check(a[5]) || !PyTuple_CheckExact(a[6]) || PyTuple_GET_SIZE(a[6]) != 4) Py_RETURN_NONE;
    const int64_t extents[4] = {d.m, d.k, d.f, d.n};
    for (int i = 0; i < 4; ++i) {
        int64_t e;
        if (!is_int(PyTuple_GET_ITEM(a[6], i), e) || e != extents[i]) Py_RETURN_NONE;
    }
    std::vector<Tensor> out = {empty({d.m, d.k}, t[0]->scalar_type(), *t[0])};
    for (int i = 1; i < 4; ++i) out.push_back(like_weight(*t[i], d.b_layout));
    d.dy = dy->data_ptr(), d.kept = THPVariable_Unpack(a[5]).data_ptr();
    d.dx = out[0].data_ptr(), d.dw1 = out[1].data_ptr(), d.dw3 = out[2].data_ptr(), d.dw2 = out[3].data_ptr();
    if (mimk_mlp_gated_train_sizes(&d, nullptr, nullptr, &d.workspace_bytes) != MIMK_OK) Py_RETURN_NONE;
    Tensor scratch = empty({int64_t(d.workspace_bytes)}, at::kByte, *dy);
    d.workspace    = scratch.data_ptr();
    const int status = unlocked([&](void* stream) { return mimk_mlp_gated_bwd(&d, stream); });
    return results(status, std::move(out));
END_OP

// x, w, targets, ignored index or None, reduction id, dloss or None, lse or None, forward, backward, lse wanted -> what of loss, lse, dx, dw is asked for
OP(linear_ce, 10)
    const Tensor *x = dense(a[0]), *w = dense(a[1], true), *dloss = a[5] == Py_None ? nullptr : dense(a[5]), *lse = a[6] == Py_None ? nullptr : dense(a[6]);
    if (!x || !w || (!dloss && a[5] != Py_None) || (!lse && a[6] != Py_None) || !THPVariable_CheckExact(a[2])) Py_RETURN_NONE;
    const Tensor& t = THPVariable_Unpack(a[2]);
    int64_t reduction, ignore = 0;
    if (!is_int(a[4], reduction) || (a[3] != Py_None && !is_int(a[3], ignore)) || !PyBool_Check(a[7]) || !PyBool_Check(a[8]) || !PyBool_Check(a[9])) Py_RETURN_NONE;
    const bool forward = a[7] == Py_True, backward = a[8] == Py_True, want_lse = a[9] == Py_True;
    const int64_t r = x->dim();
    const int layout = w->dim() == 2 ? b_layout(*w) : -1;
    if (r < 1 || layout < 0 || x->size(r - 1) != w->size(0) || x->scalar_type() != w->scalar_type()) Py_RETURN_NONE;
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.is_contiguous() || (t.scalar_type() != at::kLong && t.scalar_type() != at::kInt)) Py_RETURN_NONE;
    const at::IntArrayRef lead = x->sizes().slice(0, size_t(r - 1)), each = reduction == MIMK_REDUCTION_NONE ? lead : at::IntArrayRef();
    if (t.sizes() != lead) Py_RETURN_NONE;
    if (dloss && (dloss->scalar_type() != at::kFloat || dloss->sizes() != each)) Py_RETURN_NONE;
    if (forward == (lse != nullptr) || (lse && (lse->scalar_type() != at::kFloat || lse->sizes() != lead))) Py_RETURN_NONE;
    mimk_linear_ce_desc d = {};
    d.d = w->size(0), d.v = w->size(1), d.n = x->numel() / d.d;
    d.x = x->data_ptr(), d.w = w->data_ptr(), d.targets = t.data_ptr();
    d.dloss = dloss ? static_cast<const float*>(dloss->data_ptr()) : nullptr, d.lse = lse ? static_cast<float*>(lse->data_ptr()) : nullptr;
    d.ignore_index = ignore, d.has_ignore = a[3] != Py_None, d.reduction = int(reduction);
    d.dtype = dtype_of(x->scalar_type()), d.target_dtype = t.scalar_type() == at::kLong ? MIMK_I64 : MIMK_I32, d.w_layout = layout;
    std::vector<Tensor> out;
    if (forward) {
        out.push_back(empty(each, at::kFloat, *x));
        d.loss = static_cast<float*>(out.back().data_ptr());
        if (want_lse) out.push_back(empty(lead, at::kFloat, *x)), d.lse = static_cast<float*>(out.back().data_ptr());
    }
    if (backward) {
        out.push_back(empty(x->sizes(), x->scalar_type(), *x)), d.dx = out.back().data_ptr();
        out.push_back(like_weight(*w, layout)), d.dw = out.back().data_ptr();
    }
    if (mimk_linear_ce_workspace(&d, forward, backward, &d.workspace_bytes) != MIMK_OK) Py_RETURN_NONE;
    Tensor scratch = empty({int64_t(d.workspace_bytes)}, at::kByte, *x);
    d.workspace    = scratch.data_ptr();
    const int status = unlocked([&](void* stream) { return forward ? (backward ? mimk_linear_ce_fwd_bwd(&d, stream) : mimk_linear_ce_fwd(&d, stream)) : mimk_linear_ce_bwd(&d, stream); });
    return results(status, std::move(out));
END_OP

// a list of gradients, a list of results or None, limit or None (the norm alone), eps -> norm
OP(clip_grads, 4)
    if (!PyList_CheckExact(a[0]) || (a[1] != Py_None && !PyList_CheckExact(a[1]))) Py_RETURN_NONE;
    const Py_ssize_t count = PyList_GET_SIZE(a[0]);
    const bool clip = a[2] != Py_None;
    if (!count || (a[1] != Py_None && PyList_GET_SIZE(a[1]) != count) || (clip && (!PyFloat_CheckExact(a[2]) || !PyFloat_CheckExact(a[3])))) Py_RETURN_NONE;
    std::vector<const void*> in(count);
    std::vector<void*> out(count);
    std::vector<const Tensor*> written(count);
    std::vector<int64_t> lengths(count);
    std::vector<int32_t> dtypes(count);
    const Tensor* first = nullptr;
    for (Py_ssize_t i = 0; i < count; ++i) {
        const Tensor *t = dense(PyList_GET_ITEM(a[0], i), true), *o = a[1] == Py_None ? t : dense(PyList_GET_ITEM(a[1], i), true);
        if (!t || !o || !t->is_non_overlapping_and_dense()) Py_RETURN_NONE;
        if (o != t && (o->scalar_type() != t->scalar_type() || o->sizes() != t->sizes() || o->strides() != t->strides())) Py_RETURN_NONE;
        first = first ? first : t;
        if (t->device() != first->device() || o->device() != first->device()) Py_RETURN_NONE;
        in[i] = t->data_ptr(), out[i] = o->data_ptr(), lengths[i] = t->numel(), dtypes[i] = dtype_of(t->scalar_type()), written[i] = o;
    }
    uint64_t bytes = 0;
    if (mimk_clip_grads_workspace(count, &bytes) != MIMK_OK) Py_RETURN_NONE;
    Tensor norm = empty({}, at::kFloat, *first), scratch = empty({int64_t(bytes)}, at::kByte, *first);
    float* to = static_cast<float*>(norm.data_ptr());
    void* ws  = scratch.data_ptr();
    const int status = unlocked([&](void* stream) {
        return clip ? mimk_clip_grads(in.data(), out.data(), lengths.data(), dtypes.data(), count, float(PyFloat_AS_DOUBLE(a[2])), float(PyFloat_AS_DOUBLE(a[3])), to, ws, bytes, stream)
                    : mimk_grad_norm(in.data(), lengths.data(), dtypes.data(), count, to, ws, bytes, stream);
    });
    // a tensor that autograd has saved was changed: its version says so (an inference tensor has none)
    if (clip && status == MIMK_OK)
        for (const Tensor* o : written)
            if (!o->is_inference()) o->unsafeGetTensorImpl()->bump_version();
    return result(status, std::move(norm));
END_OP

// On the device that is current, whose stream the call is made on.
bool here(const Tensor* t) { return t && t->device().index() == c10::cuda::current_device(); }
// A dense I32 or I64 tensor on the current device, or null.
const Tensor* index_tensor(PyObject* o) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.is_contiguous() || t.numel() == 0 || (t.scalar_type() != at::kLong && t.scalar_type() != at::kInt)) return nullptr;
    return here(&t) ? &t : nullptr;
}
bool embedding_desc(mimk_embedding_desc& d, const Tensor& rows, const Tensor& ids, PyObject* scale, PyObject* ignore) {
    d = {};
    if (!PyFloat_CheckExact(scale) || (ignore != Py_None && !is_int(ignore, d.ignore_index))) return false;
    d.n = ids.numel(), d.ids = ids.data_ptr(), d.scale = float(PyFloat_AS_DOUBLE(scale)), d.has_ignore = ignore != Py_None;
    d.dtype = dtype_of(rows.scalar_type()), d.id_dtype = ids.scalar_type() == at::kLong ? MIMK_I64 : MIMK_I32;
    return true;
}

// table, ids, scale, ignored index or None, out dtype
OP(embedding, 5)
    const Tensor *table = dense(a[0]), *ids = index_tensor(a[1]);
    mimk_embedding_desc d;
    at::ScalarType t;
    if (!here(table) || !ids || table->dim() != 2 || !embedding_desc(d, *table, *ids, a[2], a[3]) || !out_type(a[4], table->scalar_type(), t)) Py_RETURN_NONE;
    std::vector<int64_t> shape(ids->sizes().begin(), ids->sizes().end());
    shape.push_back(table->size(1));
    Tensor out = empty(shape, t, *table);
    d.v = table->size(0), d.d = table->size(1), d.table = table->data_ptr(), d.out = out.data_ptr(), d.out_dtype = dtype_of(t);
    return result(unlocked([&](void* stream) { return mimk_embedding(&d, stream); }), std::move(out));
END_OP

// dy, ids, classes, scale, ignored index or None, out dtype
OP(embedding_grad, 6)
    const Tensor *dy = dense(a[0]), *ids = index_tensor(a[1]);
    mimk_embedding_desc d;
    at::ScalarType t;
    int64_t classes;
    if (!here(dy) || !ids || dy->dim() < 1 || !is_int(a[2], classes) || classes < 1 || !embedding_desc(d, *dy, *ids, a[3], a[4]) || !out_type(a[5], dy->scalar_type(), t)) Py_RETURN_NONE;
    if (dy->sizes().slice(0, size_t(dy->dim() - 1)) != ids->sizes()) Py_RETURN_NONE;
    d.v = classes, d.d = dy->size(dy->dim() - 1), d.dy = dy->data_ptr(), d.out_dtype = dtype_of(t);
    if (mimk_embedding_grad_workspace(&d, &d.workspace_bytes) != MIMK_OK) Py_RETURN_NONE;
    Tensor out = empty({classes, d.d}, t, *dy), scratch = empty({int64_t(d.workspace_bytes)}, at::kByte, *dy);
    d.dtable = out.data_ptr(), d.workspace = scratch.data_ptr();
    return result(unlocked([&](void* stream) { return mimk_embedding_grad(&d, stream); }), std::move(out));
END_OP

// The operands of residual_rmsnorm, r, h, gamma, post_gamma and gate, of which all but r may be None.
bool residual_desc(mimk_residual_rmsnorm_desc& d, PyObject* const (&o)[5], const Tensor* (&t)[5]) {
    d = {};
    for (int i = 0; i < 5; ++i) {
        t[i] = o[i] == Py_None ? nullptr : dense(o[i]);
        if ((!t[i] && (o[i] != Py_None || i == 0)) || (t[i] && !here(t[i]))) return false;
    }
    const Tensor &r = *t[0], *h = t[1], *gate = t[4];
    if (r.dim() < 1 || (h && h->sizes() != r.sizes())) return false;
    const int64_t features = r.size(r.dim() - 1);
    for (const Tensor* g : {t[2], t[3]})
        if (g && (g->dim() != 1 || g->size(0) != features)) return false;
    d.n = r.numel() / features, d.d = features, d.gate_rows = 1;
    d.r = r.data_ptr(), d.stream_dtype = d.block_dtype = dtype_of(r.scalar_type());
    if (h) d.h = h->data_ptr(), d.block_dtype = dtype_of(h->scalar_type());
    if (t[2]) d.gamma = t[2]->data_ptr(), d.gamma_dtype = dtype_of(t[2]->scalar_type());
    if (t[3]) d.post_gamma = t[3]->data_ptr(), d.post_gamma_dtype = dtype_of(t[3]->scalar_type());
    if (gate) {
        // the operands' leading axes up to one of them, and ones
        const int64_t lead = r.dim() - 1, own = gate->dim() - 1, missing = lead - own;
        if (own < 0 || missing < 0 || gate->size(own) != features) return false;
        int64_t same = 0;
        while (same < lead && (same < missing ? 1 : gate->size(same - missing)) == r.size(same)) ++same;
        for (int64_t i = same; i < lead; ++i) {
            if (i >= missing && gate->size(i - missing) != 1) return false;
            d.gate_rows *= r.size(i);
        }
        d.gate = gate->data_ptr(), d.gate_dtype = dtype_of(gate->scalar_type());
    }
    return true;
}

// r, h, gamma, post_gamma, gate, eps, residual scale, branch scale, whether bwd follows -> r' (None without h), x (None without gamma), kept
OP(residual_rmsnorm, 9)
    mimk_residual_rmsnorm_desc d;
    const Tensor* t[5];
    PyObject* const o[5] = {a[0], a[1], a[2], a[3], a[4]};
    if (!PyFloat_CheckExact(a[5]) || !PyFloat_CheckExact(a[6]) || !PyFloat_CheckExact(a[7]) || !PyBool_Check(a[8]) || !residual_desc(d, o, t)) Py_RETURN_NONE;
    d.eps = float(PyFloat_AS_DOUBLE(a[5])), d.residual_scale = float(PyFloat_AS_DOUBLE(a[6])), d.branch_scale = float(PyFloat_AS_DOUBLE(a[7]));
    std::vector<Tensor> out(3);
    if (t[1]) out[0] = empty(t[0]->sizes(), t[0]->scalar_type(), *t[0]), d.r_out = out[0].data_ptr();
    if (t[2]) out[1] = empty(t[0]->sizes(), (t[1] ? t[1] : t[0])->scalar_type(), *t[0]), d.x = out[1].data_ptr();
    if (a[8] == Py_True) out[2] = empty({2, d.n}, at::kFloat, *t[0]), d.kept = static_cast<float*>(out[2].data_ptr());
    const int status = unlocked([&](void* stream) { return mimk_residual_rmsnorm_fwd(&d, stream); });
    return results(status, std::move(out));
END_OP

// dr or None, dx or None, r, h, gamma, post_gamma, gate, the kept buffer, what the forward call was (a tuple) -> the gradients of r, h, gamma, post_gamma, gate, None for what there is not
OP(residual_rmsnorm_bwd, 9)
    mimk_residual_rmsnorm_desc d;
    const Tensor *t[5], *dr = a[0] == Py_None ? nullptr : dense(a[0]), *dx = a[1] == Py_None ? nullptr : dense(a[1]);
    PyObject* const o[5] = {a[2], a[3], a[4], a[5], a[6]};
    if ((!dr && a[0] != Py_None) || (!dx && a[1] != Py_None) || !residual_desc(d, o, t)) Py_RETURN_NONE;
    const Tensor* block = t[1] ? t[1] : t[0];
    if ((dx != nullptr) != (t[2] != nullptr) || (dr && (!here(dr) || dr->sizes() != t[0]->sizes() || dr->scalar_type() != t[0]->scalar_type()))) Py_RETURN_NONE;
    if (dx && (!here(dx) || dx->sizes() != block->sizes() || dx->scalar_type() != block->scalar_type())) Py_RETURN_NONE;
    const Tensor* kept = dense(a[7]);
    if (!here(kept) || kept->scalar_type() != at::kFloat || !PyTuple_CheckExact(a[8]) || PyTuple_GET_SIZE(a[8]) != 9) Py_RETURN_NONE;
    int64_t v;
    for (int i = 0; i < 2; ++i)
        if (!is_int(PyTuple_GET_ITEM(a[8], i), v) || v != (i ? d.d : d.n)) Py_RETURN_NONE;
    for (int i = 1; i < 5; ++i)
        if (PyTuple_GET_ITEM(a[8], 1 + i) != (t[i] ? Py_True : Py_False)) Py_RETURN_NONE;
    float f[3];
    for (int i = 0; i < 3; ++i) {
        if (!PyFloat_CheckExact(PyTuple_GET_ITEM(a[8], 6 + i))) Py_RETURN_NONE;
        f[i] = float(PyFloat_AS_DOUBLE(PyTuple_GET_ITEM(a[8], 6 + i)));
    }
    d.eps = f[0], d.residual_scale = f[1], d.branch_scale = f[2];
    if (mimk_residual_rmsnorm_workspace(&d, &d.workspace_bytes) != MIMK_OK) Py_RETURN_NONE;
    std::vector<Tensor> out(5);
    void* to[5] = {};
    for (int i = 0; i < 5; ++i)
        if (t[i]) out[i] = empty(t[i]->sizes(), t[i]->scalar_type(), *t[i]), to[i] = out[i].data_ptr();
    Tensor scratch = empty({int64_t(d.workspace_bytes)}, at::kByte, *t[0]);
    d.dr = to[0], d.dh = to[1], d.dgamma = to[2], d.dpost_gamma = to[3], d.dgate = to[4];
    d.dr_out = dr ? dr->data_ptr() : nullptr, d.dx = dx ? dx->data_ptr() : nullptr, d.kept = static_cast<float*>(kept->data_ptr()), d.workspace = scratch.data_ptr();
    const int status = unlocked([&](void* stream) { return mimk_residual_rmsnorm_bwd(&d, stream); });
    return results(status, std::move(out));
END_OP

// one tensor of matrices, steps, three coefficients (a tuple), eps, scale
OP(orthogonalize, 5)
    const Tensor* x = dense(a[0]);
    int64_t steps;
    if (!here(x) || x->dim() < 2 || !is_int(a[1], steps) || steps < 1 || steps > 64 || !PyTuple_CheckExact(a[2]) || PyTuple_GET_SIZE(a[2]) != 3) Py_RETURN_NONE;
    if (!PyFloat_CheckExact(a[3]) || !PyFloat_CheckExact(a[4])) Py_RETURN_NONE;
    float one[3], all[3 * 64];
    for (int i = 0; i < 3; ++i) {
        if (!PyFloat_CheckExact(PyTuple_GET_ITEM(a[2], i))) Py_RETURN_NONE;
        one[i] = float(PyFloat_AS_DOUBLE(PyTuple_GET_ITEM(a[2], i)));
    }
    for (int64_t i = 0; i < 3 * steps; ++i) all[i] = one[i % 3];
    mimk_orthogonalize_desc d = {};
    d.m = x->size(x->dim() - 2), d.n = x->size(x->dim() - 1), d.batch = x->numel() / (d.m * d.n);
    std::vector<const void*> each(d.batch);
    for (int64_t i = 0; i < d.batch; ++i) each[i] = static_cast<const char*>(x->data_ptr()) + i * d.m * d.n * x->element_size();
    d.x = each.data(), d.coefficients = all, d.steps = int(steps), d.dtype = dtype_of(x->scalar_type());
    d.eps = float(PyFloat_AS_DOUBLE(a[3])), d.scale = float(PyFloat_AS_DOUBLE(a[4]));
    if (mimk_orthogonalize_workspace(&d, &d.workspace_bytes) != MIMK_OK) Py_RETURN_NONE;
    Tensor out = empty(x->sizes(), at::kBFloat16, *x), scratch = empty({int64_t(d.workspace_bytes)}, at::kByte, *x);
    d.out = out.data_ptr(), d.workspace = scratch.data_ptr();
    return result(unlocked([&](void* stream) { return mimk_orthogonalize(&d, stream); }), std::move(out));
END_OP

// x, perm (a tuple of ints): the copy-style map_reduce_post that tensor.py's transpose spells
OP(transpose, 2)
    const Tensor* x = dense(a[0]);
    if (!x || !PyTuple_CheckExact(a[1]) || PyTuple_GET_SIZE(a[1]) != x->dim() || x->dim() > MIMK_MRP_MAX_RANK) Py_RETURN_NONE;
    const int r = int(x->dim());
    mimk_mrp_desc d = {};
    std::vector<int64_t> shape(r);
    bool seen[MIMK_MRP_MAX_RANK] = {};
    d.ro = d.rn = r, d.nis = 1;
    d.in_map[0].rows = d.map_out.rows = r;
    for (int i = 0; i < r; ++i) {
        int64_t p;
        if (!is_int(PyTuple_GET_ITEM(a[1], i), p) || p < 0 || p >= r || seen[p]) Py_RETURN_NONE;
        seen[p] = true, shape[i] = d.sr[i] = d.so[i] = x->size(p);
        d.in_map[0].coef[p][i] = 1, d.map_out.coef[i][i] = 1, d.in_shape[0][i] = x->size(i);
    }
    Tensor out = empty(shape, x->scalar_type(), *x);
    d.in[0] = x->data_ptr(), d.in_dtype[0] = d.out_dtype = dtype_of(x->scalar_type()), d.acc_dtype = MIMK_F32;
    d.comb = MIMK_F_FIRST, d.post = MIMK_P_ID, d.out = out.data_ptr();
    return result(unlocked([&](void* stream) { return mimk_map_reduce_post(&d, stream); }), std::move(out));
END_OP

PyMethodDef methods[] = {
#define ENTRY(NAME) {#NAME, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(NAME)), METH_FASTCALL, nullptr}
    ENTRY(product_2d), ENTRY(bmm), ENTRY(reduce), ENTRY(reduce_of_unary), ENTRY(softmax), ENTRY(rmsnorm), ENTRY(unary), ENTRY(binary), ENTRY(binary_ax),
    ENTRY(attention), ENTRY(mlp_gated), ENTRY(mlp_gated_fwd), ENTRY(mlp_gated_bwd), ENTRY(linear_ce), ENTRY(clip_grads), ENTRY(embedding), ENTRY(embedding_grad), ENTRY(residual_rmsnorm), ENTRY(residual_rmsnorm_bwd), ENTRY(orthogonalize),
    ENTRY(transpose), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__native() {
    PyObject* nn = PyImport_ImportModule("torch.nn.parameter");
    if (!nn) return nullptr;
    parameter_type = reinterpret_cast<PyTypeObject*>(PyObject_GetAttrString(nn, "Parameter"));
    Py_DECREF(nn);
    return parameter_type ? PyModule_Create(&module) : nullptr;
}
