// The common form of the operators of flexllm_b200/ops.py that are called for a few tokens, without the interpreter's share of a call: tensors are checked, outputs allocated and the
// library's entry point called here. With ctypes a call of the linear layer took 9.2 us of host time, of which the launch is 3.4
// (torch.empty from Python 2.4, five pointers 0.9, the foreign call 0.9), longer than its kernel at 128 x 2048 x 2048, and the MLP block
// of one token 20 us for 14 us of kernels. The operators over the paged cache take 9 to 14 tensors each, those of a model's layers several times that.
//
// Each function returns the output tensor, a status other than 0 as an integer, or None where the arguments are not plain contiguous CUDA
// tensors of the expected types: the caller then takes its general path, which decides what to do with them. The entry points are
// handed over as addresses (bind), so that the library that is called is the one that Python has loaded.
#include <Python.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/TensorSubclassLikeUtils.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/flexllm_b200.h"

namespace {

decltype(&flexllm_linear_prefill_i8) g_prefill = nullptr;
decltype(&flexllm_linear_decode_i8) g_decode = nullptr;
decltype(&flexllm_mlp_block_workspace) g_mlp_workspace = nullptr;
decltype(&flexllm_mlp_block_decode) g_mlp = nullptr;
decltype(&flexllm_qk_norm_rope) g_rope = nullptr;
decltype(&flexllm_attn_packed) g_packed = nullptr;
decltype(&flexllm_attn_tree) g_tree = nullptr;
decltype(&flexllm_kv_keep) g_keep = nullptr;
decltype(&flexllm_linear_w4) g_w4 = nullptr;

// A plain contiguous CUDA tensor of `dim` dimensions and type `dtype`, or nullptr.
const at::Tensor* plain(PyObject* o, at::ScalarType dtype, int64_t dim) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || t.scalar_type() != dtype || t.dim() != dim || at::isTensorSubclassLike(t) || !t.is_contiguous()) return nullptr;
    return &t;
}
at::Tensor empty_like_device(at::IntArrayRef size, at::ScalarType dtype, const at::Tensor& like) {
    return at::empty(size, at::TensorOptions().dtype(dtype).device(like.device()));
}
PyObject* general() { Py_RETURN_NONE; }
bool modes() { return c10::impl::dispatch_mode_enabled() || at::impl::torch_function_mode_enabled(); }        // someone wants to see the calls
PyObject* result(int status, at::Tensor&& y) { return status != 0 ? PyLong_FromLong(status) : THPVariable_Wrap(std::move(y)); }
bool fits(int64_t v) { return v >= 0 && v <= INT32_MAX; }

template <class F> PyObject* guarded(F f) {          // C++ exceptions as torch's own functions raise them (torch.OutOfMemoryError, torch.AcceleratorError, ...)
    try {
        return f();
    } catch (...) {
        torch::translate_exception_to_python(std::current_exception());
        return nullptr;
    }
}

// bind(prefill, decode, mlp_workspace, mlp, qk_norm_rope, attn_packed, attn_tree, kv_keep, linear_w4)
PyObject* bind(PyObject*, PyObject* args) {
    unsigned long long a, b, c, d, r, p, t, k, w;
    if (!PyArg_ParseTuple(args, "KKKKKKKKK", &a, &b, &c, &d, &r, &p, &t, &k, &w)) return nullptr;
    g_prefill = (decltype(g_prefill))a; g_decode = (decltype(g_decode))b;
    g_mlp_workspace = (decltype(g_mlp_workspace))c; g_mlp = (decltype(g_mlp))d;
    g_rope = (decltype(g_rope))r; g_packed = (decltype(g_packed))p; g_tree = (decltype(g_tree))t; g_keep = (decltype(g_keep))k; g_w4 = (decltype(g_w4))w;
    Py_RETURN_NONE;
}

// linear(decode, a [M,K] int8, s_tok [M], w [N,K] int8, s_ch [N]) -> y [M,N]
PyObject* linear(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 5 || !g_prefill || modes()) return general();
        const at::Tensor *a = plain(v[1], at::kChar, 2), *s = plain(v[2], at::kFloat, 1), *w = plain(v[3], at::kChar, 2), *c = plain(v[4], at::kFloat, 1);
        if (!a || !s || !w || !c) return general();
        const int64_t M = a->size(0), K = a->size(1), N = w->size(0);
        if (!fits(M) || !fits(K) || !fits(N)) return general();
        at::Tensor y = empty_like_device({M, N}, at::kFloat, *a);
        auto fn = v[0] == Py_True ? g_decode : g_prefill;
        const int8_t *ap = (const int8_t*)a->data_ptr(), *wp = (const int8_t*)w->data_ptr();
        const float *sp = (const float*)s->data_ptr(), *cp = (const float*)c->data_ptr();
        float* yp = (float*)y.data_ptr();
        void* stream = c10::cuda::getCurrentCUDAStream().stream();
        int status;
        Py_BEGIN_ALLOW_THREADS
        status = fn(ap, sp, wp, cp, (int)M, (int)N, (int)K, nullptr, yp, stream);
        Py_END_ALLOW_THREADS
        return result(status, std::move(y));
    });
}

// mlp_block(x [M,D], gamma [D], w_gu [2F,D] int8, s_gu [2F], w_d [D,F] int8, s_d [D], eps, order, fht_scale) -> y [M,D]
PyObject* mlp_block(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 9 || !g_mlp || modes()) return general();
        const at::Tensor *x = plain(v[0], at::kFloat, 2), *g = plain(v[1], at::kFloat, 1), *wgu = plain(v[2], at::kChar, 2), *sgu = plain(v[3], at::kFloat, 1),
                         *wd = plain(v[4], at::kChar, 2), *sd = plain(v[5], at::kFloat, 1);
        if (!x || !g || !wgu || !sgu || !wd || !sd || !PyFloat_Check(v[6]) || !PyLong_Check(v[7]) || !PyFloat_Check(v[8])) return general();
        const float eps = (float)PyFloat_AS_DOUBLE(v[6]), scale = (float)PyFloat_AS_DOUBLE(v[8]);
        const long order = PyLong_AsLong(v[7]);
        if (order == -1 && PyErr_Occurred()) { PyErr_Clear(); return general(); }
        const int64_t M = x->size(0), D = x->size(1), F = wd->size(1);
        if (!fits(M) || !fits(D) || !fits(F) || !fits(order)) return general();
        const size_t bytes = g_mlp_workspace((int)M, (int)D, (int)F);
        at::Tensor ws = empty_like_device({(int64_t)bytes}, at::kByte, *x), y = empty_like_device({M, D}, at::kFloat, *x);
        const float *xp = (const float*)x->data_ptr(), *gp = (const float*)g->data_ptr(), *sgp = (const float*)sgu->data_ptr(), *sdp = (const float*)sd->data_ptr();
        const int8_t *wgp = (const int8_t*)wgu->data_ptr(), *wdp = (const int8_t*)wd->data_ptr();
        float* yp = (float*)y.data_ptr();
        void *wsp = ws.data_ptr(), *stream = c10::cuda::getCurrentCUDAStream().stream();
        int status;
        Py_BEGIN_ALLOW_THREADS
        status = g_mlp(xp, gp, wgp, sgp, wdp, sdp, (int)M, (int)D, (int)F, eps, (int)order, scale, yp, wsp, bytes, stream);
        Py_END_ALLOW_THREADS
        return result(status, std::move(y));
    });
}

// ---- operators over packed sequences: rows of bf16 or fp32 with any row stride, everything on the current device
int code(at::ScalarType t) { return t == at::kBFloat16 ? FLEXLLM_BF16 : t == at::kFloat ? FLEXLLM_F32 : -1; }
const at::Tensor* plain_on(PyObject* o, at::ScalarType dtype, int64_t dim, const at::Tensor& like) {
    const at::Tensor* t = plain(o, dtype, dim);
    return t && t->device() == like.device() ? t : nullptr;
}
// rows [T, ...] of 2 or 3 dimensions, dense but for the row stride
const at::Tensor* rows_of(PyObject* o, int64_t dim, int64_t* ld) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || code(t.scalar_type()) < 0 || t.dim() != dim || at::isTensorSubclassLike(t) || t.numel() == 0) return nullptr;
    if (t.device().index() != c10::cuda::current_device()) return nullptr;
    const int64_t width = dim == 2 ? t.size(1) : t.size(1) * t.size(2);
    if (dim == 3 ? t.stride(2) != 1 || t.stride(1) != t.size(2) : t.stride(1) != 1) return nullptr;
    *ld = t.size(0) > 1 ? t.stride(0) : width;
    return &t;
}
bool pages_of(PyObject* ko, PyObject* vo, const at::Tensor& like, flexllm_kv_pages* out) {
    const at::Tensor *k = plain_on(ko, like.scalar_type(), 4, like), *v = plain_on(vo, like.scalar_type(), 4, like);
    if (!k || !v || k->size(2) != 64 || v->size(3) != 64 || k->size(0) != v->size(0) || k->size(1) != v->size(1)) return false;
    if (!fits(k->size(0)) || !fits(k->size(1)) || !fits(k->size(3)) || !fits(v->size(2))) return false;
    *out = {k->data_ptr(), v->data_ptr(), (int)k->size(0), (int)k->size(1), (int)k->size(3), (int)v->size(2)};
    return true;
}
struct Packed { const int32_t *table, *cu, *ctx; int max_pages, max_ctx, B; };
bool packed_of(PyObject* table, PyObject* cu, PyObject* ctx, PyObject* max_ctx, const at::Tensor& like, Packed* p) {
    const at::Tensor *t = plain_on(table, at::kInt, 2, like), *c = cu ? plain_on(cu, at::kInt, 1, like) : nullptr, *x = plain_on(ctx, at::kInt, 1, like);
    if (!t || (cu && !c) || !x || x->size(0) != t->size(0) || (c && c->size(0) != t->size(0) + 1) || !fits(t->size(0)) || !fits(t->size(1) * 64)) return false;
    long most = t->size(1) * 64 - 1;
    if (max_ctx != Py_None) {
        if (!PyLong_Check(max_ctx)) return false;
        most = PyLong_AsLong(max_ctx);
        if (most == -1 && PyErr_Occurred()) { PyErr_Clear(); return false; }
        if (!fits(most)) return false;
    }
    *p = {(const int32_t*)t->data_ptr(), c ? (const int32_t*)c->data_ptr() : nullptr, (const int32_t*)x->data_ptr(), (int)t->size(1), (int)most, (int)t->size(0)};
    return true;
}
bool small_int(PyObject* o, int* out) {
    if (!PyLong_Check(o)) return false;
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) { PyErr_Clear(); return false; }
    *out = (int)v;
    return fits(v);
}
// a vector of n floats, or None
bool maybe_floats(PyObject* o, int64_t n, const at::Tensor& like, const float** out) {
    *out = nullptr;
    if (o == Py_None) return true;
    const at::Tensor* t = plain_on(o, at::kFloat, 1, like);
    if (!t || t->size(0) != n) return false;
    *out = (const float*)t->data_ptr();
    return true;
}

// qk_norm_rope(proj, heads, pos, cos_t, sin_t, k_pages, v_pages, page_table, cu, ctx, q_gain, k_gain, eps, sections, max_ctx) -> q
PyObject* qk_norm_rope(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        int64_t ldp;
        int heads, sec[4] = {0, 0, 0, 0};
        flexllm_kv_pages kv;
        Packed s;
        if (n != 15 || !g_rope || modes()) return general();
        const at::Tensor* x = rows_of(v[0], 2, &ldp);
        if (!x || !small_int(v[1], &heads) || !pages_of(v[5], v[6], *x, &kv) || !packed_of(v[7], v[8], v[9], v[14], *x, &s) || !PyFloat_Check(v[12])) return general();
        const at::Tensor *cs = plain_on(v[3], at::kFloat, 2, *x), *sn = plain_on(v[4], at::kFloat, 2, *x), *pos = plain_on(v[2], at::kInt, 1, *x);
        if (!pos) pos = plain_on(v[2], at::kInt, 2, *x);
        const float *qg, *kg;
        if (!cs || !sn || !pos || cs->sizes() != sn->sizes() || !maybe_floats(v[10], kv.kdim, *x, &qg) || !maybe_floats(v[11], kv.kdim, *x, &kg)) return general();
        const int64_t T = x->size(0), axes = pos->dim() == 2 ? pos->size(0) : 1, width = (int64_t)heads * kv.kdim;
        if (axes < 1 || axes > 4 || pos->numel() != axes * T || !fits(T) || !fits(cs->size(0)) || !fits(cs->size(1) * 2) ||
            x->size(1) != width + (int64_t)kv.hkv * (kv.kdim + kv.vdim)) return general();
        const bool given = v[13] != Py_None;
        if (given) {
            if (!PyList_CheckExact(v[13]) || PyList_GET_SIZE(v[13]) != axes) return general();
            for (int i = 0; i < axes; i++)
                if (!small_int(PyList_GET_ITEM(v[13], i), sec + i)) return general();
        } else if (axes > 1) {
            return general();
        }
        const float eps = (float)PyFloat_AS_DOUBLE(v[12]);
        at::Tensor q = empty_like_device({T, width}, x->scalar_type(), *x);
        const void *xp = x->data_ptr(), *pp = pos->data_ptr(), *cp = cs->data_ptr(), *sp = sn->data_ptr();
        void *qp = q.data_ptr(), *stream = c10::cuda::getCurrentCUDAStream().stream();
        const int dt = code(x->scalar_type()), rot = (int)cs->size(1) * 2, len = (int)cs->size(0);
        int status;
        Py_BEGIN_ALLOW_THREADS
        status = g_rope(dt, &kv, heads, xp, ldp, qg, kg, eps, (const int32_t*)pp, (int)axes, given ? sec : nullptr, (const float*)cp, (const float*)sp, rot, len,
                        s.cu, s.ctx, s.table, s.max_pages, s.max_ctx, s.B, (int)T, qp, width, stream);
        Py_END_ALLOW_THREADS
        return result(status, std::move(q));
    });
}

// attn_paged(q [T,heads,dim], mask or None, k_pages, v_pages, page_table, cu, ctx, scale, max_ctx) -> [T,heads*vdim]
PyObject* attn_paged(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        int64_t ldq;
        flexllm_kv_pages kv;
        Packed s;
        if (n != 9 || !g_packed || modes()) return general();
        const at::Tensor* q = rows_of(v[0], 3, &ldq);
        if (!q || !pages_of(v[2], v[3], *q, &kv) || !packed_of(v[4], v[5], v[6], v[8], *q, &s) || !PyFloat_Check(v[7])) return general();
        const at::Tensor* mask = v[1] == Py_None ? nullptr : plain_on(v[1], at::kLong, 1, *q);
        const int64_t T = q->size(0), H = q->size(1);
        if ((v[1] != Py_None && (!mask || mask->size(0) != T)) || q->size(2) != kv.kdim || !fits(T) || !fits(H)) return general();
        const float scale = (float)PyFloat_AS_DOUBLE(v[7]);
        at::Tensor out = empty_like_device({T, H * kv.vdim}, q->scalar_type(), *q);
        const void *qp = q->data_ptr(), *mp = mask ? mask->data_ptr() : nullptr;
        void *op = out.data_ptr(), *stream = c10::cuda::getCurrentCUDAStream().stream();
        const int dt = code(q->scalar_type());
        int status;
        Py_BEGIN_ALLOW_THREADS
        if (mp) status = g_tree(dt, &kv, (int)H, scale, qp, ldq, (const uint64_t*)mp, s.cu, s.ctx, s.table, s.max_pages, s.max_ctx, s.B, (int)T, op, H * kv.vdim, stream);
        else status = g_packed(dt, &kv, (int)H, scale, qp, ldq, s.cu, s.ctx, s.table, s.max_pages, s.max_ctx, s.B, (int)T, op, H * kv.vdim, stream);
        Py_END_ALLOW_THREADS
        return result(status, std::move(out));
    });
}

// kv_keep([(k_pages, v_pages), ..], page_table, ctx, keep, count, max_ctx) -> status
PyObject* kv_keep(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        constexpr int kMost = 256;
        flexllm_kv_pages kv[kMost];
        Packed s;
        if (n != 6 || !g_keep || modes() || !PyList_CheckExact(v[0])) return general();
        const Py_ssize_t layers = PyList_GET_SIZE(v[0]);
        if (layers < 1 || layers > kMost) return general();
        const at::Tensor* k0 = nullptr;
        for (Py_ssize_t i = 0; i < layers; i++) {
            PyObject* l = PyList_GET_ITEM(v[0], i);
            if (!PyTuple_CheckExact(l) || PyTuple_GET_SIZE(l) != 2 || !THPVariable_CheckExact(PyTuple_GET_ITEM(l, 0))) return general();
            if (!k0) {
                k0 = &THPVariable_Unpack(PyTuple_GET_ITEM(l, 0));
                if (!k0->defined() || !k0->is_cuda() || code(k0->scalar_type()) < 0 || k0->device().index() != c10::cuda::current_device()) return general();
            }
            if (!pages_of(PyTuple_GET_ITEM(l, 0), PyTuple_GET_ITEM(l, 1), *k0, kv + i)) return general();
        }
        const at::Tensor *keep = plain_on(v[3], at::kInt, 2, *k0), *count = plain_on(v[4], at::kInt, 1, *k0);
        if (!packed_of(v[1], nullptr, v[2], v[5], *k0, &s) || !keep || !count || keep->size(0) != s.B || count->size(0) != s.B || !fits(keep->size(1))) return general();
        const int32_t *kp = (const int32_t*)keep->data_ptr(), *cp = (const int32_t*)count->data_ptr();
        const int dt = code(k0->scalar_type()), most = (int)keep->size(1);
        void* stream = c10::cuda::getCurrentCUDAStream().stream();
        int status;
        Py_BEGIN_ALLOW_THREADS
        status = g_keep(dt, kv, (int)layers, s.table, s.max_pages, s.ctx, s.max_ctx, kp, cp, most, s.B, stream);
        Py_END_ALLOW_THREADS
        return PyLong_FromLong(status);
    });
}

// linear_w4(x [M,K], w [N,K/2] uint8, scale [N,K/group], zero or None, bias or None) -> [M,N] of x's type
PyObject* linear_w4(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        int64_t lda;
        if (n != 5 || !g_w4 || modes()) return general();
        const at::Tensor* x = rows_of(v[0], 2, &lda);
        if (!x) return general();
        const at::Tensor *w = plain_on(v[1], at::kByte, 2, *x), *s = plain_on(v[2], at::kBFloat16, 2, *x);
        if (!s) s = plain_on(v[2], at::kFloat, 2, *x);
        if (!w || !s) return general();
        const at::Tensor* z = v[3] == Py_None ? nullptr : plain_on(v[3], at::kByte, 2, *x);
        const int64_t M = x->size(0), K = x->size(1), N = w->size(0), groups = s->size(1);
        const float* bias;
        if ((v[3] != Py_None && (!z || z->sizes() != s->sizes())) || s->size(0) != N || groups < 1 || K % groups || w->size(1) * 2 != K || !fits(M) || !fits(N) || !fits(K) ||
            !maybe_floats(v[4], N, *x, &bias)) return general();
        at::Tensor y = empty_like_device({M, N}, x->scalar_type(), *x);
        const void *xp = x->data_ptr(), *sp = s->data_ptr();
        const uint8_t *wp = (const uint8_t*)w->data_ptr(), *zp = z ? (const uint8_t*)z->data_ptr() : nullptr;
        void *yp = y.data_ptr(), *stream = c10::cuda::getCurrentCUDAStream().stream();
        const int dt = code(x->scalar_type()), st = code(s->scalar_type());
        int status;
        Py_BEGIN_ALLOW_THREADS
        status = g_w4(dt, xp, lda, wp, sp, st, zp, (int)(K / groups), bias, (int)M, (int)N, (int)K, yp, N, 0, stream);
        Py_END_ALLOW_THREADS
        return result(status, std::move(y));
    });
}

PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, "addresses of the library's entry points"},
                         {"linear", (PyCFunction)(void*)linear, METH_FASTCALL, "W8A8 linear layer, output fp32"},
                         {"mlp_block", (PyCFunction)(void*)mlp_block, METH_FASTCALL, "decode MLP block"},
                         {"qk_norm_rope", (PyCFunction)(void*)qk_norm_rope, METH_FASTCALL, "norm, rotation and append"},
                         {"attn_paged", (PyCFunction)(void*)attn_paged, METH_FASTCALL, "packed or tree attention"},
                         {"kv_keep", (PyCFunction)(void*)kv_keep, METH_FASTCALL, "accepted paths"},
                         {"linear_w4", (PyCFunction)(void*)linear_w4, METH_FASTCALL, "product with 4-bit weights"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_front_end", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__front_end() { return PyModule_Create(&module); }
