// The call paths of the Python package in native code: tensors are checked and described, the output is allocated and the
// C ABI is called without going back to the interpreter.  A call costs ~2 us of host time beyond the launch, where the same
// steps in Python and ctypes cost ~10: more than a small decode kernel runs.
//
// Every function here takes the plain case of its operator only -- the types, layouts and options of ordinary calls -- and
// returns None (False) for anything else; the Python implementation then takes the call, converts what it converts and
// raises what it raises.  Nothing is remembered between calls: tensors are described afresh each time, workspaces come from
// the package's own table.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include "../../include/tilegym_hip.h"

namespace {

decltype(&tg_fp8_gemm) g_gemm = nullptr;
decltype(&tg_fp8_gemm_workspace_bytes) g_gemm_workspace_bytes = nullptr;
decltype(&tg_fp8_ragged_gemm) g_ragged_gemm = nullptr;
decltype(&tg_fp8_quant_group) g_quant_group = nullptr;
decltype(&tg_fp8_fused_moe) g_fused_moe = nullptr;
decltype(&tg_fp8_fused_moe_block_m) g_fused_moe_block_m = nullptr;
decltype(&tg_fp8_fused_moe_workspace_bytes) g_fused_moe_workspace_bytes = nullptr;
decltype(&tg_fp8_rms_norm_quant) g_rms_norm_quant = nullptr;
decltype(&tg_fp8_kv_append) g_kv_append = nullptr;
decltype(&tg_fp8_kv_read) g_kv_read = nullptr;
decltype(&tg_fp8_kv_attention) g_kv_attention = nullptr;
decltype(&tg_fp8_kv_attention_workspace_bytes) g_kv_attention_workspace_bytes = nullptr;
decltype(&tg_int8_gemm) g_int8_gemm = nullptr;
decltype(&tg_int8_gemm_workspace_bytes) g_int8_gemm_workspace_bytes = nullptr;
decltype(&tg_int8_ragged_gemm) g_int8_ragged_gemm = nullptr;
decltype(&tg_int8_quant) g_int8_quant = nullptr;
decltype(&tg_last_error) g_last_error = nullptr;
decltype(&tg_moe_sort) g_moe_sort = nullptr;
decltype(&tg_moe_sort_workspace_bytes) g_moe_sort_workspace_bytes = nullptr;
decltype(&tg_moe_permute) g_moe_permute = nullptr;
decltype(&tg_moe_unpermute) g_moe_unpermute = nullptr;
decltype(&tg_moe_unpermute_backward) g_moe_unpermute_backward = nullptr;
PyObject* g_workspaces = nullptr;     // {(device, stream, under capture): [scratch tensors, newest last]}
PyObject* g_workspace_for = nullptr;  // callable(device, bytes, index, stream) -> tensor, for a new or larger one
PyObject* g_check_rc = nullptr;       // callable(rc, where): raises

constexpr int64_t kMaxMoeTokens = 32768;  // one chunk of the layer

int dtype_code(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return TG_F32;
        case at::kHalf: return TG_F16;
        case at::kBFloat16: return TG_BF16;
        case at::kInt: return TG_I32;
        case at::kLong: return TG_I64;
        case at::kFloat8_e5m2: return TG_F8E5M2;
        case at::kByte: return 6;  // (workspaces; no operand has this type)
        case at::kFloat8_e4m3fn: return TG_F8E4M3FN;
        case at::kChar: return TG_I8;
        default: return -1;
    }
}

bool describe(const at::Tensor& t, tg_tensor* d) {
    const int code = dtype_code(t.scalar_type());
    const int64_t nd = t.dim();
    if (code < 0 || nd > TG_MAX_DIMS) return false;
    *d = tg_tensor{};
    d->ptr = reinterpret_cast<uint64_t>(t.data_ptr());
    d->ndim = (int32_t)nd;
    d->dtype = code;
    for (int64_t i = 0; i < nd; ++i) {
        d->shape[i] = t.size(i);
        d->strides[i] = t.stride(i);
    }
    return true;
}

tg_tensor describe_rows(const at::Tensor& t, int64_t rows, int64_t cols) {  // a contiguous tensor as (rows, cols)
    tg_tensor d{};
    d.ptr = reinterpret_cast<uint64_t>(t.data_ptr());
    d.ndim = 2;
    d.dtype = dtype_code(t.scalar_type());
    d.shape[0] = rows; d.shape[1] = cols;
    d.strides[0] = cols; d.strides[1] = 1;
    return d;
}

const at::Tensor* tensor_of(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

bool on_gpu(const at::Tensor* t) { return t && t->is_cuda() && t->layout() == at::kStrided; }
bool plain(const at::Tensor* t, at::ScalarType type, int64_t dim) {
    return on_gpu(t) && t->scalar_type() == type && t->dim() == dim && t->is_contiguous();
}
bool io_type(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf || t == at::kFloat; }

at::Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
    return at::empty(sizes, at::TensorOptions().dtype(type).device(like.device()));
}

// The scratch buffer of the current stream, at least `bytes`, described; false with an exception set.
bool workspace(PyObject* like, int index, hipStream_t stream, int64_t bytes, tg_tensor* d) {
    const bool capturing = c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None;
    PyObject* key = Py_BuildValue("(iKO)", index, (unsigned long long)(uintptr_t)stream, capturing ? Py_True : Py_False);
    if (!key) return false;
    PyObject* held = PyDict_GetItemWithError(g_workspaces, key);
    Py_DECREF(key);
    if (held && PyList_Check(held) && PyList_GET_SIZE(held) > 0) {
        const at::Tensor* t = tensor_of(PyList_GET_ITEM(held, PyList_GET_SIZE(held) - 1));
        if (t && t->numel() >= bytes) return describe(*t, d);
    } else if (!held && PyErr_Occurred()) {
        return false;
    }
    PyObject* device = PyObject_GetAttrString(like, "device");
    if (!device) return false;
    PyObject* made = PyObject_CallFunction(g_workspace_for, "OLiK", device, (long long)bytes, index, (unsigned long long)(uintptr_t)stream);
    Py_DECREF(device);
    if (!made) return false;
    const at::Tensor* t = tensor_of(made);  // (the table keeps it alive)
    const bool ok = t && describe(*t, d);
    Py_DECREF(made);
    if (!ok && !PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "no workspace");
    return ok;
}

// Raises what check_rc raises for rc != 0; true when rc is 0.
bool succeeded(int32_t rc, const char* where) {
    if (rc == TG_OK) return true;
    PyObject* r = PyObject_CallFunction(g_check_rc, "is", (int)rc, where);
    Py_XDECREF(r);
    if (r) PyErr_SetString(PyExc_RuntimeError, where);
    return false;
}

// None -> no scale; a number -> into alpha; a tensor -> the kernel reads it.  False: not a plain scale.
bool take_scale(PyObject* o, double* alpha, const at::Tensor** t) {
    *t = nullptr;
    if (o == Py_None) return true;
    if (PyFloat_Check(o)) { *alpha *= PyFloat_AS_DOUBLE(o); return true; }
    const at::Tensor* s = tensor_of(o);
    if (!on_gpu(s) || s->scalar_type() != at::kFloat || !s->is_contiguous() || s->dim() > TG_MAX_DIMS) return false;
    *t = s;
    return true;
}

// tg_fp8_gemm on described tensors; false with an exception set.
bool run_gemm(PyObject* like, const at::Tensor& a, const tg_tensor& dc, const tg_tensor& da, const tg_tensor& db, const at::Tensor* sa,
              const at::Tensor* sb, const tg_tensor* dsa, const tg_tensor* dsb, bool trans_a, bool trans_b, double alpha, double beta, bool use_workspace) {
    const int index = a.get_device();
    const hipStream_t stream = c10::hip::getCurrentHIPStream(index).stream();
    tg_tensor tsa, tsb, dws;
    if (!dsa && sa) { if (!describe(*sa, &tsa)) { PyErr_SetString(PyExc_TypeError, "scale_a"); return false; } dsa = &tsa; }
    if (!dsb && sb) { if (!describe(*sb, &tsb)) { PyErr_SetString(PyExc_TypeError, "scale_b"); return false; } dsb = &tsb; }
    const int64_t M = da.shape[trans_a ? 1 : 0], K = da.shape[trans_a ? 0 : 1], N = db.shape[trans_b ? 0 : 1];
    const int64_t need = use_workspace && M > 0 && N > 0 && K > 0 ? g_gemm_workspace_bytes(M, N, K, trans_b, nullptr, 0) : 0;
    if (need > 0 && !workspace(like, index, stream, need, &dws)) return false;
    int32_t rc;
    Py_BEGIN_ALLOW_THREADS
    rc = g_gemm(&dc, &da, &db, dsa, dsb, trans_a, trans_b, (float)alpha, (float)beta, need > 0 ? &dws : nullptr, nullptr, 0, index,
                (uint64_t)(uintptr_t)stream);
    Py_END_ALLOW_THREADS
    return succeeded(rc, "tg_fp8_gemm");
}

// matmul(a, b, trans_a, trans_b, scale_a, scale_b, alpha, out_dtype) -> tensor, or None
PyObject* py_matmul(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 8) { PyErr_SetString(PyExc_TypeError, "matmul takes 8 arguments"); return nullptr; }
    const at::Tensor *a = tensor_of(args[0]), *b = tensor_of(args[1]), *sa, *sb;
    if (!plain(a, at::kFloat8_e4m3fn, 2) || !plain(b, at::kFloat8_e4m3fn, 2)) Py_RETURN_NONE;
    const bool trans_a = args[2] == Py_True, trans_b = args[3] == Py_True;
    double alpha = PyFloat_AsDouble(args[6]);
    if (alpha == -1.0 && PyErr_Occurred()) return nullptr;
    if (!take_scale(args[4], &alpha, &sa) || !take_scale(args[5], &alpha, &sb)) Py_RETURN_NONE;
    at::ScalarType out = at::kFloat8_e4m3fn;
    if (args[7] != Py_None) {
        if (!THPDtype_Check(args[7])) Py_RETURN_NONE;
        out = reinterpret_cast<THPDtype*>(args[7])->scalar_type;
        if (!io_type(out) && out != at::kFloat8_e4m3fn) Py_RETURN_NONE;
    }
    const int64_t M = a->size(trans_a ? 1 : 0), K = a->size(trans_a ? 0 : 1), N = b->size(trans_b ? 0 : 1), Kb = b->size(trans_b ? 1 : 0);
    if (K != Kb || a->device() != b->device()) Py_RETURN_NONE;
    at::Tensor c = new_tensor({M, N}, out, *a);
    tg_tensor dc, da, db;
    if (!describe(c, &dc) || !describe(*a, &da) || !describe(*b, &db)) Py_RETURN_NONE;
    if (!run_gemm(args[0], *a, dc, da, db, sa, sb, nullptr, nullptr, trans_a, trans_b, alpha, 0.0, true)) return nullptr;
    return THPVariable_Wrap(std::move(c));
    END_HANDLE_TH_ERRORS
}

// gemm(c, a, b, scale_a, scale_b, trans_a, trans_b, alpha, beta, use_workspace) -> True, or False
PyObject* py_gemm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 10) { PyErr_SetString(PyExc_TypeError, "gemm takes 10 arguments"); return nullptr; }
    const at::Tensor *c = tensor_of(args[0]), *a = tensor_of(args[1]), *b = tensor_of(args[2]);
    const at::Tensor *sa = args[3] == Py_None ? nullptr : tensor_of(args[3]), *sb = args[4] == Py_None ? nullptr : tensor_of(args[4]);
    if (!on_gpu(c) || !on_gpu(a) || !on_gpu(b) || (args[3] != Py_None && !on_gpu(sa)) || (args[4] != Py_None && !on_gpu(sb))) Py_RETURN_FALSE;
    tg_tensor dc, da, db, dsa, dsb;
    if (a->dim() != 2 || b->dim() != 2 || !describe(*c, &dc) || !describe(*a, &da) || !describe(*b, &db) || (sa && !describe(*sa, &dsa)) ||
        (sb && !describe(*sb, &dsb)))
        Py_RETURN_FALSE;
    const double alpha = PyFloat_AsDouble(args[7]), beta = PyFloat_AsDouble(args[8]);
    if (PyErr_Occurred()) return nullptr;
    if (!run_gemm(args[1], *a, dc, da, db, nullptr, nullptr, sa ? &dsa : nullptr, sb ? &dsb : nullptr, args[5] == Py_True, args[6] == Py_True, alpha,
                  beta, args[9] == Py_True))
        return nullptr;
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// block_matmul(A, B, As, Bs, out_dtype) -> tensor, or None: 128 x 128 quantization blocks
PyObject* py_block_matmul(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 5) { PyErr_SetString(PyExc_TypeError, "block_matmul takes 5 arguments"); return nullptr; }
    const at::Tensor *a = tensor_of(args[0]), *b = tensor_of(args[1]), *as = tensor_of(args[2]), *bs = tensor_of(args[3]);
    if (!on_gpu(a) || a->dim() < 1 || !plain(a, at::kFloat8_e4m3fn, a->dim()) || !plain(b, at::kFloat8_e4m3fn, 2) || !on_gpu(as) ||
        !plain(as, at::kFloat, a->dim()) || !plain(bs, at::kFloat, 2) || !THPDtype_Check(args[4]))
        Py_RETURN_NONE;
    const at::ScalarType out = reinterpret_cast<THPDtype*>(args[4])->scalar_type;
    const int64_t nd = a->dim(), K = a->size(nd - 1), N = b->size(0), kb = (K + 127) / 128;
    if (!io_type(out) || b->size(1) != K || K == 0 || a->numel() == 0 || as->size(nd - 1) != kb || bs->size(0) != (N + 127) / 128 ||
        bs->size(1) != kb || a->device() != b->device())
        Py_RETURN_NONE;
    c10::SmallVector<int64_t, 4> sizes(a->sizes().begin(), a->sizes().end());
    for (int64_t i = 0; i + 1 < nd; ++i)
        if (as->size(i) != sizes[i]) Py_RETURN_NONE;
    sizes[nd - 1] = N;
    const int64_t M = a->numel() / K;
    at::Tensor c = new_tensor(sizes, out, *a);
    const tg_tensor dc = describe_rows(c, M, N), da = describe_rows(*a, M, K), db = describe_rows(*b, N, K), das = describe_rows(*as, M, kb),
                    dbs = describe_rows(*bs, bs->size(0), kb);
    if (!run_gemm(args[0], *a, dc, da, db, nullptr, nullptr, &das, &dbs, false, true, 1.0, 0.0, true)) return nullptr;
    return THPVariable_Wrap(std::move(c));
    END_HANDLE_TH_ERRORS
}

// act_quant(x, group_size, eps, rule) -> (q e4m3, scales row-major), or None
PyObject* py_act_quant(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4) { PyErr_SetString(PyExc_TypeError, "act_quant takes 4 arguments"); return nullptr; }
    const at::Tensor* x = tensor_of(args[0]);
    const long group = PyLong_AsLong(args[1]), rule = PyLong_AsLong(args[3]);
    const double eps = PyFloat_AsDouble(args[2]);
    if (PyErr_Occurred()) return nullptr;
    if (!on_gpu(x) || !io_type(x->scalar_type()) || !x->is_contiguous() || x->dim() < 1 || x->dim() > TG_MAX_DIMS || group <= 0 ||
        x->size(x->dim() - 1) % group != 0)
        Py_RETURN_NONE;
    at::Tensor q = new_tensor(x->sizes(), at::kFloat8_e4m3fn, *x);
    c10::SmallVector<int64_t, 4> sizes(x->sizes().begin(), x->sizes().end());
    sizes.back() /= group;
    at::Tensor scales = new_tensor(sizes, at::kFloat, *x);
    tg_tensor dq, ds, dx;
    if (!describe(q, &dq) || !describe(scales, &ds) || !describe(*x, &dx)) Py_RETURN_NONE;
    const int index = x->get_device();
    const hipStream_t stream = c10::hip::getCurrentHIPStream(index).stream();
    int32_t rc;
    Py_BEGIN_ALLOW_THREADS
    rc = g_quant_group(&dq, &ds, &dx, (int32_t)group, (float)eps, (int32_t)rule, index, (uint64_t)(uintptr_t)stream);
    Py_END_ALLOW_THREADS
    if (!succeeded(rc, "tg_fp8_quant_group")) return nullptr;
    PyObject* tuple = PyTuple_New(2);
    if (!tuple) return nullptr;
    PyTuple_SET_ITEM(tuple, 0, THPVariable_Wrap(std::move(q)));
    PyTuple_SET_ITEM(tuple, 1, THPVariable_Wrap(std::move(scales)));
    return tuple;
    END_HANDLE_TH_ERRORS
}

// ragged_matmul(a, b, a_scale, b_scale, m_indptr, out_dtype) -> tensor, or None: 128 x 128 quantization blocks
PyObject* py_ragged_matmul(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6) { PyErr_SetString(PyExc_TypeError, "ragged_matmul takes 6 arguments"); return nullptr; }
    const at::Tensor *a = tensor_of(args[0]), *b = tensor_of(args[1]), *as = tensor_of(args[2]), *bs = tensor_of(args[3]), *ptr = tensor_of(args[4]);
    if (!plain(a, at::kFloat8_e4m3fn, 2) || !plain(b, at::kFloat8_e4m3fn, 3) || !plain(as, at::kFloat, 2) || !plain(bs, at::kFloat, 3) ||
        !plain(ptr, at::kInt, 1))
        Py_RETURN_NONE;
    at::ScalarType out = at::kBFloat16;
    if (args[5] != Py_None) {
        if (!THPDtype_Check(args[5])) Py_RETURN_NONE;
        out = reinterpret_cast<THPDtype*>(args[5])->scalar_type;
    }
    const int64_t M = a->size(0), K = a->size(1), E = b->size(0), N = b->size(1), kb = (K + 127) / 128;
    if (!io_type(out) || b->size(2) != K || ptr->size(0) != E + 1 || bs->size(0) != E || bs->size(1) != (N + 127) / 128 || bs->size(2) != kb ||
        as->size(0) != M || as->size(1) != kb || a->device() != b->device())
        Py_RETURN_NONE;
    at::Tensor c = new_tensor({M, N}, out, *a);
    tg_tensor dc, da, db, das, dbs, dptr;
    if (!describe(c, &dc) || !describe(*a, &da) || !describe(*b, &db) || !describe(*as, &das) || !describe(*bs, &dbs) || !describe(*ptr, &dptr))
        Py_RETURN_NONE;
    const int index = a->get_device();
    const hipStream_t stream = c10::hip::getCurrentHIPStream(index).stream();
    int32_t rc;
    Py_BEGIN_ALLOW_THREADS
    rc = g_ragged_gemm(&dc, &da, &db, &das, &dbs, &dptr, nullptr, 0, index, (uint64_t)(uintptr_t)stream);
    Py_END_ALLOW_THREADS
    if (!succeeded(rc, "tg_fp8_ragged_gemm")) return nullptr;
    return THPVariable_Wrap(std::move(c));
    END_HANDLE_TH_ERRORS
}

// fused_moe(hidden, w1, w2, topk_weights, topk_ids, w1_scale, w2_scale, inplace, max_experts) -> tensor, or None: the whole layer
// when tg_fp8_fused_moe takes it as one chunk
PyObject* py_fused_moe(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 9) { PyErr_SetString(PyExc_TypeError, "fused_moe takes 9 arguments"); return nullptr; }
    const at::Tensor *x = tensor_of(args[0]), *w1 = tensor_of(args[1]), *w2 = tensor_of(args[2]), *tw = tensor_of(args[3]), *ids = tensor_of(args[4]),
                     *s1 = tensor_of(args[5]), *s2 = tensor_of(args[6]);
    const long max_experts = PyLong_AsLong(args[8]);
    if (PyErr_Occurred()) return nullptr;
    if (!on_gpu(x) || (x->scalar_type() != at::kBFloat16 && x->scalar_type() != at::kHalf) || x->dim() != 2 || !x->is_contiguous() ||
        !plain(w1, at::kFloat8_e4m3fn, 3) || !plain(w2, at::kFloat8_e4m3fn, 3) || !plain(tw, at::kFloat, 2) || !on_gpu(ids) ||
        (ids->scalar_type() != at::kInt && ids->scalar_type() != at::kLong) || ids->dim() != 2 || !ids->is_contiguous() || !plain(s1, at::kFloat, 3) ||
        !plain(s2, at::kFloat, 3))
        Py_RETURN_NONE;
    const int64_t T = x->size(0), H = x->size(1), E = w1->size(0), I2 = w1->size(1), k = ids->size(1);
    if (T < 1 || T > kMaxMoeTokens || E < 1 || E > max_experts || k < 1 || H % 128 != 0 || H < 128 || H > 65536 || I2 % 256 != 0 || I2 == 0 ||
        w1->size(2) != H || w2->size(0) != E || w2->size(1) != H || w2->size(2) != I2 / 2 || ids->size(0) != T || tw->sizes() != ids->sizes() ||
        x->device() != w1->device() || x->device() != w2->device())
        Py_RETURN_NONE;
    const int block_m = g_fused_moe_block_m(T, k, E, I2 / 2);
    const bool inplace = args[7] == Py_True;
    at::Tensor out = inplace ? *x : new_tensor({T, H}, x->scalar_type(), *x);
    tg_tensor dout, dx, dw1, dw2, ds1, ds2, dtw, dids, dws;
    if (!describe(out, &dout) || !describe(*x, &dx) || !describe(*w1, &dw1) || !describe(*w2, &dw2) || !describe(*s1, &ds1) || !describe(*s2, &ds2) ||
        !describe(*tw, &dtw) || !describe(*ids, &dids))
        Py_RETURN_NONE;
    const int index = x->get_device();
    const hipStream_t stream = c10::hip::getCurrentHIPStream(index).stream();
    if (!workspace(args[0], index, stream, g_fused_moe_workspace_bytes(T, k, E, H, I2 / 2, block_m), &dws)) return nullptr;
    int32_t rc;
    Py_BEGIN_ALLOW_THREADS
    rc = g_fused_moe(&dout, &dx, &dw1, &dw2, &ds1, &ds2, &dtw, &dids, &dws, block_m, index, (uint64_t)(uintptr_t)stream);
    Py_END_ALLOW_THREADS
    if (!succeeded(rc, "tg_fp8_fused_moe")) return nullptr;
    if (inplace) {
        Py_INCREF(args[0]);
        return args[0];
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// An optional tensor of the first tensor's device: described into *d and *p set; a None leaves *p null.  False: not plain.
bool optional_tensor(PyObject* o, const at::Tensor& like, tg_tensor* d, const tg_tensor** p) {
    *p = nullptr;
    if (o == Py_None) return true;
    const at::Tensor* t = tensor_of(o);
    if (!on_gpu(t) || t->device() != like.device() || !describe(*t, d)) return false;
    *p = d;
    return true;
}

// rms_norm_quant(x, weight, eps, residual, group_size, scale, residual_out, return_norm) -> tuple, or None.  group_size 0 with a scale
PyObject* py_rms_norm_quant(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 8) { PyErr_SetString(PyExc_TypeError, "rms_norm_quant takes 8 arguments"); return nullptr; }
    const at::Tensor* x = tensor_of(args[0]);
    const double eps = PyFloat_AsDouble(args[2]);
    const long group = PyLong_AsLong(args[4]);
    const int with_norm = PyObject_IsTrue(args[7]);
    if (PyErr_Occurred()) return nullptr;
    const bool given = args[5] != Py_None;
    if (!on_gpu(x) || !io_type(x->scalar_type()) || !x->is_contiguous() || x->dim() < 1 || x->dim() > TG_MAX_DIMS ||
        (!given && (group <= 0 || x->size(x->dim() - 1) % group != 0)))
        Py_RETURN_NONE;
    tg_tensor dx, dw, dr, dro, dsc, dq, ds, dn;
    const tg_tensor *w, *r, *ro, *sc;
    if (!describe(*x, &dx) || !optional_tensor(args[1], *x, &dw, &w) || !w || !optional_tensor(args[3], *x, &dr, &r) || !optional_tensor(args[6], *x, &dro, &ro) ||
        !optional_tensor(args[5], *x, &dsc, &sc))
        Py_RETURN_NONE;
    if ((r && tensor_of(args[3])->sizes() != x->sizes()) || (ro && (!r || tensor_of(args[6])->sizes() != x->sizes()))) Py_RETURN_NONE;
    at::Tensor q = new_tensor(x->sizes(), at::kFloat8_e4m3fn, *x), scales, made_residual, norm;
    if (!describe(q, &dq)) Py_RETURN_NONE;
    if (!given) {
        c10::SmallVector<int64_t, 4> sizes(x->sizes().begin(), x->sizes().end());
        sizes.back() /= group;
        scales = new_tensor(sizes, at::kFloat, *x);
        if (!describe(scales, &ds)) Py_RETURN_NONE;
    }
    if (r && !ro) {
        made_residual = new_tensor(x->sizes(), x->scalar_type(), *x);
        if (!describe(made_residual, &dro)) Py_RETURN_NONE;
        ro = &dro;
    }
    if (with_norm) {
        norm = new_tensor(x->sizes(), x->scalar_type(), *x);
        if (!describe(norm, &dn)) Py_RETURN_NONE;
    }
    const int index = x->get_device();
    const hipStream_t stream = c10::hip::getCurrentHIPStream(index).stream();
    int32_t rc;
    Py_BEGIN_ALLOW_THREADS
    rc = g_rms_norm_quant(&dq, given ? nullptr : &ds, with_norm ? &dn : nullptr, ro, &dx, w, r, sc, (float)eps, (int32_t)group, index,
                          (uint64_t)(uintptr_t)stream);
    Py_END_ALLOW_THREADS
    if (!succeeded(rc, "tg_fp8_rms_norm_quant")) return nullptr;
    PyObject* tuple = PyTuple_New(2 + (r != nullptr) + (with_norm != 0));
    if (!tuple) return nullptr;
    int at = 0;
    auto borrowed = [](PyObject* o) { Py_INCREF(o); return o; };
    PyTuple_SET_ITEM(tuple, at++, THPVariable_Wrap(std::move(q)));
    PyTuple_SET_ITEM(tuple, at++, given ? borrowed(args[5]) : THPVariable_Wrap(std::move(scales)));
    if (r) PyTuple_SET_ITEM(tuple, at++, made_residual.defined() ? THPVariable_Wrap(std::move(made_residual)) : borrowed(args[6]));
    if (with_norm) PyTuple_SET_ITEM(tuple, at++, THPVariable_Wrap(std::move(norm)));
    return tuple;
    END_HANDLE_TH_ERRORS
}

// A paged cache's four tensors, described; null: not four tensors of one device.
const at::Tensor* describe_cache(PyObject* o, tg_tensor d[4]) {
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) return nullptr;
    const at::Tensor* first = nullptr;
    for (int i = 0; i < 4; ++i) {
        const at::Tensor* t = tensor_of(PyTuple_GET_ITEM(o, i));
        if (!on_gpu(t) || (first && t->device() != first->device()) || !describe(*t, &d[i])) return nullptr;
        if (!first) first = t;
    }
    return first->dim() == 4 ? first : nullptr;
}

// kv_append(cache, k, v, block_table, seq_lens, indptr, q, rope, interleaved) -> (q turned or None,), or None
PyObject* py_kv_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 9) { PyErr_SetString(PyExc_TypeError, "kv_append takes 9 arguments"); return nullptr; }
    tg_tensor dc[4], d[7], dq_out;
    const tg_tensor* p[7];
    const at::Tensor* first = describe_cache(args[0], dc);
    if (!first) Py_RETURN_NONE;
    for (int i = 0; i < 7; ++i)
        if (!optional_tensor(args[1 + i], *first, &d[i], &p[i]) || (i < 5 && !p[i])) Py_RETURN_NONE;
    const tg_tensor *q = p[5], *rope = p[6];
    if (q && !rope) Py_RETURN_NONE;
    at::Tensor q_out;
    if (q) {
        const at::Tensor* t = tensor_of(args[6]);
        q_out = new_tensor(t->sizes(), t->scalar_type(), *t);
        if (!describe(q_out, &dq_out)) Py_RETURN_NONE;
    }
    const int index = first->get_device();
    const hipStream_t stream = c10::hip::getCurrentHIPStream(index).stream();
    const int interleaved = PyObject_IsTrue(args[8]);
    if (interleaved < 0) return nullptr;
    int32_t rc;
    Py_BEGIN_ALLOW_THREADS
    rc = g_kv_append(&dc[0], &dc[1], &dc[2], &dc[3], p[0], p[1], p[2], p[3], p[4], q ? &dq_out : nullptr, q, rope, interleaved, index,
                     (uint64_t)(uintptr_t)stream);
    Py_END_ALLOW_THREADS
    if (!succeeded(rc, "tg_fp8_kv_append")) return nullptr;
    PyObject* tuple = PyTuple_New(1);
    if (!tuple) return nullptr;
    if (q) {
        PyTuple_SET_ITEM(tuple, 0, THPVariable_Wrap(std::move(q_out)));
    } else {
        Py_INCREF(Py_None);
        PyTuple_SET_ITEM(tuple, 0, Py_None);
    }
    return tuple;
    END_HANDLE_TH_ERRORS
}

// kv_read(cache, block_table, indptr, total_tokens, out_dtype) -> (k, v), or None
PyObject* py_kv_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 5) { PyErr_SetString(PyExc_TypeError, "kv_read takes 5 arguments"); return nullptr; }
    tg_tensor dc[4], dt, di, dk, dv;
    const tg_tensor *table, *indptr;
    const at::Tensor* first = describe_cache(args[0], dc);
    const long long total = PyLong_AsLongLong(args[3]);
    if (total == -1 && PyErr_Occurred()) return nullptr;
    if (!first || !optional_tensor(args[1], *first, &dt, &table) || !table || !optional_tensor(args[2], *first, &di, &indptr) || !indptr || total < 0 ||
        !THPDtype_Check(args[4]))
        Py_RETURN_NONE;
    const at::ScalarType type = reinterpret_cast<THPDtype*>(args[4])->scalar_type;
    if (!io_type(type)) Py_RETURN_NONE;
    at::Tensor k = new_tensor({total, first->size(1), first->size(3)}, type, *first), v = new_tensor({total, first->size(1), first->size(3)}, type, *first);
    if (!describe(k, &dk) || !describe(v, &dv)) Py_RETURN_NONE;
    const int index = first->get_device();
    const hipStream_t stream = c10::hip::getCurrentHIPStream(index).stream();
    int32_t rc;
    Py_BEGIN_ALLOW_THREADS
    rc = g_kv_read(&dk, &dv, &dc[0], &dc[1], &dc[2], &dc[3], table, indptr, index, (uint64_t)(uintptr_t)stream);
    Py_END_ALLOW_THREADS
    if (!succeeded(rc, "tg_fp8_kv_read")) return nullptr;
    PyObject* tuple = PyTuple_New(2);
    if (!tuple) return nullptr;
    PyTuple_SET_ITEM(tuple, 0, THPVariable_Wrap(std::move(k)));
    PyTuple_SET_ITEM(tuple, 1, THPVariable_Wrap(std::move(v)));
    return tuple;
    END_HANDLE_TH_ERRORS
}

// kv_attention(q, cache, block_table, seq_lens, indptr, sm_scale, window, sink_tokens, out) -> out, or None.  The scratch memory
// is the call's own: torch's allocator orders its reuse by stream and keeps a graph's apart
PyObject* py_kv_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 9) { PyErr_SetString(PyExc_TypeError, "kv_attention takes 9 arguments"); return nullptr; }
    const at::Tensor* q = tensor_of(args[0]);
    tg_tensor dc[4], dq, dout, dt, dl, di, dws;
    const tg_tensor *table, *lens, *indptr, *given;
    const at::Tensor* first = describe_cache(args[1], dc);
    const double scale = PyFloat_AsDouble(args[5]);
    const long window = PyLong_AsLong(args[6]), sinks = PyLong_AsLong(args[7]);
    if (PyErr_Occurred()) return nullptr;
    if (!on_gpu(q) || !first || q->dim() != 3 || q->device() != first->device() || !describe(*q, &dq) || !optional_tensor(args[2], *q, &dt, &table) || !table ||
        !optional_tensor(args[3], *q, &dl, &lens) || !lens || !optional_tensor(args[4], *q, &di, &indptr) || !indptr ||
        !optional_tensor(args[8], *q, &dout, &given) || dt.ndim != 2 || window < 0 || window > INT32_MAX || sinks < 0 || sinks > INT32_MAX)
        Py_RETURN_NONE;
    at::Tensor out, ws;
    if (!given) {
        out = new_tensor(q->sizes(), q->scalar_type(), *q);
        if (!describe(out, &dout)) Py_RETURN_NONE;
    }
    const int64_t need = g_kv_attention_workspace_bytes(q->size(0), q->size(1), dt.shape[0], first->size(1), first->size(3), first->size(2), dt.shape[1],
                                                        (int32_t)window, (int32_t)sinks);
    if (need > 0) {
        ws = new_tensor({need}, at::kByte, *q);
        if (!describe(ws, &dws)) Py_RETURN_NONE;
    }
    const int index = q->get_device();
    const hipStream_t stream = c10::hip::getCurrentHIPStream(index).stream();
    int32_t rc;
    Py_BEGIN_ALLOW_THREADS
    rc = g_kv_attention(&dout, &dq, &dc[0], &dc[1], &dc[2], &dc[3], table, lens, indptr, (float)scale, (int32_t)window, (int32_t)sinks,
                        need > 0 ? &dws : nullptr, index, (uint64_t)(uintptr_t)stream);
    Py_END_ALLOW_THREADS
    if (!succeeded(rc, "tg_fp8_kv_attention")) return nullptr;
    if (given) {
        Py_INCREF(args[8]);
        return args[8];
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// Calls f(device, stream) without the interpreter's lock; false with an exception set.
template <typename F>
bool launched(const at::Tensor& like, const char* where, F f) {
    const int index = like.get_device();
    const uint64_t stream = (uint64_t)(uintptr_t)c10::hip::getCurrentHIPStream(index).stream();
    int32_t rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f(index, stream);
    Py_END_ALLOW_THREADS
    return succeeded(rc, where);
}

PyObject* tuple_of(std::initializer_list<at::Tensor*> tensors) {
    PyObject* tuple = PyTuple_New((Py_ssize_t)tensors.size());
    if (!tuple) return nullptr;
    Py_ssize_t at = 0;
    for (at::Tensor* t : tensors) PyTuple_SET_ITEM(tuple, at++, THPVariable_Wrap(std::move(*t)));
    return tuple;
}

// The given `out` (contiguous, of these sizes and type), or a new tensor.  False: not plain.
bool out_tensor(PyObject* given, at::IntArrayRef sizes, PyObject* dtype, const at::Tensor& like, at::Tensor* out) {
    if (!THPDtype_Check(dtype)) return false;
    const at::ScalarType type = reinterpret_cast<THPDtype*>(dtype)->scalar_type;
    if (!io_type(type)) return false;
    if (given == Py_None) {
        *out = new_tensor(sizes, type, like);
        return true;
    }
    const at::Tensor* t = tensor_of(given);
    if (!on_gpu(t) || t->scalar_type() != type || t->sizes() != sizes || !t->is_contiguous() || t->device() != like.device()) return false;
    *out = *t;
    return true;
}
PyObject* out_or_given(PyObject* given, at::Tensor&& out) {
    if (given == Py_None) return THPVariable_Wrap(std::move(out));
    Py_INCREF(given);
    return given;
}

// int8_matmul(a, b, scale_a, scale_b, bias, out_dtype, out) -> out, or None.  The scratch memory is the call's own
PyObject* py_int8_matmul(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 7) { PyErr_SetString(PyExc_TypeError, "int8_matmul takes 7 arguments"); return nullptr; }
    const at::Tensor *a = tensor_of(args[0]), *b = tensor_of(args[1]);
    if (!on_gpu(a) || a->dim() < 1 || !plain(a, at::kChar, a->dim()) || !plain(b, at::kChar, 2) || a->device() != b->device()) Py_RETURN_NONE;
    const int64_t K = a->size(a->dim() - 1), N = b->size(0);
    if (b->size(1) != K || K == 0) Py_RETURN_NONE;
    const int64_t M = a->numel() / K;
    tg_tensor dsa, dsb, dbias, dws;
    const tg_tensor *sa, *sb, *bias;
    if (!optional_tensor(args[2], *a, &dsa, &sa) || !sa || !optional_tensor(args[3], *a, &dsb, &sb) || !sb || !optional_tensor(args[4], *a, &dbias, &bias))
        Py_RETURN_NONE;
    c10::SmallVector<int64_t, 4> sizes(a->sizes().begin(), a->sizes().end());
    sizes.back() = N;
    at::Tensor c, ws;
    if (!out_tensor(args[6], sizes, args[5], *a, &c)) Py_RETURN_NONE;
    const int64_t need = g_int8_gemm_workspace_bytes(M, N, K, nullptr, 0);
    if (need > 0) {
        ws = new_tensor({need}, at::kByte, *a);
        dws = describe_rows(ws, 1, need);
    }
    const tg_tensor dc = describe_rows(c, M, N), da = describe_rows(*a, M, K), db = describe_rows(*b, N, K);
    if (!launched(*a, "tg_int8_gemm", [&](int32_t device, uint64_t stream) {
            return g_int8_gemm(&dc, &da, &db, sa, sb, bias, need > 0 ? &dws : nullptr, nullptr, 0, device, stream);
        }))
        return nullptr;
    return out_or_given(args[6], std::move(c));
    END_HANDLE_TH_ERRORS
}

// ragged_int8_matmul(a, b, scale_a, scale_b, m_indptr, out_dtype, out) -> out, or None
PyObject* py_ragged_int8_matmul(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 7) { PyErr_SetString(PyExc_TypeError, "ragged_int8_matmul takes 7 arguments"); return nullptr; }
    const at::Tensor *a = tensor_of(args[0]), *b = tensor_of(args[1]);
    if (!plain(a, at::kChar, 2) || !plain(b, at::kChar, 3) || a->device() != b->device() || a->size(1) != b->size(2)) Py_RETURN_NONE;
    tg_tensor dc, da, db, dsa, dsb, dptr;
    const tg_tensor *sa, *sb, *ptr;
    if (!optional_tensor(args[2], *a, &dsa, &sa) || !sa || !optional_tensor(args[3], *a, &dsb, &sb) || !sb || !optional_tensor(args[4], *a, &dptr, &ptr) || !ptr)
        Py_RETURN_NONE;
    at::Tensor c;
    if (!out_tensor(args[6], {a->size(0), b->size(1)}, args[5], *a, &c) || !describe(c, &dc) || !describe(*a, &da) || !describe(*b, &db)) Py_RETURN_NONE;
    if (!launched(*a, "tg_int8_ragged_gemm",
                  [&](int32_t device, uint64_t stream) { return g_int8_ragged_gemm(&dc, &da, &db, sa, sb, ptr, nullptr, 0, device, stream); }))
        return nullptr;
    return out_or_given(args[6], std::move(c));
    END_HANDLE_TH_ERRORS
}

// int8_quant(x, rows, silu_mul) -> (q, scales), or None: rows (T, k) carries each row of x (T, H) to its k places, None leaves them in order
PyObject* py_int8_quant(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 3) { PyErr_SetString(PyExc_TypeError, "int8_quant takes 3 arguments"); return nullptr; }
    const at::Tensor* x = tensor_of(args[0]);
    if (!on_gpu(x) || !io_type(x->scalar_type()) || !x->is_contiguous() || x->dim() < 1 || x->dim() > TG_MAX_DIMS) Py_RETURN_NONE;
    tg_tensor dq, ds, dx, dplace;
    const tg_tensor* place;
    if (!optional_tensor(args[1], *x, &dplace, &place)) Py_RETURN_NONE;
    const bool silu_mul = args[2] == Py_True;
    c10::SmallVector<int64_t, 4> sizes(x->sizes().begin(), x->sizes().end());
    if (place) {
        if (dplace.ndim != 2 || x->dim() != 2 || dplace.shape[0] != sizes[0]) Py_RETURN_NONE;
        sizes[0] *= dplace.shape[1];
    }
    if (silu_mul) {
        if (sizes.back() % 2 != 0) Py_RETURN_NONE;
        sizes.back() /= 2;
    }
    at::Tensor q = new_tensor(sizes, at::kChar, *x), scales = new_tensor(at::IntArrayRef(sizes.data(), sizes.size() - 1), at::kFloat, *x);
    if (!describe(q, &dq) || !describe(scales, &ds) || !describe(*x, &dx)) Py_RETURN_NONE;
    if (!launched(*x, "tg_int8_quant", [&](int32_t device, uint64_t stream) { return g_int8_quant(&dq, &ds, &dx, place, silu_mul, device, stream); }))
        return nullptr;
    return tuple_of({&q, &scales});
    END_HANDLE_TH_ERRORS
}

// moe_sort(ids, num_experts) -> (indptr, rows, slots), or None.  The scratch memory is the call's own
PyObject* py_moe_sort(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 2) { PyErr_SetString(PyExc_TypeError, "moe_sort takes 2 arguments"); return nullptr; }
    const at::Tensor* ids = tensor_of(args[0]);
    const long experts = PyLong_AsLong(args[1]);
    if (PyErr_Occurred()) return nullptr;
    if (!on_gpu(ids) || ids->dim() != 2 || !ids->is_contiguous() || experts < 1 || experts > 512) Py_RETURN_NONE;
    at::Tensor indptr = new_tensor({experts + 1}, at::kInt, *ids), rows = new_tensor(ids->sizes(), at::kInt, *ids), slots = new_tensor({ids->numel()}, at::kInt, *ids);
    tg_tensor di, dp, dr, ds, dws;
    at::Tensor ws;
    const int64_t need = g_moe_sort_workspace_bytes(ids->numel(), (int32_t)experts);
    if (need > 0) {
        ws = new_tensor({need}, at::kByte, *ids);
        dws = describe_rows(ws, 1, need);
    }
    if (!describe(*ids, &di) || !describe(indptr, &dp) || !describe(rows, &dr) || !describe(slots, &ds)) Py_RETURN_NONE;
    if (!launched(*ids, "tg_moe_sort", [&](int32_t device, uint64_t stream) {
            return g_moe_sort(&di, (int32_t)experts, &dp, &dr, &ds, need > 0 ? &dws : nullptr, device, stream);
        }))
        return nullptr;
    return tuple_of({&indptr, &rows, &slots});
    END_HANDLE_TH_ERRORS
}

// A dual tensor of forward-mode differentiation: not plain, the Python implementation refuses it.
bool dual(const at::Tensor* t) { return t && t->_fw_grad(0).defined(); }

// The x (rows, H) and the places (T, k) of the ways there and back; false: not plain.
bool route_operands(PyObject* x, PyObject* rows, const at::Tensor** px, const at::Tensor** prows, tg_tensor* dx, tg_tensor* drows) {
    const at::Tensor *tx = tensor_of(x), *tr = tensor_of(rows);
    if (!on_gpu(tx) || !io_type(tx->scalar_type()) || tx->dim() != 2 || !plain(tr, at::kInt, 2) || tx->device() != tr->device() || dual(tx)) return false;
    *px = tx;
    *prows = tr;
    return describe(*tx, dx) && describe(*tr, drows);
}

// moe_permute(x, rows) -> tensor, or None
PyObject* py_moe_permute(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 2) { PyErr_SetString(PyExc_TypeError, "moe_permute takes 2 arguments"); return nullptr; }
    const at::Tensor *x, *rows;
    tg_tensor dout, dx, drows;
    if (!route_operands(args[0], args[1], &x, &rows, &dx, &drows) || x->size(0) != rows->size(0)) Py_RETURN_NONE;
    at::Tensor out = new_tensor({rows->numel(), x->size(1)}, x->scalar_type(), *x);
    if (!describe(out, &dout)) Py_RETURN_NONE;
    if (!launched(*x, "tg_moe_permute", [&](int32_t device, uint64_t stream) { return g_moe_permute(&dout, &dx, &drows, device, stream); })) return nullptr;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// moe_unpermute(x, rows, weights) -> tensor, or None
PyObject* py_moe_unpermute(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 3) { PyErr_SetString(PyExc_TypeError, "moe_unpermute takes 3 arguments"); return nullptr; }
    const at::Tensor *x, *rows;
    tg_tensor dout, dx, drows, dw;
    const tg_tensor* weights;
    if (!route_operands(args[0], args[1], &x, &rows, &dx, &drows) || x->size(0) != rows->numel() || !optional_tensor(args[2], *x, &dw, &weights) || dual(tensor_of(args[2])))
        Py_RETURN_NONE;
    at::Tensor out = new_tensor({rows->size(0), x->size(1)}, x->scalar_type(), *x);
    if (!describe(out, &dout)) Py_RETURN_NONE;
    if (!launched(*x, "tg_moe_unpermute", [&](int32_t device, uint64_t stream) { return g_moe_unpermute(&dout, &dx, &drows, weights, device, stream); }))
        return nullptr;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// moe_unpermute_backward(grad_out, x, rows, weights) -> (grad_x, grad_weights), or None
PyObject* py_moe_unpermute_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4) { PyErr_SetString(PyExc_TypeError, "moe_unpermute_backward takes 4 arguments"); return nullptr; }
    const at::Tensor *x, *rows, *grad = tensor_of(args[0]), *weights = tensor_of(args[3]);
    tg_tensor dgx, dgw, dgrad, dx, drows, dw;
    if (!route_operands(args[1], args[2], &x, &rows, &dx, &drows) || !on_gpu(grad) || grad->device() != x->device() || !grad->is_contiguous() ||
        !on_gpu(weights) || weights->device() != x->device() || !io_type(weights->scalar_type()) || dual(grad) || dual(weights) || !describe(*grad, &dgrad) || !describe(*weights, &dw))
        Py_RETURN_NONE;
    at::Tensor gx = new_tensor(x->sizes(), x->scalar_type(), *x), gw = new_tensor(weights->sizes(), weights->scalar_type(), *x);
    if (!describe(gx, &dgx) || !describe(gw, &dgw)) Py_RETURN_NONE;
    if (!launched(*x, "tg_moe_unpermute_backward", [&](int32_t device, uint64_t stream) {
            return g_moe_unpermute_backward(&dgx, &dgw, &dgrad, &dx, &drows, &dw, device, stream);
        }))
        return nullptr;
    return tuple_of({&gx, &gw});
    END_HANDLE_TH_ERRORS
}

// int8_moe(x, w1, w2, w1_scale, w2_scale, topk_weights, topk_ids) -> tensor, or None: the layer's six launches one after the other, what lies between
// them in one allocation of the call's own
PyObject* py_int8_moe(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 7) { PyErr_SetString(PyExc_TypeError, "int8_moe takes 7 arguments"); return nullptr; }
    const at::Tensor *x = tensor_of(args[0]), *w1 = tensor_of(args[1]), *w2 = tensor_of(args[2]), *s1 = tensor_of(args[3]), *s2 = tensor_of(args[4]),
                     *tw = tensor_of(args[5]), *ids = tensor_of(args[6]);
    if (!on_gpu(x) || (x->scalar_type() != at::kBFloat16 && x->scalar_type() != at::kHalf) || x->dim() != 2 || !x->is_contiguous() || !plain(w1, at::kChar, 3) ||
        !plain(w2, at::kChar, 3) || !on_gpu(s1) || !plain(s1, at::kFloat, s1->dim()) || !on_gpu(s2) || !plain(s2, at::kFloat, s2->dim()) || !on_gpu(tw) ||
        tw->dim() != 2 || !io_type(tw->scalar_type()) || !tw->is_contiguous() || !on_gpu(ids) || ids->dim() != 2 || !ids->is_contiguous() ||
        (ids->scalar_type() != at::kInt && ids->scalar_type() != at::kLong))
        Py_RETURN_NONE;
    for (const at::Tensor* t : {w1, w2, s1, s2, tw, ids})
        if (t->device() != x->device()) Py_RETURN_NONE;
    const int64_t T = x->size(0), H = x->size(1), E = w1->size(0), I = w2->size(2), k = ids->size(1), rows = T * k;
    if (T < 1 || k < 1 || H < 1 || I < 1 || E < 1 || E > 512 || rows > INT32_MAX || ids->size(0) != T || tw->sizes() != ids->sizes() || w1->size(1) != 2 * I ||
        w1->size(2) != H || w2->size(0) != E || w2->size(1) != H)
        Py_RETURN_NONE;
    tg_tensor dx, dw1, dw2, ds1, ds2, dtw, dids, dout;
    at::Tensor out = new_tensor({T, H}, x->scalar_type(), *x);
    if (!describe(*x, &dx) || !describe(*w1, &dw1) || !describe(*w2, &dw2) || !describe(*s1, &ds1) || !describe(*s2, &ds2) || !describe(*tw, &dtw) ||
        !describe(*ids, &dids) || !describe(out, &dout))
        Py_RETURN_NONE;
    const int io = dtype_code(x->scalar_type());
    const int64_t sort_bytes = g_moe_sort_workspace_bytes(rows, (int32_t)E);
    // (at, shape, type) of what lies between; a buffer is used again once what it held has been read
    int64_t bytes = 0;
    auto room = [&](int64_t size) { const int64_t at = bytes; bytes += (size + 255) / 256 * 256; return at; };
    auto matrix = [](int64_t at, int64_t r, int64_t c, int type) {
        tg_tensor d{};
        d.ptr = (uint64_t)at;
        d.ndim = 2;
        d.dtype = type;
        d.shape[0] = r, d.shape[1] = c;
        d.strides[0] = c, d.strides[1] = 1;
        return d;
    };
    auto vector = [&](int64_t at, int64_t r, int type) {
        tg_tensor d = matrix(at, r, 1, type);
        d.ndim = 1;
        d.strides[0] = 1, d.shape[1] = d.strides[1] = 0;
        return d;
    };
    tg_tensor dptr = vector(room((E + 1) * 4), E + 1, TG_I32), drows = matrix(room(rows * 4), T, k, TG_I32), dslots = vector(room(rows * 4), rows, TG_I32);
    tg_tensor dsort = vector(room(sort_bytes), sort_bytes, 6);
    const int64_t codes = room(rows * std::max(H, I)), scales = room(rows * 4), wide = room(rows * std::max(2 * I, H) * 2);
    tg_tensor dq = matrix(codes, rows, H, TG_I8), ds = vector(scales, rows, TG_F32), dh = matrix(wide, rows, 2 * I, io);
    // (dy in x's type: one more rounding of each row for half the bytes of what is written and gathered; rows_dtype asks for them whole, one operator after the other)
    tg_tensor dq2 = matrix(codes, rows, I, TG_I8), dy = matrix(wide, rows, H, io);
    at::Tensor scratch = new_tensor({bytes}, at::kByte, *x);
    const uint64_t base = reinterpret_cast<uint64_t>(scratch.data_ptr());
    for (tg_tensor* d : {&dptr, &drows, &dslots, &dsort, &dq, &ds, &dh, &dq2, &dy}) d->ptr += base;
    const char* where = "";
    const int index = x->get_device();
    const uint64_t stream = (uint64_t)(uintptr_t)c10::hip::getCurrentHIPStream(index).stream();
    int32_t rc = TG_OK;
    Py_BEGIN_ALLOW_THREADS
    auto step = [&](const char* name, auto f) {
        if (rc == TG_OK) where = name, rc = f();
    };
    step("tg_moe_sort", [&] { return g_moe_sort(&dids, (int32_t)E, &dptr, &drows, &dslots, sort_bytes > 0 ? &dsort : nullptr, index, stream); });
    step("tg_int8_quant", [&] { return g_int8_quant(&dq, &ds, &dx, &drows, 0, index, stream); });
    step("tg_int8_ragged_gemm", [&] { return g_int8_ragged_gemm(&dh, &dq, &dw1, &ds, &ds1, &dptr, nullptr, 0, index, stream); });
    step("tg_int8_quant", [&] { return g_int8_quant(&dq2, &ds, &dh, nullptr, 1, index, stream); });
    step("tg_int8_ragged_gemm", [&] { return g_int8_ragged_gemm(&dy, &dq2, &dw2, &ds, &ds2, &dptr, nullptr, 0, index, stream); });
    step("tg_moe_unpermute", [&] { return g_moe_unpermute(&dout, &dy, &drows, &dtw, index, stream); });
    Py_END_ALLOW_THREADS
    if (!succeeded(rc, where)) return nullptr;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// ---- the ways there and back with their gradients.  Their backward passes run in torch's threads, without the interpreter: nothing below calls into it
uint64_t stream_of(const at::Tensor& t) { return (uint64_t)(uintptr_t)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
tg_tensor described(const at::Tensor& t) {
    tg_tensor d;
    TORCH_CHECK(describe(t, &d), "not a tensor of the C ABI");
    return d;
}
void check(int32_t rc, const char* where) { TORCH_CHECK(rc == TG_OK, where, ": rc=", rc, ": ", g_last_error()); }

at::Tensor permuted(const at::Tensor& x, const at::Tensor& rows) {
    at::Tensor out = new_tensor({rows.numel(), x.size(1)}, x.scalar_type(), x);
    const tg_tensor dout = described(out), dx = described(x), drows = described(rows);
    check(g_moe_permute(&dout, &dx, &drows, x.get_device(), stream_of(x)), "tg_moe_permute");
    return out;
}
at::Tensor unpermuted(const at::Tensor& x, const at::Tensor& rows, const at::Tensor& weights) {
    at::Tensor out = new_tensor({rows.size(0), x.size(1)}, x.scalar_type(), x);
    const tg_tensor dout = described(out), dx = described(x), drows = described(rows), dw = weights.defined() ? described(weights) : tg_tensor{};
    check(g_moe_unpermute(&dout, &dx, &drows, weights.defined() ? &dw : nullptr, x.get_device(), stream_of(x)), "tg_moe_unpermute");
    return out;
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A backward pass has no gradient of its own: where a graph of it is made, it ends in an error.
variable_list once(variable_list made) {
    if (!c10::GradMode::is_enabled()) return made;
    variable_list ends;
    for (at::Tensor& t : made)
        if (t.defined()) ends.push_back(t.detach().requires_grad_());
    auto error = std::make_shared<torch::autograd::DelayedError>("the gradients of moe_permute and moe_unpermute cannot be differentiated again", (int64_t)ends.size());
    ends = (*error)(std::move(ends));
    size_t at = 0;
    for (at::Tensor& t : made)
        if (t.defined()) t = ends[at++];
    return made;
}

struct Permute : torch::autograd::Function<Permute> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& rows) {
        ctx->save_for_backward({rows});
        return permuted(x, rows);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        return once({unpermuted(grads[0].contiguous(), ctx->get_saved_variables()[0], at::Tensor()), at::Tensor()});
    }
};
struct Unpermute : torch::autograd::Function<Unpermute> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& rows, const std::optional<at::Tensor>& weights) {
        ctx->save_for_backward(weights ? variable_list{rows, x, *weights} : variable_list{rows});
        return unpermuted(x, rows, weights ? *weights : at::Tensor());
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const at::Tensor grad = grads[0].contiguous();
        if (saved.size() == 1) return once({permuted(grad, saved[0]), at::Tensor(), at::Tensor()});
        const at::Tensor &rows = saved[0], &x = saved[1], &weights = saved[2];
        at::Tensor gx = new_tensor(x.sizes(), x.scalar_type(), x), gw = new_tensor(weights.sizes(), weights.scalar_type(), x);
        const tg_tensor dgx = described(gx), dgw = described(gw), dgrad = described(grad), dx = described(x), drows = described(rows), dw = described(weights);
        check(g_moe_unpermute_backward(&dgx, &dgw, &dgrad, &dx, &drows, &dw, x.get_device(), stream_of(x)), "tg_moe_unpermute_backward");
        return once({gx, at::Tensor(), gw});
    }
};

// moe_permute_grad(x, rows) -> tensor with a gradient, or None
PyObject* py_moe_permute_grad(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 2) { PyErr_SetString(PyExc_TypeError, "moe_permute_grad takes 2 arguments"); return nullptr; }
    const at::Tensor *x, *rows;
    tg_tensor dx, drows;
    if (!route_operands(args[0], args[1], &x, &rows, &dx, &drows) || !x->is_contiguous() || x->size(0) != rows->size(0)) Py_RETURN_NONE;
    return THPVariable_Wrap(Permute::apply(*x, *rows));
    END_HANDLE_TH_ERRORS
}

// moe_unpermute_grad(x, rows, weights) -> tensor with a gradient, or None
PyObject* py_moe_unpermute_grad(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 3) { PyErr_SetString(PyExc_TypeError, "moe_unpermute_grad takes 3 arguments"); return nullptr; }
    const at::Tensor *x, *rows, *weights = args[2] == Py_None ? nullptr : tensor_of(args[2]);
    tg_tensor dx, drows;
    if (!route_operands(args[0], args[1], &x, &rows, &dx, &drows) || !x->is_contiguous() || x->size(0) != rows->numel() ||
        (args[2] != Py_None && (!on_gpu(weights) || dual(weights) || weights->device() != x->device() || !io_type(weights->scalar_type()) || !weights->is_contiguous() ||
                                weights->sizes() != rows->sizes())))
        Py_RETURN_NONE;
    return THPVariable_Wrap(Unpermute::apply(*x, *rows, weights ? std::optional<at::Tensor>(*weights) : std::nullopt));
    END_HANDLE_TH_ERRORS
}

// leaf_held(t) -> whether a graph that still lives accumulates into the leaf t on another stream than the current one
PyObject* py_leaf_held(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const at::Tensor* t = n == 1 ? tensor_of(args[0]) : nullptr;
    if (!t) { PyErr_SetString(PyExc_TypeError, "leaf_held takes a tensor"); return nullptr; }
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    if (!node) Py_RETURN_FALSE;
    const auto stream = node->stream();
    // (the node's stream is one of the tensor's device type, and equal only to such a one: not to a HIPStream's own c10::Stream)
    if (t->is_cuda() && stream && *stream == c10::impl::VirtualGuardImpl(t->device().type()).getStream(t->device())) Py_RETURN_FALSE;
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// set_up({name: address}, workspaces, workspace_for, check_rc)
PyObject* py_set_up(PyObject*, PyObject* args) {
    PyObject *table, *workspaces, *workspace_for, *check_rc;
    if (!PyArg_ParseTuple(args, "O!O!OO", &PyDict_Type, &table, &PyDict_Type, &workspaces, &workspace_for, &check_rc)) return nullptr;
    auto find = [&](const char* name, auto* slot) {
        PyObject* o = PyDict_GetItemString(table, name);
        const unsigned long long address = o ? PyLong_AsUnsignedLongLong(o) : 0;
        if (!address && !PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "no address for %s", name);
        *slot = reinterpret_cast<std::remove_pointer_t<decltype(slot)>>((uintptr_t)address);
        return !PyErr_Occurred();
    };
    if (!find("tg_fp8_gemm", &g_gemm) || !find("tg_fp8_gemm_workspace_bytes", &g_gemm_workspace_bytes) || !find("tg_fp8_ragged_gemm", &g_ragged_gemm) ||
        !find("tg_fp8_quant_group", &g_quant_group) || !find("tg_fp8_fused_moe", &g_fused_moe) ||
        !find("tg_fp8_rms_norm_quant", &g_rms_norm_quant) || !find("tg_fp8_kv_append", &g_kv_append) || !find("tg_fp8_kv_read", &g_kv_read) ||
        !find("tg_fp8_kv_attention", &g_kv_attention) || !find("tg_fp8_kv_attention_workspace_bytes", &g_kv_attention_workspace_bytes) ||
        !find("tg_fp8_fused_moe_block_m", &g_fused_moe_block_m) || !find("tg_fp8_fused_moe_workspace_bytes", &g_fused_moe_workspace_bytes) ||
        !find("tg_int8_gemm", &g_int8_gemm) || !find("tg_int8_gemm_workspace_bytes", &g_int8_gemm_workspace_bytes) ||
        !find("tg_int8_ragged_gemm", &g_int8_ragged_gemm) || !find("tg_int8_quant", &g_int8_quant) || !find("tg_moe_sort", &g_moe_sort) ||
        !find("tg_last_error", &g_last_error) || !find("tg_moe_sort_workspace_bytes", &g_moe_sort_workspace_bytes) ||
        !find("tg_moe_permute", &g_moe_permute) || !find("tg_moe_unpermute", &g_moe_unpermute) ||
        !find("tg_moe_unpermute_backward", &g_moe_unpermute_backward))
        return nullptr;
    for (auto [slot, o] : {std::pair{&g_workspaces, workspaces}, std::pair{&g_workspace_for, workspace_for}, std::pair{&g_check_rc, check_rc}}) {
        Py_INCREF(o);
        Py_XDECREF(*slot);
        *slot = o;
    }
    Py_RETURN_NONE;
}

#define TG_FAST(name, fn) {name, (PyCFunction)(void (*)(void))fn, METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {TG_FAST("matmul", py_matmul),
                          TG_FAST("gemm", py_gemm),
                          TG_FAST("block_matmul", py_block_matmul),
                          TG_FAST("act_quant", py_act_quant),
                          TG_FAST("ragged_matmul", py_ragged_matmul),
                          TG_FAST("fused_moe", py_fused_moe),
                          TG_FAST("rms_norm_quant", py_rms_norm_quant),
                          TG_FAST("kv_append", py_kv_append),
                          TG_FAST("kv_read", py_kv_read),
                          TG_FAST("kv_attention", py_kv_attention),
                          TG_FAST("int8_matmul", py_int8_matmul),
                          TG_FAST("ragged_int8_matmul", py_ragged_int8_matmul),
                          TG_FAST("int8_quant", py_int8_quant),
                          TG_FAST("moe_sort", py_moe_sort),
                          TG_FAST("moe_permute", py_moe_permute),
                          TG_FAST("moe_unpermute", py_moe_unpermute),
                          TG_FAST("moe_unpermute_backward", py_moe_unpermute_backward),
                          TG_FAST("int8_moe", py_int8_moe),
                          TG_FAST("moe_permute_grad", py_moe_permute_grad),
                          TG_FAST("moe_unpermute_grad", py_moe_unpermute_grad),
                          TG_FAST("leaf_held", py_leaf_held),
                          {"set_up", py_set_up, METH_VARARGS, nullptr},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native() { return PyModule_Create(&kModule); }
