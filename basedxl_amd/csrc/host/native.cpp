// The host path of an ordinary eager call in one C++ function: checks, result tensor, stream, workspace and the call
// into libcascmm.so.
//
// A UNet step makes some 500 of these calls, most of them on kernels of 5 - 15 us; issued from Python (argument checks,
// views, torch.empty, a ctypes call of twenty arguments) each took 13 - 21 us of host time, so the GPU waited for the
// host.  Everything here is a short cut: a function returns None whenever a call is not the ordinary case (another
// device, unusual strides, a workspace that has to grow, a status other than 0, ...) and the Python code, which holds
// all rules and raises all errors, takes it from the start.  Nothing is remembered about a tensor.
#include "native_common.h"

#include "native_operators.h"

using namespace native;

namespace {

// matmul(a, b, bias | None, lowp | None, terms | None, products) -> Tensor | None: b a raw [K, N] tensor
PyObject* matmul(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 6) Py_RETURN_NONE;
  try {
    const int device = c10::hip::current_device();
    const at::Tensor *a = gpu_tensor(args[0], device), *b = gpu_tensor(args[1], device);
    if (!a || !b || b->dim() != 2 || b->scalar_type() != a->scalar_type() || !b->is_contiguous()) Py_RETURN_NONE;
    const int dt = dtype_code(*a);
    // the default cascade: two bf16 terms for fp32, one term of their own format for 16-bit tensors
    const int fmt = args[3] != Py_None ? format_code(args[3]) : dt == CASCMM_DT_F16 ? CASCMM_FMT_FP16 : CASCMM_FMT_BF16;
    const int terms = args[4] != Py_None ? (PyLong_Check(args[4]) ? (int)PyLong_AsLong(args[4]) : -1) : dt == CASCMM_DT_F32 ? 2 : 1;
    const int products = products_code(args[5]);
    int64_t M, K, lda;
    const void* bias;
    if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
    if (dt < 0 || fmt < 0 || terms < 1 || products < 0 || !rows_of(*a, M, K, lda) || b->size(0) != K || b->size(1) <= 0) Py_RETURN_NONE;
    const int64_t N = b->size(1);
    if (!bias_of(args[2], *a, N, device, bias)) Py_RETURN_NONE;
    const hipStream_t stream = c10::hip::getCurrentHIPStream(device).stream();
    at::Tensor hold;
    void* ws;
    size_t ws_bytes;
    if (!workspace_of(workspace_need({M, N, K, dt, fmt, terms, products}), device, stream, hold, ws, ws_bytes)) Py_RETURN_NONE;
    at::Tensor out = result_like(*a, N);
    const void *ap = a->const_data_ptr(), *bp = b->const_data_ptr();
    void* cp = out.data_ptr();
    int st;
    Py_BEGIN_ALLOW_THREADS
    st = cascmm_gemm_variant(ap, bp, cp, bias, M, N, K, lda, N, N, dt, fmt, terms, products, nullptr, ws, ws_bytes, stream, -1);
    Py_END_ALLOW_THREADS
    if (st != CASCMM_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

// prepared(a, slots, bias | None, K, N, fmt, terms, products, dtype of the weight, glu, min_rows) -> Tensor | None: the
// operand slots of a PreparedWeight (not fp8); fp32 problems of fewer than min_rows rows are left to the caller
PyObject* prepared(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 11) Py_RETURN_NONE;
  try {
    const int device = c10::hip::current_device();
    const at::Tensor *a = gpu_tensor(args[0], device), *slots = gpu_tensor(args[1], device);
    if (!a || !slots) Py_RETURN_NONE;
    const int64_t wk = PyLong_AsLongLong(args[3]), N = PyLong_AsLongLong(args[4]);
    const int fmt = (int)PyLong_AsLong(args[5]), terms = (int)PyLong_AsLong(args[6]), products = products_code(args[7]);
    const int w_dt = (int)PyLong_AsLong(args[8]), glu = PyObject_IsTrue(args[9]);
    const int64_t min_rows = PyLong_AsLongLong(args[10]);
    if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
    const int dt = dtype_code(*a);
    int64_t M, K, lda;
    const void* bias;
    if (dt < 0 || fmt == CASCMM_FMT_FP8 || products < 0 || N <= 0 || !rows_of(*a, M, K, lda) || K != wk) Py_RETURN_NONE;
    if (!bias_of(args[2], *a, N, device, bias)) Py_RETURN_NONE;
    const size_t slot_bytes = cascmm_prepared_bytes(wk, N, fmt, terms);
    if (slots->nbytes() != (slot_bytes > 16 ? slot_bytes : 16)) Py_RETURN_NONE;   // (not this layout: the wrapper raises)
    const uintptr_t at0 = (uintptr_t)a->const_data_ptr();
    if (at0 % 16 != 0 || (size_t)lda * a->element_size() % 16 != 0) Py_RETURN_NONE;   // (the wrapper copies such rows)
    if (dt == CASCMM_DT_F32) {
      const bool any_rows = fmt == CASCMM_FMT_BF16 && terms == 2 && !glu && K % 8 == 0;
      if (M < min_rows || (!any_rows && (K % 64 != 0 || N % 4 != 0))) Py_RETURN_NONE;
    } else if (dt != w_dt || terms != 1 || K % 8 != 0) {
      Py_RETURN_NONE;
    }
    const hipStream_t stream = c10::hip::getCurrentHIPStream(device).stream();
    at::Tensor hold;
    void* ws = nullptr;
    size_t ws_bytes = 0;
    if (!glu &&
        !workspace_of(workspace_need({M, N, K, dt, fmt, terms, products}), device, stream, hold, ws, ws_bytes))
      Py_RETURN_NONE;
    const int64_t NO = glu ? N / 2 : N;
    at::Tensor out = result_like(*a, NO);
    const void *ap = (const void*)at0, *bp = slots->const_data_ptr();
    void* cp = out.data_ptr();
    int st;
    Py_BEGIN_ALLOW_THREADS
    st = glu ? cascmm_gemm_prepared_glu(1, &ap, &bp, &cp, bias ? &bias : nullptr, M, N, K, lda, NO, dt, fmt, terms, products, nullptr, stream, -1)
             : cascmm_gemm_prepared(1, &ap, &bp, &cp, bias ? &bias : nullptr, M, N, K, lda, NO, dt, fmt, terms, products, nullptr, ws, ws_bytes,
                                    stream, -1);
    Py_END_ALLOW_THREADS
    if (st != CASCMM_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

// fp8(a, b, bias | None, b_exp | None, K, N, terms, products, b is slots) -> Tensor | None: fp8 terms of fp32 tensors, the scale of a found
// in the call; b a raw [K, N] tensor or the operand slots of a PreparedWeight, b_exp its scale exponent (None, raw only: found too)
PyObject* fp8(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 9) Py_RETURN_NONE;
  try {
    const int device = c10::hip::current_device();
    const at::Tensor *a = gpu_tensor(args[0], device), *b = gpu_tensor(args[1], device);
    if (!a || !b) Py_RETURN_NONE;
    int64_t wk = PyLong_AsLongLong(args[4]), N = PyLong_AsLongLong(args[5]);   // (of slots)
    const int terms = PyLong_Check(args[6]) ? (int)PyLong_AsLong(args[6]) : -1, products = products_code(args[7]), slots = PyObject_IsTrue(args[8]);
    if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
    if (!slots) {
      if (b->dim() != 2 || b->scalar_type() != at::kFloat || !b->is_contiguous()) Py_RETURN_NONE;
      wk = b->size(0);
      N = b->size(1);
    }
    const at::Tensor* exp = args[3] == Py_None ? nullptr : gpu_tensor(args[3], device);
    if ((args[3] != Py_None || slots) && (!exp || exp->scalar_type() != at::kInt || exp->numel() != 1)) Py_RETURN_NONE;
    int64_t M, K, lda;
    const void* bias;
    if (a->scalar_type() != at::kFloat || terms < 1 || products < 0 || N <= 0 || !rows_of(*a, M, K, lda) || K != wk) Py_RETURN_NONE;
    if (!bias_of(args[2], *a, N, device, bias)) Py_RETURN_NONE;
    if (slots) {
      const size_t bytes = cascmm_prepared_bytes(wk, N, CASCMM_FMT_FP8, terms);
      if (b->nbytes() != (bytes > 16 ? bytes : 16)) Py_RETURN_NONE;                                    // (not this layout: the wrapper raises)
      if ((uintptr_t)a->const_data_ptr() % 16 != 0 || lda % 4 != 0 || K % 64 != 0 || N % 4 != 0) Py_RETURN_NONE;   // (the wrapper copies such rows)
    }
    const hipStream_t stream = c10::hip::getCurrentHIPStream(device).stream();
    at::Tensor hold, hold_scratch;
    void* ws;
    size_t ws_bytes;
    int32_t* scratch;
    if (!scale_scratch_of(device, stream, hold_scratch, scratch) ||
        !workspace_of(workspace_need({M, N, K, CASCMM_DT_F32, CASCMM_FMT_FP8, terms, products}), device, stream, hold, ws, ws_bytes))
      Py_RETURN_NONE;
    at::Tensor out = result_like(*a, N);
    at::Tensor exps = at::empty({2}, at::TensorOptions().dtype(at::kInt).device(a->device()));
    const void *ap = a->const_data_ptr(), *bp = b->const_data_ptr();
    const int32_t* b_exp = exp ? (const int32_t*)exp->const_data_ptr() : nullptr;
    void* cp = out.data_ptr();
    int32_t* ep = (int32_t*)exps.data_ptr();
    int st;
    Py_BEGIN_ALLOW_THREADS
    if (b_exp) {
      st = cascmm_gemm_fp8_autoscale(ap, bp, slots, cp, bias, M, N, K, lda, N, N, terms, products, b_exp, ep, scratch, ws, ws_bytes, stream);
    } else {
      st = cascmm_tensor_exps(ap, M, K, lda, CASCMM_DT_F32, nullptr, ep, scratch, stream);
      if (st == CASCMM_OK) st = cascmm_tensor_exps(bp, K, N, N, CASCMM_DT_F32, nullptr, ep + 1, scratch, stream);
      if (st == CASCMM_OK) st = cascmm_gemm_variant(ap, bp, cp, bias, M, N, K, lda, N, N, CASCMM_DT_F32, CASCMM_FMT_FP8, terms, products, ep, ws, ws_bytes, stream, -1);
    }
    Py_END_ALLOW_THREADS
    if (st != CASCMM_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

// init_scales(scratch): the dict to look the scale searches' scratch up in
PyObject* init_scales(PyObject*, PyObject* d) {
  if (!PyDict_Check(d)) {
    PyErr_SetString(PyExc_TypeError, "init_scales takes the dict of scale scratch");
    return nullptr;
  }
  Py_INCREF(d);
  Py_XDECREF(g_scales);
  g_scales = d;
  Py_RETURN_NONE;
}

// init(workspaces): the dict to look workspaces up in
PyObject* init(PyObject*, PyObject* d) {
  if (!PyDict_Check(d)) {
    PyErr_SetString(PyExc_TypeError, "init takes the dict of workspaces");
    return nullptr;
  }
  Py_INCREF(d);
  Py_XDECREF(g_workspaces);
  g_workspaces = d;
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"matmul", (PyCFunction)(void (*)(void))matmul, METH_FASTCALL, "raw operands; None: not the ordinary case"},
    {"prepared", (PyCFunction)(void (*)(void))prepared, METH_FASTCALL, "prepared weight; None: not the ordinary case"},
    {"fp8", (PyCFunction)(void (*)(void))fp8, METH_FASTCALL, "fp8 terms, scale found in the call; None: not the ordinary case"},
    {"layer_norm", (PyCFunction)(void (*)(void))layer_norm, METH_FASTCALL, "layer norm, differentiable; None: not the ordinary case"},
    {"add_layer_norm", (PyCFunction)(void (*)(void))add_layer_norm, METH_FASTCALL, "residual add and layer norm, differentiable; None: not the ordinary case"},
    {"epilogue", (PyCFunction)(void (*)(void))epilogue, METH_FASTCALL, "raw operands and an epilogue, differentiable; None: not the ordinary case"},
    {"epilogue_prepared", (PyCFunction)(void (*)(void))epilogue_prepared, METH_FASTCALL, "prepared weight and an epilogue; None: not the ordinary case"},
    {"init_scales", init_scales, METH_O, "hands over the dict of the scale searches' scratch"},
    {"init", init, METH_O, "hands over the workspaces' dict"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_native", "host path of ordinary eager calls", -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&kModule); }
