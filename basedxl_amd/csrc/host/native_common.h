// What the functions of the host extension share: looking at arguments, workspaces, results.
#pragma once
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <tuple>
#include <unordered_map>

#include "../../../include/cascmm.h"

namespace native {


inline PyObject* g_scales = nullptr;       // the dict {(device index, stream handle): int32[2] tensor} of the fp8 scale searches' scratch
inline PyObject* g_workspaces = nullptr;   // the dict {(device index, stream handle): uint8 tensor} of the Python wrapper

struct Need {
  int64_t M, N, K;
  int dt, fmt, terms, products;
  bool operator==(const Need& o) const {
    return M == o.M && N == o.N && K == o.K && dt == o.dt && fmt == o.fmt && terms == o.terms && products == o.products;
  }
};
struct NeedHash {
  size_t operator()(const Need& n) const {
    uint64_t h = 1469598103934665603ull;
    for (uint64_t v : {(uint64_t)n.M, (uint64_t)n.N, (uint64_t)n.K, (uint64_t)(n.dt | n.fmt << 8 | n.terms << 16 | n.products << 24)})
      h = (h ^ v) * 1099511628211ull;
    return (size_t)h;
  }
};
// cascmm_workspace_bytes per problem (it walks the whole variant table); guarded by the interpreter lock
inline size_t workspace_need(const Need& n) {
  static std::unordered_map<Need, size_t, NeedHash> memo;
  auto it = memo.find(n);
  if (it != memo.end()) return it->second;
  if (memo.size() >= 4096) memo.clear();
  return memo[n] = cascmm_workspace_bytes(n.M, n.N, n.K, n.dt, n.fmt, n.terms, n.products);
}

inline int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return CASCMM_DT_F32;
    case at::kHalf: return CASCMM_DT_F16;
    case at::kBFloat16: return CASCMM_DT_BF16;
    default: return -1;
  }
}
inline int format_code(PyObject* s) {
  if (!PyUnicode_Check(s)) return -1;
  if (PyUnicode_CompareWithASCIIString(s, "bf16") == 0) return CASCMM_FMT_BF16;
  if (PyUnicode_CompareWithASCIIString(s, "fp16") == 0) return CASCMM_FMT_FP16;
  return -1;   // (fp8 products find scales first: a function of their own)
}
inline int products_code(PyObject* s) {
  if (!PyUnicode_Check(s)) return -1;
  if (PyUnicode_CompareWithASCIIString(s, "tri") == 0) return CASCMM_PROD_TRI;
  if (PyUnicode_CompareWithASCIIString(s, "full") == 0) return CASCMM_PROD_FULL;
  return -1;
}

// A native function's answer to an exception, in its handler: None, so that the Python code decides, but for one that Python code raised within the call (a hook of saved tensors, by which
// activation checkpointing ends its second run; a dispatch mode): that is the caller's, and Python code behind it would run the hook once more.
inline PyObject* not_ordinary() {
  try {
    throw;
  } catch (python_error& e) {
    e.restore();
    if (PyErr_Occurred()) return nullptr;
  } catch (...) {
  }
  PyErr_Clear();
  Py_RETURN_NONE;
}

// a plain torch.Tensor or Parameter on the current GPU (no subclass: those may not own memory)
inline const at::Tensor* gpu_tensor(PyObject* o, int device) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.get_device() == device && t.has_storage() ? &t : nullptr;
}
// the left operand as rows of K elements: false where it is not a view of such rows
inline bool rows_of(const at::Tensor& a, int64_t& M, int64_t& K, int64_t& lda) {
  if (a.dim() < 1) return false;
  K = a.size(-1);
  if (K <= 0 || a.numel() == 0) return false;
  M = a.numel() / K;
  if (a.is_contiguous()) lda = K;
  else if (a.dim() == 2 && a.stride(1) == 1 && a.stride(0) >= K) lda = a.stride(0);
  else return false;
  if (M == 1) lda = K;
  return true;
}
// a bias the kernels can read (None: no bias); false: not the ordinary case
inline bool bias_of(PyObject* o, const at::Tensor& a, int64_t n, int device, const void*& ptr) {
  ptr = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* b = gpu_tensor(o, device);
  if (!b || b->dim() != 1 || b->size(0) != n || b->scalar_type() != a.scalar_type() || !b->is_contiguous()) return false;
  ptr = b->const_data_ptr();
  return true;
}
// the stream's workspace if it holds `need` bytes already (eager launches: a recorded one takes the Python path).
// `hold` keeps it until the launch: another thread may replace the dict's entry while this one has given up the lock, and
// memory freed before the launch could be written by work that was enqueued in between
inline bool workspace_of(size_t need, int device, hipStream_t stream, at::Tensor& hold, void*& ptr, size_t& bytes) {
  ptr = nullptr;
  bytes = 0;
  if (need == 0) return true;
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(stream, &cap) != hipSuccess || cap != hipStreamCaptureStatusNone) return false;
  PyObject* key = Py_BuildValue("(iK)", device, (unsigned long long)(uintptr_t)stream);
  if (!key) { PyErr_Clear(); return false; }
  PyObject* ws = PyDict_GetItem(g_workspaces, key);   // borrowed
  Py_DECREF(key);
  if (!ws || !THPVariable_Check(ws)) return false;
  hold = THPVariable_Unpack(ws);
  if ((size_t)hold.numel() < need) return false;
  ptr = hold.data_ptr();
  bytes = (size_t)hold.numel();
  return true;
}
// the stream's scratch of the scale searches, if it exists already and nothing is being recorded; `hold` as above
inline bool scale_scratch_of(int device, hipStream_t stream, at::Tensor& hold, int32_t*& ptr) {
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  if (!g_scales || hipStreamIsCapturing(stream, &cap) != hipSuccess || cap != hipStreamCaptureStatusNone) return false;
  PyObject* key = Py_BuildValue("(iK)", device, (unsigned long long)(uintptr_t)stream);
  if (!key) { PyErr_Clear(); return false; }
  PyObject* t = PyDict_GetItem(g_scales, key);   // borrowed
  Py_DECREF(key);
  if (!t || !THPVariable_Check(t)) return false;
  hold = THPVariable_Unpack(t);
  if (hold.numel() != 2 || hold.scalar_type() != at::kInt) return false;
  ptr = (int32_t*)hold.data_ptr();
  return true;
}
inline at::Tensor result_like(const at::Tensor& a, int64_t n) {
  c10::SmallVector<int64_t, 6> sizes(a.sizes().begin(), a.sizes().end());
  sizes.back() = n;
  return at::empty(sizes, at::TensorOptions().dtype(a.scalar_type()).device(a.device()));
}

}  // namespace native
