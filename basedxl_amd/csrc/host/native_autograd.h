// What the differentiable functions of the host extension share.
#pragma once
#include "native_common.h"

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <optional>

namespace native {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

inline void check(int st, const char* where) { TORCH_CHECK(st == CASCMM_OK, where, " failed: ", cascmm_strerror(st), " (status ", st, ")"); }

inline hipStream_t stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
inline const void* data_of(const at::Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
inline at::Tensor scratch(size_t bytes, const at::Tensor& like) { return at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(like.device())); }
inline at::Tensor fresh(at::IntArrayRef sizes, const at::Tensor& like) { return at::empty(sizes, at::TensorOptions().dtype(like.scalar_type()).device(like.device())); }

// rows of `t` (all of it known not to be empty), copied where its strides are not those of rows
inline at::Tensor as_rows(const at::Tensor& t, int64_t& rows, int64_t& cols, int64_t& ld) {
  if (rows_of(t, rows, cols, ld)) return t;
  at::Tensor c = t.contiguous();
  rows_of(c, rows, cols, ld);
  return c;
}

inline bool differentiated(std::initializer_list<const at::Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : tensors)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
// gradients that are asked to be differentiated again say so when they are (what once_differentiable does for a Python function)
inline variable_list once(variable_list grads, const char* name, bool again) {
  if (!again) return grads;
  at::AutoGradMode enabled(true);
  for (at::Tensor& g : grads)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  auto raise = std::make_shared<torch::autograd::DelayedError>(std::string("trying to differentiate twice a function that is differentiable once: ") + name, (int64_t)grads.size());
  return (*raise)(std::move(grads));
}

// An optional input of a node: those that are there count among the node's edges, in the order of the arguments
typedef std::optional<at::Tensor> Optional;
inline Optional optional_of(const at::Tensor& t) { return t.defined() ? Optional(t) : std::nullopt; }
inline at::Tensor tensor_of(const Optional& t) { return t ? *t : at::Tensor(); }
struct Wanted {
  AutogradContext* ctx;
  size_t edge = 0;
  bool next(bool there = true) { return there && ctx->needs_input_grad(edge++); }
};

// a tensor whose forward-mode tangent would be lost here (the wrapper raises)
inline bool dual(std::initializer_list<const at::Tensor*> tensors) {
  for (const at::Tensor* t : tensors)
    if (t->defined() && t->_fw_grad(0).defined()) return true;
  return false;
}

// a tensor or None (undefined); false: not the ordinary case
inline bool optional_tensor(PyObject* o, int device, at::Tensor& t) {
  if (o == Py_None) return true;
  const at::Tensor* p = gpu_tensor(o, device);
  if (!p) return false;
  t = *p;
  return true;
}

}  // namespace native
