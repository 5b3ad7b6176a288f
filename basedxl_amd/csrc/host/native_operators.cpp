// The host path of ordinary eager calls of layer norm and of products with an epilogue, and of their gradients.
//
// A norm of a transformer block is 5 - 10 us on the GPU; issued from Python (checks, views, a ctypes call of twenty arguments) it took 15 us of host
// time, and a forward and backward pass through Python autograd functions 180.  As in native.cpp everything here is a short cut: a function
// returns None whenever a call is not the ordinary case and the Python code, which holds all rules and raises all errors, takes it from the start.
// The gradients' nodes are the counterparts of the Python autograd functions (layer_norm.py, matmul_epilogue.py), and like them differentiable once.
#include "native_autograd.h"

#include "native_operators.h"

#include <mutex>

namespace native {
namespace {

// 16-bit operands off dwords: what the library copies of them beyond what cascmm_workspace_bytes counts, and copies made here where the library makes none (_copied_bytes
// and _kernel_rows of matmul_epilogue.py)
bool off_dwords(const at::Tensor& t, int64_t cols, int64_t ld, int unit) {
  return t.element_size() == 2 && cols % unit == 0 && ((uintptr_t)t.const_data_ptr() % 4 != 0 || ld % 2 != 0);
}
int64_t copied_rows(const at::Tensor& a, int64_t M, int64_t K, int64_t lda) { return off_dwords(a, K, lda, 8) ? M * ((2 * K + 127) / 128 * 128) + 256 : 0; }
int64_t copied_weight(const at::Tensor& b, int64_t K, int64_t N) { return off_dwords(b, N, N, 2) ? (K + 31) / 32 * 64 * N + 256 : 0; }
at::Tensor kernel_rows(const at::Tensor& t, int64_t cols, int64_t& ld, bool copy) {
  if (t.element_size() != 2 || (!copy && (ld == cols || ld * 2 * 512 < INT32_MAX))) return t;
  ld = cols;
  return t.clone(at::MemoryFormat::Contiguous);
}

// ---------------------------------------------------------------------------------------
// layer norm
// ---------------------------------------------------------------------------------------
struct Normed { at::Tensor y, sum, mean, rstd; };

int weight_code(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias) {
  return dtype_code(weight.defined() ? weight : bias.defined() ? bias : x);
}

Normed norm_forward(const at::Tensor& x, const at::Tensor& residual, const at::Tensor& weight, const at::Tensor& bias, double eps, bool keep) {
  Normed n;
  int64_t rows, cols, ldx, rows_r, cols_r, ldr = 0;
  rows_of(x, rows, cols, ldx);
  n.y = fresh(x.sizes(), x);
  if (residual.defined()) {
    rows_of(residual, rows_r, cols_r, ldr);
    n.sum = fresh(x.sizes(), x);
  }
  if (keep) {
    const auto f32 = at::TensorOptions().dtype(at::kFloat).device(x.device());
    n.mean = at::empty({rows}, f32);
    n.rstd = at::empty({rows}, f32);
  }
  check(cascmm_layer_norm(x.const_data_ptr(), data_of(residual), data_of(weight), data_of(bias), n.y.data_ptr(), n.sum.defined() ? n.sum.data_ptr() : nullptr,
                          keep ? (float*)n.mean.data_ptr() : nullptr, keep ? (float*)n.rstd.data_ptr() : nullptr, rows, cols, ldx, ldr, cols, cols, (float)eps,
                          dtype_code(x), weight_code(x, weight, bias), stream_of(x)),
        "cascmm_layer_norm");
  return n;
}

// {dx, dweight, dbias}, undefined where not wanted; s: what was normed
variable_list norm_backward(const at::Tensor& dy, const at::Tensor& ds, const at::Tensor& s, const at::Tensor& weight, const at::Tensor& bias, const at::Tensor& mean,
                            const at::Tensor& rstd, bool want_x, bool want_weight, bool want_bias) {
  variable_list out(3);
  if (!want_x && !want_weight && !want_bias) return out;
  int64_t rows, cols, lds, lddy, ldds = 0;
  const at::Tensor s2 = as_rows(s, rows, cols, lds), dy2 = as_rows(dy, rows, cols, lddy);
  at::Tensor ds2, ws;
  if (ds.defined()) ds2 = as_rows(ds, rows, cols, ldds);
  if (want_x) out[0] = fresh(s.sizes(), s);
  if (want_weight) out[1] = fresh({cols}, weight);
  if (want_bias) out[2] = fresh({cols}, bias);
  if (want_weight || want_bias) ws = scratch(cascmm_layer_norm_workspace_bytes(rows, cols, dtype_code(s)), s);
  auto ptr = [](const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
  check(cascmm_layer_norm_backward(dy2.const_data_ptr(), data_of(ds2), s2.const_data_ptr(), data_of(weight), (const float*)mean.const_data_ptr(),
                                   (const float*)rstd.const_data_ptr(), ptr(out[0]), ptr(out[1]), ptr(out[2]), rows, cols, lddy, ldds, lds, cols, dtype_code(s),
                                   weight_code(s, weight, bias), ptr(ws), ws.defined() ? ws.nbytes() : 0, stream_of(s)),
        "cascmm_layer_norm_backward");
  return out;
}

struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const Optional& w, const Optional& b, double eps) {
    const at::Tensor weight = tensor_of(w), bias = tensor_of(b);
    Normed n = norm_forward(x, at::Tensor(), weight, bias, eps, true);
    ctx->save_for_backward({x, weight, bias, n.mean, n.rstd});
    return n.y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list v = ctx->get_saved_variables();
    const bool again = at::GradMode::is_enabled();
    at::NoGradGuard none;
    Wanted wanted{ctx};
    const bool want_x = wanted.next(), want_weight = wanted.next(v[1].defined()), want_bias = wanted.next(v[2].defined());
    variable_list g = norm_backward(grads[0], at::Tensor(), v[0], v[1], v[2], v[3], v[4], want_x, want_weight, want_bias);
    return once({g[0], g[1], g[2], at::Tensor()}, "layer_norm", again);
  }
};

struct AddLayerNormNode : torch::autograd::Function<AddLayerNormNode> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& residual, const Optional& w, const Optional& b, double eps) {
    const at::Tensor weight = tensor_of(w), bias = tensor_of(b);
    Normed n = norm_forward(x, residual, weight, bias, eps, true);
    ctx->save_for_backward({n.sum, weight, bias, n.mean, n.rstd});
    ctx->set_materialize_grads(false);
    return {n.y, n.sum};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    Wanted wanted{ctx};
    const bool want_x = wanted.next(), want_r = wanted.next();
    const at::Tensor none;
    if (!grads[0].defined())   // (the norm's result was not used: the sum's gradient passes through)
      return {want_x ? grads[1] : none, want_r ? grads[1] : none, none, none, none};
    const variable_list v = ctx->get_saved_variables();
    const bool want_weight = wanted.next(v[1].defined()), want_bias = wanted.next(v[2].defined()), again = at::GradMode::is_enabled();
    at::NoGradGuard guard;
    variable_list g = norm_backward(grads[0], grads[1], v[0], v[1], v[2], v[3], v[4], want_x || want_r, want_weight, want_bias);
    return once({want_x ? g[0] : none, want_r ? g[0] : none, g[1], g[2], none}, "add_layer_norm", again);
  }
};

// the checks of layer_norm.py; false: not the ordinary case
bool norm_arguments(PyObject* const* args, int device, const at::Tensor*& x, at::Tensor& weight, at::Tensor& bias, PyObject* eps_arg, double& eps) {
  x = gpu_tensor(args[0], device);
  int64_t rows, cols, ld;
  if (!x || dtype_code(*x) < 0 || !rows_of(*x, rows, cols, ld)) return false;
  eps = PyFloat_AsDouble(eps_arg);
  if (PyErr_Occurred()) { PyErr_Clear(); return false; }
  if (!(eps >= 0) || !(eps < 1e30)) return false;
  if ((weight.defined() && bias.defined() && weight.scalar_type() != bias.scalar_type()) || dual({x, &weight, &bias})) return false;
  for (const at::Tensor* t : {&weight, &bias})
    if (t->defined() && (t->dim() != 1 || t->size(0) != cols || !t->is_contiguous() || (t->scalar_type() != x->scalar_type() && t->scalar_type() != at::kFloat))) return false;
  return true;
}

// ---------------------------------------------------------------------------------------
// products with an epilogue
// ---------------------------------------------------------------------------------------
// (the backward pass runs without the interpreter lock, which guards workspace_need's memory)
size_t workspace_need_anywhere(const Need& n) {
  static std::mutex mu;
  static std::unordered_map<Need, size_t, NeedHash> memo;
  std::lock_guard<std::mutex> lock(mu);
  auto it = memo.find(n);
  if (it != memo.end()) return it->second;
  if (memo.size() >= 4096) memo.clear();
  return memo[n] = cascmm_workspace_bytes(n.M, n.N, n.K, n.dt, n.fmt, n.terms, n.products);
}

// C = A . B of raw operands with a workspace of the call's own
void product(const void* A, int64_t lda, const void* B, int64_t ldb, at::Tensor& C, int64_t M, int64_t N, int64_t K, int fmt, int terms, int products) {
  const int dt = dtype_code(C);
  const size_t need = workspace_need_anywhere({M, N, K, dt, fmt, terms, products});
  at::Tensor ws;
  if (need) ws = scratch(need, C);
  check(cascmm_gemm(A, B, C.data_ptr(), nullptr, M, N, K, lda, ldb, N, dt, fmt, terms, products, nullptr, need ? ws.data_ptr() : nullptr, need, stream_of(C)), "cascmm_gemm");
}

struct EpilogueNode : torch::autograd::Function<EpilogueNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& a, const at::Tensor& b, const Optional& bias_in, const Optional& residual_in, int64_t act, int64_t fmt,
                            int64_t terms, int64_t products) {
    const at::Tensor bias = tensor_of(bias_in), residual = tensor_of(residual_in);
    int64_t M, K, lda, rows_r, cols_r, ldr = 0;
    rows_of(a, M, K, lda);
    int64_t N = b.size(1), ldb = N;
    const at::Tensor a_rows = kernel_rows(a, K, lda, copied_rows(a, M, K, lda) > INT32_MAX), b_rows = kernel_rows(b, N, ldb, copied_weight(b, K, N) > INT32_MAX);
    if (residual.defined()) rows_of(residual, rows_r, cols_r, ldr);
    at::Tensor out = result_like(a, N), preact, ws;
    if (act) preact = fresh({M, N}, a);
    const int dt = dtype_code(a);
    const size_t need = workspace_need_anywhere({M, N, K, dt, (int)fmt, (int)terms, (int)products}) + copied_rows(a_rows, M, K, lda) + copied_weight(b_rows, K, N);
    if (need) ws = scratch(need, a);
    check(cascmm_gemm_epilogue(a_rows.const_data_ptr(), b_rows.const_data_ptr(), 0, out.data_ptr(), data_of(bias), data_of(residual), act ? preact.data_ptr() : nullptr, M, N, K, lda, N,
                               N, ldr, N, dt, (int)fmt, (int)terms, (int)products, (int)act, nullptr, need ? ws.data_ptr() : nullptr, need, stream_of(a)),
          "cascmm_gemm_epilogue");
    ctx->save_for_backward({a, b, preact});
    ctx->saved_data["how"] = std::vector<int64_t>{act, fmt, terms, products, bias.defined(), residual.defined()};
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list v = ctx->get_saved_variables();
    const std::vector<int64_t> how = ctx->saved_data["how"].toIntVector();
    const int act = (int)how[0], fmt = (int)how[1], terms = (int)how[2], products = (int)how[3];
    Wanted wanted{ctx};
    const bool want_a = wanted.next(), want_b = wanted.next(), want_bias = wanted.next(how[4] != 0), want_residual = wanted.next(how[5] != 0);
    const at::Tensor& b = v[1];
    variable_list out(8);
    {
      at::NoGradGuard none;
      int64_t M, N, K, lda, lddz;
      const at::Tensor a = as_rows(v[0], M, K, lda), dy = as_rows(grads[0], M, N, lddz);
      const int dt = dtype_code(a);
      const hipStream_t stream = stream_of(a);
      // dz, dbias and the products' other operands in one launch
      const bool slope = act && (want_a || want_b);
      at::Tensor dz = dy, ws, at, bt;
      const int64_t lddy = lddz;
      if (slope) {
        dz = fresh({M, N}, a);
        lddz = N;
      }
      if (want_bias) {
        out[2] = fresh({N}, a);
        ws = scratch(cascmm_epilogue_workspace_bytes(M, N, dt), a);
      }
      if (want_b) at = fresh({K, M}, a);
      if (want_a) bt = fresh({N, K}, b);
      auto ptr = [](const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
      check(cascmm_epilogue_backward_operands(dy.const_data_ptr(), data_of(v[2]), slope ? dz.data_ptr() : nullptr, ptr(out[2]), a.const_data_ptr(), ptr(at), b.const_data_ptr(),
                                              ptr(bt), M, N, K, lddy, N, N, lda, M, N, K, act, dt, ptr(ws), ws.defined() ? ws.nbytes() : 0, stream),
            "cascmm_epilogue_backward_operands");
      if (want_a || want_b) dz = kernel_rows(dz, N, lddz, off_dwords(dz, N, lddz, 2));
      if (want_a) {
        out[0] = fresh(v[0].sizes(), a);
        product(dz.const_data_ptr(), lddz, bt.const_data_ptr(), K, out[0], M, K, N, fmt, terms, products);
      }
      if (want_b) {
        out[1] = fresh({K, N}, b);
        product(at.const_data_ptr(), M, dz.const_data_ptr(), lddz, out[1], K, N, M, fmt, terms, products);
      }
    }
    if (want_residual) out[3] = grads[0];
    return once(std::move(out), "cascaded_lowp_matmul_epilogue", at::GradMode::is_enabled());
  }
};

// What both forms of the product ask of their common arguments: rows of a, a bias, a residual like the result; false: not the ordinary case
struct Product {
  const at::Tensor* a;
  at::Tensor bias, residual;
  int64_t M, K, lda, ldr;
  int dt, act;
};
bool product_arguments(PyObject* a, PyObject* bias, PyObject* residual, PyObject* act, int device, Product& p) {
  p.a = gpu_tensor(a, device);
  if (!p.a || (p.dt = dtype_code(*p.a)) < 0 || !rows_of(*p.a, p.M, p.K, p.lda)) return false;
  p.act = PyLong_Check(act) ? (int)PyLong_AsLong(act) : -1;
  if (PyErr_Occurred()) { PyErr_Clear(); return false; }
  return p.act >= CASCMM_ACT_NONE && p.act <= CASCMM_ACT_SILU && optional_tensor(bias, device, p.bias) && optional_tensor(residual, device, p.residual);
}
bool result_arguments(Product& p, int64_t N) {
  const at::Tensor& a = *p.a;
  if (p.bias.defined() && (p.bias.dim() != 1 || p.bias.size(0) != N || p.bias.scalar_type() != a.scalar_type() || !p.bias.is_contiguous())) return false;
  p.ldr = 0;
  if (dual({&a, &p.bias, &p.residual})) return false;
  if (!p.residual.defined()) return true;
  int64_t rows, cols;
  if (p.residual.scalar_type() != a.scalar_type() || p.residual.dim() != a.dim() || !rows_of(p.residual, rows, cols, p.ldr) || cols != N) return false;
  for (int64_t d = 0; d + 1 < a.dim(); ++d)
    if (p.residual.size(d) != a.size(d)) return false;
  return true;
}
// (copied: bytes of the workspace for a copy of B)
PyObject* run_product(Product& p, const void* B, int prepared, int64_t copied, int64_t N, int fmt, int terms, int products, int device) {
  const hipStream_t stream = c10::hip::getCurrentHIPStream(device).stream();
  at::Tensor hold;
  void* ws;
  size_t ws_bytes;
  const at::Tensor rows = kernel_rows(*p.a, p.K, p.lda, copied_rows(*p.a, p.M, p.K, p.lda) > INT32_MAX);
  copied += copied_rows(rows, p.M, p.K, p.lda);
  if (!workspace_of(workspace_need({p.M, N, p.K, p.dt, fmt, terms, products}) + copied, device, stream, hold, ws, ws_bytes)) Py_RETURN_NONE;
  at::Tensor out = result_like(*p.a, N);
  const void *A = rows.const_data_ptr(), *bias = data_of(p.bias), *residual = data_of(p.residual);
  void* C = out.data_ptr();
  int st;
  Py_BEGIN_ALLOW_THREADS
  st = cascmm_gemm_epilogue(A, B, prepared, C, bias, residual, nullptr, p.M, N, p.K, p.lda, N, N, p.ldr, 0, p.dt, fmt, terms, products, p.act, nullptr, ws, ws_bytes, stream);
  Py_END_ALLOW_THREADS
  if (st != CASCMM_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
}

}  // namespace

// layer_norm(x, weight | None, bias | None, eps) -> Tensor | None
PyObject* layer_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 4) Py_RETURN_NONE;
  try {
    const int device = c10::hip::current_device();
    const at::Tensor* x;
    at::Tensor weight, bias;
    double eps;
    if (!optional_tensor(args[1], device, weight) || !optional_tensor(args[2], device, bias) || !norm_arguments(args, device, x, weight, bias, args[3], eps)) Py_RETURN_NONE;
    at::Tensor y = differentiated({x, &weight, &bias}) ? LayerNormNode::apply(*x, optional_of(weight), optional_of(bias), eps) : norm_forward(*x, at::Tensor(), weight, bias, eps, false).y;
    return THPVariable_Wrap(std::move(y));
  } catch (...) {
    return not_ordinary();
  }
}

// add_layer_norm(x, residual, weight | None, bias | None, eps) -> (Tensor, Tensor) | None
PyObject* add_layer_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 5) Py_RETURN_NONE;
  try {
    const int device = c10::hip::current_device();
    const at::Tensor *x, *residual = gpu_tensor(args[1], device);
    at::Tensor weight, bias;
    double eps;
    int64_t rows, cols, ld;
    if (!residual || !optional_tensor(args[2], device, weight) || !optional_tensor(args[3], device, bias) || !norm_arguments(args, device, x, weight, bias, args[4], eps))
      Py_RETURN_NONE;
    if (residual->scalar_type() != x->scalar_type() || residual->sizes() != x->sizes() || dual({residual}) || !rows_of(*residual, rows, cols, ld)) Py_RETURN_NONE;
    at::Tensor y, s;
    if (differentiated({x, residual, &weight, &bias})) {
      variable_list both = AddLayerNormNode::apply(*x, *residual, optional_of(weight), optional_of(bias), eps);
      y = both[0];
      s = both[1];
    } else {
      Normed n = norm_forward(*x, *residual, weight, bias, eps, false);
      y = n.y;
      s = n.sum;
    }
    PyObject* py = THPVariable_Wrap(std::move(y));
    PyObject* ps = py ? THPVariable_Wrap(std::move(s)) : nullptr;
    PyObject* both = ps ? PyTuple_Pack(2, py, ps) : nullptr;
    Py_XDECREF(py);
    Py_XDECREF(ps);
    return both;
  } catch (...) {
    return not_ordinary();
  }
}

// epilogue(a, b, bias | None, residual | None, activation, lowp | None, terms | None, products) -> Tensor | None: b a raw [K, N] tensor
PyObject* epilogue(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 8) Py_RETURN_NONE;
  try {
    const int device = c10::hip::current_device();
    Product p;
    const at::Tensor* b = gpu_tensor(args[1], device);
    if (!b || !product_arguments(args[0], args[2], args[3], args[4], device, p)) Py_RETURN_NONE;
    if (b->dim() != 2 || b->scalar_type() != p.a->scalar_type() || !b->is_contiguous() || b->size(0) != p.K || b->size(1) <= 0) Py_RETURN_NONE;
    const int fmt = args[5] != Py_None ? format_code(args[5]) : p.dt == CASCMM_DT_F16 ? CASCMM_FMT_FP16 : CASCMM_FMT_BF16;
    const int terms = args[6] != Py_None ? (PyLong_Check(args[6]) ? (int)PyLong_AsLong(args[6]) : -1) : p.dt == CASCMM_DT_F32 ? 2 : 1;
    const int products = products_code(args[7]);
    if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
    const int64_t N = b->size(1);
    if (fmt < 0 || terms < 1 || products < 0 || !result_arguments(p, N) || dual({b})) Py_RETURN_NONE;
    if (differentiated({p.a, b, &p.bias, &p.residual}))
      return THPVariable_Wrap(EpilogueNode::apply(*p.a, *b, optional_of(p.bias), optional_of(p.residual), (int64_t)p.act, (int64_t)fmt, (int64_t)terms, (int64_t)products));
    int64_t ldb = N;
    const at::Tensor weight = kernel_rows(*b, N, ldb, copied_weight(*b, p.K, N) > INT32_MAX);
    return run_product(p, weight.const_data_ptr(), 0, copied_weight(weight, p.K, N), N, fmt, terms, products, device);
  } catch (...) {
    return not_ordinary();
  }
}

// epilogue_prepared(a, slots, bias | None, residual | None, activation, K, N, fmt, terms, products, dtype of the weight) -> Tensor | None: the operand slots
// of a plain PreparedWeight (not fp8); without gradients
PyObject* epilogue_prepared(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 11) Py_RETURN_NONE;
  try {
    const int device = c10::hip::current_device();
    Product p;
    const at::Tensor* slots = gpu_tensor(args[1], device);
    if (!slots || !product_arguments(args[0], args[2], args[3], args[4], device, p)) Py_RETURN_NONE;
    const int64_t wk = PyLong_AsLongLong(args[5]), N = PyLong_AsLongLong(args[6]);
    const int fmt = (int)PyLong_AsLong(args[7]), terms = (int)PyLong_AsLong(args[8]), products = products_code(args[9]), w_dt = (int)PyLong_AsLong(args[10]);
    if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
    if (fmt == CASCMM_FMT_FP8 || products < 0 || N <= 0 || p.K != wk || p.dt != w_dt || !result_arguments(p, N) || differentiated({p.a, &p.bias, &p.residual})) Py_RETURN_NONE;
    const size_t slot_bytes = cascmm_prepared_bytes(wk, N, fmt, terms);
    if (slots->nbytes() != (slot_bytes > 16 ? slot_bytes : 16)) Py_RETURN_NONE;   // (not this layout: the wrapper raises)
    if (p.dt == CASCMM_DT_F32) {
      if ((uintptr_t)p.a->const_data_ptr() % 16 != 0 || p.lda % 4 != 0) Py_RETURN_NONE;   // (the wrapper copies such rows)
      if (!(fmt == CASCMM_FMT_BF16 && terms == 2 && p.K % 8 == 0) && (p.K % 64 != 0 || N % 4 != 0)) Py_RETURN_NONE;
    } else if (terms != 1 || fmt != (p.dt == CASCMM_DT_F16 ? CASCMM_FMT_FP16 : CASCMM_FMT_BF16)) {   // (rows of any alignment)
      Py_RETURN_NONE;
    }
    return run_product(p, slots->const_data_ptr(), 1, 0, N, fmt, terms, products, device);
  } catch (...) {
    return not_ordinary();
  }
}

}  // namespace native
