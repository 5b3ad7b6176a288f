// The host path of ordinary eager calls of block-scaled products, of the norms around a residual add, with their gradients, and of the gradients' norm.
//
// As in native_operators.cpp everything here is a short cut: a function returns None whenever a call is not the ordinary case and the Python code, which holds all rules and raises
// all errors, takes it from the start.  The gradients' nodes are the counterparts of the Python autograd functions (block_scaled.py, gated_norm.py), and like them
// differentiable once.  (From Python a forward and backward pass took 230 us of host time, a call with two operands 30, the table of 400 gradients 600.)
#include "native_autograd.h"

#include "native_operators.h"

#include <ATen/ops/zeros_like.h>

#include <cmath>
#include <vector>

namespace native {
namespace {

constexpr int64_t kMostK = (int64_t)1 << 22;
void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
PyObject* pair(at::Tensor a, at::Tensor b) {
  PyObject* pa = THPVariable_Wrap(std::move(a));
  PyObject* pb = pa ? THPVariable_Wrap(std::move(b)) : nullptr;
  PyObject* both = pb ? PyTuple_Pack(2, pa, pb) : nullptr;
  Py_XDECREF(pa);
  Py_XDECREF(pb);
  return both;
}

// ---------------------------------------------------------------------------------------
// block-scaled products
// ---------------------------------------------------------------------------------------
// a rounded operand: values and, behind them, scales in one piece of memory
struct Held {
  at::Tensor memory;
  int64_t rows = 0, k = 0;
  size_t values_bytes() const { return (cascmm_block_values_bytes(rows, k) + 255) / 256 * 256; }
  void* values() const { return ptr(memory); }
  void* scales() const { return memory.defined() ? (char*)memory.data_ptr() + values_bytes() : nullptr; }
};
Held space(int64_t rows, int64_t k, const at::Tensor& like) {
  Held h{at::Tensor(), rows, k};
  h.memory = scratch(h.values_bytes() + cascmm_block_scales_bytes(rows, k), like);
  return h;
}

struct Rounded { Held along, across; at::Tensor sums; };
Rounded round_rows(const at::Tensor& x, int64_t rows, int64_t cols, int64_t ld, bool square, bool along, bool across, bool sums) {
  Rounded r;
  at::Tensor ws;
  if (along) r.along = space(rows, cols, x);
  if (across) r.across = space(cols, rows, x);
  if (sums) {
    r.sums = fresh({cols}, x);
    ws = scratch(cascmm_block_round_workspace_bytes(rows, cols), x);
  }
  check(cascmm_block_round(x.const_data_ptr(), rows, cols, ld, dtype_code(x), square, r.along.values(), r.along.scales(), r.across.values(), r.across.scales(), ptr(r.sums), ptr(ws),
                           ws.defined() ? ws.nbytes() : 0, stream_of(x)),
        "cascmm_block_round");
  return r;
}
// the order in which a right operand [K, N] lies: rows of it, or of its transpose; false: neither
bool weight_order(const at::Tensor& b, bool& turned, int64_t& ld) {
  const int64_t K = b.size(0), N = b.size(1);
  turned = false;
  if (b.stride(1) == 1 && (K == 1 || b.stride(0) >= N)) { ld = K == 1 ? N : b.stride(0); return true; }
  turned = true;
  if (b.stride(0) == 1 && b.stride(1) >= K) { ld = b.stride(1); return true; }
  return false;
}
struct RoundedWeight { Held forward, backward; };
RoundedWeight round_weight(const at::Tensor& b, bool turned, int64_t ld, bool backward) {
  const int64_t K = b.size(0), N = b.size(1);
  Rounded r = turned ? round_rows(b, N, K, ld, true, true, backward, false) : round_rows(b, K, N, ld, true, backward, true, false);
  if (turned) return {r.along, r.across};
  return {r.across, r.along};
}
void multiply(const Held& a, const Held& b, at::Tensor& out, const void* bias, int64_t M, int64_t N, int64_t K) {
  check(cascmm_block_gemm(a.values(), a.scales(), b.values(), b.scales(), out.data_ptr(), bias, M, N, K, N, dtype_code(out), stream_of(out)), "cascmm_block_gemm");
}
void linear(const at::Tensor& a, int64_t M, int64_t K, int64_t lda, const void* values, const void* scales, at::Tensor& out, const void* bias, int64_t N) {
  const size_t need = cascmm_block_linear_workspace_bytes(M, K, dtype_code(a));
  at::Tensor ws;
  if (need) ws = scratch(need, a);
  check(cascmm_block_linear(a.const_data_ptr(), values, scales, out.data_ptr(), bias, M, N, K, lda, N, dtype_code(a), ptr(ws), need, stream_of(a)), "cascmm_block_linear");
}

struct BlockScaledNode : torch::autograd::Function<BlockScaledNode> {
  // (a's rows and b's order are known to be ordinary)
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& a, const at::Tensor& b, const Optional& bias) {
    int64_t M, K, lda, ldb;
    bool turned;
    rows_of(a, M, K, lda);
    weight_order(b, turned, ldb);
    const int64_t N = b.size(1);
    const at::Tensor add = tensor_of(bias);
    at::Tensor out = result_like(a, N);
    const Rounded left = round_rows(a, M, K, lda, false, true, b.requires_grad(), false);
    const RoundedWeight right = round_weight(b, turned, ldb, a.requires_grad());
    multiply(left.along, right.forward, out, data_of(add), M, N, K);
    ctx->save_for_backward({left.across.memory, right.backward.memory});
    ctx->saved_data["K"] = K;
    ctx->saved_data["bias"] = add.defined();
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list v = ctx->get_saved_variables();
    const bool again = at::GradMode::is_enabled();
    at::NoGradGuard none;
    const int64_t K = ctx->saved_data["K"].toInt();
    Wanted wanted{ctx};
    const bool want_a = wanted.next(), want_b = wanted.next(), want_bias = wanted.next(ctx->saved_data["bias"].toBool());
    int64_t M, N, ld;
    const at::Tensor dy = as_rows(grads[0], M, N, ld);
    Rounded r = round_rows(dy, M, N, ld, false, want_a, want_b, want_bias);
    at::Tensor da, db;
    if (want_a) {
      da = result_like(grads[0], K);
      multiply(r.along, Held{v[1], K, N}, da, nullptr, M, K, N);
    }
    if (want_b) {
      db = fresh({K, N}, dy);
      multiply(Held{v[0], K, M}, r.across, db, nullptr, K, N, M);
    }
    return once({da, db, r.sums}, "block_scaled_matmul", again);
  }
};

// ---------------------------------------------------------------------------------------
// norms around a residual add
// ---------------------------------------------------------------------------------------
struct GatedHow { bool post; int64_t norm; double eps, alpha; };
enum { kWeight, kBias, kGate, kScale, kPostWeight, kPostBias, kParameters };
typedef std::array<at::Tensor, kParameters> Parameters;

// whether a parameter is one row, or one for each entry of x's first axis at any distance from each other (parts of a wider row, as a conditioning's are)
bool parameter_of(const at::Tensor& x, const at::Tensor& t, bool may_group) {
  const int64_t cols = x.size(-1);
  if ((t.scalar_type() != x.scalar_type() && t.scalar_type() != at::kFloat) || t.dim() < 1 || t.size(-1) != cols || (cols > 1 && t.stride(-1) != 1)) return false;
  if (t.numel() == cols) return t.dim() == 1 || t.dim() <= x.dim();
  return may_group && t.dim() == x.dim() && t.size(0) == x.size(0) && t.numel() == t.size(0) * cols && t.stride(0) >= cols;
}
cascmm_gated_norm gated_arguments(const at::Tensor& s, const Parameters& p, const GatedHow& how) {
  cascmm_gated_norm a;
  std::memset(&a, 0, sizeof(a));
  const int64_t cols = s.size(-1), rows = s.numel() / cols;
  bool grouped = false;
  int code = dtype_code(s);
  for (const at::Tensor& t : p)
    if (t.defined()) {
      code = dtype_code(t);
      grouped = grouped || t.numel() > cols;
    }
  auto ld = [&](const at::Tensor& t) { return t.defined() && t.numel() > cols ? t.stride(0) : 0; };
  a.weight = data_of(p[kWeight]); a.bias = data_of(p[kBias]); a.gate = data_of(p[kGate]); a.scale = data_of(p[kScale]);
  a.post_weight = data_of(p[kPostWeight]); a.post_bias = data_of(p[kPostBias]);
  a.rows = rows; a.cols = cols; a.group_rows = grouped ? rows / s.size(0) : rows;
  a.weight_ld = ld(p[kWeight]); a.bias_ld = ld(p[kBias]); a.gate_ld = ld(p[kGate]); a.scale_ld = ld(p[kScale]);
  a.residual_scale = how.alpha; a.eps = how.eps; a.norm = (int)how.norm; a.post = how.post; a.dtype = dtype_code(s); a.weight_dtype = code;
  return a;
}
struct Gated { at::Tensor y, s, stats; };
Gated gated_forward(const at::Tensor& x, const at::Tensor& residual, const Parameters& p, const GatedHow& how, bool keep) {
  Gated g{fresh(x.sizes(), x), fresh(x.sizes(), x), at::Tensor()};
  cascmm_gated_norm a = gated_arguments(g.s, p, how);
  int64_t rows, cols;
  rows_of(x, rows, cols, a.ldx);
  rows_of(residual, rows, cols, a.ldr);
  if (keep) g.stats = at::empty({4, rows}, at::TensorOptions().dtype(at::kFloat).device(x.device()));
  a.x = x.const_data_ptr(); a.residual = residual.const_data_ptr(); a.y = g.y.data_ptr(); a.sum = g.s.data_ptr(); a.stats = (float*)ptr(g.stats);
  a.ldy = a.lds = cols;
  check(cascmm_gated_norm_forward(&a, stream_of(x)), "cascmm_gated_norm_forward");
  return g;
}

struct GatedNode : torch::autograd::Function<GatedNode> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& residual, const Optional& weight, const Optional& bias, const Optional& gate, const Optional& scale,
                               const Optional& post_weight, const Optional& post_bias, bool post, int64_t norm, double eps, double alpha) {
    const Parameters p = {tensor_of(weight), tensor_of(bias), tensor_of(gate), tensor_of(scale), tensor_of(post_weight), tensor_of(post_bias)};
    Gated g = gated_forward(x, residual, p, {post, norm, eps, alpha}, true);
    ctx->save_for_backward({post || p[kGate].defined() ? x : at::Tensor(), p[kScale].defined() ? residual : at::Tensor(), g.s, g.stats, p[0], p[1], p[2], p[3], p[4], p[5]});
    ctx->set_materialize_grads(false);
    ctx->saved_data["post"] = post;
    ctx->saved_data["norm"] = norm;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["alpha"] = alpha;
    return {g.y, g.s};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(12);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    const variable_list v = ctx->get_saved_variables();
    const bool again = at::GradMode::is_enabled();
    at::NoGradGuard none;
    const GatedHow how = {ctx->saved_data["post"].toBool(), ctx->saved_data["norm"].toInt(), ctx->saved_data["eps"].toDouble(), ctx->saved_data["alpha"].toDouble()};
    const Parameters p = {v[4], v[5], v[6], v[7], v[8], v[9]};
    const at::Tensor& s = v[2];
    cascmm_gated_norm a = gated_arguments(s, p, how);
    int64_t rows, cols;
    Wanted wanted{ctx};
    const bool want_x = wanted.next(), want_r = wanted.next();
    // (neither gate, scale nor norm in front of the sum: its gradient is that of both)
    const bool same = !how.post && !p[kGate].defined() && !p[kScale].defined() && how.alpha == 1.0;
    const at::Tensor dy = as_rows(grads[0].defined() ? grads[0] : at::zeros_like(s), rows, cols, a.lddy);
    at::Tensor ds, x, residual, dx, dr;
    if (grads[1].defined()) ds = as_rows(grads[1], rows, cols, a.ldds);
    if (v[0].defined()) x = as_rows(v[0], rows, cols, a.ldx);
    if (v[1].defined()) residual = as_rows(v[1], rows, cols, a.ldr);
    const at::Tensor sum = as_rows(s, rows, cols, a.lds);
    if (want_x && !same) dx = fresh(s.sizes(), s);
    if (want_r || (want_x && same)) dr = fresh(s.sizes(), s);
    void** const to[kParameters] = {&a.dweight, &a.dbias, &a.dgate, &a.dscale, &a.dpost_weight, &a.dpost_bias};
    for (int i = 0; i < kParameters; ++i)
      if (wanted.next(p[i].defined())) {
        out[2 + i] = fresh(p[i].sizes(), p[i]);
        *to[i] = out[2 + i].data_ptr();
      }
    a.dy = dy.const_data_ptr(); a.ds = data_of(ds); a.x = data_of(x); a.residual = data_of(residual); a.sum = sum.data_ptr(); a.stats = (float*)v[3].data_ptr();
    a.dx = ptr(dx); a.dresidual = ptr(dr);
    a.lddx = a.lddr = cols;
    if (residual.defined()) rows_of(residual, rows, cols, a.ldr);
    const at::Tensor ws = scratch(cascmm_gated_norm_backward_bytes(&a), s);
    check(cascmm_gated_norm_backward(&a, ws.data_ptr(), ws.nbytes(), stream_of(s)), "cascmm_gated_norm_backward");
    if (want_x) out[0] = same ? dr : dx;
    if (want_r) out[1] = dr;
    return once(std::move(out), "gated_add_norm", again);
  }
};

}  // namespace

// block_scaled(a, b, None, 0, 0, 0, bias | None) -> Tensor | None: b a raw [K, N] tensor;
// block_scaled(a, values, scales, K, N, dtype, bias | None): a held weight
PyObject* block_scaled(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 7) Py_RETURN_NONE;
  try {
    const int device = c10::hip::current_device();
    const at::Tensor *a = gpu_tensor(args[0], device), *b = gpu_tensor(args[1], device);
    at::Tensor scales, bias;
    int64_t M, K, lda;
    if (!a || !b || dtype_code(*a) < 0 || !rows_of(*a, M, K, lda) || K > kMostK || !optional_tensor(args[2], device, scales) || !optional_tensor(args[6], device, bias) || dual({a, b, &bias}))
      Py_RETURN_NONE;
    const bool held = scales.defined();
    int64_t N, ldb = 0;
    bool turned = false;
    if (held) {
      if (PyLong_AsLongLong(args[3]) != K || PyLong_AsLong(args[5]) != dtype_code(*a)) { PyErr_Clear(); Py_RETURN_NONE; }
      N = PyLong_AsLongLong(args[4]);
      if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
      if (N <= 0 || b->scalar_type() != at::kByte || scales.scalar_type() != at::kByte || !b->is_contiguous() || !scales.is_contiguous() || b->nbytes() < cascmm_block_values_bytes(N, K) ||
          scales.nbytes() < cascmm_block_scales_bytes(N, K))
        Py_RETURN_NONE;
    } else {
      if (b->dim() != 2 || b->scalar_type() != a->scalar_type() || b->size(0) != K || b->size(1) <= 0 || !weight_order(*b, turned, ldb)) Py_RETURN_NONE;
      N = b->size(1);
    }
    if (bias.defined() && (bias.dim() != 1 || bias.size(0) != N || bias.scalar_type() != a->scalar_type() || !bias.is_contiguous())) Py_RETURN_NONE;
    if (held ? differentiated({a, &bias}) : differentiated({a, b, &bias})) {
      if (held || M > kMostK || N > kMostK) Py_RETURN_NONE;
      return THPVariable_Wrap(BlockScaledNode::apply(*a, *b, optional_of(bias)));
    }
    at::Tensor out = result_like(*a, N);
    if (held) {
      linear(*a, M, K, lda, b->const_data_ptr(), scales.const_data_ptr(), out, data_of(bias), N);
    } else {
      const RoundedWeight w = round_weight(*b, turned, ldb, false);
      linear(*a, M, K, lda, w.forward.values(), w.forward.scales(), out, data_of(bias), N);
    }
    return THPVariable_Wrap(std::move(out));
  } catch (...) {
    return not_ordinary();
  }
}

// gated_add_norm(x, residual, weight, bias, gate, residual_scale, post_weight, post_bias, post_norm, norm, eps) -> (Tensor, Tensor) | None
PyObject* gated_add_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 11) Py_RETURN_NONE;
  try {
    const int device = c10::hip::current_device();
    const at::Tensor *x = gpu_tensor(args[0], device), *residual = gpu_tensor(args[1], device);
    int64_t rows, cols, ld;
    if (!x || !residual || dtype_code(*x) < 0 || residual->scalar_type() != x->scalar_type() || residual->sizes() != x->sizes() || !rows_of(*x, rows, cols, ld) ||
        !rows_of(*residual, rows, cols, ld) || dual({x, residual}))
      Py_RETURN_NONE;
    GatedHow how{false, PyLong_Check(args[9]) ? PyLong_AsLong(args[9]) : -1, 0, 1.0};
    if (!PyBool_Check(args[8]) || how.norm < 0 || how.norm > 1) { PyErr_Clear(); Py_RETURN_NONE; }
    how.post = args[8] == Py_True;
    how.eps = PyFloat_AsDouble(args[10]);
    Parameters p;
    PyObject* const at_[kParameters] = {args[2], args[3], args[4], nullptr, args[6], args[7]};
    for (int i = 0; i < kParameters; ++i)
      if (at_[i] && !optional_tensor(at_[i], device, p[i])) Py_RETURN_NONE;
    if (PyFloat_Check(args[5]) || PyLong_Check(args[5])) how.alpha = PyFloat_AsDouble(args[5]);
    else if (args[5] == Py_None || !optional_tensor(args[5], device, p[kScale])) Py_RETURN_NONE;
    if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
    if (!(how.eps >= 0) || !(how.eps < 1e30) || !std::isfinite(how.alpha) || (!how.post && (p[kPostWeight].defined() || p[kPostBias].defined()))) Py_RETURN_NONE;
    at::ScalarType type = at::ScalarType::Undefined;
    for (int i = 0; i < kParameters; ++i) {
      if (!p[i].defined()) continue;
      if (!parameter_of(*x, p[i], i < kPostWeight) || (type != at::ScalarType::Undefined && p[i].scalar_type() != type) || dual({&p[i]})) Py_RETURN_NONE;
      type = p[i].scalar_type();
    }
    if (differentiated({x, residual, &p[0], &p[1], &p[2], &p[3], &p[4], &p[5]})) {
      variable_list both = GatedNode::apply(*x, *residual, optional_of(p[0]), optional_of(p[1]), optional_of(p[2]), optional_of(p[3]), optional_of(p[4]), optional_of(p[5]), how.post, how.norm, how.eps,
                                            how.alpha);
      return pair(both[0], both[1]);
    }
    Gated g = gated_forward(*x, *residual, p, how, false);
    return pair(std::move(g.y), std::move(g.s));
  } catch (...) {
    return not_ordinary();
  }
}

// clip_gradients(gradients, results | None, norm type, max_norm) -> Tensor | None; lists of tensors (None: the norm alone)
PyObject* clip_gradients(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 4) Py_RETURN_NONE;
  try {
    const int device = c10::hip::current_device();
    const bool clip = args[1] != Py_None;
    if (!PyList_CheckExact(args[0]) || (clip && !PyList_CheckExact(args[1])) || !PyLong_Check(args[2])) Py_RETURN_NONE;
    const Py_ssize_t count = PyList_GET_SIZE(args[0]);
    const long type = PyLong_AsLong(args[2]);
    const double max_norm = PyFloat_AsDouble(args[3]);
    if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
    if (count == 0 || count > (1 << 20) || (clip && PyList_GET_SIZE(args[1]) != count) || type < 0 || type > 2 || !(max_norm >= 0)) Py_RETURN_NONE;
    std::vector<cascmm_gradient> table((size_t)count);
    std::vector<const at::Tensor*> written;
    if (clip) written.reserve((size_t)count);
    const at::Tensor* first = nullptr;
    for (Py_ssize_t i = 0; i < count; ++i) {
      const at::Tensor* g = gpu_tensor(PyList_GET_ITEM(args[0], i), device);
      if (!g || dtype_code(*g) < 0 || !g->is_non_overlapping_and_dense()) Py_RETURN_NONE;
      cascmm_gradient& entry = table[(size_t)i];
      entry = {g->const_data_ptr(), nullptr, g->numel(), dtype_code(*g), 0};
      if (!first) first = g;
      if (!clip) continue;
      const at::Tensor* o = g;
      if (PyList_GET_ITEM(args[1], i) != PyList_GET_ITEM(args[0], i)) {
        o = gpu_tensor(PyList_GET_ITEM(args[1], i), device);
        if (!o || o->sizes() != g->sizes() || o->strides() != g->strides() || (o->scalar_type() != g->scalar_type() && o->scalar_type() != at::kFloat) || (o->requires_grad() && o->is_leaf()))
          Py_RETURN_NONE;
      }
      if (o->is_inference()) Py_RETURN_NONE;
      entry.out = o->data_ptr();
      entry.out_dtype = dtype_code(*o);
      written.push_back(o);
    }
    at::Tensor norm = at::empty({}, at::TensorOptions().dtype(at::kFloat).device(first->device()));
    const at::Tensor ws = scratch(cascmm_gradients_workspace_bytes((int)count, table.data()), *first);
    if (cascmm_clip_gradients((int)count, table.data(), (int)type, max_norm, (float*)norm.data_ptr(), ws.data_ptr(), ws.nbytes(), stream_of(*first)) != CASCMM_OK) Py_RETURN_NONE;
    for (const at::Tensor* o : written) o->unsafeGetTensorImpl()->bump_version();   // (written behind autograd's back)
    return THPVariable_Wrap(std::move(norm));
  } catch (...) {
    return not_ordinary();
  }
}

}  // namespace native
