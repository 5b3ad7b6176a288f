// extern "C" entry points of the norms around a residual add (cascmm_gated_kernel.h): argument checks, parts and the choice of kernel.
#include <cstring>

#include "cascmm_gated_launch.h"

namespace cascmm {

CASCMM_GATED_OF(extern, CASCMM_DT_F32)
CASCMM_GATED_OF(extern, CASCMM_DT_F16)
CASCMM_GATED_OF(extern, CASCMM_DT_BF16)

static bool gated_aligned(const void* p, int64_t a) { return (uintptr_t)p % (uintptr_t)a == 0; }
static int64_t gated_size(int dtype) { return dtype == CASCMM_DT_F32 ? 4 : 2; }
static bool gated_dtype(int dtype) { return dtype == CASCMM_DT_F32 || dtype == CASCMM_DT_F16 || dtype == CASCMM_DT_BF16; }

struct GatedPlan {
  int64_t groups, part_rows;
  int parts, lanes;
  bool rich;
};
static int gated_plan(const cascmm_gated_norm& a, bool backward, GatedPlan& plan) {
  if (!gated_dtype(a.dtype) || (a.weight_dtype != a.dtype && a.weight_dtype != CASCMM_DT_F32)) return CASCMM_ERR_BAD_DTYPE;
  if (a.norm != CASCMM_NORM_LAYER && a.norm != CASCMM_NORM_RMS) return CASCMM_ERR_BAD_FORMAT;
  if (a.rows < 0 || a.cols < 0 || a.group_rows < 0 || (a.rows > 0 && (a.group_rows == 0 || a.rows % a.group_rows != 0))) return CASCMM_ERR_BAD_SHAPE;
  if (!(a.eps >= 0)) return CASCMM_ERR_BAD_SHAPE;
  for (const int64_t ld : {a.gate_ld, a.scale_ld, a.weight_ld, a.bias_ld})
    if (ld != 0 && ld < a.cols) return CASCMM_ERR_BAD_SHAPE;
  if (a.rows > INT32_MAX || a.cols > kFinishMostCols) return CASCMM_ERR_TOO_LARGE;
  plan.groups = a.rows ? a.rows / a.group_rows : 0;
  plan.lanes = gated_shape(a.cols, backward, 16 / gated_size(a.dtype)).lanes;
  plan.rich = a.scale || (a.post && a.post_bias);
  gated_parts(plan.groups, a.group_rows, plan.lanes, backward, plan.parts, plan.part_rows);
  // (a launch has fewer than 2^32 threads)
  if (plan.groups * plan.parts > (plan.lanes ? (1 << 24) - 1 : INT32_MAX)) return CASCMM_ERR_TOO_LARGE;
  return CASCMM_OK;
}
static bool gated_sums(const cascmm_gated_norm& a) { return a.dgate || a.dscale || a.dpost_weight || a.dpost_bias || a.dweight || a.dbias; }
// five sums where there is a row of the residual's scales or a bias of the first norm, and of rows without registers, else three
static size_t gated_sum_bytes(const cascmm_gated_norm& a, const GatedPlan& plan) {
  return (size_t)plan.groups * (size_t)plan.parts * (plan.lanes && !plan.rich ? 3 : 5) * (size_t)a.cols * sizeof(float);
}
static size_t gated_bytes(const cascmm_gated_norm& a, const GatedPlan& plan, bool sums) {
  return (sums ? gated_sum_bytes(a, plan) + (plan.lanes ? 0 : 2 * (size_t)a.rows * sizeof(float)) : 0) + 16;
}
static bool gated_pointers(const cascmm_gated_norm& a) {
  const int64_t es = gated_size(a.dtype), ws = gated_size(a.weight_dtype);
  for (const void* p : {(const void*)a.x, a.residual, (const void*)a.y, (const void*)a.sum, a.dy, a.ds, (const void*)a.dx, (const void*)a.dresidual})
    if (!gated_aligned(p, es)) return false;
  for (const void* p : {a.gate, a.scale, a.post_weight, a.post_bias, a.weight, a.bias, (const void*)a.dgate, (const void*)a.dscale, (const void*)a.dpost_weight, (const void*)a.dpost_bias,
                        (const void*)a.dweight, (const void*)a.dbias})
    if (!gated_aligned(p, ws)) return false;
  return gated_aligned(a.stats, 4);
}
static GatedParams gated_params(const cascmm_gated_norm& a, const GatedPlan& plan) {
  GatedParams p;
  memset(&p, 0, sizeof(p));
  p.x = a.x; p.residual = a.residual; p.gate = a.gate; p.scale = a.scale; p.weight = a.weight; p.bias = a.bias;
  if (a.post) {
    p.post_weight = a.post_weight;
    p.post_bias = a.post_bias;
  }
  p.y = a.y; p.sum = a.sum; p.stats = a.stats; p.dy = a.dy; p.ds = a.ds; p.dx = a.dx; p.dresidual = a.dresidual;
  p.rows = a.rows; p.group_rows = a.group_rows; p.part_rows = plan.part_rows;
  p.ldx = a.ldx; p.ldr = a.ldr; p.ldy = a.ldy; p.lds = a.lds; p.lddy = a.lddy; p.ldds = a.ldds; p.lddx = a.lddx; p.lddr = a.lddr;
  p.gate_ld = a.gate_ld; p.scale_ld = a.scale_ld; p.weight_ld = a.weight_ld; p.bias_ld = a.bias_ld;
  p.cols = (int)a.cols; p.parts = plan.parts;
  p.f32 = a.weight_dtype == CASCMM_DT_F32;
  p.centred = a.norm == CASCMM_NORM_LAYER;
  p.eps = (float)a.eps;
  p.inv_cols = 1.0f / (float)a.cols;
  p.alpha = (float)a.residual_scale;
  return p;
}

}  // namespace cascmm

using namespace cascmm;

extern "C" {

int cascmm_gated_norm_forward(const cascmm_gated_norm* args, void* stream) {
  if (!args) return CASCMM_ERR_NULL_POINTER;
  const cascmm_gated_norm& a = *args;
  GatedPlan plan;
  const int st = gated_plan(a, false, plan);
  if (st != CASCMM_OK) return st;
  if (a.ldx < a.cols || a.ldr < a.cols || a.ldy < a.cols || a.lds < a.cols) return CASCMM_ERR_BAD_SHAPE;
  if (a.rows == 0 || a.cols == 0) return CASCMM_OK;
  if (!a.x || !a.residual || !a.y || !a.sum) return CASCMM_ERR_NULL_POINTER;
  if (!gated_pointers(a)) return CASCMM_ERR_ALIGNMENT;
  const GatedParams p = gated_params(a, plan);
  const hipStream_t s = (hipStream_t)stream;
  const bool post = a.post != 0;
  const hipError_t err = a.dtype == CASCMM_DT_F32   ? gated_forward<CASCMM_DT_F32>(p, plan.groups, post, plan.rich, s)
                         : a.dtype == CASCMM_DT_F16 ? gated_forward<CASCMM_DT_F16>(p, plan.groups, post, plan.rich, s)
                                                    : gated_forward<CASCMM_DT_BF16>(p, plan.groups, post, plan.rich, s);
  return err == hipSuccess ? CASCMM_OK : CASCMM_ERR_LAUNCH;
}

size_t cascmm_gated_norm_workspace_bytes(const cascmm_gated_norm* args) {
  GatedPlan plan;
  return args && gated_plan(*args, true, plan) == CASCMM_OK ? gated_bytes(*args, plan, true) : 0;
}
size_t cascmm_gated_norm_backward_bytes(const cascmm_gated_norm* args) {
  GatedPlan plan;
  return args && gated_plan(*args, true, plan) == CASCMM_OK ? gated_bytes(*args, plan, gated_sums(*args)) : 0;
}

int cascmm_gated_norm_backward(const cascmm_gated_norm* args, void* workspace, size_t workspace_bytes, void* stream) {
  if (!args) return CASCMM_ERR_NULL_POINTER;
  const cascmm_gated_norm& a = *args;
  GatedPlan plan;
  const int st = gated_plan(a, true, plan);
  if (st != CASCMM_OK) return st;
  const bool sums = gated_sums(a), reads_x = a.post || a.gate;
  if (a.lddy < a.cols || a.lds < a.cols || (reads_x && a.ldx < a.cols) || (a.scale && a.ldr < a.cols) || (a.ds && a.ldds < a.cols) || (a.dx && a.lddx < a.cols) ||
      (a.dresidual && a.lddr < a.cols))
    return CASCMM_ERR_BAD_SHAPE;
  // (a gradient without what it is the gradient of)
  if ((a.dgate && !a.gate) || (a.dscale && !a.scale) || (a.dpost_weight && (!a.post || !a.post_weight)) || (a.dpost_bias && (!a.post || !a.post_bias)) || (a.dweight && !a.weight) ||
      (a.dbias && !a.bias))
    return CASCMM_ERR_NULL_POINTER;
  if (a.cols == 0 || (!a.dx && !a.dresidual && !sums) || (a.rows == 0 && !sums)) return CASCMM_OK;
  if (a.rows > 0 && (!a.dy || !a.sum || !a.stats || (reads_x && !a.x) || (a.scale && !a.residual))) return CASCMM_ERR_NULL_POINTER;
  if (!gated_pointers(a)) return CASCMM_ERR_ALIGNMENT;
  if (!workspace || workspace_bytes < gated_bytes(a, plan, sums)) return CASCMM_ERR_WORKSPACE;
  if (!gated_aligned(workspace, 16)) return CASCMM_ERR_ALIGNMENT;
  GatedParams p = gated_params(a, plan);
  p.partials = sums ? (float*)workspace : nullptr;
  if (!plan.lanes && sums) p.row_means = (float*)((char*)workspace + gated_sum_bytes(a, plan));
  const hipStream_t s = (hipStream_t)stream;
  const bool post = a.post != 0;
  hipError_t err = hipSuccess;
  if (a.rows > 0)
    err = a.dtype == CASCMM_DT_F32   ? gated_backward<CASCMM_DT_F32>(p, plan.groups, post, plan.rich, s)
          : a.dtype == CASCMM_DT_F16 ? gated_backward<CASCMM_DT_F16>(p, plan.groups, post, plan.rich, s)
                                     : gated_backward<CASCMM_DT_BF16>(p, plan.groups, post, plan.rich, s);
  if (sums && err == hipSuccess) {
    GatedFinish f;
    memset(&f, 0, sizeof(f));
    f.partials = p.partials;
    f.gate = a.gate; f.post_weight = p.post_weight; f.post_bias = p.post_bias;
    f.dgate = a.dgate; f.dscale = a.dscale; f.dpost_weight = a.dpost_weight; f.dpost_bias = a.dpost_bias; f.dweight = a.dweight; f.dbias = a.dbias;
    f.groups = plan.groups;
    f.gate_ld = a.gate_ld;
    f.parts = a.rows > 0 ? plan.parts : 0;
    f.cols = (int)a.cols;
    const bool rich = plan.lanes == 0 || plan.rich;     // (the sums of rows without registers are always five)
    f.gate_grouped = a.gate_ld != 0; f.scale_grouped = a.scale_ld != 0; f.weight_grouped = a.weight_ld != 0; f.bias_grouped = a.bias_ld != 0;
    f.shared = a.dpost_weight || a.dpost_bias || (a.dgate && !f.gate_grouped) || (a.dscale && !f.scale_grouped) || (a.dweight && !f.weight_grouped) || (a.dbias && !f.bias_grouped);
    // (rows of threads on a group: as many as leave one for each group; where no gradient runs over the groups there are more workgroups, and eight rows add the parts of each of four groups)
    f.share = f.shared ? 32 : plan.parts >= 4 ? 8 : 1;
    while (f.shared && f.share > 1 && 32 / f.share < plan.groups) f.share /= 2;
    err = a.weight_dtype == CASCMM_DT_F32   ? gated_finish<CASCMM_DT_F32>(f, rich, s)
          : a.weight_dtype == CASCMM_DT_F16 ? gated_finish<CASCMM_DT_F16>(f, rich, s)
                                            : gated_finish<CASCMM_DT_BF16>(f, rich, s);
  }
  return err == hipSuccess ? CASCMM_OK : CASCMM_ERR_LAUNCH;
}

}  // extern "C"
