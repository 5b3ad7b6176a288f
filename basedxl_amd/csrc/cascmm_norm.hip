// extern "C" entry points of layer norm (cascmm_norm_kernel.h): argument checks and the choice of kernel.
#include "cascmm_norm_kernel.h"

#include <cstring>

#include <algorithm>

namespace cascmm {

static bool norm_aligned(const void* p, size_t a) { return (uintptr_t)p % a == 0; }
static size_t norm_size(int dtype) { return dtype == CASCMM_DT_F32 ? 4 : 2; }
static bool norm_dtype(int dtype) { return dtype == CASCMM_DT_F32 || dtype == CASCMM_DT_F16 || dtype == CASCMM_DT_BF16; }
constexpr int64_t kNormMostCols = 1 << 30;   // (column numbers and a step beyond the last are 32-bit)

// workgroups (rows of partial sums) of the backward pass
static int64_t norm_parts(int64_t rows, int64_t) { return std::max<int64_t>(1, std::min<int64_t>((rows + 15) / 16, 512)); }

static int norm_check(int64_t rows, int64_t cols, int dtype, int weight_dtype) {
  if (!norm_dtype(dtype) || (weight_dtype != dtype && weight_dtype != CASCMM_DT_F32)) return CASCMM_ERR_BAD_DTYPE;
  if (rows < 0 || cols < 0) return CASCMM_ERR_BAD_SHAPE;
  if (rows > INT32_MAX || cols > kNormMostCols) return CASCMM_ERR_TOO_LARGE;
  return CASCMM_OK;
}

template <int IODT> static hipError_t norm_forward(const NormParams& p, hipStream_t s) {
  hipError_t err = hipSuccess;
  if (p.residual) CASCMM_LAUNCH(err, (cascmm_layer_norm_wide_kernel<IODT, true>), dim3((unsigned)p.rows), dim3(kNormWide), 0, s, p);
  else CASCMM_LAUNCH(err, (cascmm_layer_norm_wide_kernel<IODT, false>), dim3((unsigned)p.rows), dim3(kNormWide), 0, s, p);
  return err;
}

template <int IODT> static hipError_t norm_backward(const NormParams& p, void* dweight, void* dbias, int weight_dtype, hipStream_t s) {
  hipError_t err = hipSuccess;
  if (p.y && p.rows > 0) CASCMM_LAUNCH(err, (cascmm_layer_norm_backward_wide_kernel<IODT>), dim3((unsigned)p.rows), dim3(kNormWide), 0, s, p);
  if (!p.partials) return err;
  const int parts = (int)norm_parts(p.rows, p.cols);
  CASCMM_LAUNCH(err, (cascmm_layer_norm_sums_kernel<IODT>), dim3((unsigned)((p.cols + 255) / 256), (unsigned)parts), dim3(256), 0, s, p);
  const dim3 grid((unsigned)((p.cols + kFinishCols - 1) / kFinishCols), 2);
  if (weight_dtype == CASCMM_DT_F32)
    CASCMM_LAUNCH(err, (cascmm_column_finish_kernel<CASCMM_DT_F32>), grid, dim3(1024), 0, s, (const float*)p.partials, parts, 2, (int64_t)p.cols, dweight, dbias);
  else
    CASCMM_LAUNCH(err, (cascmm_column_finish_kernel<IODT>), grid, dim3(1024), 0, s, (const float*)p.partials, parts, 2, (int64_t)p.cols, dweight, dbias);
  return err;
}

}  // namespace cascmm

using namespace cascmm;

extern "C" {

int cascmm_layer_norm(const void* x, const void* residual, const void* weight, const void* bias, void* y, void* sum, float* mean, float* rstd,
                      int64_t rows, int64_t cols, int64_t ldx, int64_t ldr, int64_t ldy, int64_t lds, float eps, int dtype, int weight_dtype, void* stream) {
  const int st = norm_check(rows, cols, dtype, weight_dtype);
  if (st != CASCMM_OK) return st;
  if (ldx < cols || ldy < cols || (residual && (ldr < cols || lds < cols)) || !(eps >= 0.f)) return CASCMM_ERR_BAD_SHAPE;
  if (rows == 0 || cols == 0) return CASCMM_OK;
  if (!x || !y || (residual != nullptr) != (sum != nullptr) || (mean != nullptr) != (rstd != nullptr)) return CASCMM_ERR_NULL_POINTER;
  const size_t es = norm_size(dtype), ws = norm_size(weight_dtype);
  if (!norm_aligned(x, es) || !norm_aligned(y, es) || !norm_aligned(residual, es) || !norm_aligned(sum, es) || !norm_aligned(weight, ws) ||
      !norm_aligned(bias, ws) || !norm_aligned(mean, 4) || !norm_aligned(rstd, 4))
    return CASCMM_ERR_ALIGNMENT;
  NormParams p;
  memset(&p, 0, sizeof(p));
  p.x = x; p.residual = residual; p.weight = weight; p.bias = bias; p.y = y; p.sum = sum; p.mean = mean; p.rstd = rstd;
  p.rows = rows; p.cols = (int)cols; p.ldx = ldx; p.ldr = ldr; p.ldy = ldy; p.lds = lds;
  p.weight_f32 = weight_dtype == CASCMM_DT_F32;
  p.eps = eps;
  p.inv_cols = 1.0f / (float)cols;
  const hipStream_t s = (hipStream_t)stream;
  const hipError_t err = dtype == CASCMM_DT_F32   ? norm_forward<CASCMM_DT_F32>(p, s)
                         : dtype == CASCMM_DT_F16 ? norm_forward<CASCMM_DT_F16>(p, s)
                                                  : norm_forward<CASCMM_DT_BF16>(p, s);
  return err == hipSuccess ? CASCMM_OK : CASCMM_ERR_LAUNCH;
}

size_t cascmm_layer_norm_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0 || rows > INT32_MAX || cols > kNormMostCols) return 0;
  return (size_t)norm_parts(rows, cols) * 2 * (size_t)cols * sizeof(float);
}

int cascmm_layer_norm_backward(const void* dy, const void* ds, const void* x, const void* weight, const float* mean, const float* rstd, void* dx,
                               void* dweight, void* dbias, int64_t rows, int64_t cols, int64_t lddy, int64_t ldds, int64_t ldx, int64_t lddx, int dtype,
                               int weight_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const int st = norm_check(rows, cols, dtype, weight_dtype);
  if (st != CASCMM_OK) return st;
  if (lddy < cols || ldx < cols || (ds && ldds < cols) || (dx && lddx < cols)) return CASCMM_ERR_BAD_SHAPE;
  const bool sums = dweight || dbias;
  if (cols == 0 || (!dx && !sums) || (rows == 0 && !sums)) return CASCMM_OK;
  if (rows > 0 && (!dy || !x || !mean || !rstd)) return CASCMM_ERR_NULL_POINTER;
  const size_t es = norm_size(dtype), ws = norm_size(weight_dtype);
  if (!norm_aligned(dy, es) || !norm_aligned(ds, es) || !norm_aligned(x, es) || !norm_aligned(dx, es) || !norm_aligned(weight, ws) ||
      !norm_aligned(dweight, ws) || !norm_aligned(dbias, ws) || !norm_aligned(mean, 4) || !norm_aligned(rstd, 4))
    return CASCMM_ERR_ALIGNMENT;
  if (sums) {
    if (!workspace || workspace_bytes < cascmm_layer_norm_workspace_bytes(rows, cols)) return CASCMM_ERR_WORKSPACE;
    if (!norm_aligned(workspace, 16)) return CASCMM_ERR_ALIGNMENT;
  }
  NormParams p;
  memset(&p, 0, sizeof(p));
  p.dy = dy; p.ds = ds; p.x = x; p.weight = weight; p.mean = const_cast<float*>(mean); p.rstd = const_cast<float*>(rstd); p.y = dx;
  p.partials = sums ? (float*)workspace : nullptr;
  p.rows = rows; p.cols = (int)cols; p.ldx = ldx; p.ldy = lddx; p.lddy = lddy; p.ldds = ldds;
  p.weight_f32 = weight_dtype == CASCMM_DT_F32;
  p.inv_cols = 1.0f / (float)cols;
  const hipStream_t s = (hipStream_t)stream;
  const hipError_t err = dtype == CASCMM_DT_F32   ? norm_backward<CASCMM_DT_F32>(p, dweight, dbias, weight_dtype, s)
                         : dtype == CASCMM_DT_F16 ? norm_backward<CASCMM_DT_F16>(p, dweight, dbias, weight_dtype, s)
                                                  : norm_backward<CASCMM_DT_BF16>(p, dweight, dbias, weight_dtype, s);
  return err == hipSuccess ? CASCMM_OK : CASCMM_ERR_LAUNCH;
}

}  // extern "C"
