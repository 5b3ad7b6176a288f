// extern "C" entry points of layer norm (cascmm_norm_kernel.h): argument checks and the choice of kernel.
#include "cascmm_norm_kernel.h"

#include <cstring>

#include <algorithm>

namespace cascmm {

static bool norm_aligned(const void* p, size_t a) { return (uintptr_t)p % a == 0; }
static size_t norm_size(int dtype) { return dtype == CASCMM_DT_F32 ? 4 : 2; }
static bool norm_dtype(int dtype) { return dtype == CASCMM_DT_F32 || dtype == CASCMM_DT_F16 || dtype == CASCMM_DT_BF16; }

// The lanes of a row and the elements of a lane: four lanes take rows shorter than a chunk of 16 bytes, eight rows of up to 64 columns, sixteen up to 256, a wave up to 2048 (in the backward pass, which
// holds the sums beside a row, 1536), four of them up to 8192; none: longer rows
struct NormShape { int lanes, values; };
static NormShape norm_shape(int64_t cols, bool backward, int64_t chunk) {
  const auto fit = [&](int lanes) { return (int)std::min<int64_t>((cols + 8 * lanes - 1) / (8 * lanes) * 8, 1 << 20); };
  if (cols < chunk) return {4, 8};
  if (cols <= 64) return {8, 8};
  if (fit(16) <= 16) return {16, fit(16)};
  if (fit(64) <= (backward ? 24 : 32)) return {64, fit(64)};
  if (fit(256) <= 32) return {256, fit(256)};
  return {0, 0};
}
// Workgroups that walk over the rows: four on a CU forward and for short rows, backward else two, one where four waves hold a row (as many as their
// registers leave room for; 65536 x 1280 bf16 backward 98 us, 256 workgroups 97, 768 111, 1024 105; 8192 x 640 fp16 15.0, 15.3, 16.1, 18.2), and backward two rows
// at least for each of a workgroup's, since what a workgroup sums is written and read again.
static int64_t norm_groups(int64_t rows, int lanes, bool backward) {
  const int64_t at_a_time = 256 / lanes * (backward ? 2 : 1), most = backward ? (lanes == 256 ? 256 : lanes == 64 ? 512 : 1024) : 1024;
  return std::max<int64_t>(1, std::min<int64_t>((rows + at_a_time - 1) / at_a_time, most));
}
// (a launch has fewer than 2^32 threads)
static unsigned norm_wide_groups(int64_t rows) { return (unsigned)std::min<int64_t>(rows, 1 << 20); }
// rows of partial sums of the backward pass
static int64_t norm_parts(int64_t rows, int64_t cols, int dtype) {
  const NormShape f = norm_shape(cols, true, 16 / (int64_t)norm_size(dtype));
  return f.lanes ? norm_groups(rows, f.lanes, true) : std::max<int64_t>(1, std::min<int64_t>((rows + 15) / 16, 512));
}

static int norm_check(int64_t rows, int64_t cols, int dtype, int weight_dtype) {
  if (!norm_dtype(dtype) || (weight_dtype != dtype && weight_dtype != CASCMM_DT_F32)) return CASCMM_ERR_BAD_DTYPE;
  if (rows < 0 || cols < 0) return CASCMM_ERR_BAD_SHAPE;
  if (rows > INT32_MAX || cols > kFinishMostCols) return CASCMM_ERR_TOO_LARGE;
  return CASCMM_OK;
}

template <int IODT, bool ADD> static hipError_t norm_forward(const NormParams& p, hipStream_t s) {
  hipError_t err = hipSuccess;
  const NormShape f = norm_shape(p.cols, false, NormRow<IODT>::VEC);
  const dim3 grid(f.lanes ? (unsigned)norm_groups(p.rows, f.lanes, false) : 1u);
#define NORM_CASE(LPR, NV) \
  case (LPR) * 100 + (NV): CASCMM_LAUNCH(err, (cascmm_layer_norm_kernel<IODT, NV, LPR, ADD>), grid, dim3(256), 0, s, p); break
  switch (f.lanes * 100 + f.values) {
    NORM_CASE(4, 8);
    NORM_CASE(8, 8);
    NORM_CASE(16, 8);
    NORM_CASE(16, 16);
    NORM_CASE(64, 8);
    NORM_CASE(64, 16);
    NORM_CASE(64, 24);
    NORM_CASE(64, 32);
    NORM_CASE(256, 16);
    NORM_CASE(256, 24);
    NORM_CASE(256, 32);
    default: CASCMM_LAUNCH(err, (cascmm_layer_norm_wide_kernel<IODT, ADD>), dim3(norm_wide_groups(p.rows)), dim3(kNormWide), 0, s, p);
  }
#undef NORM_CASE
  return err;
}

template <int IODT, bool DS, bool SUMS> static hipError_t norm_backward_rows(const NormParams& p, hipStream_t s) {
  hipError_t err = hipSuccess;
  const NormShape f = norm_shape(p.cols, true, NormRow<IODT>::VEC);
  const dim3 grid((unsigned)norm_groups(p.rows, f.lanes, true));
#define NORM_CASE(LPR, NV) \
  case (LPR) * 100 + (NV): CASCMM_LAUNCH(err, (cascmm_layer_norm_backward_kernel<IODT, NV, LPR, DS, SUMS>), grid, dim3(256), 0, s, p); break
  switch (f.lanes * 100 + f.values) {
    NORM_CASE(4, 8);
    NORM_CASE(8, 8);
    NORM_CASE(16, 8);
    NORM_CASE(16, 16);
    NORM_CASE(64, 8);
    NORM_CASE(64, 16);
    NORM_CASE(64, 24);
    NORM_CASE(256, 8);
    NORM_CASE(256, 16);
    NORM_CASE(256, 24);
    NORM_CASE(256, 32);
    default: return hipErrorInvalidValue;
  }
#undef NORM_CASE
  return err;
}

template <int IODT> static hipError_t norm_backward(const NormParams& p, void* dweight, void* dbias, int weight_dtype, hipStream_t s) {
  hipError_t err = hipSuccess;
  const int parts = (int)norm_parts(p.rows, p.cols, IODT);
  // (no dx wanted: nothing but the sums.  No rows: sums of zeros)
  const bool rows = p.y && p.rows > 0, wide = norm_shape(p.cols, true, NormRow<IODT>::VEC).lanes == 0;
  if (rows && wide) CASCMM_LAUNCH(err, (cascmm_layer_norm_backward_wide_kernel<IODT>), dim3(norm_wide_groups(p.rows)), dim3(kNormWide), 0, s, p);
  else if (rows && p.partials) err = p.ds ? norm_backward_rows<IODT, true, true>(p, s) : norm_backward_rows<IODT, false, true>(p, s);
  else if (rows) err = p.ds ? norm_backward_rows<IODT, true, false>(p, s) : norm_backward_rows<IODT, false, false>(p, s);
  if (!p.partials) return err;
  if (!rows || wide)
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
  const hipError_t err = dtype == CASCMM_DT_F32   ? (residual ? norm_forward<CASCMM_DT_F32, true>(p, s) : norm_forward<CASCMM_DT_F32, false>(p, s))
                         : dtype == CASCMM_DT_F16 ? (residual ? norm_forward<CASCMM_DT_F16, true>(p, s) : norm_forward<CASCMM_DT_F16, false>(p, s))
                                                  : (residual ? norm_forward<CASCMM_DT_BF16, true>(p, s) : norm_forward<CASCMM_DT_BF16, false>(p, s));
  return err == hipSuccess ? CASCMM_OK : CASCMM_ERR_LAUNCH;
}

size_t cascmm_layer_norm_workspace_bytes(int64_t rows, int64_t cols, int dtype) {
  if (rows < 0 || cols < 0 || rows > INT32_MAX || cols > kFinishMostCols || !norm_dtype(dtype)) return 0;
  return (size_t)norm_parts(rows, cols, dtype) * 2 * (size_t)cols * sizeof(float);
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
    if (!workspace || workspace_bytes < cascmm_layer_norm_workspace_bytes(rows, cols, dtype)) return CASCMM_ERR_WORKSPACE;
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
