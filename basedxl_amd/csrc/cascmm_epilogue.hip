// extern "C" entry points of the passes in cascmm_epilogue_kernel.h.
#include "cascmm_epilogue_kernel.h"

#include <algorithm>

#include "cascmm_epilogue.h"

namespace cascmm {

static bool ep_aligned(const void* p, size_t a) { return (uintptr_t)p % a == 0; }
static size_t ep_size(int dtype) { return dtype == CASCMM_DT_F32 ? 4 : 2; }
static bool ep_dtype(int dtype) { return dtype == CASCMM_DT_F32 || dtype == CASCMM_DT_F16 || dtype == CASCMM_DT_BF16; }

template <int IODT>
static int launch_epilogue_of(const void* src, int64_t lds, const void* residual, int64_t ldr, void* dst, int64_t ldd, int64_t rows, int64_t cols, int act, hipStream_t s) {
  const int64_t per_row = (cols + NormRow<IODT>::VEC - 1) / NormRow<IODT>::VEC;
  if (per_row > (int64_t)(UINT32_MAX - 256) / rows) return CASCMM_ERR_TOO_LARGE;
  const int64_t total = rows * per_row;
  hipError_t err = hipSuccess;
  CASCMM_LAUNCH(err, (cols < NormRow<IODT>::VEC ? cascmm_epilogue_kernel<IODT, true> : cascmm_epilogue_kernel<IODT, false>), dim3((unsigned)((total + 255) / 256)), dim3(256), 0, s, src, lds, residual, ldr, dst, ldd, (int)cols,
                (unsigned)per_row, (unsigned)total, act);
  return err == hipSuccess ? CASCMM_OK : CASCMM_ERR_LAUNCH;
}
int launch_epilogue(const void* src, int64_t lds, const void* residual, int64_t ldr, void* dst, int64_t ldd, int64_t rows, int64_t cols, int act, int dtype,
                    hipStream_t s) {
  return dtype == CASCMM_DT_F32   ? launch_epilogue_of<CASCMM_DT_F32>(src, lds, residual, ldr, dst, ldd, rows, cols, act, s)
         : dtype == CASCMM_DT_F16 ? launch_epilogue_of<CASCMM_DT_F16>(src, lds, residual, ldr, dst, ldd, rows, cols, act, s)
                                  : launch_epilogue_of<CASCMM_DT_BF16>(src, lds, residual, ldr, dst, ldd, rows, cols, act, s);
}

// The lanes on a row, and the workgroups that share the rows of a band of columns: four for a CU, as their registers allow, four rows at least for each of
// their groups of lanes (what a workgroup sums is written and read again)
static int ep_lanes(int64_t cols, int dtype) { return cols <= 16 * (int64_t)(16 / ep_size(dtype)) ? 16 : 64; }
static int64_t ep_parts(int64_t rows, int64_t cols, int dtype) {
  const int lanes = ep_lanes(cols, dtype);
  const int64_t bands = (cols + lanes * (16 / (int64_t)ep_size(dtype)) - 1) / (lanes * (16 / (int64_t)ep_size(dtype)));
  return std::max<int64_t>(1, std::min<int64_t>((rows + 4 * (256 / lanes) - 1) / (4 * (256 / lanes)), (1024 + bands - 1) / bands));
}

template <int IODT, int LANES>
static hipError_t ep_backward_lanes(const void* dy, int64_t lddy, const void* z, int64_t ldz, void* dz, int64_t lddz, float* partials, int64_t rows, int64_t cols, int parts,
                                    int act, hipStream_t s) {
  hipError_t err = hipSuccess;
  constexpr int BAND = LANES * NormRow<IODT>::VEC;
  CASCMM_LAUNCH(err, (LANES == 16 && cols < NormRow<IODT>::VEC ? cascmm_epilogue_backward_kernel<IODT, LANES, LANES == 16> : cascmm_epilogue_backward_kernel<IODT, LANES, false>), dim3((unsigned)((cols + BAND - 1) / BAND), (unsigned)parts), dim3(256), 0, s, dy, lddy, z, ldz, dz,
                lddz, partials, rows, (int)cols, act);
  return err;
}
template <int IODT>
static hipError_t ep_backward(const void* dy, int64_t lddy, const void* z, int64_t ldz, void* dz, int64_t lddz, void* dbias, float* partials, int64_t rows, int64_t cols,
                              int act, hipStream_t s) {
  const int parts = (int)ep_parts(rows, cols, IODT);
  hipError_t err = ep_lanes(cols, IODT) == 16 ? ep_backward_lanes<IODT, 16>(dy, lddy, z, ldz, dz, lddz, partials, rows, cols, parts, act, s)
                                              : ep_backward_lanes<IODT, 64>(dy, lddy, z, ldz, dz, lddz, partials, rows, cols, parts, act, s);
  if (partials)
    CASCMM_LAUNCH(err, (cascmm_column_finish_kernel<IODT>), dim3((unsigned)((cols + kFinishCols - 1) / kFinishCols), 1), dim3(1024), 0, s, (const float*)partials, parts, 1,
                  cols, dbias, (void*)nullptr);
  return err;
}

}  // namespace cascmm

using namespace cascmm;

extern "C" {

size_t cascmm_epilogue_workspace_bytes(int64_t rows, int64_t cols, int dtype) {
  if (rows < 0 || cols <= 0 || rows > INT32_MAX || cols > kFinishMostCols || !ep_dtype(dtype)) return 0;
  return (size_t)ep_parts(rows, cols, dtype) * (size_t)cols * sizeof(float);
}

int cascmm_epilogue_backward(const void* dy, const void* z, void* dz, void* dbias, int64_t rows, int64_t cols, int64_t lddy, int64_t ldz, int64_t lddz, int activation,
                             int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (!ep_dtype(dtype)) return CASCMM_ERR_BAD_DTYPE;
  if (activation < CASCMM_ACT_NONE || activation > CASCMM_ACT_SILU) return CASCMM_ERR_BAD_FORMAT;
  if (rows < 0 || cols < 0 || lddy < cols || (activation && ldz < cols) || (dz && lddz < cols)) return CASCMM_ERR_BAD_SHAPE;
  if (rows > INT32_MAX || cols > kFinishMostCols) return CASCMM_ERR_TOO_LARGE;
  if (cols == 0 || (!dz && !dbias) || (rows == 0 && !dbias)) return CASCMM_OK;
  if (rows > 0 && (!dy || (activation && !z))) return CASCMM_ERR_NULL_POINTER;
  const size_t es = ep_size(dtype);
  if (!ep_aligned(dy, es) || !ep_aligned(z, es) || !ep_aligned(dz, es) || !ep_aligned(dbias, es)) return CASCMM_ERR_ALIGNMENT;
  if (dbias) {
    if (!workspace || workspace_bytes < cascmm_epilogue_workspace_bytes(rows, cols, dtype)) return CASCMM_ERR_WORKSPACE;
    if (!ep_aligned(workspace, 16)) return CASCMM_ERR_ALIGNMENT;
  }
  float* partials = dbias ? (float*)workspace : nullptr;
  const hipStream_t s = (hipStream_t)stream;
  const hipError_t err = dtype == CASCMM_DT_F32   ? ep_backward<CASCMM_DT_F32>(dy, lddy, z, ldz, dz, lddz, dbias, partials, rows, cols, activation, s)
                         : dtype == CASCMM_DT_F16 ? ep_backward<CASCMM_DT_F16>(dy, lddy, z, ldz, dz, lddz, dbias, partials, rows, cols, activation, s)
                                                  : ep_backward<CASCMM_DT_BF16>(dy, lddy, z, ldz, dz, lddz, dbias, partials, rows, cols, activation, s);
  return err == hipSuccess ? CASCMM_OK : CASCMM_ERR_LAUNCH;
}

int cascmm_transpose(const void* x, void* out, int64_t rows, int64_t cols, int64_t ldx, int64_t ldo, int dtype, void* stream) {
  if (!ep_dtype(dtype)) return CASCMM_ERR_BAD_DTYPE;
  if (rows < 0 || cols < 0 || ldx < cols || ldo < rows) return CASCMM_ERR_BAD_SHAPE;
  if (rows == 0 || cols == 0) return CASCMM_OK;
  if (!x || !out) return CASCMM_ERR_NULL_POINTER;
  const size_t es = ep_size(dtype);
  if (!ep_aligned(x, es) || !ep_aligned(out, es)) return CASCMM_ERR_ALIGNMENT;
  if (rows > (1 << 30) || cols > (1 << 30)) return CASCMM_ERR_TOO_LARGE;
  // (workgroups are counted in 32 bits, and their threads too)
  const int64_t across = (cols + 63) / 64, tiles = (rows + 63) / 64 * across;
  if (tiles > UINT32_MAX / 256) return CASCMM_ERR_TOO_LARGE;
  hipError_t err = hipSuccess;
  if (es == 4)
    CASCMM_LAUNCH(err, (cascmm_transpose_kernel<unsigned>), dim3((unsigned)tiles), dim3(256), 0, (hipStream_t)stream, (const unsigned*)x, ldx, (unsigned*)out, ldo, (int)rows,
                  (int)cols, (unsigned)across);
  else
    CASCMM_LAUNCH(err, (cascmm_transpose_kernel<unsigned short>), dim3((unsigned)tiles), dim3(256), 0, (hipStream_t)stream, (const unsigned short*)x, ldx,
                  (unsigned short*)out, ldo, (int)rows, (int)cols, (unsigned)across);
  return err == hipSuccess ? CASCMM_OK : CASCMM_ERR_LAUNCH;
}

}  // extern "C"
