// extern "C" entry points of the passes in cascmm_epilogue_kernel.h.
#include "cascmm_epilogue_kernel.h"

#include <cstring>

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

template <int IODT, int LANES, bool TINY>
static hipError_t ep_backward_launch(const SlopeParams& p, unsigned bands, unsigned parts, const TransposeParams& a, const TransposeParams& b, hipStream_t s) {
  hipError_t err = hipSuccess;
  if (a.tiles + b.tiles > 0)
    CASCMM_LAUNCH(err, (cascmm_epilogue_operands_kernel<IODT, LANES, TINY>), dim3(bands * parts + a.tiles + b.tiles), dim3(256), 0, s, p, bands, parts, a, b);
  else
    CASCMM_LAUNCH(err, (cascmm_epilogue_backward_kernel<IODT, LANES, TINY>), dim3(bands, parts), dim3(256), 0, s, p);
  return err;
}
// (slopes: dz or the sums are wanted; else the transpositions alone)
template <int IODT> static hipError_t ep_backward(const SlopeParams& p, bool slopes, void* dbias, const TransposeParams& a, const TransposeParams& b, hipStream_t s) {
  typedef NormRow<IODT> R;
  hipError_t err = hipSuccess;
  if (!slopes) {
    typedef typename std::conditional<sizeof(typename IoType<IODT>::T) == 4, unsigned, unsigned short>::type E;
    CASCMM_LAUNCH(err, (cascmm_transpose_kernel<E>), dim3(a.tiles + b.tiles), dim3(256), 0, s, a, b);
    return err;
  }
  const int parts = (int)ep_parts(p.rows, p.cols, IODT), lanes = ep_lanes(p.cols, IODT);
  const unsigned bands = (unsigned)((p.cols + lanes * R::VEC - 1) / (lanes * R::VEC));
  err = lanes == 64         ? ep_backward_launch<IODT, 64, false>(p, bands, (unsigned)parts, a, b, s)
        : p.cols < R::VEC ? ep_backward_launch<IODT, 16, true>(p, bands, (unsigned)parts, a, b, s)
                            : ep_backward_launch<IODT, 16, false>(p, bands, (unsigned)parts, a, b, s);
  if (p.partials)
    CASCMM_LAUNCH(err, (cascmm_column_finish_kernel<IODT>), dim3((unsigned)((p.cols + kFinishCols - 1) / kFinishCols), 1), dim3(1024), 0, s, (const float*)p.partials, parts, 1,
                  (int64_t)p.cols, dbias, (void*)nullptr);
  return err;
}

// one transposition's arguments; x NULL: none is wanted
static int transpose_of(const void* x, void* out, int64_t rows, int64_t cols, int64_t ldx, int64_t ldo, int dtype, TransposeParams& p) {
  memset(&p, 0, sizeof(p));
  if (rows < 0 || cols < 0 || ldx < cols || ldo < rows) return CASCMM_ERR_BAD_SHAPE;
  if (rows == 0 || cols == 0) return CASCMM_OK;
  if (!x || !out) return CASCMM_ERR_NULL_POINTER;
  if (!ep_aligned(x, ep_size(dtype)) || !ep_aligned(out, ep_size(dtype))) return CASCMM_ERR_ALIGNMENT;
  if (rows > (1 << 30) || cols > (1 << 30)) return CASCMM_ERR_TOO_LARGE;
  // (workgroups are counted in 32 bits, and their threads too)
  const int64_t across = (cols + 63) / 64, tiles = (rows + 63) / 64 * across;
  if (tiles > UINT32_MAX / 256 / 4) return CASCMM_ERR_TOO_LARGE;
  p = {x, out, ldx, ldo, (int)rows, (int)cols, (unsigned)across, (unsigned)tiles};
  return CASCMM_OK;
}

// cascmm_epilogue_backward with up to two transpositions beside it
static int epilogue_backward_with(const void* dy, const void* z, void* dz, void* dbias, int64_t rows, int64_t cols, int64_t lddy, int64_t ldz, int64_t lddz, int activation,
                                  int dtype, const TransposeParams& a, const TransposeParams& b, void* workspace, size_t workspace_bytes, hipStream_t s) {
  if (activation < CASCMM_ACT_NONE || activation > CASCMM_ACT_SILU) return CASCMM_ERR_BAD_FORMAT;
  if (rows < 0 || cols < 0 || lddy < cols || (activation && ldz < cols) || (dz && lddz < cols)) return CASCMM_ERR_BAD_SHAPE;
  if (rows > INT32_MAX || cols > kFinishMostCols) return CASCMM_ERR_TOO_LARGE;
  const bool slopes = cols > 0 && ((dz && rows > 0) || dbias);
  if (!slopes && a.tiles + b.tiles == 0) return CASCMM_OK;
  if (slopes) {
    if (rows > 0 && (!dy || (activation && !z))) return CASCMM_ERR_NULL_POINTER;
    const size_t es = ep_size(dtype);
    if (!ep_aligned(dy, es) || !ep_aligned(z, es) || !ep_aligned(dz, es) || !ep_aligned(dbias, es)) return CASCMM_ERR_ALIGNMENT;
    if (dbias) {
      if (!workspace || workspace_bytes < cascmm_epilogue_workspace_bytes(rows, cols, dtype)) return CASCMM_ERR_WORKSPACE;
      if (!ep_aligned(workspace, 16)) return CASCMM_ERR_ALIGNMENT;
    }
  }
  const SlopeParams p{dy, z, dz, slopes && dbias ? (float*)workspace : nullptr, lddy, ldz, lddz, rows, (int)cols, activation};
  const hipError_t err = dtype == CASCMM_DT_F32   ? ep_backward<CASCMM_DT_F32>(p, slopes, dbias, a, b, s)
                         : dtype == CASCMM_DT_F16 ? ep_backward<CASCMM_DT_F16>(p, slopes, dbias, a, b, s)
                                                  : ep_backward<CASCMM_DT_BF16>(p, slopes, dbias, a, b, s);
  return err == hipSuccess ? CASCMM_OK : CASCMM_ERR_LAUNCH;
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
  TransposeParams none;
  memset(&none, 0, sizeof(none));
  return epilogue_backward_with(dy, z, dz, dbias, rows, cols, lddy, ldz, lddz, activation, dtype, none, none, workspace, workspace_bytes, (hipStream_t)stream);
}

int cascmm_epilogue_backward_operands(const void* dy, const void* z, void* dz, void* dbias, const void* A, void* At, const void* B, void* Bt, int64_t M, int64_t N, int64_t K,
                                      int64_t lddy, int64_t ldz, int64_t lddz, int64_t lda, int64_t ldat, int64_t ldb, int64_t ldbt, int activation, int dtype,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  if (!ep_dtype(dtype)) return CASCMM_ERR_BAD_DTYPE;
  TransposeParams a, b;
  memset(&a, 0, sizeof(a));
  memset(&b, 0, sizeof(b));
  int st = K < 0 ? (int)CASCMM_ERR_BAD_SHAPE : CASCMM_OK;
  if (st == CASCMM_OK && At) st = transpose_of(A, At, M, K, lda, ldat, dtype, a);
  if (st == CASCMM_OK && Bt) st = transpose_of(B, Bt, K, N, ldb, ldbt, dtype, b);
  if (st != CASCMM_OK) return st;
  return epilogue_backward_with(dy, z, dz, dbias, M, N, lddy, ldz, lddz, activation, dtype, a, b, workspace, workspace_bytes, (hipStream_t)stream);
}

int cascmm_transpose(const void* x, void* out, int64_t rows, int64_t cols, int64_t ldx, int64_t ldo, int dtype, void* stream) {
  if (!ep_dtype(dtype)) return CASCMM_ERR_BAD_DTYPE;
  TransposeParams p;
  const int st = transpose_of(x, out, rows, cols, ldx, ldo, dtype, p);
  if (st != CASCMM_OK || p.tiles == 0) return st;
  TransposeParams none;
  memset(&none, 0, sizeof(none));
  return epilogue_backward_with(nullptr, nullptr, nullptr, nullptr, 0, 0, 0, 0, 0, CASCMM_ACT_NONE, dtype, p, none, nullptr, 0, (hipStream_t)stream);
}

}  // extern "C"
