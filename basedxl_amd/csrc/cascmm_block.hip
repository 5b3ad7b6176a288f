// extern "C" entry points of the block-scaled products (cascmm_block_kernel.h): argument checks and the choice of kernel.
#include "cascmm_block_kernel.h"

#include <cstring>

#include <algorithm>

#include "cascmm_norm_kernel.h"

namespace cascmm {

static bool block_aligned(const void* p, size_t a) { return (uintptr_t)p % a == 0; }
static size_t block_size(int dtype) { return dtype == CASCMM_DT_F32 ? 4 : 2; }
static bool block_dtype(int dtype) { return dtype == CASCMM_DT_F32 || dtype == CASCMM_DT_F16 || dtype == CASCMM_DT_BF16; }
// (a tile's rows are addressed in 31 bits: 256 of them)
constexpr int64_t kBlockMostK = 1 << 22;

template <int IODT> static hipError_t block_round(const BlockRoundParams& p, bool square, unsigned tiles, hipStream_t s) {
  hipError_t err = hipSuccess;
  CASCMM_LAUNCH(err, (square ? cascmm_block_round_kernel<IODT, true> : cascmm_block_round_kernel<IODT, false>), dim3(tiles), dim3(256), 0, s, p);
  return err;
}

template <int IODT, int MT, int NT> static hipError_t block_gemm(BlockGemmParams p, hipStream_t s) {
  hipError_t err = hipSuccess;
  constexpr int BM = 64 * MT, BN = 64 * NT, LDS = 2 * (BM + BN) * 128;
  p.tiles_m = (p.M + BM - 1) / BM;
  p.tiles_n = (p.N + BN - 1) / BN;
  CASCMM_LAUNCH(err, (cascmm_block_gemm_kernel<IODT, MT, NT, IODT == CASCMM_DT_F32>), dim3((unsigned)p.tiles_m * (unsigned)p.tiles_n), dim3(256), LDS, s, p);
  return err;
}

}  // namespace cascmm

using namespace cascmm;

extern "C" {

size_t cascmm_block_values_bytes(int64_t rows, int64_t k) {
  if (rows < 0 || k < 0 || rows > INT32_MAX || k > INT32_MAX) return 0;
  return (size_t)(rows * block_padded(k));
}
size_t cascmm_block_scales_bytes(int64_t rows, int64_t k) {
  if (rows < 0 || k < 0 || rows > INT32_MAX || k > INT32_MAX) return 0;
  return (size_t)block_scale_bytes(rows, k);
}
size_t cascmm_block_round_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0 || rows > INT32_MAX || cols > kFinishMostCols) return 0;
  return (size_t)((rows + kBlock - 1) / kBlock * cols) * sizeof(float);
}

int cascmm_block_round(const void* x, int64_t rows, int64_t cols, int64_t ldx, int dtype, int square, void* values, void* scales, void* values_t, void* scales_t, void* sums,
                       void* workspace, size_t workspace_bytes, void* stream) {
  if (!block_dtype(dtype)) return CASCMM_ERR_BAD_DTYPE;
  if (rows < 0 || cols < 0 || ldx < cols) return CASCMM_ERR_BAD_SHAPE;
  if (rows > INT32_MAX || cols > kFinishMostCols) return CASCMM_ERR_TOO_LARGE;
  if ((values != nullptr) != (scales != nullptr) || (values_t != nullptr) != (scales_t != nullptr)) return CASCMM_ERR_NULL_POINTER;
  if (cols == 0 || (rows == 0 && !sums) || (!values && !values_t && !sums)) return CASCMM_OK;
  if (rows > 0 && !x) return CASCMM_ERR_NULL_POINTER;
  const size_t es = block_size(dtype);
  if (!block_aligned(x, es) || !block_aligned(values, 16) || !block_aligned(scales, 4) || !block_aligned(values_t, 16) || !block_aligned(scales_t, 4) || !block_aligned(sums, es))
    return CASCMM_ERR_ALIGNMENT;
  if (sums) {
    if (!workspace && rows > 0) return CASCMM_ERR_WORKSPACE;
    if (workspace_bytes < cascmm_block_round_workspace_bytes(rows, cols)) return CASCMM_ERR_WORKSPACE;
    if (!block_aligned(workspace, 16)) return CASCMM_ERR_ALIGNMENT;
  }
  const int64_t down = (rows + kBlock - 1) / kBlock, across = (cols + kBlock - 1) / kBlock;
  if (down * across > (1 << 24) - 1) return CASCMM_ERR_TOO_LARGE;      // (a launch has fewer than 2^32 threads)
  BlockRoundParams p;
  memset(&p, 0, sizeof(p));
  p.x = x; p.q = (unsigned char*)values; p.s = (unsigned char*)scales; p.qt = (unsigned char*)values_t; p.st = (unsigned char*)scales_t;
  p.sums = sums ? (float*)workspace : nullptr;
  p.rows = rows; p.cols = cols; p.ldx = ldx; p.across = (unsigned)across;
  const hipStream_t s = (hipStream_t)stream;
  hipError_t err = hipSuccess;
  if (rows > 0)
    err = dtype == CASCMM_DT_F32   ? block_round<CASCMM_DT_F32>(p, square != 0, (unsigned)(down * across), s)
          : dtype == CASCMM_DT_F16 ? block_round<CASCMM_DT_F16>(p, square != 0, (unsigned)(down * across), s)
                                   : block_round<CASCMM_DT_BF16>(p, square != 0, (unsigned)(down * across), s);
  if (sums && err == hipSuccess) {
    const dim3 grid((unsigned)((cols + kFinishCols - 1) / kFinishCols), 1);
    if (dtype == CASCMM_DT_F32)
      CASCMM_LAUNCH(err, (cascmm_column_finish_kernel<CASCMM_DT_F32>), grid, dim3(1024), 0, s, (const float*)workspace, (int)down, 1, cols, sums, (void*)nullptr);
    else if (dtype == CASCMM_DT_F16)
      CASCMM_LAUNCH(err, (cascmm_column_finish_kernel<CASCMM_DT_F16>), grid, dim3(1024), 0, s, (const float*)workspace, (int)down, 1, cols, sums, (void*)nullptr);
    else
      CASCMM_LAUNCH(err, (cascmm_column_finish_kernel<CASCMM_DT_BF16>), grid, dim3(1024), 0, s, (const float*)workspace, (int)down, 1, cols, sums, (void*)nullptr);
  }
  return err == hipSuccess ? CASCMM_OK : CASCMM_ERR_LAUNCH;
}

int cascmm_block_gemm(const void* a, const void* a_scales, const void* b, const void* b_scales, void* C, const void* bias, int64_t M, int64_t N, int64_t K, int64_t ldc, int dtype,
                      void* stream) {
  if (!block_dtype(dtype)) return CASCMM_ERR_BAD_DTYPE;
  if (M < 0 || N < 0 || K < 0 || ldc < N) return CASCMM_ERR_BAD_SHAPE;
  if (M > INT32_MAX || N > INT32_MAX || K > kBlockMostK) return CASCMM_ERR_TOO_LARGE;
  if (M == 0 || N == 0) return CASCMM_OK;
  if (!C || (K > 0 && (!a || !a_scales || !b || !b_scales))) return CASCMM_ERR_NULL_POINTER;
  const size_t es = block_size(dtype);
  if (!block_aligned(C, es) || !block_aligned(bias, es) || !block_aligned(a, 16) || !block_aligned(b, 16) || !block_aligned(a_scales, 4) || !block_aligned(b_scales, 4))
    return CASCMM_ERR_ALIGNMENT;
  if ((M + 127) / 128 * ((N + 127) / 128) > (1 << 24) - 1) return CASCMM_ERR_TOO_LARGE;
  BlockGemmParams p;
  memset(&p, 0, sizeof(p));
  p.a = (const unsigned char*)a; p.b = (const unsigned char*)b; p.sa = (const unsigned*)a_scales; p.sb = (const unsigned*)b_scales;
  p.c = C; p.bias = bias; p.ldc = ldc;
  p.M = (int)M; p.N = (int)N; p.blocks = (int)(block_padded(K) / kBlock);
  const hipStream_t s = (hipStream_t)stream;
  const hipError_t err = dtype == CASCMM_DT_F32   ? block_gemm<CASCMM_DT_F32, 2, 2>(p, s)
                         : dtype == CASCMM_DT_F16 ? block_gemm<CASCMM_DT_F16, 2, 2>(p, s)
                                                  : block_gemm<CASCMM_DT_BF16, 2, 2>(p, s);
  return err == hipSuccess ? CASCMM_OK : CASCMM_ERR_LAUNCH;
}

}  // extern "C"
