// extern "C" entry points of the block-scaled products (cascmm_block_kernel.h): argument checks and the choice of kernel.
#include "cascmm_block_kernel.h"

#include <cstring>

#include <algorithm>
#include <cmath>

#include "cascmm_norm_kernel.h"
#include "cascmm_variants.h"

namespace cascmm {

static bool block_aligned(const void* p, size_t a) { return (uintptr_t)p % a == 0; }
static size_t block_size(int dtype) { return dtype == CASCMM_DT_F32 ? 4 : 2; }
static bool block_dtype(int dtype) { return dtype == CASCMM_DT_F32 || dtype == CASCMM_DT_F16 || dtype == CASCMM_DT_BF16; }
// (a tile's rows are addressed in 31 bits: 256 of them)
constexpr int64_t kBlockMostK = 1 << 22;

template <int IODT> static hipError_t block_round(const BlockRoundParams& p, bool square, unsigned tiles, hipStream_t s) {
  hipError_t err = hipSuccess;
  const int64_t strips = (p.rows + 15) / 16 * p.across;
  if (!square && !p.qt && !p.sums && strips < (1 << 24)) {
    CASCMM_LAUNCH(err, cascmm_block_round_rows_kernel<IODT>, dim3((unsigned)strips), dim3(256), 0, s, p);
    return err;
  }
  CASCMM_LAUNCH(err, (square ? cascmm_block_round_kernel<IODT, true> : cascmm_block_round_kernel<IODT, false>), dim3(tiles), dim3(256), 0, s, p);
  return err;
}

// The tiles: estimated microseconds from what was measured (us in a graph, 8192 x 8192 x 8192 bf16 / 8192 x 1280 x 5120 / 2048 x 10240 x 1280 / 1024 x 1280 x 5120 / 154 x 5120 x 1280):
// 256 x 256 on eight waves, one workgroup on a CU, 409 / 52.6 / 37.0 / 48.1 / 15.1; 128 x 128, two on a CU, so that one's stores hide behind the other's products, 480 / 68.2 / 34.6 /
// 31.2 / 7.9; 128 x 64, three stages deep, 640 / 68.2 / 42.8 / 17.4 / 6.7; 64 x 64, as deep, 825 / 90.5 / 51.3 / 18.8 / 5.7 (two deep 816 / 88.8 / 50.8 / 22.9 / 5.9 with the weights in the caches,
// and 1.6 more of 154 x 5120 x 1280 with them in memory); 64 x 64 with k dealt to two groups of waves, four stages deep, 977 / 115 / 96.9 / 23.9 / 6.1, and for 640 x 640 x 8192 17.0 where the
// others take 70, 42, 24 and 20.  Of 25 sizes the estimate's tile is the best or within 5 % for 24, 13 % behind for one.  In the terms: what a block of k and a tile's beginning and end take,
// times the tiles that fall to a CU.  Where the last turn of 256 x 256 tiles would leave half of the CUs or more without one, its tiles are cut in pieces, four (128 x 128) up to a quarter of a
// turn and two (128 x 256) up to a half: 2048 x 10240 x 1280 33.5 where 128 x 128 takes 35.2 and 256 x 256 38.9, 4096 x 5120 x 2560 51.1, 61.9 and 62.3, 2304 x 8192 x 4096 69.8, 88.8 and 90.6,
// 8192 x 5120 x 1280, in twos, 59.2, 73 and 62.1; of twelve such sizes the rule's is the best for eleven, 9 % behind for one.
typedef BlockTile<2, 2, 1, 1, 3, 1> BlockTile64;
typedef BlockTile<2, 2, 1, 1, 4, 2> BlockTile64Shares;
typedef BlockTile<2, 2, 2, 1, 3, 1> BlockTile128x64;
typedef BlockTile<2, 2, 2, 2, 2, 1> BlockTile128;
typedef BlockTile<2, 4, 4, 2, 2, 1> BlockTile256;
typedef BlockTile<2, 4, 2, 1, 3, 1> BlockPiece128;     // (on the waves of a 256 x 256 tile)
typedef BlockTile<2, 4, 2, 2, 2, 1> BlockPiece128x256;
enum { kTile64, kTile64Shares, kTile128x64, kTile128, kTile256, kTile256Pieces, kTiles };
static int block_tile(int64_t M, int64_t N, int64_t blocks, bool fine) {
  const auto tiles = [&](int64_t bm, int64_t bn) { return ((M + bm - 1) / bm) * ((N + bn - 1) / bn); };
  const double k = (double)blocks;
  double cost[kTiles];
  const int64_t small = tiles(64, 64), n64 = (small + 255) / 256, n128x64 = (tiles(128, 64) + 255) / 256, n128 = (tiles(128, 128) + 255) / 256, t256 = tiles(256, 256), n256 = (t256 + 255) / 256;
  cost[kTile64] = std::max(n64 * (0.22 * k + 0.9), 0.3 * k + 1.0);
  cost[kTile64Shares] = n64 * (0.23 * k + 1.9);
  cost[kTile128x64] = n128x64 <= 1 ? 0.36 * k + 1.2 : n128x64 * (0.31 * k + 1.0);
  cost[kTile128] = n128 <= 1 ? 0.62 * k + 1.5 : n128 == 2 ? 2 * (0.45 * k + 1.5) : n128 * (0.5 * k + 2.0);
  cost[kTile256] = t256 <= 256 ? (t256 <= 128 ? 1.05 : 1.2) * k + 3.5 : n256 * (1.4 * k + 5.5);
  cost[kTile256Pieces] = t256 > 256 && t256 % 256 != 0 && t256 % 256 <= 128 ? (n256 - 1) * (1.4 * k + 5.5) + (t256 % 256 <= 64 ? 0.45 : 0.75) * k + 8.0 : INFINITY;
  int best = kTile64;
  for (int i = 0; i < kTiles; ++i)
    if (cost[i] < cost[best] && !(fine && i >= kTile256)) best = i;     // (widened fragments do not fit beside 128 x 64 sums of a wave)
  return best;
}

// Launches of fewer than 2^32 threads, and scales that 31 bits of an offset span
static bool block_too_large(int64_t M, int64_t N, int64_t K, bool fine) {
  if (M > INT32_MAX || N > INT32_MAX || K > kBlockMostK || block_scale_bytes(std::max(M, N), K) > INT32_MAX) return true;
  const int tile = block_tile(M, N, block_padded(K) / kBlock, fine);
  const int64_t bm = tile <= kTile64Shares ? 64 : tile >= kTile256 ? 256 : 128, bn = tile <= kTile128x64 ? 64 : tile >= kTile256 ? 256 : 128;
  return ((M + bm - 1) / bm) * ((N + bn - 1) / bn) > (int64_t)UINT32_MAX / 512 - 256;     // (pieces: up to 192 more)
}

template <int IODT, typename T> static hipError_t block_gemm_tile(BlockGemmParams p, hipStream_t s) {
  hipError_t err = hipSuccess;
  constexpr bool FINE = IODT == CASCMM_DT_F32;
  static LdsFlags done;
  if (T::LDS > 64 * 1024 && !ensure_lds((const void*)cascmm_block_gemm_kernel<IODT, T, FINE>, T::LDS, done)) return hipErrorInvalidValue;
  p.tiles_m = (p.M + T::BM - 1) / T::BM;
  p.tiles_n = (p.N + T::BN - 1) / T::BN;
  CASCMM_LAUNCH(err, (cascmm_block_gemm_kernel<IODT, T, FINE>), dim3((unsigned)p.tiles_m * (unsigned)p.tiles_n), dim3(T::THREADS), T::LDS, s, p);
  return err;
}
template <int IODT, typename T, typename R> static hipError_t block_gemm_pieces(BlockGemmParams p, hipStream_t s) {
  hipError_t err = hipSuccess;
  static LdsFlags done;
  if (!ensure_lds((const void*)cascmm_block_gemm_pieces_kernel<IODT, T, R>, T::LDS, done)) return hipErrorInvalidValue;
  p.tiles_m = (p.M + T::BM - 1) / T::BM;
  p.tiles_n = (p.N + T::BN - 1) / T::BN;
  const unsigned tiles = (unsigned)p.tiles_m * (unsigned)p.tiles_n;
  p.whole = (int)(tiles / 256 * 256);
  const unsigned pieces = (tiles - (unsigned)p.whole) * (T::BM / R::BM) * (T::BN / R::BN);
  CASCMM_LAUNCH(err, (cascmm_block_gemm_pieces_kernel<IODT, T, R>), dim3((unsigned)p.whole + pieces), dim3(T::THREADS), T::LDS, s, p);
  return err;
}
template <int IODT> static hipError_t block_gemm(const BlockGemmParams& p, hipStream_t s) {
  constexpr bool FINE = IODT == CASCMM_DT_F32;
  switch (block_tile(p.M, p.N, p.blocks, FINE)) {
    case kTile64: return block_gemm_tile<IODT, BlockTile64>(p, s);
    case kTile64Shares: return block_gemm_tile<IODT, BlockTile64Shares>(p, s);
    case kTile128x64: return block_gemm_tile<IODT, BlockTile128x64>(p, s);
    case kTile128: return block_gemm_tile<IODT, BlockTile128>(p, s);
    case kTile256:
      if constexpr (!FINE) return block_gemm_tile<IODT, BlockTile256>(p, s);
      return hipErrorInvalidValue;
    default:
      if constexpr (!FINE) {
        const int64_t left = (int64_t)((p.M + 255) / 256) * ((p.N + 255) / 256) % 256;
        return left <= 64 ? block_gemm_pieces<IODT, BlockTile256, BlockPiece128>(p, s) : block_gemm_pieces<IODT, BlockTile256, BlockPiece128x256>(p, s);
      }
      return hipErrorInvalidValue;
  }
}

template <int IODT, int WAVES> static hipError_t block_rows_waves(const BlockRowsParams& p, hipStream_t s) {
  hipError_t err = hipSuccess;
  const dim3 grid((unsigned)(p.N + 15) / 16, (unsigned)(p.M + 15) / 16), threads(64 * WAVES);
  if (p.M <= 4) CASCMM_LAUNCH(err, (cascmm_block_rows_kernel<IODT, WAVES, 1>), grid, threads, 0, s, p);
  else if (p.M <= 8) CASCMM_LAUNCH(err, (cascmm_block_rows_kernel<IODT, WAVES, 2>), grid, threads, 0, s, p);
  else CASCMM_LAUNCH(err, (cascmm_block_rows_kernel<IODT, WAVES, 4>), grid, threads, 0, s, p);
  return err;
}
// Sixteen waves where no CU gets a second workgroup, eight behind that (us, 16 waves / 8: 1 x 5120 x 1280 5.3 / 5.4, 16 x 5120 x 1280 8.2 / 9.2; 1 x 1280 x 10240 7.7 / 5.5, 16 x 1280 x 5120
// 7.5 / 6.0, 8 x 10240 x 10240 33.5 / 29.9)
static int64_t block_rows_groups(int64_t M, int64_t N) { return (M + 15) / 16 * ((N + 15) / 16); }
template <int IODT> static hipError_t block_rows(const BlockRowsParams& p, hipStream_t s) {
  return block_rows_groups(p.M, p.N) <= 256 ? block_rows_waves<IODT, 16>(p, s) : block_rows_waves<IODT, 8>(p, s);
}
// Which products take that one launch: those of sixteen rows, and of more while two workgroups fall to a CU (us, so / rounded in a launch of its own, then tiles: 48 x 5120 x 1280 8.3 / 13.9,
// 90 x 640 x 640 3.8 / 6.4, 8192 x 640 x 16 4.4 / 9.5, 77 x 2048 x 1280 7.5 / 9.4, 64 x 40960 x 640 45 / 108, 128 x 10240 x 640 21.3 / 23.1; with three, 512 x 640 x 384 6.3 / 6.6 but
// 154 x 1280 x 1280 9.8 / 8.1).  fp32 results come from the 16-bit instruction, which this kernel does not use.
constexpr int64_t kBlockRowsMost = 512;
static bool block_few_rows(int64_t M, int64_t N, int64_t K, int dtype) { return (M <= 16 || block_rows_groups(M, N) <= kBlockRowsMost) && K > 0 && dtype != CASCMM_DT_F32; }
static size_t block_slice(size_t bytes) { return (bytes + 255) / 256 * 256; }

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
  if (block_too_large(M, N, K, dtype == CASCMM_DT_F32)) return CASCMM_ERR_TOO_LARGE;
  if (M == 0 || N == 0) return CASCMM_OK;
  if (!C || (K > 0 && (!a || !a_scales || !b || !b_scales))) return CASCMM_ERR_NULL_POINTER;
  const size_t es = block_size(dtype);
  if (!block_aligned(C, es) || !block_aligned(bias, es) || !block_aligned(a, 16) || !block_aligned(b, 16) || !block_aligned(a_scales, 4) || !block_aligned(b_scales, 4))
    return CASCMM_ERR_ALIGNMENT;
  BlockGemmParams p;
  memset(&p, 0, sizeof(p));
  p.a = (const unsigned char*)a; p.b = (const unsigned char*)b; p.sa = (const unsigned*)a_scales; p.sb = (const unsigned*)b_scales;
  p.c = C; p.bias = bias; p.ldc = ldc;
  p.M = (int)M; p.N = (int)N; p.blocks = (int)(block_padded(K) / kBlock);
  const hipStream_t s = (hipStream_t)stream;
  const hipError_t err = dtype == CASCMM_DT_F32   ? block_gemm<CASCMM_DT_F32>(p, s)
                         : dtype == CASCMM_DT_F16 ? block_gemm<CASCMM_DT_F16>(p, s)
                                                  : block_gemm<CASCMM_DT_BF16>(p, s);
  return err == hipSuccess ? CASCMM_OK : CASCMM_ERR_LAUNCH;
}

size_t cascmm_block_linear_workspace_bytes(int64_t M, int64_t K, int dtype) {
  if (M < 0 || K < 0 || M > INT32_MAX || K > kBlockMostK || !block_dtype(dtype) || (M <= 16 && block_few_rows(M, 0, K, dtype))) return 0;
  return block_slice((size_t)(M * block_padded(K))) + (size_t)block_scale_bytes(M, K);
}

int cascmm_block_linear(const void* x, const void* b, const void* b_scales, void* C, const void* bias, int64_t M, int64_t N, int64_t K, int64_t ldx, int64_t ldc, int dtype,
                        void* workspace, size_t workspace_bytes, void* stream) {
  if (!block_dtype(dtype)) return CASCMM_ERR_BAD_DTYPE;
  if (M < 0 || N < 0 || K < 0 || ldx < K || ldc < N) return CASCMM_ERR_BAD_SHAPE;
  if (M > INT32_MAX || N > INT32_MAX || K > kBlockMostK) return CASCMM_ERR_TOO_LARGE;
  if (M == 0 || N == 0) return CASCMM_OK;
  // (whichever kernel takes the call: what a caller has to bring depends on M and K alone)
  const size_t need = cascmm_block_linear_workspace_bytes(M, K, dtype);
  if (need && (!workspace || workspace_bytes < need)) return CASCMM_ERR_WORKSPACE;
  if (need && !block_aligned(workspace, 16)) return CASCMM_ERR_ALIGNMENT;
  if (!block_few_rows(M, N, K, dtype)) {
    void* const scales = (char*)workspace + block_slice((size_t)(M * block_padded(K)));
    // (everything is checked before the first launch: the product's own checks see the same arguments)
    if (!C || (K > 0 && (!x || !b || !b_scales))) return CASCMM_ERR_NULL_POINTER;
    if (block_too_large(M, N, K, dtype == CASCMM_DT_F32)) return CASCMM_ERR_TOO_LARGE;
    if (!block_aligned(C, block_size(dtype)) || !block_aligned(bias, block_size(dtype)) || !block_aligned(b, 16) || !block_aligned(b_scales, 4)) return CASCMM_ERR_ALIGNMENT;
    const int st = K > 0 ? cascmm_block_round(x, M, K, ldx, dtype, 0, workspace, scales, nullptr, nullptr, nullptr, nullptr, 0, stream) : (int)CASCMM_OK;
    return st != CASCMM_OK ? st : cascmm_block_gemm(workspace, scales, b, b_scales, C, bias, M, N, K, ldc, dtype, stream);
  }
  if (!C || !x || !b || !b_scales) return CASCMM_ERR_NULL_POINTER;
  const size_t es = block_size(dtype);
  if (!block_aligned(C, es) || !block_aligned(bias, es) || !block_aligned(x, es) || !block_aligned(b, 16) || !block_aligned(b_scales, 4)) return CASCMM_ERR_ALIGNMENT;
  if ((N + 15) / 16 > (1 << 22) - 1) return CASCMM_ERR_TOO_LARGE;
  BlockRowsParams p;
  memset(&p, 0, sizeof(p));
  p.x = x; p.b = (const unsigned char*)b; p.sb = (const unsigned*)b_scales; p.c = C; p.bias = bias; p.ldx = ldx; p.ldc = ldc;
  p.M = (int)M; p.N = (int)N; p.K = (int)K; p.blocks = (int)(block_padded(K) / kBlock);
  const hipError_t err = dtype == CASCMM_DT_F16 ? block_rows<CASCMM_DT_F16>(p, (hipStream_t)stream) : block_rows<CASCMM_DT_BF16>(p, (hipStream_t)stream);
  return err == hipSuccess ? CASCMM_OK : CASCMM_ERR_LAUNCH;
}

}  // extern "C"
