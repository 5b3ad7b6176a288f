// Products of 8-bit floating-point operands with a scale for each block of 128 (gfx950): the operands' rounding and the product.
//
//   q = e4m3(x 2^-e), nearest, ties to even;   C[m][n] = sum over blocks of k of 2^(ea[m][block] + eb[n][block]) sum over the block of qa[m][k] qb[n][k]  (+ bias[n])
//
// The scale of a block is the smallest power of two with max|x| <= 448 * 2^e over its finite elements: scaling is exact, and the matrix instruction
// applies it by itself (one E8M0 byte a lane), so that all blocks of a row meet in one fp32 accumulator and nothing is added to the loop for the scales.
// Infinities and NaN become NaN.
//
// Operands lie as rows of bytes along k, [rows][k rounded up to 128], what is behind k zero; the scales as bytes [block / 4][rows][4], so that a lane
// fetches those of its row for four blocks at once.  Both operands have this form: a right operand [K][N] is stored transposed.
#pragma once
#include <type_traits>

#include "cascmm_common.h"

namespace cascmm {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kBlock = 128;
inline __host__ __device__ int64_t block_padded(int64_t k) { return (k + kBlock - 1) / kBlock * kBlock; }
inline __host__ __device__ int64_t block_scale_bytes(int64_t rows, int64_t k) { return (block_padded(k) / kBlock + 3) / 4 * rows * 4; }

// ---------------------------------------------------------------------------------------
// rounding
// ---------------------------------------------------------------------------------------
struct BlockRoundParams {
  const void* x;         // [rows][cols], row stride ldx
  unsigned char* q;      // NULL or [rows][cols padded]: blocks along the columns
  unsigned char* s;      // its scales
  unsigned char* qt;     // NULL or [cols][rows padded]: the transposed, blocks along the rows
  unsigned char* st;
  float* sums;           // NULL or [tiles of rows][cols]: sums over a tile's rows
  int64_t rows, cols, ldx;
  unsigned across;       // tiles in a row of tiles
};

template <int CTRL> __device__ __forceinline__ unsigned block_dpp(unsigned v) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true); }
__device__ __forceinline__ unsigned block_larger(unsigned a, unsigned b) { return a > b ? a : b; }
// the largest over the sixteen lanes of a row of lanes, in each of them
__device__ __forceinline__ unsigned block_row_max(unsigned v) {
  v = block_larger(v, block_dpp<0xB1>(v));
  v = block_larger(v, block_dpp<0x4E>(v));
  v = block_larger(v, block_dpp<0x141>(v));
  return block_larger(v, block_dpp<0x140>(v));
}
// the scale's E8M0 byte from the bits of max|x| (finite): 448 = 1.75 * 2^8, so a mantissa beyond 1.75 takes one more
__device__ __forceinline__ unsigned block_scale(unsigned most) {
  const int byte = (int)((most + 0x1FFFFFu) >> 23) - 8;
  return most == 0 ? 127u : byte < 0 ? 0u : (unsigned)byte;
}
__device__ __forceinline__ float block_inverse(unsigned byte) { return __builtin_bit_cast(float, (254u - byte) << 23); }   // (2^-e, e from -127 to 120: a normal number)
__device__ __forceinline__ u32x2 block_pack(const float (&v)[8], float f) {
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * f, v[1] * f, lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * f, v[3] * f, lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * f, v[5] * f, hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * f, v[7] * f, hi, true);
  return (u32x2){(unsigned)lo, (unsigned)hi};
}

// A tile of 128 x 128 a workgroup, read once: a thread holds 8 rows of 8 columns, sixteen threads a row of the tile.
// SQUARE: one scale for the whole tile; else one for each of its rows (q) and of its columns (qt).
template <int IODT, bool SQUARE>
__global__ __launch_bounds__(256) void cascmm_block_round_kernel(const BlockRoundParams p) {
  typedef typename IoType<IODT>::T E;
  typedef E chunk __attribute__((ext_vector_type(8), aligned(sizeof(E))));   // (rows start on elements, not on 16 bytes)
  __shared__ unsigned col_most[4][kBlock];
  __shared__ float col_sum[4][kBlock];
  __shared__ u32x2 turned[kBlock][16];       // [column][eight rows], the eights of a column in the order i ^ (column / 8): writes and reads without conflicts
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, wave = tid >> 6;
  const int64_t tile_row = blockIdx.x / p.across, tile_col = blockIdx.x % p.across;
  const int64_t row0 = tile_row * kBlock + ty * 8, col0 = tile_col * kBlock + tx * 8;
  const E* src = (const E*)p.x + row0 * p.ldx + col0;
  float v[8][8];
  const int64_t left = p.cols - col0;
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    if (row0 + r < p.rows && left >= 8) {
      const chunk c = *(const chunk*)(src + r * p.ldx);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[r][e] = (float)c[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[r][e] = row0 + r < p.rows && e < left ? (float)src[r * p.ldx + e] : 0.f;
    }
  }
  if (p.sums) {
    // sums over the tile's rows: eight in a thread, four threads of a wave, four waves, in this order
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float s = 0.f;
#pragma unroll
      for (int r = 0; r < 8; ++r) s += v[r][e];
      s += __shfl_xor(s, 16, 64);
      s += __shfl_xor(s, 32, 64);
      if ((tid & 63) < 16) col_sum[wave][tx * 8 + e] = s;
    }
  }
  unsigned row_most[8], most[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) most[e] = 0;
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    row_most[r] = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned bits = __builtin_bit_cast(unsigned, v[r][e]) & 0x7FFFFFFFu;
      const bool finite = bits < 0x7F800000u;
      v[r][e] = finite ? v[r][e] : __builtin_nanf("");
      const unsigned b = finite ? bits : 0u;
      row_most[r] = block_larger(row_most[r], b);
      most[e] = block_larger(most[e], b);
    }
  }
  unsigned square = 0;
  if (SQUARE) {
#pragma unroll
    for (int r = 0; r < 8; ++r) square = block_larger(square, row_most[r]);
    square = block_row_max(square);
    square = block_larger(square, (unsigned)__shfl_xor((int)square, 16, 64));
    square = block_larger(square, (unsigned)__shfl_xor((int)square, 32, 64));
    if ((tid & 63) == 0) col_most[wave][0] = square;
    __syncthreads();
    square = block_scale(block_larger(block_larger(col_most[0][0], col_most[1][0]), block_larger(col_most[2][0], col_most[3][0])));
  }
  if (p.q) {
    const int64_t padded = block_padded(p.cols);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const unsigned byte = SQUARE ? square : block_scale(block_row_max(row_most[r]));
      if (row0 + r < p.rows) {
        *(u32x2*)(p.q + (row0 + r) * padded + col0) = block_pack(v[r], block_inverse(byte));
        if (tx == 0) p.s[((tile_col >> 2) * p.rows + row0 + r) * 4 + (tile_col & 3)] = (unsigned char)byte;
      }
    }
  }
  if (!p.qt && !p.sums) return;
  if (!SQUARE && p.qt) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      most[e] = block_larger(most[e], (unsigned)__shfl_xor((int)most[e], 16, 64));
      most[e] = block_larger(most[e], (unsigned)__shfl_xor((int)most[e], 32, 64));
      if ((tid & 63) < 16) col_most[wave][tx * 8 + e] = most[e];
    }
  }
  __syncthreads();
  if (p.sums && tid < kBlock && tile_col * kBlock + tid < p.cols)
    p.sums[tile_row * p.cols + tile_col * kBlock + tid] = (col_sum[0][tid] + col_sum[1][tid]) + (col_sum[2][tid] + col_sum[3][tid]);
  if (!p.qt) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int c = tx * 8 + e;
    const unsigned byte = SQUARE ? square : block_scale(block_larger(block_larger(col_most[0][c], col_most[1][c]), block_larger(col_most[2][c], col_most[3][c])));
    const float column[8] = {v[0][e], v[1][e], v[2][e], v[3][e], v[4][e], v[5][e], v[6][e], v[7][e]};
    turned[c][ty ^ tx] = block_pack(column, block_inverse(byte));
    if (ty == 0 && col0 + e < p.cols) p.st[((tile_row >> 2) * p.cols + col0 + e) * 4 + (tile_row & 3)] = (unsigned char)byte;
  }
  __syncthreads();
  const int64_t padded = block_padded(p.rows);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = i * 32 + (tid >> 3), k = tid & 7, turn = (c >> 3) & 15;
    const int64_t col = tile_col * kBlock + c;
    const u32x2 lo = turned[c][(2 * k) ^ turn], hi = turned[c][(2 * k + 1) ^ turn];
    if (col < p.cols) *(u32x4*)(p.qt + col * padded + tile_row * kBlock + k * 16) = (u32x4){lo[0], lo[1], hi[0], hi[1]};
  }
}

// ---------------------------------------------------------------------------------------
// product
// ---------------------------------------------------------------------------------------
struct BlockGemmParams {
  const unsigned char *a, *b;      // [M][K padded], [N][K padded]
  const unsigned *sa, *sb;         // [blocks / 4][M], [blocks / 4][N], four bytes each
  void* c;                         // [M][N], row stride ldc
  const void* bias;                // NULL or [N] of the type of c
  int64_t ldc;
  int M, N, blocks;                // blocks of 128 along k
  int tiles_m, tiles_n;
};

typedef __attribute__((address_space(3))) void* block_lds_ptr;
__device__ __forceinline__ void block_load_lds(__amdgpu_buffer_rsrc_t rsrc, unsigned char* dst, int voffset, int soffset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (block_lds_ptr)dst, 16, voffset, soffset, 0, 0);
}

// 2 x 2 waves, each MT x NT blocks of 32 x 32.  A stage is one block of k: rows of 128 bytes in LDS, the eight 16-byte pieces of row r in the order i ^ (r % 8), so that
// the lanes of a fragment read, 32 rows apart by 128 bytes, hit all banks.  The copy to LDS writes in order; the order is made by the addresses it reads.
// FINE: products and sums by the 16-bit matrix instruction, to fp32's accuracy.  The 8-bit one cuts the products inside an instruction at about 2^-15 of the largest: 1.5e-5
// of the result's size, unbiased and the same for every depth, which 16-bit results do not show and fp32 ones would.  (bf16 holds the scaled values exactly, but for those
// below 2^-126, which the instruction takes as zeros.)
template <int IODT, int MT, int NT, bool FINE>
__global__ __launch_bounds__(256) void cascmm_block_gemm_kernel(const BlockGemmParams p) {
  typedef typename IoType<IODT>::T E;
  constexpr int BM = 64 * MT, BN = 64 * NT, STAGE = (BM + BN) * 128, LOADS = (BM + BN) / 8 / 4;
  extern __shared__ __attribute__((aligned(1024))) unsigned char block_smem[];
  const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tile_m = blockIdx.x / p.tiles_n, tile_n = blockIdx.x % p.tiles_n;
  const int m0 = tile_m * BM, n0 = tile_n * BN, wm = (wave >> 1) * 32 * MT, wn = (wave & 1) * 32 * NT;
  const int64_t kp = (int64_t)p.blocks * kBlock;
  // (a tile's rows lie below 2 GiB from its first: host-checked)
  const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc((void*)(p.a + m0 * kp), 0, 0x7FFFFFFF, 0x00020000);
  const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc((void*)(p.b + n0 * kp), 0, 0x7FFFFFFF, 0x00020000);
  int from[LOADS];
#pragma unroll
  for (int j = 0; j < LOADS; ++j) {
    int r = (wave + 4 * j) * 8 + (lane >> 3);
    const bool second = r >= BM;
    r -= second ? BM : 0;
    const int last = (second ? p.N - n0 : p.M - m0) - 1, row = r < last ? r : last;     // (rows past the edge: the last one again)
    from[j] = (int)(row * kp) + (((lane & 7) ^ (r & 7)) << 4);
  }
  auto issue = [&](int step) {
    unsigned char* to = block_smem + (step & 1) * STAGE;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) block_load_lds((wave + 4 * j) * 8 >= BM ? rb : ra, to + (wave + 4 * j) * 1024, from[j], step * kBlock);
  };
  const unsigned *sa[MT], *sb[NT];
#pragma unroll
  for (int i = 0; i < MT; ++i) sa[i] = p.sa + (m0 + wm + 32 * i + l31 < p.M ? m0 + wm + 32 * i + l31 : p.M - 1);
#pragma unroll
  for (int i = 0; i < NT; ++i) sb[i] = p.sb + (n0 + wn + 32 * i + l31 < p.N ? n0 + wn + 32 * i + l31 : p.N - 1);
  unsigned a_scale[MT], b_scale[NT], a_next[MT], b_next[NT];
  auto scales = [&](int four) {
#pragma unroll
    for (int i = 0; i < MT; ++i) a_next[i] = sa[i][(int64_t)four * p.M];
#pragma unroll
    for (int i = 0; i < NT; ++i) b_next[i] = sb[i][(int64_t)four * p.N];
  };
  f32x16 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  if (p.blocks > 0) {     // (else: nothing but the bias)
    issue(0);
    scales(0);
  }
  for (int step = 0; step < p.blocks; ++step) {
    __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0), lgkmcnt(0): this stage has landed, the last one is read
    __syncthreads();
    if ((step & 3) == 0) {
#pragma unroll
      for (int i = 0; i < MT; ++i) a_scale[i] = a_next[i];
#pragma unroll
      for (int i = 0; i < NT; ++i) b_scale[i] = b_next[i];
    }
    if (step + 1 < p.blocks) {
      issue(step + 1);
      if ((step & 3) == 0 && step + 4 < p.blocks) scales((step >> 2) + 1);
    }
    const unsigned char* stage = block_smem + (step & 1) * STAGE;
    auto fragment = [&](int r, int half) {
      const u32x4 lo = *(const u32x4*)(stage + r * 128 + (((4 * half + 2 * h) ^ (r & 7)) << 4));
      const u32x4 hi = *(const u32x4*)(stage + r * 128 + (((4 * half + 2 * h + 1) ^ (r & 7)) << 4));
      return (i32x8){(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
    };
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      i32x8 a[MT], b[NT];
#pragma unroll
      for (int i = 0; i < MT; ++i) a[i] = fragment(wm + 32 * i + l31, half);
#pragma unroll
      for (int j = 0; j < NT; ++j) b[j] = fragment(BM + wn + 32 * j + l31, half);
      if constexpr (!FINE) {
        // (the right operand first: a lane's registers are then neighbours along a row of c)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b[j], a[i], acc[i][j], 0, 0, 0, (int)b_scale[j], 0, (int)a_scale[i]);
      } else {
        auto wide = [&](i32x8 q, int g, unsigned byte) {     // eight values, scaled
          const float f = __builtin_bit_cast(float, byte << 23);
          typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
          u32x4 w;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const unsigned word = (unsigned)q[2 * g + (e >> 1)];
            const bf16x2 two = e & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, f, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, f, false);
            w[e] = __builtin_bit_cast(unsigned, two);
          }
          return __builtin_bit_cast(bf16x8, w);
        };
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          bf16x8 aw[MT], bw[NT];
#pragma unroll
          for (int i = 0; i < MT; ++i) aw[i] = wide(a[i], g, a_scale[i] & 255u);
#pragma unroll
          for (int j = 0; j < NT; ++j) bw[j] = wide(b[j], g, b_scale[j] & 255u);
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bw[j], aw[i], acc[i][j], 0, 0, 0);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) a_scale[i] >>= 8;
#pragma unroll
    for (int i = 0; i < NT; ++i) b_scale[i] >>= 8;
  }
  // a lane holds row l31 of a block of c, columns 8 q + 4 h + e
  typedef E four __attribute__((ext_vector_type(4), aligned(sizeof(E))));
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int n = n0 + wn + 32 * j + 8 * q + 4 * h;
      float bias[4] = {0.f, 0.f, 0.f, 0.f};
      if (p.bias) {
#pragma unroll
        for (int e = 0; e < 4; ++e) bias[e] = IoType<IODT>::load((const E*)p.bias + (n + e < p.N ? n + e : p.N - 1));
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int m = m0 + wm + 32 * i + l31;
        E* row = (E*)p.c + m * p.ldc;
        four o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (E)(acc[i][j][4 * q + e] + bias[e]);
        if (m < p.M && n + 4 <= p.N) {
          *(four*)(row + n) = o;
        } else if (m < p.M) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < p.N) row[n + e] = o[e];
        }
      }
    }
}

}  // namespace cascmm
