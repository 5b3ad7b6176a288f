// Products of 8-bit floating-point operands with a scale for each block of 128 (gfx950): the operands' rounding and the product.
//
//   q = e4m3(x 2^-e), nearest, ties to even;   C[m][n] = sum over blocks of k of 2^(ea[m][block] + eb[n][block]) sum over the block of qa[m][k] qb[n][k]  (+ bias[n])
//
// The scale of a block is the smallest power of two with max|x| <= 448 * 2^e over its finite elements: scaling is exact, and the matrix instruction
// applies it by itself (one E8M0 byte a lane), so that all blocks of a row meet in one fp32 accumulator and nothing is added to the loop for the scales.
// Infinities and NaN become NaN.
//
// The rounding is bound by memory.  The product, over 8192 k, by the matrix units at the clock that the card holds under them (82 % of the busy cycles of the CUs at 1.6 GHz); over 1280 k by
// tiles that begin and end every ten blocks, while nothing else runs on their CU (46 to 53 % busy; 76 % over 5120 k on 160 CUs), at 1.75 to 1.85 GHz: 8192 x 1280 x 5120 takes the same time on 160 CUs
// (256 x 256 tiles) as on all 256 (256 x 160).  Measured (us in a graph): 8192 x 8192 x 8192 bf16 393 to 409 (2.7 PF; registers alone reach 4.1 to 4.4), 8192 x 5120 x 1280 59 to 61,
// 2048 x 10240 x 1280 33.5 to 34.4, 154 x 5120 x 1280 5.7; fp32 8192 x 8192 x 8192 865 (1.27 PF), 8192 x 5120 x 1280 112, 8192 x 1280 x 1280 35.6 (bf16 20.3);
// rounding 8192 x 5120 bf16 in both orders with its sums 37.5 (168 MB, 4.5 TB/s), 2048 x 1280 along rows 3.7 (a launch of 32 tiles, which turns them too, 5.4).  Tried and left out: four waves on 256 x 320 (the sums no longer fit the
// accumulation registers and are moved about: 2.3 us a block of k for 1.25 of instructions), stages of half a block in deeper rings (8192 x 8192 x 8192 620), 256 x 128 tiles (490).
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

// Eight elements, as the rounding handles them.  fp32: numbers; 16 bits: pairs, whose magnitudes are compared as whole numbers two at a time and which an instruction divides by the
// scale and rounds two at a time (all patterns under all scales: the same bytes as by fp32; infinities become NaN there too).
template <int IODT> struct BlockEight {
  typedef typename IoType<IODT>::T E;
  typedef float Values[8];
  typedef unsigned Most[8];                   // magnitudes of eight columns
  static __device__ __forceinline__ void clear(Most& m) {
#pragma unroll
    for (int e = 0; e < 8; ++e) m[e] = 0;
  }
  static __device__ __forceinline__ void load(Values& v, const E* src, bool whole, int left) {
    typedef E chunk __attribute__((ext_vector_type(8), aligned(sizeof(E))));   // (rows start on elements, not on 16 bytes)
    if (whole) {
      const chunk c = *(const chunk*)src;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = c[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = e < left ? src[e] : 0.f;
    }
  }
  static __device__ __forceinline__ float value(const Values& v, int e) { return v[e]; }
  // folds the finite magnitudes into those of the columns; returns the largest of the eight, as bits of a float
  static __device__ __forceinline__ unsigned fold(Values& v, Most& columns) {
    unsigned most = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned bits = __builtin_bit_cast(unsigned, v[e]) & 0x7FFFFFFFu;
      const bool finite = bits < 0x7F800000u;
      v[e] = finite ? v[e] : __builtin_nanf("");
      const unsigned b = finite ? bits : 0u;
      columns[e] = block_larger(columns[e], b);
      most = block_larger(most, b);
    }
    return most;
  }
  static __device__ __forceinline__ unsigned column(const Most& m, int e) { return m[e]; }
  static __device__ __forceinline__ u32x2 pack(const Values& v, unsigned byte) { return block_pack(v, block_inverse(byte)); }
  static __device__ __forceinline__ u32x2 pack_column(const Values (&v)[8], int e, unsigned byte) {
    const float column[8] = {v[0][e], v[1][e], v[2][e], v[3][e], v[4][e], v[5][e], v[6][e], v[7][e]};
    return block_pack(column, block_inverse(byte));
  }
};
template <int IODT> struct BlockEight16 {
  typedef typename IoType<IODT>::T E;
  typedef E pair __attribute__((ext_vector_type(2)));
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  typedef u32x4 Values;
  typedef unsigned Most[4];
  static constexpr unsigned kInf = IODT == CASCMM_DT_BF16 ? 0x7F80u : 0x7C00u;
  static __device__ __forceinline__ void clear(Most& m) {
#pragma unroll
    for (int c = 0; c < 4; ++c) m[c] = 0;
  }
  static __device__ __forceinline__ void load(Values& v, const E* src, bool whole, int left) {
    typedef E chunk __attribute__((ext_vector_type(8), aligned(sizeof(E))));
    chunk c;
    if (whole) {
      c = *(const chunk*)src;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) c[e] = e < left ? src[e] : (E)0.f;
    }
    v = __builtin_bit_cast(u32x4, c);
  }
  static __device__ __forceinline__ float value(const Values& v, int e) {
    const unsigned w = v[e >> 1];      // (a number of its own: a cast of a vector's element takes the vector's first)
    return (float)__builtin_bit_cast(pair, w)[e & 1];
  }
  static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b) {
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
  }
  static __device__ __forceinline__ unsigned bits(unsigned half) {   // of the float
    return IODT == CASCMM_DT_BF16 ? half << 16 : __builtin_bit_cast(unsigned, (float)__builtin_bit_cast(_Float16, (unsigned short)half));
  }
  static __device__ __forceinline__ unsigned fold(Values& v, Most& columns) {
    unsigned m[4], most = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      m[c] = v[c] & 0x7FFF7FFFu;
      most = larger(most, m[c]);
    }
    if ((most >> 16) >= kInf || (most & 0xFFFFu) >= kInf) {   // (hardly ever)
      most = 0;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        m[c] = ((m[c] >> 16) >= kInf ? 0u : m[c] & 0xFFFF0000u) | ((m[c] & 0xFFFFu) >= kInf ? 0u : m[c] & 0xFFFFu);
        most = larger(most, m[c]);
      }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) columns[c] = larger(columns[c], m[c]);
    return bits((most >> 16) > (most & 0xFFFFu) ? most >> 16 : most & 0xFFFFu);
  }
  static __device__ __forceinline__ unsigned column(const Most& m, int e) { return bits(e & 1 ? m[e >> 1] >> 16 : m[e >> 1] & 0xFFFFu); }
  static __device__ __forceinline__ s16x2 two(s16x2 old, unsigned w, float scale, bool high) {
    if constexpr (IODT == CASCMM_DT_BF16)
      return high ? __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(old, __builtin_bit_cast(pair, w), scale, true) : __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(old, __builtin_bit_cast(pair, w), scale, false);
    else
      return high ? __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(old, __builtin_bit_cast(pair, w), scale, true) : __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(old, __builtin_bit_cast(pair, w), scale, false);
  }
  static __device__ __forceinline__ u32x2 pack4(unsigned w0, unsigned w1, unsigned w2, unsigned w3, unsigned byte) {
    const float scale = __builtin_bit_cast(float, byte << 23);      // (its exponent is the scale: a byte of 0 is 2^-127)
    const s16x2 zero = {0, 0};
    return (u32x2){__builtin_bit_cast(unsigned, two(two(zero, w0, scale, false), w1, scale, true)), __builtin_bit_cast(unsigned, two(two(zero, w2, scale, false), w3, scale, true))};
  }
  static __device__ __forceinline__ u32x2 pack(const Values& v, unsigned byte) { return pack4(v[0], v[1], v[2], v[3], byte); }
  static __device__ __forceinline__ u32x2 pack_column(const Values (&v)[8], int e, unsigned byte) {
    const unsigned which = e & 1 ? 0x07060302u : 0x05040100u;
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_perm(v[2 * i + 1][e >> 1], v[2 * i][e >> 1], which);
    return pack4(w[0], w[1], w[2], w[3], byte);
  }
};
template <> struct BlockEight<CASCMM_DT_F16> : BlockEight16<CASCMM_DT_F16> {};
template <> struct BlockEight<CASCMM_DT_BF16> : BlockEight16<CASCMM_DT_BF16> {};

// A tile of 128 x 128 a workgroup, read once: a thread holds 8 rows of 8 columns, sixteen threads a row of the tile.
// SQUARE: one scale for the whole tile; else one for each of its rows (q) and of its columns (qt).
template <int IODT, bool SQUARE>
__global__ __launch_bounds__(256) void cascmm_block_round_kernel(const BlockRoundParams p) {
  typedef BlockEight<IODT> V;
  typedef typename V::E E;
  constexpr int MOST = sizeof(typename V::Most) / 4;      // words of eight columns' magnitudes
  __shared__ unsigned col_most[4][16][MOST];
  __shared__ float col_sum[4][kBlock];
  __shared__ u32x2 turned[kBlock][16];       // [column][eight rows], the eights of a column in the order i ^ (column / 8): writes and reads without conflicts
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, wave = tid >> 6;
  const int64_t tile_row = blockIdx.x / p.across, tile_col = blockIdx.x % p.across;
  const int64_t row0 = tile_row * kBlock + ty * 8, col0 = tile_col * kBlock + tx * 8;
  const E* src = (const E*)p.x + row0 * p.ldx + col0;
  typename V::Values v[8];
  const int left = p.cols - col0 < 8 ? (int)(p.cols - col0) : 8, down = p.rows - row0 < 8 ? (int)(p.rows - row0) : 8;
  if (left == 8 && down == 8) {
#pragma unroll
    for (int r = 0; r < 8; ++r) V::load(v[r], src + r * p.ldx, true, 8);
  } else {
#pragma unroll
    for (int r = 0; r < 8; ++r) V::load(v[r], src + r * p.ldx, r < down && left == 8, r < down ? left : 0);
  }
  if (p.sums) {
    // sums over the tile's rows: eight in a thread, four threads of a wave, four waves, in this order
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float s = 0.f;
#pragma unroll
      for (int r = 0; r < 8; ++r) s += V::value(v[r], e);
      s += __shfl_xor(s, 16, 64);
      s += __shfl_xor(s, 32, 64);
      if ((tid & 63) < 16) col_sum[wave][tx * 8 + e] = s;
    }
  }
  unsigned row_most[8];
  typename V::Most most;
  V::clear(most);
#pragma unroll
  for (int r = 0; r < 8; ++r) row_most[r] = V::fold(v[r], most);
  unsigned square = 0;
  if (SQUARE) {
    __shared__ unsigned all[4];
#pragma unroll
    for (int r = 0; r < 8; ++r) square = block_larger(square, row_most[r]);
    square = block_row_max(square);
    square = block_larger(square, (unsigned)__shfl_xor((int)square, 16, 64));
    square = block_larger(square, (unsigned)__shfl_xor((int)square, 32, 64));
    if ((tid & 63) == 0) all[wave] = square;
    __syncthreads();
    square = block_scale(block_larger(block_larger(all[0], all[1]), block_larger(all[2], all[3])));
  }
  if (p.q) {
    const int64_t padded = block_padded(p.cols);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const unsigned byte = SQUARE ? square : block_scale(block_row_max(row_most[r]));
      if (r < down) {
        *(u32x2*)(p.q + (row0 + r) * padded + col0) = V::pack(v[r], byte);
        if (tx == 0) p.s[((tile_col >> 2) * p.rows + row0 + r) * 4 + (tile_col & 3)] = (unsigned char)byte;
      }
    }
  }
  if (!p.qt && !p.sums) return;
  auto join = [&](unsigned a, unsigned b) {
    if constexpr (MOST == 4) return V::larger(a, b);
    else return block_larger(a, b);
  };
  if (!SQUARE && p.qt) {
#pragma unroll
    for (int c = 0; c < MOST; ++c) {
      most[c] = join(most[c], (unsigned)__shfl_xor((int)most[c], 16, 64));
      most[c] = join(most[c], (unsigned)__shfl_xor((int)most[c], 32, 64));
      if ((tid & 63) < 16) col_most[wave][tx][c] = most[c];
    }
  }
  __syncthreads();
  if (p.sums && tid < kBlock && tile_col * kBlock + tid < p.cols)
    p.sums[tile_row * p.cols + tile_col * kBlock + tid] = (col_sum[0][tid] + col_sum[1][tid]) + (col_sum[2][tid] + col_sum[3][tid]);
  if (!p.qt) return;
  if (!SQUARE) {
#pragma unroll
    for (int c = 0; c < MOST; ++c) most[c] = join(join(col_most[0][tx][c], col_most[1][tx][c]), join(col_most[2][tx][c], col_most[3][tx][c]));
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const unsigned byte = SQUARE ? square : block_scale(V::column(most, e));
    turned[tx * 8 + e][ty ^ tx] = V::pack_column(v, e, byte);
    if (ty == 0 && e < left) p.st[((tile_row >> 2) * p.cols + col0 + e) * 4 + (tile_row & 3)] = (unsigned char)byte;
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

// Blocks along the rows alone: sixteen rows of one block of columns a workgroup, eight elements a thread.  Few and short loads for each, so that few rows are spread over many workgroups
template <int IODT>
__global__ __launch_bounds__(256) void cascmm_block_round_rows_kernel(const BlockRoundParams p) {
  typedef BlockEight<IODT> V;
  typedef typename V::E E;
  const int tid = threadIdx.x, tx = tid & 15;
  const int64_t tile_row = blockIdx.x / p.across, tile_col = blockIdx.x % p.across;
  const int64_t row = tile_row * 16 + (tid >> 4), col0 = tile_col * kBlock + tx * 8;
  if (row >= p.rows) return;       // (sixteen lanes of a row or none)
  const int left = p.cols - col0 < 8 ? (int)(p.cols - col0) : 8;
  typename V::Values v;
  V::load(v, (const E*)p.x + row * p.ldx + col0, left == 8, left);
  typename V::Most columns;
  V::clear(columns);
  const unsigned byte = block_scale(block_row_max(V::fold(v, columns)));
  *(u32x2*)(p.q + row * block_padded(p.cols) + col0) = V::pack(v, byte);
  if (tx == 0) p.s[((tile_col >> 2) * p.rows + row) * 4 + (tile_col & 3)] = (unsigned char)byte;
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
  int whole;                       // (pieces) tiles that stay whole
};

typedef __attribute__((address_space(3))) void* block_lds_ptr;
__device__ __forceinline__ void block_load_lds(__amdgpu_buffer_rsrc_t rsrc, unsigned char* dst, int voffset, int soffset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (block_lds_ptr)dst, 16, voffset, soffset, 0, 0);
}

// WM x WN waves, each MT x NT blocks of 32 x 32.  A stage is one block of k: rows of 128 bytes in LDS, the eight 16-byte pieces of a row turned (block_turn), so that
// the lanes of a fragment read, 32 rows apart by 128 bytes, hit all banks, and the rows' scales of the block's four.  The copy to LDS writes in order; the order is made by the
// addresses it reads.
// A stage is multiplied in two halves of 64 k.  The fragments of one half are read behind the matrix instructions of the other, so that no wave waits for LDS: behind the first
// half's the second's; then the barrier, which the stage has been read in front of and the next one has landed at; behind the second half's instructions the next stage's first
// fragments, and the loads of the stage DEEP on, into the place of the one just read: they have DEEP - 1 stages' instructions to land.
// SHARES: the blocks of k are dealt to as many groups of WM x WN waves, each with stages of its own, for few tiles and a long k; their sums meet in LDS, in order.
// FINE: products and sums by the 16-bit matrix instruction, to fp32's accuracy.  The 8-bit one cuts the products inside an instruction at about 2^-15 of the largest: 1.5e-5
// of the result's size (rms of ordinary data), unbiased and the same for every depth: less than a 16-bit result's rounding, of which it turns one in some dozens (fp16) or hundreds (bf16) the
// other way, while fp32 results would show nothing else.  At worst it is 2^-10 of the largest product of every sixteen, where large ones cancel.  (bf16 holds the scaled values exactly, but for
// those below 2^-126, which the instruction takes as zeros, and for 2^128, which is infinite there.)
constexpr int block_waitcnt(int vm, int lgkm) { return 0x70 | (vm & 15) | (vm >> 4) << 14 | lgkm << 8; }
template <int WM_, int WN_, int MT_, int NT_, int DEEP_, int SHARES_> struct BlockTile {
  static constexpr int WM = WM_, WN = WN_, MT = MT_, NT = NT_, DEEP = DEEP_, SHARES = SHARES_, WAVES = WM * WN, THREADS = 64 * WAVES * SHARES;
  static constexpr int BM = 32 * MT * WM, BN = 32 * NT * WN, ROWS = BM + BN;
  static constexpr int STAGE = ROWS * 132, LDS = DEEP * STAGE * SHARES, BAND = BM >= 256 ? 4 : 8;
  static constexpr int LOADS = ROWS / 8 / WAVES, SCALES = (ROWS / 64 + WAVES - 1) / WAVES;    // a wave's, of a stage: 1 KB (256 bytes) each
  static_assert(ROWS % (8 * WAVES) == 0 && ROWS % 64 == 0 && BM % 64 == 0 && LDS <= 160 * 1024, "tile");
};

// Workgroup w runs on die w % 8, each with a cache of its own: a die takes tiles that follow each other, in bands of `band` tiles down and all the way across, so that those at work
// at a time share rows of both operands
__device__ __forceinline__ unsigned block_order(unsigned w, unsigned total) {
  const unsigned die = w & 7u, each = total >> 3, more = total & 7u;
  return die * each + (die < more ? die : more) + (w >> 3);
}
__device__ __forceinline__ void block_place(unsigned id, int tiles_m, int tiles_n, int band, int& tile_m, int& tile_n) {
  const unsigned across = (unsigned)band * (unsigned)tiles_n, which = id / across, in = id % across;
  const unsigned down = (unsigned)tiles_m - which * band < (unsigned)band ? (unsigned)tiles_m - which * band : (unsigned)band;    // (the last band may be lower)
  tile_m = (int)(which * band + in % down);
  tile_n = (int)(in / down);
}

// The order of a row's 16-byte pieces in LDS: piece i lies at i ^ turn.  Sixteen lanes are served at a time, from 64 banks: two rows side by side, and eight pairs of them in eight places (measured,
// cycles of a read by sixteen waves: 4.4 so, 8.1 with r % 8)
__device__ __forceinline__ int block_turn(int r) { return (r >> 1) & 7; }

// A wave's loads of a stage: 1 KB of rows each, and 256 bytes of scales
template <typename T> struct BlockLoads {
  __amdgpu_buffer_rsrc_t ra, rb, rsa, rsb;
  int from[T::LOADS], scale_from[T::SCALES], wave;
  __device__ __forceinline__ BlockLoads(const BlockGemmParams& p, int m0, int n0, int wave_, int lane) : wave(wave_) {
    const int64_t kp = (int64_t)p.blocks * kBlock;
    // (a tile's rows lie below 2 GiB from its first: host-checked)
    ra = __builtin_amdgcn_make_buffer_rsrc((void*)(p.a + m0 * kp), 0, 0x7FFFFFFF, 0x00020000);
    rb = __builtin_amdgcn_make_buffer_rsrc((void*)(p.b + n0 * kp), 0, 0x7FFFFFFF, 0x00020000);
    rsa = __builtin_amdgcn_make_buffer_rsrc((void*)(p.sa + m0), 0, 0x7FFFFFFF, 0x00020000);
    rsb = __builtin_amdgcn_make_buffer_rsrc((void*)(p.sb + n0), 0, 0x7FFFFFFF, 0x00020000);
    const int last_m = p.M - m0 - 1, last_n = p.N - n0 - 1;     // (rows past the edge: the last one again)
#pragma unroll
    for (int j = 0; j < T::LOADS; ++j) {
      const int r = (wave + T::WAVES * j) * 8 + (lane >> 3), row = r < T::BM ? (r < last_m ? r : last_m) : (r - T::BM < last_n ? r - T::BM : last_n);
      from[j] = (int)(row * kp) + (((lane & 7) ^ block_turn(r)) << 4);
    }
#pragma unroll
    for (int j = 0; j < T::SCALES; ++j) {
      const int r = (wave + T::WAVES * j) % (T::ROWS / 64) * 64 + lane;
      scale_from[j] = 4 * (r < T::BM ? (r < last_m ? r : last_m) : (r - T::BM < last_n ? r - T::BM : last_n));
    }
  }
  // load j of block `block` of k to the stage at `to`, the first ones those of the scales
  __device__ __forceinline__ void issue(const BlockGemmParams& p, int block, unsigned char* to, int j) const {
    if (j < T::SCALES) {
      const int run = (wave + T::WAVES * j) % (T::ROWS / 64);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(run * 64 < T::BM ? rsa : rsb, (block_lds_ptr)(to + T::ROWS * 128 + run * 256), 4, scale_from[j], (block >> 2) * 4 * (run * 64 < T::BM ? p.M : p.N), 0, 0);
    } else {
      const int run = wave + T::WAVES * (j - T::SCALES);
      block_load_lds(run * 8 < T::BM ? ra : rb, to + run * 1024, from[j - T::SCALES], block * kBlock);
    }
  }
};

template <int IODT, typename T>
__device__ __forceinline__ void block_store(const BlockGemmParams& p, const f32x16 (&acc)[T::MT][T::NT], unsigned char* smem, int m0, int n0, int wave, int lane) {
  typedef typename IoType<IODT>::T E;
  constexpr int MT = T::MT, NT = T::NT;
  const int l31 = lane & 31, h = lane >> 5, wm = (wave / T::WN) * 32 * MT, wn = (wave % T::WN) * 32 * NT;
  // A lane holds row l31 of a block, columns 8 q + 4 h + e: sixteen bytes of a row and less.  Through LDS, in a place of each wave's own, 32 rows of the wave's width at a time, so that
  // what is stored are whole pieces of rows.
  typedef E four __attribute__((ext_vector_type(4), aligned(4 * sizeof(E))));
  constexpr int VEC = 16 / (int)sizeof(E), WIDTH = 32 * NT, PITCH = WIDTH + VEC, PIECES = WIDTH / VEC, STORES = 32 * PIECES / 64;   // (elements; pieces of a row; stores of a lane)
  static_assert(32 * PIECES % 64 == 0 && T::WAVES * 32 * PITCH * (int)sizeof(E) <= T::LDS, "the rows of a store");
  typedef E chunk __attribute__((ext_vector_type(VEC), aligned(sizeof(E))));
  E* const mine = (E*)smem + wave * 32 * PITCH;
  float bias[NT][4][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = n0 + wn + 32 * j + 8 * q + 4 * h + e;
        bias[j][q][e] = p.bias ? IoType<IODT>::load((const E*)p.bias + (n < p.N ? n : p.N - 1)) : 0.f;
      }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        four o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (E)(acc[i][j][4 * q + e] + bias[j][q][e]);
        *(four*)(mine + l31 * PITCH + 32 * j + 8 * q + 4 * h) = o;
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int k = 0; k < STORES; ++k) {
      const int id = k * 64 + lane, r = id / PIECES, m = m0 + wm + 32 * i + r, column = n0 + wn + id % PIECES * VEC;
      const chunk o = *(const chunk*)__builtin_assume_aligned(mine + r * PITCH + id % PIECES * VEC, 16);
      E* to = (E*)p.c + m * p.ldc + column;
      if (m < p.M && column + VEC <= p.N) {
        *(chunk*)to = o;
      } else if (m < p.M) {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (column + e < p.N) to[e] = o[e];
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// the tile of c at (m0, n0)
template <int IODT, typename T, bool FINE> __device__ __forceinline__ void block_product(const BlockGemmParams& p, unsigned char* block_smem, int m0, int n0) {
  constexpr int MT = T::MT, NT = T::NT, BM = T::BM;
  const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) % T::WAVES, share = __builtin_amdgcn_readfirstlane(tid >> 6) / T::WAVES;
  const int wm = (wave / T::WN) * 32 * MT, wn = (wave % T::WN) * 32 * NT;
  // this share's blocks; all shares take as many steps, those past the last block without products
  const int steps = (p.blocks + T::SHARES - 1) / T::SHARES, first = share * steps, live = p.blocks - first < steps ? p.blocks - first : steps;
  unsigned char* const ring = block_smem + share * T::DEEP * T::STAGE;
  const BlockLoads<T> loads(p, m0, n0, wave, lane);
  // (past the end: the last block again, so that every share waits for as many)
  auto issue = [&](int step, unsigned char* to, int j) { loads.issue(p, first + step < p.blocks ? first + step : p.blocks - 1, to, j); };
  constexpr int ISSUES = T::LOADS + T::SCALES, GAPS = MT * NT, READS = 2 * (MT + NT);
  f32x16 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  u32x4 f[2][MT + NT][2];              // fragments of both halves: rows of a, then of b; 32 k in two pieces
  unsigned scale[MT + NT], scale_next[MT + NT];
  // read k of a half: the pieces of b and a in turn, as the instructions want them
  const int at[2] = {(wm + l31) * 128, (BM + wn + l31) * 128}, turn = block_turn(l31);
  auto read = [&](const unsigned char* stage, int half, int k) {
    const int g = k >> 1, piece = k & 1;
    const int base = g < MT ? at[0] + g * 4096 : at[1] + (g - MT) * 4096;
    f[half][g][piece] = *(const u32x4*)(stage + base + (((4 * half + 2 * h + piece) ^ turn) << 4));
  };
  auto read_scale = [&](const unsigned char* stage, int g) {
    scale_next[g] = *(const unsigned*)(stage + T::ROWS * 128 + (g < MT ? wm + 32 * g + l31 : BM + wn + 32 * (g - MT) + l31) * 4);
  };
  auto whole = [&](int half, int g) {
    const u32x4 lo = f[half][g][0], hi = f[half][g][1];
    return (i32x8){(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
  };
  // product t of a half
  auto multiply = [&](int half, int t) {
    const int i = t / NT, j = t % NT;
    if constexpr (!FINE) {
      // (the right operand first: a lane's registers are then neighbours along a row of c)
      acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(whole(half, MT + j), whole(half, i), acc[i][j], 0, 0, 0, (int)scale[MT + j], 0, (int)scale[i]);
    } else {
      typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
      auto wide = [&](int g, int part) {     // eight values, scaled (once for a half, whatever the products it enters: 128 conversions beside 32 products of a 128 x 128 tile's block)
        const float s = __builtin_bit_cast(float, (scale[g] & 255u) << 23);
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned word = f[half][g][part >> 1][2 * (part & 1) + (e >> 1)];
          const bf16x2 two = e & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, s, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, s, false);
          w[e] = __builtin_bit_cast(unsigned, two);
        }
        return __builtin_bit_cast(bf16x8, w);
      };
#pragma unroll
      for (int part = 0; part < 4; ++part) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wide(MT + j, part), wide(i, part), acc[i][j], 0, 0, 0);
    }
  };
#define BLOCK_FENCE() __builtin_amdgcn_sched_barrier(0)
  if (p.blocks > 0) {     // (else: nothing but the bias)
#pragma unroll
    for (int s = 0; s < T::DEEP; ++s)
#pragma unroll
      for (int j = 0; j < ISSUES; ++j) issue(s, ring + s * T::STAGE, j);
    __builtin_amdgcn_s_waitcnt(block_waitcnt(ISSUES * (T::DEEP - 1), 15));
    __builtin_amdgcn_s_barrier();
    BLOCK_FENCE();
#pragma unroll
    for (int g = 0; g < MT + NT; ++g) read_scale(ring, g);
#pragma unroll
    for (int k = 0; k < READS; ++k) read(ring, 0, k);
    int here = 0;
    for (int step = 0; step < steps; ++step) {
      unsigned char* const stage = ring + here;
      here = here + T::STAGE < T::DEEP * T::STAGE ? here + T::STAGE : 0;
      unsigned char* const other = ring + here;
      const bool counts = T::SHARES == 1 || step < live;
#pragma unroll
      for (int g = 0; g < MT + NT; ++g) scale[g] = scale_next[g] >> (((first + step) & 3) * 8);
#pragma unroll
      for (int t = 0; t < GAPS; ++t) {
        if (counts) multiply(0, t);
        BLOCK_FENCE();
#pragma unroll
        for (int k = READS * t / GAPS; k < READS * (t + 1) / GAPS; ++k) read(stage, 1, k);
        BLOCK_FENCE();
      }
      __builtin_amdgcn_s_waitcnt(block_waitcnt(ISSUES * (T::DEEP - 2), 0));    // own loads of the next stage have landed, own reads of this one are back
      __builtin_amdgcn_s_barrier();          // everybody's
      BLOCK_FENCE();
#pragma unroll
      for (int t = 0; t < GAPS; ++t) {
        if (counts) multiply(1, t);
        BLOCK_FENCE();
#pragma unroll
        for (int k = READS * t / GAPS; k < READS * (t + 1) / GAPS; ++k) read(other, 0, k);
#pragma unroll
        for (int g = (MT + NT) * t / GAPS; g < (MT + NT) * (t + 1) / GAPS; ++g) read_scale(other, g);
#pragma unroll
        for (int j = ISSUES * t / GAPS; j < ISSUES * (t + 1) / GAPS; ++j) issue(step + T::DEEP, stage, j);
        BLOCK_FENCE();
      }
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);      // (the redundant loads land before LDS is given up)
  }
#undef BLOCK_FENCE
  __syncthreads();
  if constexpr (T::SHARES > 1) {
    float* const meet = (float*)block_smem + (wave * MT * NT * 16) * 64 + lane;
    constexpr int ALL = T::WAVES * MT * NT * 16 * 64;
    static_assert((T::SHARES - 1) * ALL * 4 <= T::LDS, "the sums of the shares");
    if (share > 0) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) meet[(share - 1) * ALL + ((i * NT + j) * 16 + e) * 64] = acc[i][j][e];
    }
    __syncthreads();
    if (share == 0) {
#pragma unroll
      for (int o = 0; o < T::SHARES - 1; ++o)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] += meet[o * ALL + ((i * NT + j) * 16 + e) * 64];
    }
    __syncthreads();
    if (share > 0) return;
  }
  block_store<IODT, T>(p, acc, block_smem, m0, n0, wave, lane);
}
template <int IODT, typename T, bool FINE> __global__ __launch_bounds__(T::THREADS) void cascmm_block_gemm_kernel(const BlockGemmParams p) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char block_smem[];
  int tile_m, tile_n;
  block_place(block_order(blockIdx.x, gridDim.x), p.tiles_m, p.tiles_n, T::BAND, tile_m, tile_n);
  block_product<IODT, T, FINE>(p, block_smem, tile_m * T::BM, tile_n * T::BN);
}
// The first p.whole tiles by a workgroup each, those behind them in pieces of R's size: where the last turn of tiles would leave most of the CUs without one
template <int IODT, typename T, typename R> __global__ __launch_bounds__(T::THREADS) void cascmm_block_gemm_pieces_kernel(const BlockGemmParams p) {
  static_assert(R::THREADS == T::THREADS && R::LDS <= T::LDS && T::BM % R::BM == 0 && T::BN % R::BN == 0, "pieces");
  extern __shared__ __attribute__((aligned(1024))) unsigned char block_smem[];
  constexpr unsigned PIECES = (T::BM / R::BM) * (T::BN / R::BN);
  const unsigned whole = (unsigned)p.whole;
  int tile_m, tile_n;
  if (blockIdx.x < whole) {
    block_place(block_order(blockIdx.x, whole), p.tiles_m, p.tiles_n, T::BAND, tile_m, tile_n);
    block_product<IODT, T, false>(p, block_smem, tile_m * T::BM, tile_n * T::BN);
  } else {
    const unsigned id = block_order(blockIdx.x - whole, gridDim.x - whole), piece = id % PIECES;
    block_place(whole + id / PIECES, p.tiles_m, p.tiles_n, T::BAND, tile_m, tile_n);
    const int m0 = tile_m * T::BM + (int)(piece / (T::BN / R::BN)) * R::BM, n0 = tile_n * T::BN + (int)(piece % (T::BN / R::BN)) * R::BN;
    if (m0 < p.M && n0 < p.N) block_product<IODT, R, false>(p, block_smem, m0, n0);
  }
}

// ---------------------------------------------------------------------------------------
// few rows: c [M][N], x rounded here
// ---------------------------------------------------------------------------------------
// Sixteen columns and rows a workgroup, a block of k at a time a wave; every workgroup rounds the rows itself, which costs less than a launch in front of it (1 x 5120 x 1280 bf16 5.3 us a call in a
// graph; a launch each 5 and 11).  Bound by what a CU's vector memory takes in: the weights' fragments come straight from memory, sixteen bytes a lane, and a load of the rows is four of
// them whole, sixteen lanes a row, turned into fragments in the wave's own LDS (loaded as fragments, sixteen rows whatever M is, 6.9 us, and 43 instead of 30 for 8 x 10240 x 10240).  The
// next block's loads are under way while one is multiplied, with no branch between them (a load that a branch may skip makes every wait one for all); two blocks ahead gain nothing (5.4).
// The waves' sums meet in LDS, in order.  A lane's 32 k are the pieces i and i + 4 of a block's eight, of both operands.
struct BlockRowsParams {
  const void* x;                   // [M][K], row stride ldx
  const unsigned char* b;
  const unsigned* sb;
  void* c;
  const void* bias;
  int64_t ldx, ldc;
  int M, N, K, blocks;
};
template <int IODT, int WAVES, int QUADS>
__global__ __launch_bounds__(64 * WAVES) void cascmm_block_rows_kernel(const BlockRowsParams p) {
  typedef BlockEight<IODT> V;
  typedef typename V::E E;
  constexpr int PITCH = kBlock + 16;                // (the scale stands behind a row; sixteen rows' pieces on banks of their own)
  __shared__ __attribute__((aligned(16))) unsigned char rounded[WAVES][16 * PITCH];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l15 = lane & 15, part = lane >> 4;
  const int n = blockIdx.x * 16 + l15, row_b = n < p.N ? n : p.N - 1;
  const unsigned char* const b = p.b + (int64_t)row_b * p.blocks * kBlock + part * 16;
  unsigned char* const mine = rounded[wave];
  const int m0 = blockIdx.y * 16, rows = p.M - m0 < 16 ? p.M - m0 : 16;
  const E* x[QUADS];
#pragma unroll
  for (int i = 0; i < QUADS; ++i) {
    const int row = 4 * i + part;
    x[i] = (const E*)p.x + (m0 + (row < rows ? row : rows - 1)) * p.ldx + l15 * 8;
  }
  struct Piece {
    u32x4 b[2];
    unsigned scale;
    typename V::Values x[QUADS];
  };
  auto fetch = [&](Piece& to, int block, bool whole) {
    to.b[0] = *(const u32x4*)(b + (int64_t)block * kBlock);
    to.b[1] = *(const u32x4*)(b + (int64_t)block * kBlock + 64);
    to.scale = p.sb[(int64_t)(block >> 2) * p.N + row_b] >> ((block & 3) * 8);
    const int left = p.K - block * kBlock - l15 * 8;
#pragma unroll
    for (int i = 0; i < QUADS; ++i) V::load(to.x[i], x[i] + (int64_t)block * kBlock, whole || left >= 8, left);
  };
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](Piece& cur) {
#pragma unroll
    for (int i = 0; i < QUADS; ++i) {
      typename V::Most columns;
      V::clear(columns);
      unsigned most = V::fold(cur.x[i], columns);
#pragma unroll
      for (int o = 1; o < 16; o *= 2) most = block_larger(most, (unsigned)__shfl_xor((int)most, o, 64));
      const unsigned byte = block_scale(most);
      *(u32x2*)(mine + (4 * i + part) * PITCH + l15 * 8) = V::pack(cur.x[i], byte);
      if (l15 == 0) mine[(4 * i + part) * PITCH + kBlock] = (unsigned char)byte;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const u32x4 a0 = *(const u32x4*)(mine + l15 * PITCH + part * 16), a1 = *(const u32x4*)(mine + l15 * PITCH + 64 + part * 16);
    const unsigned byte = mine[l15 * PITCH + kBlock];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const i32x8 a = {(int)a0[0], (int)a0[1], (int)a0[2], (int)a0[3], (int)a1[0], (int)a1[1], (int)a1[2], (int)a1[3]};
    const i32x8 w = {(int)cur.b[0][0], (int)cur.b[0][1], (int)cur.b[0][2], (int)cur.b[0][3], (int)cur.b[1][0], (int)cur.b[1][1], (int)cur.b[1][2], (int)cur.b[1][3]};
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, acc, 0, 0, 0, (int)cur.scale, 0, (int)byte);
  };
  const int whole = p.K / kBlock;
  int block = wave;
  if (block < whole) {
    Piece next;
    fetch(next, block, true);
    while ((block += WAVES) < whole) {
      Piece cur = next;
      fetch(next, block, true);
      add(cur);
    }
    add(next);
  }
  if (whole < p.blocks && wave == whole % WAVES) {
    Piece last;
    fetch(last, whole, false);
    add(last);
  }
  f32x4* const sums = (f32x4*)mine;
  sums[lane] = acc;
  __syncthreads();
  // a lane holds row l15 of c, columns 4 part + e: a thread for each of the 256
  if (tid < 256) {
    const int from = tid >> 2, e = tid & 3, m = from & 15, column = blockIdx.x * 16 + 4 * (from >> 4) + e;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) s += ((const f32x4*)rounded[w])[from][e];
    if (m < rows && column < p.N) {
      if (p.bias) s += IoType<IODT>::load((const E*)p.bias + column);
      IoType<IODT>::store((E*)p.c + (int64_t)(m0 + m) * p.ldc + column, s);
    }
  }
}

}  // namespace cascmm
