// Layer norm over the last axis, forward and backward, alone or behind the residual add in front of it (gfx950).
//
//   s = x + residual, rounded to the tensors' type (or s = x);   xhat = (s - mean(s)) / sqrt(var(s) + eps);   y = xhat * weight + bias
//   dx = rstd (g - mean(g) - xhat mean(g xhat)) + ds,  g = dy * weight;   dweight = sum over rows of dy * xhat,  dbias = sum over rows of dy
//
// The norm is of the sum as it is stored: what the block goes on with, and what the backward pass reads.  Everything between a load and a
// store is fp32: statistics, xhat, the sums over rows; results are rounded once.  The variance is the mean of the squared differences from
// the mean, in a second run over registers, so rows far from zero lose nothing.
//
// Bound by memory.  A row lies in the registers of one wave (of four where it is longer), so every element is read once: a lane holds
// chunks of 16 bytes, 64 (256) of them side by side.  A wave keeps weight and bias in registers and walks over rows a grid apart, the
// next row's loads in flight while this one is reduced.  The backward pass adds the weight's and bias' gradients up in registers on its
// way, the waves of a workgroup meet in LDS, and a second kernel adds the workgroups' sums: in a fixed order, without atomics, so that
// the same call gives the same bits.
//
// Measured (graph replay, us; a large copy reaches 5.2 TB/s): 65536 x 1280 bf16 forward 60.9 (5.5 TB/s), backward with both sums 95.9 (5.25); 8192 x 640 fp16 7.0
// (3.0) and 14.3, fp32 8.8 (4.8) and 18.4; 1976 x 1280 bf16 4.4, with the residual 6.3 (3.2), backward 11.5; 8192 x 1001 bf16, rows off 16 bytes,
// backward 18.9; 4096 x 8192 bf16, four waves a row, 27.9 (4.8) and 52.2 (3.9); 2 x 1280 fp32 2.5, the launch and two trips to memory.  Backward the second kernel is 4 to 5 of them, mostly its launch and latency.
#pragma once
#include "cascmm_common.h"

namespace cascmm {

struct NormParams {
  const void* x;         // [rows][cols], row stride ldx (backward: the s that was normed)
  const void* residual;  // forward: NULL or [rows][cols]
  const void* weight;    // [cols] or NULL (ones)
  const void* bias;      // [cols] or NULL (zeros)
  void* y;               // forward: result; backward: dx
  void* sum;             // forward with a residual: s
  float* mean;           // [rows]; forward: written unless NULL; backward: read
  float* rstd;
  const void* dy;        // backward
  const void* ds;        // backward: NULL or the gradient that reaches s past the norm
  float* partials;       // backward: [workgroups][2][cols] sums for dweight, dbias; NULL: not wanted
  int64_t rows, ldx, ldr, ldy, lds, lddy, ldds;
  int cols, weight_f32;  // weight_f32: weight and bias are fp32 whatever the elements are
  float eps, inv_cols;
};

// sum over the 64 lanes, in every lane: inside rows of sixteen by DPP moves, then the four rows in order
template <int CTRL> __device__ __forceinline__ float norm_dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ float norm_wave_sum(float v) {
  v += norm_dpp<0xB1>(v);    // lane ^ 1
  v += norm_dpp<0x4E>(v);    // lane ^ 2
  v += norm_dpp<0x141>(v);   // the other four of eight
  v += norm_dpp<0x140>(v);   // the other eight of sixteen
  const int b = __builtin_bit_cast(int, v);
  float s = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 0));
  s += __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 16));
  s += __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 32));
  s += __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 48));
  return s;
}
// sum over four, eight or the sixteen lanes of a DPP row
template <int LANES> __device__ __forceinline__ float norm_few_sum(float v) {
  v += norm_dpp<0xB1>(v);
  v += norm_dpp<0x4E>(v);
  if (LANES > 4) v += norm_dpp<0x141>(v);
  if (LANES > 8) v += norm_dpp<0x140>(v);
  return v;
}
// N sums over the LPR lanes of a row: four, eight, sixteen, a wave or the waves of a workgroup.  `turn` counts the reductions: two sets of slots take turns, so one barrier each is enough
// (a wave writes a set again only behind the barrier that all readers of it have passed).
template <int LPR, int N> __device__ __forceinline__ void norm_sums(float (&v)[N], float* slots, int& turn) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (LPR < 64) v[i] = norm_few_sum<LPR>(v[i]);
    else v[i] = norm_wave_sum(v[i]);
  }
  if constexpr (LPR > 64) {
    constexpr int WPR = LPR / 64;
    float* set = slots + (turn & 1) * (2 * WPR);
    ++turn;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) set[i * WPR + (threadIdx.x >> 6)] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < WPR; ++w) s += set[i * WPR + w];
      v[i] = s;
    }
  }
}

// 16 bytes of a row as fp32.  Rows start on element boundaries, not always on 16 bytes: the type says so to the compiler.
// TINY: rows shorter than 16 bytes, element by element.
template <int IODT, bool TINY = false> struct NormRow {
  typedef typename IoType<IODT>::T E;
  static constexpr int VEC = 16 / (int)sizeof(E);
  typedef E chunk __attribute__((ext_vector_type(VEC), aligned(sizeof(E))));
  // The chunk at column c of a row of `cols` (past the end: zeros), in two steps, the load and what settle() does to it where it is used.  A chunk that hangs over
  // the end is loaded as the row's last whole one and shifted: element by element its parts would be put together behind the load, and every load in
  // front of it waited for there (8192 x 1001 bf16 backward 22.7 us, so 19.3; rows of whole chunks too, whose code it was: 65536 x 1280 110 us, so 96).
  static __device__ __forceinline__ chunk load(const E* row, int c, int cols) {
    chunk v;
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = (E)0.f;
    if constexpr (TINY) {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (c + e < cols) v[e] = row[c + e];
    } else if (c < cols) {
      v = *(const chunk*)(row + (c < cols - VEC ? c : cols - VEC));
    }
    return v;
  }
  static __device__ __forceinline__ bool ragged(int cols) { return !TINY && cols % VEC != 0; }
  // TURN: what lies behind the end are elements from in front of the lane's own, not zeros.
  template <bool TURN = false> static __device__ __forceinline__ chunk settle(chunk v, int c, int cols) {
    if (!ragged(cols)) return v;
    const int s = c > cols - VEC && c < cols ? c - (cols - VEC) : 0;   // elements in front of the lane's own
    const int dwords = sizeof(E) == 2 ? s >> 1 : s;
    u32x4 w = __builtin_bit_cast(u32x4, v);
    if (dwords & 1) w = (u32x4){w[1], w[2], w[3], TURN ? w[0] : 0u};
    if (dwords & 2) w = (u32x4){w[2], w[3], TURN ? w[0] : 0u, TURN ? w[1] : 0u};
    if (sizeof(E) == 2 && (s & 1))
      w = (u32x4){__builtin_amdgcn_alignbit(w[1], w[0], 16), __builtin_amdgcn_alignbit(w[2], w[1], 16), __builtin_amdgcn_alignbit(w[3], w[2], 16),
                  TURN ? __builtin_amdgcn_alignbit(w[0], w[3], 16) : w[3] >> 16};
    return __builtin_bit_cast(chunk, w);
  }
  // ... of a chunk that no row of this kernel ends in (whole: known at compile time)
  static __device__ __forceinline__ chunk load(const E* row, int c, int cols, bool whole) { return whole ? *(const chunk*)(row + c) : load(row, c, cols); }
  static __device__ __forceinline__ void store(E* row, int c, int cols, chunk v, bool whole) {
    if (whole) *(chunk*)(row + c) = v;
    else store(row, c, cols, v);
  }
  static __device__ __forceinline__ chunk load_settled(const E* row, int c, int cols) { return settle(load(row, c, cols), c, cols); }
  static __device__ __forceinline__ chunk load_turned(const E* row, int c, int cols) { return settle<true>(load(row, c, cols), c, cols); }
  static __device__ __forceinline__ void store(E* row, int c, int cols, chunk v) {
    if (c + VEC <= cols) {
      *(chunk*)(row + c) = v;
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (c + e < cols) row[c + e] = v[e];
    }
  }
  // CH chunks of weight or bias, `step` columns apart: all of them asked for before the first is looked at
  template <int FULL, int CH> static __device__ __forceinline__ void load_weight(float (&w)[CH][VEC], const void* p, int f32, int c0, int step, int cols, float otherwise) {
    if (!p) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < VEC; ++e) w[c][e] = otherwise;
    } else if (f32 && sizeof(E) == 2) {
      const float* q = (const float*)p;
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int col = c0 + c * step + e;
          w[c][e] = col < cols ? q[col] : 0.f;
        }
    } else if constexpr (TINY) {
      static_assert(CH <= 2, "a row of one chunk");
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int col = c0 + c * step + e;
          w[c][e] = col < cols ? (float)((const E*)p)[col] : 0.f;
        }
    } else {
      chunk v[CH];
#pragma unroll
      for (int c = 0; c < CH; ++c) v[c] = load((const E*)p, c0 + c * step, cols, c < FULL);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if (c >= FULL) v[c] = settle(v[c], c0 + c * step, cols);
#pragma unroll
        for (int e = 0; e < VEC; ++e) w[c][e] = (float)v[c][e];
      }
    }
  }
};

// Rows of up to LPR NV columns, NV a multiple of 8: LPR lanes a row (eight, sixteen, a wave, or all four waves of a workgroup; four: rows
// shorter than 16 bytes), NV elements a lane.
template <int IODT, int NV, int LPR, bool ADD>
__global__ __launch_bounds__(256) void cascmm_layer_norm_kernel(const NormParams p) {
  typedef NormRow<IODT, LPR == 4> R;
  typedef typename R::E E;
  typedef typename R::chunk chunk;
  constexpr int VEC = R::VEC, CH = NV / VEC, STEP = LPR * VEC, ROWS = 256 / LPR;   // ROWS: of a workgroup at a time
  constexpr int FULL = CH - 8 / VEC;   // chunks that lie inside every row: a shorter one has a kernel of fewer values
  __shared__ float slots[16];
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  int cols = p.cols;
  const E *x_at = (const E*)p.x, *r_at = (const E*)p.residual;
  E *y_at = (E*)p.y, *s_at = (E*)p.sum;
  const void *weight = p.weight, *bias = p.bias;
  int64_t rows = p.rows, ldx = p.ldx, ldr = p.ldr;
  // (the arguments are requested together: left to themselves the reads sink to their uses and wait one behind the other, 1.2 us of 2 x 1280's 5.0 with a residual)
  asm volatile("" : "+s"(cols), "+s"(x_at), "+s"(weight), "+s"(bias), "+s"(rows), "+s"(ldx));
  if constexpr (ADD) asm volatile("" : "+s"(r_at), "+s"(ldr));
  const int col0 = lane * VEC;
  const int64_t stride = (int64_t)gridDim.x * ROWS;
  int64_t row = (int64_t)blockIdx.x * ROWS + (LPR == 64 ? __builtin_amdgcn_readfirstlane(group) : group);
  int turn = 0;
  if (row >= rows) return;   // (of a row's lanes all or none, so every barrier has its waves)
  chunk x[CH], r[ADD ? CH : 1];
  auto fetch = [&](int64_t at) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      x[c] = R::load(x_at + at * ldx, col0 + c * STEP, cols, c < FULL);
      if constexpr (ADD) r[c] = R::load(r_at + at * ldr, col0 + c * STEP, cols, c < FULL);
    }
  };
  fetch(row);
  float w[CH][VEC], b[CH][VEC];
  R::template load_weight<FULL>(w, weight, p.weight_f32, col0, STEP, cols, 1.f);
  R::template load_weight<FULL>(b, bias, p.weight_f32, col0, STEP, cols, 0.f);
  for (;;) {
    float v[CH][VEC], total[1] = {0.f};
    if (R::ragged(cols)) {
#pragma unroll
      for (int c = FULL; c < CH; ++c) {
        x[c] = R::settle(x[c], col0 + c * STEP, cols);
        if constexpr (ADD) r[c] = R::settle(r[c], col0 + c * STEP, cols);
      }
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if constexpr (ADD) {
        chunk s;
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[e] = (E)((float)x[c][e] + (float)r[c][e]);
        R::store(s_at + row * p.lds, col0 + c * STEP, cols, s, c < FULL);
        x[c] = s;
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        v[c][e] = (float)x[c][e];
        total[0] += v[c][e];
      }
    }
    const int64_t next = row + stride;
    if (next < rows) fetch(next);
    norm_sums<LPR>(total, slots, turn);
    const float mean = total[0] / (float)cols;
    float square[1] = {0.f};
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        v[c][e] = c < FULL || col0 + c * STEP + e < cols ? v[c][e] - mean : 0.f;
        square[0] = __builtin_fmaf(v[c][e], v[c][e], square[0]);
      }
    norm_sums<LPR>(square, slots, turn);
    const float rstd = rsqrtf(square[0] * p.inv_cols + p.eps);
    if (p.mean && lane == 0) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      chunk y;
#pragma unroll
      for (int e = 0; e < VEC; ++e) y[e] = (E)__builtin_fmaf(v[c][e] * rstd, w[c][e], b[c][e]);
      R::store(y_at + row * p.ldy, col0 + c * STEP, cols, y, c < FULL);
    }
    if (next >= rows) return;
    row = next;
  }
}

// longer rows: a workgroup a row, three runs over it (the second and third mostly from the caches): 2048 x 16384 bf16 38.3 us, 25.8 for its bytes at a copy's rate
constexpr int kNormWide = 1024;
template <int IODT, bool ADD>
__global__ __launch_bounds__(kNormWide) void cascmm_layer_norm_wide_kernel(const NormParams p) {
  typedef NormRow<IODT> R;
  typedef typename R::E E;
  typedef typename R::chunk chunk;
  constexpr int VEC = R::VEC, STEP = kNormWide * VEC;
  __shared__ float slots[kNormWide / 16];
  const int cols = p.cols, col0 = threadIdx.x * VEC;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const E* x = (const E*)p.x + row * p.ldx;
    float total[1] = {0.f};
    for (int64_t c = col0; c < cols; c += STEP) {
      chunk v = R::load_settled(x, (int)c, cols);
      if constexpr (ADD) {
        const chunk r = R::load_settled((const E*)p.residual + row * p.ldr, (int)c, cols);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = (E)((float)v[e] + (float)r[e]);
        R::store((E*)p.sum + row * p.lds, (int)c, cols, v);
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) total[0] += (float)v[e];
    }
    // (a thread reads back what it has written itself)
    const E* s = ADD ? (const E*)p.sum + row * p.lds : x;
    norm_sums<kNormWide>(total, slots, turn);
    const float mean = total[0] / (float)p.cols;
    float square[1] = {0.f};
    for (int64_t c = col0; c < cols; c += STEP) {
      const chunk v = R::load_settled(s, (int)c, cols);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = c + e < cols ? (float)v[e] - mean : 0.f;
        square[0] = __builtin_fmaf(d, d, square[0]);
      }
    }
    norm_sums<kNormWide>(square, slots, turn);
    const float rstd = rsqrtf(square[0] * p.inv_cols + p.eps);
    if (p.mean && threadIdx.x == 0) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
    for (int64_t c = col0; c < cols; c += STEP) {
      const chunk v = R::load_settled(s, (int)c, cols);
      float w[1][VEC], b[1][VEC];
      R::template load_weight<0>(w, p.weight, p.weight_f32, (int)c, 0, cols, 1.f);
      R::template load_weight<0>(b, p.bias, p.weight_f32, (int)c, 0, cols, 0.f);
      chunk y;
#pragma unroll
      for (int e = 0; e < VEC; ++e) y[e] = (E)__builtin_fmaf(((float)v[e] - mean) * rstd, w[0][e], b[0][e]);
      R::store((E*)p.y + row * p.ldy, (int)c, cols, y);
    }
  }
}

// Backward.  SUMS: the sums for dweight and dbias too, a workgroup's at partials[blockIdx.x].
template <int IODT, int NV, int LPR, bool DS, bool SUMS>
__global__ __launch_bounds__(256) void cascmm_layer_norm_backward_kernel(const NormParams p) {
  typedef NormRow<IODT, LPR == 4> R;
  typedef typename R::E E;
  typedef typename R::chunk chunk;
  constexpr int VEC = R::VEC, CH = NV / VEC, STEP = LPR * VEC, ROWS = 256 / LPR;
  constexpr int FULL = CH - 8 / VEC;   // (as above)
  __shared__ float slots[16];
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  int cols = p.cols;
  const E *x_at = (const E*)p.x, *dy_at = (const E*)p.dy, *ds_at = (const E*)p.ds;
  E* dx_at = (E*)p.y;
  const void* weight = p.weight;
  const float *mean_at = p.mean, *rstd_at = p.rstd;
  int64_t rows = p.rows, ldx = p.ldx, lddy = p.lddy, ldds = p.ldds;
  asm volatile("" : "+s"(cols), "+s"(x_at), "+s"(dy_at), "+s"(weight), "+s"(mean_at), "+s"(rstd_at), "+s"(rows), "+s"(ldx), "+s"(lddy));
  if constexpr (DS) asm volatile("" : "+s"(ds_at), "+s"(ldds));
  const int col0 = lane * VEC;
  const int64_t stride = (int64_t)gridDim.x * ROWS;
  int64_t row = (int64_t)blockIdx.x * ROWS + (LPR == 64 ? __builtin_amdgcn_readfirstlane(group) : group);
  int turn = 0;
  struct Row {
    chunk x[CH], dy[CH], ds[DS ? CH : 1];
    float mean, rstd;
  } next;
  auto fetch = [&](int64_t at) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      next.x[c] = R::load(x_at + at * ldx, col0 + c * STEP, cols, c < FULL);
      next.dy[c] = R::load(dy_at + at * lddy, col0 + c * STEP, cols, c < FULL);
      if constexpr (DS) next.ds[c] = R::load(ds_at + at * ldds, col0 + c * STEP, cols, c < FULL);
    }
    next.mean = mean_at[at];
    next.rstd = rstd_at[at];
  };
  float w[CH][VEC], dw[SUMS ? CH : 1][VEC], db[SUMS ? CH : 1][VEC];
  R::template load_weight<FULL>(w, weight, p.weight_f32, col0, STEP, cols, 1.f);
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    if constexpr (SUMS) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) dw[c][e] = db[c][e] = 0.f;
    }
  }
  if (row < rows) fetch(row);
  while (row < rows) {
    Row cur = next;
    if (R::ragged(cols)) {
#pragma unroll
      for (int c = FULL; c < CH; ++c) {
        cur.x[c] = R::settle(cur.x[c], col0 + c * STEP, cols);
        cur.dy[c] = R::settle(cur.dy[c], col0 + c * STEP, cols);
        if constexpr (DS) cur.ds[c] = R::settle(cur.ds[c], col0 + c * STEP, cols);
      }
    }
    const int64_t at = row;
    row += stride;
    if (row < rows) fetch(row);
    float sums[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        // (behind the last column x, dy and with it g are zeros; xhat, which the mean is taken from, is held to zero too: of a row far from zero the
        // mean times rstd may be infinite there, and zero times that is no zero)
        const float xhat = ((float)cur.x[c][e] - cur.mean) * cur.rstd, d = (float)cur.dy[c][e], g = d * w[c][e];
        sums[0] += g;
        sums[1] = __builtin_fmaf(g, c < FULL || col0 + c * STEP + e < cols ? xhat : 0.f, sums[1]);
        if constexpr (SUMS) {
          dw[c][e] = __builtin_fmaf(d, xhat, dw[c][e]);
          db[c][e] += d;
        }
      }
    norm_sums<LPR>(sums, slots, turn);
    const float c1 = sums[0] * p.inv_cols, c2 = sums[1] * p.inv_cols;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      chunk out;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float xhat = ((float)cur.x[c][e] - cur.mean) * cur.rstd;
        float d = cur.rstd * ((float)cur.dy[c][e] * w[c][e] - c1 - xhat * c2);
        if constexpr (DS) d += (float)cur.ds[c][e];
        out[e] = (E)d;
      }
      R::store(dx_at + at * p.ldy, col0 + c * STEP, cols, out, c < FULL);
    }
  }
  if constexpr (SUMS) {
    float* part = p.partials + (int64_t)blockIdx.x * 2 * cols;
    if constexpr (LPR <= 64) {
      // a wave's rows of lanes, then the four waves in order, in LDS (a lane's elements LPR apart: side by side over the lanes)
      __shared__ float meet[4][2][LPR * NV];
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          float a = dw[c][e], b = db[c][e];
#pragma unroll
          for (int off = LPR; off < 64; off *= 2) {
            a += __shfl_xor(a, off, 64);
            b += __shfl_xor(b, off, 64);
          }
          if (LPR == 64 || (threadIdx.x & 63) < LPR) {
            meet[threadIdx.x >> 6][0][(c * VEC + e) * LPR + lane] = a;
            meet[threadIdx.x >> 6][1][(c * VEC + e) * LPR + lane] = b;
          }
        }
      __syncthreads();
      for (int i = threadIdx.x; i < LPR * NV; i += 256) {
        const int col = i / STEP * STEP + (i % LPR) * VEC + i % STEP / LPR;
        if (col < cols) {
          part[col] = ((meet[0][0][i] + meet[1][0][i]) + meet[2][0][i]) + meet[3][0][i];
          part[cols + col] = ((meet[0][1][i] + meet[1][1][i]) + meet[2][1][i]) + meet[3][1][i];
        }
      }
    } else {
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int col = col0 + c * STEP + e;
          if (col < cols) {
            part[col] = dw[c][e];
            part[cols + col] = db[c][e];
          }
        }
    }
  }
}

// longer rows: dx with a workgroup a row, two runs over x and dy, which the sums read once more: 2048 x 16384 bf16 93 us all together, 38.7 for the bytes ...
template <int IODT>
__global__ __launch_bounds__(kNormWide) void cascmm_layer_norm_backward_wide_kernel(const NormParams p) {
  typedef NormRow<IODT> R;
  typedef typename R::E E;
  typedef typename R::chunk chunk;
  constexpr int VEC = R::VEC, STEP = kNormWide * VEC;
  __shared__ float slots[kNormWide / 16];
  const int cols = p.cols, col0 = threadIdx.x * VEC;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const E *x = (const E*)p.x + row * p.ldx, *dy = (const E*)p.dy + row * p.lddy, *ds = p.ds ? (const E*)p.ds + row * p.ldds : nullptr;
    const float mean = p.mean[row], rstd = p.rstd[row];
    float sums[2] = {0.f, 0.f};
    for (int64_t c = col0; c < cols; c += STEP) {
      // (behind the last column xhat meets a zero of dy; of turned chunks it is some other column's there, and finite where the row's are)
      const chunk v = R::load_turned(x, (int)c, cols), d = R::load_settled(dy, (int)c, cols);
      float w[1][VEC];
      R::template load_weight<0>(w, p.weight, p.weight_f32, (int)c, 0, cols, 1.f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float g = (float)d[e] * w[0][e];
        sums[0] += g;
        sums[1] = __builtin_fmaf(g, ((float)v[e] - mean) * rstd, sums[1]);
      }
    }
    norm_sums<kNormWide>(sums, slots, turn);
    const float c1 = sums[0] * p.inv_cols, c2 = sums[1] * p.inv_cols;
    for (int64_t c = col0; c < cols; c += STEP) {
      const chunk v = R::load_settled(x, (int)c, cols), d = R::load_settled(dy, (int)c, cols);
      float w[1][VEC];
      R::template load_weight<0>(w, p.weight, p.weight_f32, (int)c, 0, cols, 1.f);
      chunk z, out;
      if (ds) z = R::load_settled(ds, (int)c, cols);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float o = rstd * ((float)d[e] * w[0][e] - c1 - ((float)v[e] - mean) * rstd * c2);
        if (ds) o += (float)z[e];
        out[e] = (E)o;
      }
      R::store((E*)p.y + row * p.ldy, (int)c, cols, out);
    }
  }
}
// ... and the sums with a thread a column over every gridDim.y-th row
template <int IODT>
__global__ __launch_bounds__(256) void cascmm_layer_norm_sums_kernel(const NormParams p) {
  typedef typename IoType<IODT>::T E;
  const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (col >= p.cols) return;
  float dw = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const float d = (float)((const E*)p.dy)[row * p.lddy + col];
    dw = __builtin_fmaf(d, ((float)((const E*)p.x)[row * p.ldx + col] - p.mean[row]) * p.rstd[row], dw);
    db += d;
  }
  float* part = p.partials + (int64_t)blockIdx.y * 2 * p.cols;
  part[col] = dw;
  part[p.cols + col] = db;
}

// out[col] (and out2[col], the second half of a partial row) = sum over `parts` rows of partials, [parts][halves][cols].  Thirty-two columns a
// workgroup, its 32 rows of threads a share of the parts each; they meet in LDS in order.
constexpr int kFinishCols = 32;
constexpr int64_t kFinishMostCols = 1 << 26;   // (a launch has fewer than 2^32 threads; column numbers and a step beyond the last stay in 32 bits)
template <int ODT>
__global__ __launch_bounds__(1024) void cascmm_column_finish_kernel(const float* __restrict__ partials, int parts, int halves, int64_t cols, void* out, void* out2) {
  typedef typename IoType<ODT>::T E;
  __shared__ float meet[32][kFinishCols + 1];
  const int c = threadIdx.x & 31, r = threadIdx.x >> 5, half = blockIdx.y;
  const int64_t col = (int64_t)blockIdx.x * kFinishCols + c;
  float s = 0.f;
  if (col < cols) {
    const float* src = partials + (int64_t)half * cols + col;
    const int64_t step = (int64_t)halves * cols;
    for (int i = r; i < parts; i += 32 * 16) {   // (sixteen loads in flight: a workgroup runs through its partial sums once, bound by their latency)
      float v[16];
#pragma unroll
      for (int u = 0; u < 16; ++u) v[u] = i + 32 * u < parts ? src[(i + 32 * u) * step] : 0.f;
#pragma unroll
      for (int u = 0; u < 16; ++u) s += v[u];
    }
  }
  meet[r][c] = s;
  __syncthreads();
  if (r == 0 && col < cols) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) t += meet[i][c];
    E* dst = (E*)(half ? out2 : out);
    if (dst) IoType<ODT>::store(dst + col, t);
  }
}

}  // namespace cascmm
