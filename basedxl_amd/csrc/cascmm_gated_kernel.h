// The norms on both sides of a block's residual add, with the add, its gate and the residual's scale, forward and backward (gfx950).
//
//   p = norm(x) post_weight + post_bias (or p = x);   s = scale * residual + gate * p, rounded to the tensors' type;   y = norm(s) weight + bias
//   norm(v) = (v - mean) / sqrt(var + eps) ("layer"), v / sqrt(mean of v^2 + eps) ("rms", written below with a mean of zero)
// Backward, with shat and xhat what the norms give and [..] of a layer norm only:
//   D = ds + rstd2 (dy weight - [mean(dy weight)] - shat mean(dy weight shat));   dresidual = scale D
//   q = D gate post_weight;   dx = rstd1 (q - [mean(q)] - xhat mean(q xhat)), without the first norm dx = D gate
//   sums over the rows that share an element:  S1 = D xhat (of x itself without the first norm),  S2 = D,  S3 = D residual,  S4 = dy shat,  S5 = dy;
//   dgate = post_weight S1 + post_bias S2,  dpost_weight = sum of gate S1,  dpost_bias = sum of gate S2,  dscale = S3,  dweight = S4,  dbias = S5
//
// Gate, scale, weight and bias are one row for all rows or one for each group of consecutive rows (a sample's tokens); a workgroup stays within a group and
// keeps them in registers, the gate multiplied into the first norm's weight.  The second norm is of s as it is stored: what the block goes on with, and what the
// backward pass reads.  Everything between a load and a store is fp32.
//
// Bound by memory.  As in cascmm_norm_kernel.h, whose rows and sums these are, a row lies in the registers of sixteen lanes, a wave or four waves, so every element is
// read once; the backward pass adds the five sums up in registers on its way over a workgroup's rows, and one more kernel adds the workgroups' sums
// in a fixed order, without atomics.
//
// Measured (us; a large copy reaches 4.9 TB/s): 32768 x 1280 bf16, gated and modulated for each of 32 samples, 63.2 (5.3 TB/s) and backward 106 (4.7) + 8.6 for the sums, most of
// that latency; 8192 x 640 bf16, norms on both sides, 10.9 (3.8); 2331 x 457 fp32, all six sums, 8.8 and 12.9 + 7.3; 2 x 1280 fp16 3.6.
#pragma once
#include "cascmm_norm_kernel.h"

namespace cascmm {

struct GatedParams {
  const void *x, *residual;           // [rows][cols]
  const void *gate, *scale, *post_weight, *post_bias, *weight, *bias;   // NULL: ones (bias: zeros)
  void *y, *sum;                      // forward: results; backward (sum: what was stored)
  float* stats;                       // [4][rows]: mean and 1 / deviation of x, of s; forward: NULL or written
  const void *dy, *ds;                // backward; ds may be NULL
  void *dx, *dresidual;               // NULL: not wanted
  float* partials;                    // [groups][parts][sums][cols]; NULL: not wanted
  float* row_means;                   // rows without registers: [2][rows], mean(g) and mean(g shat) of the second norm
  int64_t rows, group_rows, part_rows;            // part_rows: of a workgroup
  int64_t ldx, ldr, ldy, lds, lddy, ldds, lddx, lddr;
  int64_t gate_ld, scale_ld, weight_ld, bias_ld;  // from a group's row to the next's; 0: shared
  int cols, parts, f32;               // f32: gate, scale, weights and biases are fp32 whatever the elements are
  int centred;                        // layer norms
  float eps, inv_cols, alpha;         // alpha: the residual's scale where there is no row of them
};

// a parameter's row of a group
__device__ __forceinline__ const void* gated_row(const void* p, int64_t at, int size) { return p ? (const char*)p + at * size : nullptr; }

template <int IODT, int LPR, int NV, bool POST, bool RICH> struct GatedRow {
  typedef NormRow<IODT> R;
  typedef typename R::E E;
  typedef typename R::chunk chunk;
  static constexpr int VEC = R::VEC, CH = NV / VEC, STEP = LPR * VEC, ROWS = 256 / LPR, FULL = CH - 8 / VEC;
  // the factor of xhat (of x), what is added with it, and the residual's scale
  float P[CH][VEC], Q[RICH ? CH : 1][VEC], A[RICH ? CH : 1][VEC];
  __device__ __forceinline__ void load(const GatedParams& p, int64_t group, int col0) {
    const int size = p.f32 ? 4 : (int)sizeof(E), cols = p.cols;
    R::template load_weight<FULL>(P, gated_row(p.gate, group * p.gate_ld, size), p.f32, col0, STEP, cols, 1.f);
    if constexpr (RICH) {
      R::template load_weight<FULL>(A, gated_row(p.scale, group * p.scale_ld, size), p.f32, col0, STEP, cols, p.alpha);
      R::template load_weight<FULL>(Q, p.post_bias, p.f32, col0, STEP, cols, 0.f);
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < VEC; ++e) Q[c][e] *= P[c][e];
    }
    if constexpr (POST) {
      float w[CH][VEC];
      R::template load_weight<FULL>(w, p.post_weight, p.f32, col0, STEP, cols, 1.f);
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < VEC; ++e) P[c][e] *= w[c][e];
    }
  }
};

// RICH: a row of the residual's scales or the first norm's bias is there.  Rows as cascmm_layer_norm_kernel holds them.
template <int IODT, int NV, int LPR, bool POST, bool RICH>
__global__ __launch_bounds__(256) void cascmm_gated_norm_kernel(const GatedParams p) {
  typedef GatedRow<IODT, LPR, NV, POST, RICH> G;
  typedef typename G::R R;
  typedef typename G::E E;
  typedef typename G::chunk chunk;
  constexpr int VEC = G::VEC, CH = G::CH, STEP = G::STEP, ROWS = G::ROWS, FULL = G::FULL;
  __shared__ float slots[16];
  const int lane = threadIdx.x % LPR, col0 = lane * VEC, cols = p.cols;
  const int64_t group = blockIdx.x / p.parts, first = (int64_t)(blockIdx.x % p.parts) * p.part_rows;
  const int64_t end = group * p.group_rows + (first + p.part_rows < p.group_rows ? first + p.part_rows : p.group_rows);
  int64_t row = group * p.group_rows + first + (LPR == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / LPR) : threadIdx.x / LPR);
  int turn = 0;
  if (row >= end) return;   // (of a row's lanes all or none, so every barrier has its waves)
  chunk x[CH], r[CH];
  auto fetch = [&](int64_t at) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      x[c] = R::load((const E*)p.x + at * p.ldx, col0 + c * STEP, cols, c < FULL);
      r[c] = R::load((const E*)p.residual + at * p.ldr, col0 + c * STEP, cols, c < FULL);
    }
  };
  fetch(row);
  G g;
  float w[CH][VEC], b[CH][VEC];
  g.load(p, group, col0);
  const int size = p.f32 ? 4 : (int)sizeof(E);
  R::template load_weight<FULL>(w, gated_row(p.weight, group * p.weight_ld, size), p.f32, col0, STEP, cols, 1.f);
  R::template load_weight<FULL>(b, gated_row(p.bias, group * p.bias_ld, size), p.f32, col0, STEP, cols, 0.f);
  auto inside = [&](int c, int e) { return c < FULL || col0 + c * STEP + e < cols; };
  for (;;) {
    float v[CH][VEC];
    if (R::ragged(cols)) {
#pragma unroll
      for (int c = FULL; c < CH; ++c) {
        x[c] = R::settle(x[c], col0 + c * STEP, cols);
        r[c] = R::settle(r[c], col0 + c * STEP, cols);
      }
    }
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[c][e] = (float)x[c][e];
    // v -> (v - mean) rstd, zero behind the last column
    auto normed = [&](float& mean, float& rstd) {
      mean = 0.f;
      if (p.centred) {
        float total[1] = {0.f};
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int e = 0; e < VEC; ++e) total[0] += v[c][e];
        norm_sums<LPR>(total, slots, turn);
        mean = total[0] / (float)cols;
      }
      float square[1] = {0.f};
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          v[c][e] = inside(c, e) ? v[c][e] - mean : 0.f;
          square[0] = __builtin_fmaf(v[c][e], v[c][e], square[0]);
        }
      norm_sums<LPR>(square, slots, turn);
      rstd = rsqrtf(square[0] * p.inv_cols + p.eps);
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[c][e] *= rstd;
    };
    float mean1 = 0.f, rstd1 = 1.f, mean2, rstd2;
    if constexpr (POST) normed(mean1, rstd1);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      chunk s;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float t = (float)r[c][e] * (RICH ? g.A[c][e] : p.alpha);
        if constexpr (RICH) t += g.Q[c][e];
        s[e] = (E)__builtin_fmaf(v[c][e], g.P[c][e], t);
        v[c][e] = inside(c, e) ? (float)s[e] : 0.f;
      }
      R::store((E*)p.sum + row * p.lds, col0 + c * STEP, cols, s, c < FULL);
    }
    const int64_t at = row;
    row += ROWS;
    if (row < end) fetch(row);
    normed(mean2, rstd2);
    if (p.stats && lane == 0) {
      p.stats[at] = mean1;
      p.stats[p.rows + at] = rstd1;
      p.stats[2 * p.rows + at] = mean2;
      p.stats[3 * p.rows + at] = rstd2;
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      chunk y;
#pragma unroll
      for (int e = 0; e < VEC; ++e) y[e] = (E)__builtin_fmaf(v[c][e], w[c][e], b[c][e]);
      R::store((E*)p.y + at * p.ldy, col0 + c * STEP, cols, y, c < FULL);
    }
    if (row >= end) return;
  }
}

// RICH: five sums, else S1, S4 and S5.
template <int IODT, int NV, int LPR, bool POST, bool RICH>
__global__ __launch_bounds__(256) void cascmm_gated_norm_backward_kernel(const GatedParams p) {
  typedef GatedRow<IODT, LPR, NV, POST, RICH> G;
  typedef typename G::R R;
  typedef typename G::E E;
  typedef typename G::chunk chunk;
  constexpr int VEC = G::VEC, CH = G::CH, STEP = G::STEP, ROWS = G::ROWS, FULL = G::FULL, NS = RICH ? 5 : 3;
  __shared__ float slots[16];
  const int lane = threadIdx.x % LPR, col0 = lane * VEC, cols = p.cols;
  const int64_t group = blockIdx.x / p.parts, first = (int64_t)(blockIdx.x % p.parts) * p.part_rows;
  const int64_t end = group * p.group_rows + (first + p.part_rows < p.group_rows ? first + p.part_rows : p.group_rows);
  int64_t row = group * p.group_rows + first + (LPR == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / LPR) : threadIdx.x / LPR);
  int turn = 0;
  G g;
  float w[CH][VEC], sum[NS][CH][VEC];
  g.load(p, group, col0);
  R::template load_weight<FULL>(w, gated_row(p.weight, group * p.weight_ld, p.f32 ? 4 : (int)sizeof(E)), p.f32, col0, STEP, cols, 1.f);
#pragma unroll
  for (int i = 0; i < NS; ++i)
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum[i][c][e] = 0.f;
  const bool reads_x = POST || p.gate, reads_r = RICH && p.scale;
  struct Row {
    chunk x[CH], s[CH], dy[CH], ds[CH], r[RICH ? CH : 1];
    float mean1, rstd1, mean2, rstd2;
  } next;
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      next.x[c][e] = next.ds[c][e] = (E)0.f;
      if (RICH) next.r[c][e] = (E)0.f;
    }
  auto fetch = [&](int64_t at) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = col0 + c * STEP;
      next.s[c] = R::load((const E*)p.sum + at * p.lds, col, cols, c < FULL);
      next.dy[c] = R::load((const E*)p.dy + at * p.lddy, col, cols, c < FULL);
      if (reads_x) next.x[c] = R::load((const E*)p.x + at * p.ldx, col, cols, c < FULL);
      if (p.ds) next.ds[c] = R::load((const E*)p.ds + at * p.ldds, col, cols, c < FULL);
      if constexpr (RICH)
        if (reads_r) next.r[c] = R::load((const E*)p.residual + at * p.ldr, col, cols, c < FULL);
    }
    next.mean1 = p.stats[at];
    next.rstd1 = p.stats[p.rows + at];
    next.mean2 = p.stats[2 * p.rows + at];
    next.rstd2 = p.stats[3 * p.rows + at];
  };
  auto inside = [&](int c, int e) { return c < FULL || col0 + c * STEP + e < cols; };
  if (row < end) fetch(row);
  while (row < end) {
    Row cur = next;
    if (R::ragged(cols)) {
#pragma unroll
      for (int c = FULL; c < CH; ++c) {
        const int col = col0 + c * STEP;
        cur.s[c] = R::settle(cur.s[c], col, cols);
        cur.dy[c] = R::settle(cur.dy[c], col, cols);
        cur.x[c] = R::settle(cur.x[c], col, cols);
        cur.ds[c] = R::settle(cur.ds[c], col, cols);
        if constexpr (RICH) cur.r[c] = R::settle(cur.r[c], col, cols);
      }
    }
    const int64_t at = row;
    row += ROWS;
    if (row < end) fetch(row);
    // (behind the last column dy, ds, x and residual are zeros, and what a mean is taken from is held to zero too: of a row far from zero the mean times rstd
    // may be infinite there)
    float means[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float shat = inside(c, e) ? ((float)cur.s[c][e] - cur.mean2) * cur.rstd2 : 0.f, d = (float)cur.dy[c][e], q = d * w[c][e];
        means[0] += q;
        means[1] = __builtin_fmaf(q, shat, means[1]);
        sum[NS - 2][c][e] = __builtin_fmaf(d, shat, sum[NS - 2][c][e]);
        sum[NS - 1][c][e] += d;
      }
    norm_sums<LPR>(means, slots, turn);
    const float c1 = p.centred ? means[0] * p.inv_cols : 0.f, c2 = means[1] * p.inv_cols;
    float D[POST ? CH : 1][VEC], post[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      chunk out, dx;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float shat = ((float)cur.s[c][e] - cur.mean2) * cur.rstd2;
        const float d = inside(c, e) ? (float)cur.ds[c][e] + cur.rstd2 * ((float)cur.dy[c][e] * w[c][e] - c1 - shat * c2) : 0.f;
        const float xhat = POST ? (inside(c, e) ? ((float)cur.x[c][e] - cur.mean1) * cur.rstd1 : 0.f) : (float)cur.x[c][e];
        out[e] = (E)(d * (RICH ? g.A[c][e] : p.alpha));
        sum[0][c][e] = __builtin_fmaf(d, xhat, sum[0][c][e]);
        if constexpr (RICH) {
          sum[1][c][e] += d;
          sum[2][c][e] = __builtin_fmaf(d, (float)cur.r[c][e], sum[2][c][e]);
        }
        const float q = d * g.P[c][e];
        if constexpr (POST) {
          D[c][e] = q;
          post[0] += q;
          post[1] = __builtin_fmaf(q, xhat, post[1]);
        } else {
          dx[e] = (E)q;
        }
      }
      if (p.dresidual) R::store((E*)p.dresidual + at * p.lddr, col0 + c * STEP, cols, out, c < FULL);
      if constexpr (!POST)
        if (p.dx) R::store((E*)p.dx + at * p.lddx, col0 + c * STEP, cols, dx, c < FULL);
    }
    if constexpr (POST) {
      if (!p.dx) continue;   // (of all lanes)
      norm_sums<LPR>(post, slots, turn);
      const float c3 = p.centred ? post[0] * p.inv_cols : 0.f, c4 = post[1] * p.inv_cols;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        chunk out;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float xhat = ((float)cur.x[c][e] - cur.mean1) * cur.rstd1;
          out[e] = (E)(cur.rstd1 * (D[c][e] - c3 - xhat * c4));
        }
        R::store((E*)p.dx + at * p.lddx, col0 + c * STEP, cols, out, c < FULL);
      }
    }
  }
  if (!p.partials) return;
  float* part = p.partials + (int64_t)blockIdx.x * NS * cols;
  if constexpr (LPR <= 64) {
    // a wave's rows of lanes, then the four waves in order, in LDS, one sum at a time
    __shared__ float meet[4][LPR * NV];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      if (i) __syncthreads();
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          float a = sum[i][c][e];
#pragma unroll
          for (int off = LPR; off < 64; off *= 2) a += __shfl_xor(a, off, 64);
          if (LPR == 64 || (threadIdx.x & 63) < LPR) meet[threadIdx.x >> 6][(c * VEC + e) * LPR + lane] = a;
        }
      __syncthreads();
      for (int k = threadIdx.x; k < LPR * NV; k += 256) {
        const int col = k / STEP * STEP + (k % LPR) * VEC + k % STEP / LPR;
        if (col < cols) part[i * (int64_t)cols + col] = ((meet[0][k] + meet[1][k]) + meet[2][k]) + meet[3][k];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int col = col0 + c * STEP + e;
          if (col < cols) part[i * (int64_t)cols + col] = sum[i][c][e];
        }
  }
}

// ---------------------------------------------------------------------------------------
// rows that no registers hold, and rows shorter than 16 bytes (TINY): a workgroup a row, several runs over it
// ---------------------------------------------------------------------------------------
constexpr int kGatedWide = 1024;
template <int IODT, bool TINY> struct GatedWide {
  typedef NormRow<IODT, TINY> R;
  typedef typename R::E E;
  typedef typename R::chunk chunk;
  static constexpr int VEC = R::VEC, STEP = kGatedWide * VEC;
  static __device__ __forceinline__ void values(float (&v)[VEC], const void* row, int c, int cols) {
    const chunk k = R::load_settled((const E*)row, c, cols);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = (float)k[e];
  }
  static __device__ __forceinline__ void weights(float (&v)[VEC], const void* p, int64_t at, const GatedParams& q, int c, float otherwise) {
    float w[1][VEC];
    R::template load_weight<0>(w, gated_row(p, at, q.f32 ? 4 : (int)sizeof(E)), q.f32, c, 0, q.cols, otherwise);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = w[0][e];
  }
  static __device__ __forceinline__ void put(void* row, int c, int cols, const float (&v)[VEC]) {
    chunk k;
#pragma unroll
    for (int e = 0; e < VEC; ++e) k[e] = (E)v[e];
    R::store((E*)row, c, cols, k);
  }
  // mean and 1 / deviation of a row
  static __device__ __forceinline__ void statistics(const void* row, const GatedParams& p, float* slots, int& turn, float& mean, float& rstd) {
    float v[VEC];
    mean = 0.f;
    if (p.centred) {
      float total[1] = {0.f};
      for (int64_t c = threadIdx.x * VEC; c < p.cols; c += STEP) {
        values(v, row, (int)c, p.cols);
#pragma unroll
        for (int e = 0; e < VEC; ++e) total[0] += v[e];
      }
      norm_sums<kGatedWide>(total, slots, turn);
      mean = total[0] / (float)p.cols;
    }
    float square[1] = {0.f};
    for (int64_t c = threadIdx.x * VEC; c < p.cols; c += STEP) {
      values(v, row, (int)c, p.cols);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = c + e < p.cols ? v[e] - mean : 0.f;
        square[0] = __builtin_fmaf(d, d, square[0]);
      }
    }
    norm_sums<kGatedWide>(square, slots, turn);
    rstd = rsqrtf(square[0] * p.inv_cols + p.eps);
  }
};

template <int IODT, bool TINY>
__global__ __launch_bounds__(kGatedWide) void cascmm_gated_norm_wide_kernel(const GatedParams p, int post) {
  typedef GatedWide<IODT, TINY> W;
  typedef typename W::E E;
  constexpr int VEC = W::VEC, STEP = W::STEP;
  __shared__ float slots[kGatedWide / 16];
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const int64_t group = row / p.group_rows;
    const E *x = (const E*)p.x + row * p.ldx, *r = (const E*)p.residual + row * p.ldr;
    E* s = (E*)p.sum + row * p.lds;
    float mean1 = 0.f, rstd1 = 1.f, mean2, rstd2;
    if (post) W::statistics(x, p, slots, turn, mean1, rstd1);
    for (int64_t c = threadIdx.x * VEC; c < p.cols; c += STEP) {
      float v[VEC], t[VEC], gate[VEC], scale[VEC], w[VEC], b[VEC];
      W::values(v, x, (int)c, p.cols);
      W::values(t, r, (int)c, p.cols);
      W::weights(gate, p.gate, group * p.gate_ld, p, (int)c, 1.f);
      W::weights(scale, p.scale, group * p.scale_ld, p, (int)c, p.alpha);
      W::weights(w, post ? p.post_weight : nullptr, 0, p, (int)c, 1.f);
      W::weights(b, post ? p.post_bias : nullptr, 0, p, (int)c, 0.f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = __builtin_fmaf((v[e] - mean1) * rstd1, gate[e] * w[e], __builtin_fmaf(t[e], scale[e], gate[e] * b[e]));
      W::put(s, (int)c, p.cols, v);
    }
    // (a thread reads back what it has written itself)
    W::statistics(s, p, slots, turn, mean2, rstd2);
    if (p.stats && threadIdx.x == 0) {
      p.stats[row] = mean1;
      p.stats[p.rows + row] = rstd1;
      p.stats[2 * p.rows + row] = mean2;
      p.stats[3 * p.rows + row] = rstd2;
    }
    for (int64_t c = threadIdx.x * VEC; c < p.cols; c += STEP) {
      float v[VEC], w[VEC], b[VEC];
      W::values(v, s, (int)c, p.cols);
      W::weights(w, p.weight, group * p.weight_ld, p, (int)c, 1.f);
      W::weights(b, p.bias, group * p.bias_ld, p, (int)c, 0.f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = __builtin_fmaf((v[e] - mean2) * rstd2, w[e], b[e]);
      W::put((E*)p.y + row * p.ldy, (int)c, p.cols, v);
    }
  }
}

template <int IODT, bool TINY>
__global__ __launch_bounds__(kGatedWide) void cascmm_gated_norm_backward_wide_kernel(const GatedParams p, int post) {
  typedef GatedWide<IODT, TINY> W;
  typedef typename W::E E;
  constexpr int VEC = W::VEC, STEP = W::STEP;
  __shared__ float slots[kGatedWide / 16];
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const int64_t group = row / p.group_rows;
    const E *s = (const E*)p.sum + row * p.lds, *dy = (const E*)p.dy + row * p.lddy, *x = (const E*)p.x + row * p.ldx, *ds = p.ds ? (const E*)p.ds + row * p.ldds : nullptr;
    const float mean1 = p.stats[row], rstd1 = p.stats[p.rows + row], mean2 = p.stats[2 * p.rows + row], rstd2 = p.stats[3 * p.rows + row];
    float means[2] = {0.f, 0.f};
    for (int64_t c = threadIdx.x * VEC; c < p.cols; c += STEP) {
      float v[VEC], d[VEC], w[VEC];
      W::values(v, s, (int)c, p.cols);
      W::values(d, dy, (int)c, p.cols);
      W::weights(w, p.weight, group * p.weight_ld, p, (int)c, 1.f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float q = d[e] * w[e];
        means[0] += q;
        means[1] = __builtin_fmaf(q, c + e < p.cols ? (v[e] - mean2) * rstd2 : 0.f, means[1]);
      }
    }
    norm_sums<kGatedWide>(means, slots, turn);
    const float c1 = p.centred ? means[0] * p.inv_cols : 0.f, c2 = means[1] * p.inv_cols;
    if (p.row_means && threadIdx.x == 0) {
      p.row_means[row] = c1;
      p.row_means[p.rows + row] = c2;
    }
    // D gate post_weight and xhat of a piece of the row
    auto piece = [&](int c, float (&q)[VEC], float (&xhat)[VEC], bool store) {
      float v[VEC], d[VEC], w[VEC], z[VEC], gate[VEC], scale[VEC], pw[VEC], out[VEC];
      W::values(v, s, c, p.cols);
      W::values(d, dy, c, p.cols);
      W::weights(w, p.weight, group * p.weight_ld, p, c, 1.f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) z[e] = 0.f;
      if (ds) W::values(z, ds, c, p.cols);
      W::weights(gate, p.gate, group * p.gate_ld, p, c, 1.f);
      W::weights(scale, p.scale, group * p.scale_ld, p, c, p.alpha);
      W::weights(pw, post ? p.post_weight : nullptr, 0, p, c, 1.f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) xhat[e] = 0.f;
      if (post) W::values(xhat, x, c, p.cols);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const bool in = c + e < p.cols;
        const float D = in ? z[e] + rstd2 * (d[e] * w[e] - c1 - (v[e] - mean2) * rstd2 * c2) : 0.f;
        xhat[e] = in ? (xhat[e] - mean1) * rstd1 : 0.f;
        out[e] = D * scale[e];
        q[e] = D * gate[e] * pw[e];
      }
      if (store) W::put((E*)p.dresidual + row * p.lddr, c, p.cols, out);
    };
    float together[2] = {0.f, 0.f};
    for (int64_t c = threadIdx.x * VEC; c < p.cols; c += STEP) {
      float q[VEC], xhat[VEC];
      piece((int)c, q, xhat, p.dresidual != nullptr);
      if (!post && p.dx) W::put((E*)p.dx + row * p.lddx, (int)c, p.cols, q);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        together[0] += q[e];
        together[1] = __builtin_fmaf(q[e], xhat[e], together[1]);
      }
    }
    if (!post || !p.dx) continue;
    norm_sums<kGatedWide>(together, slots, turn);
    const float c3 = p.centred ? together[0] * p.inv_cols : 0.f, c4 = together[1] * p.inv_cols;
    for (int64_t c = threadIdx.x * VEC; c < p.cols; c += STEP) {
      float q[VEC], xhat[VEC];
      piece((int)c, q, xhat, false);
#pragma unroll
      for (int e = 0; e < VEC; ++e) q[e] = rstd1 * (q[e] - c3 - xhat[e] * c4);
      W::put((E*)p.dx + row * p.lddx, (int)c, p.cols, q);
    }
  }
}
// ... and the five sums with a thread a column over a part's rows; `all` parts of all groups, which the grid's second axis goes through
template <int IODT>
__global__ __launch_bounds__(256) void cascmm_gated_norm_sums_kernel(const GatedParams p, int64_t all, int post) {
  typedef typename IoType<IODT>::T E;
  const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (col >= p.cols) return;
  for (int64_t at = blockIdx.y; at < all; at += gridDim.y) {
    const int64_t group = at / p.parts, first = at % p.parts * p.part_rows;
    const int64_t end = group * p.group_rows + (first + p.part_rows < p.group_rows ? first + p.part_rows : p.group_rows);
    const int64_t wat = group * p.weight_ld + col;
    const float w = !p.weight ? 1.f : p.f32 ? ((const float*)p.weight)[wat] : (float)((const E*)p.weight)[wat];
    float sum[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
    for (int64_t row = group * p.group_rows + first; row < end; ++row) {
      const float mean1 = p.stats[row], rstd1 = p.stats[p.rows + row], mean2 = p.stats[2 * p.rows + row], rstd2 = p.stats[3 * p.rows + row];
      const float d = (float)((const E*)p.dy)[row * p.lddy + col], shat = ((float)((const E*)p.sum)[row * p.lds + col] - mean2) * rstd2;
      float D = rstd2 * (d * w - p.row_means[row] - shat * p.row_means[p.rows + row]);
      if (p.ds) D += (float)((const E*)p.ds)[row * p.ldds + col];
      if (post || p.gate) sum[0] = __builtin_fmaf(D, ((float)((const E*)p.x)[row * p.ldx + col] - mean1) * rstd1, sum[0]);
      sum[1] += D;
      if (p.scale) sum[2] = __builtin_fmaf(D, (float)((const E*)p.residual)[row * p.ldr + col], sum[2]);
      sum[3] = __builtin_fmaf(d, shat, sum[3]);
      sum[4] += d;
    }
#pragma unroll
    for (int i = 0; i < 5; ++i) p.partials[(at * 5 + i) * p.cols + col] = sum[i];
  }
}

// The gradients from the workgroups' sums.  Thirty-two columns a workgroup; of its 32 rows of threads `share` (a power of two) add a group's parts between them, so that
// 32 / share groups are at hand at a time; a group's gradients are written, those that groups share added up over the groups, in order.
struct GatedFinish {
  const float* partials;         // [groups][parts][five sums, or S1, S4, S5][cols]
  const void *gate, *post_weight, *post_bias;
  void *dgate, *dscale, *dpost_weight, *dpost_bias, *dweight, *dbias;   // NULL: not wanted
  int64_t groups, gate_ld;
  int parts, cols, share;        // parts 0: there are no rows
  int shared;                    // a gradient over all groups is wanted: one workgroup of the grid's second axis, else 32 / share groups each
  int gate_grouped, scale_grouped, weight_grouped, bias_grouped;        // a gradient for each group
};
template <int ODT, bool RICH>
__global__ __launch_bounds__(1024) void cascmm_gated_norm_finish_kernel(const GatedFinish p) {
  typedef typename IoType<ODT>::T E;
  constexpr int NS = RICH ? 5 : 3;
  __shared__ float meet[NS][32][33];
  const int c = threadIdx.x & 31, r = threadIdx.x >> 5, slot = r / p.share, sub = r % p.share, at_a_time = 32 / p.share;
  const int64_t col = (int64_t)blockIdx.x * 32 + c;
  const bool in = col < p.cols;
  float total[6] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f};    // gate, scale, post_weight, post_bias, weight, bias
  const float w1 = in && p.post_weight ? (float)((const E*)p.post_weight)[col] : 1.f, b1 = in && p.post_bias ? (float)((const E*)p.post_bias)[col] : 0.f;
  auto store = [&](void* to, int64_t at, float v) {
    if (to && in) IoType<ODT>::store((E*)to + at, v);
  };
  for (int64_t base = p.shared ? 0 : (int64_t)blockIdx.y * at_a_time; base < p.groups; base += p.shared ? at_a_time : (int64_t)gridDim.y * at_a_time) {
    const int64_t group = base + slot;
    float s[NS], gate = 1.f;
#pragma unroll
    for (int k = 0; k < NS; ++k) s[k] = 0.f;
    if (in && group < p.groups) {
      if (p.gate) gate = (float)((const E*)p.gate)[group * p.gate_ld + col];
      const float* src = p.partials + group * p.parts * NS * p.cols + col;
      for (int i = sub; i < p.parts; i += p.share * 8) {   // (loads of eight parts in flight, the last part again past the end: a load under a condition is waited for by itself)
        float v[8][NS];
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
          for (int k = 0; k < NS; ++k) v[u][k] = src[((int64_t)(i + u * p.share < p.parts ? i + u * p.share : p.parts - 1) * NS + k) * p.cols];
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
          for (int k = 0; k < NS; ++k) s[k] += i + u * p.share < p.parts ? v[u][k] : 0.f;
      }
    }
    if (p.share > 1) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NS; ++k) meet[k][r][c] = s[k];
      __syncthreads();
      if (sub == 0) {
#pragma unroll
        for (int k = 0; k < NS; ++k)
          for (int i = 1; i < p.share; ++i) s[k] += meet[k][r + i][c];
      }
    }
    if (sub == 0 && group < p.groups) {
      const float s2 = RICH ? s[1] : 0.f, s3 = RICH ? s[2] : 0.f, s4 = s[NS - 2], s5 = s[NS - 1];
      const float dgate = w1 * s[0] + b1 * s2;
      if (p.gate_grouped) store(p.dgate, group * p.cols + col, dgate);
      if (p.scale_grouped) store(p.dscale, group * p.cols + col, s3);
      if (p.weight_grouped) store(p.dweight, group * p.cols + col, s4);
      if (p.bias_grouped) store(p.dbias, group * p.cols + col, s5);
      total[0] += dgate;
      total[1] += s3;
      total[2] += gate * s[0];
      total[3] += gate * s2;
      total[4] += s4;
      total[5] += s5;
    }
  }
  if (!p.shared) return;
  if (p.groups <= 1) {
    if (r != 0) return;
    void* const to[6] = {p.gate_grouped ? nullptr : p.dgate, p.scale_grouped ? nullptr : p.dscale, p.dpost_weight, p.dpost_bias, p.weight_grouped ? nullptr : p.dweight,
                         p.bias_grouped ? nullptr : p.dbias};
#pragma unroll
    for (int k = 0; k < 6; ++k) store(to[k], col, total[k]);
    return;
  }
  // over the groups, one gradient at a time (they share the first slots of the memory)
#pragma unroll
  for (int k = 0; k < 6; ++k) {
    __syncthreads();
    meet[0][r][c] = sub == 0 ? total[k] : 0.f;
    __syncthreads();
    if (r == 0) {
      float v = 0.f;
      for (int i = 0; i < 32; ++i) v += meet[0][i][c];
      if (k == 0 && !p.gate_grouped) store(p.dgate, col, v);
      if (k == 1 && !p.scale_grouped) store(p.dscale, col, v);
      if (k == 2) store(p.dpost_weight, col, v);
      if (k == 3) store(p.dpost_bias, col, v);
      if (k == 4 && !p.weight_grouped) store(p.dweight, col, v);
      if (k == 5 && !p.bias_grouped) store(p.dbias, col, v);
    }
  }
}

}  // namespace cascmm
