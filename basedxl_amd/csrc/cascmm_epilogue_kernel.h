// What follows a product in a Linear layer:  y = act(z) + residual,  z = A . B + bias,  as a pass of its own behind kernels that store z, and
// its backward pass:  dz = dy act'(z),  dbias = sum over rows of dz.  fp32 between a load and a store whatever the elements are.
//
//   relu       max(z, 0)                                    z > 0
//   gelu       z Phi(z)                                     Phi(z) + z phi(z)
//   gelu_tanh  z s(2 u), u = sqrt(2 / pi) (z + 0.044715 z^3)   s + 2 z s (1 - s) u',  s = s(2 u)
//   silu       z s(z)                                       s (1 + z (1 - s)),  s(x) = 1 / (1 + exp(-x))
//
// (z s(2 u) is z (1 + tanh u) / 2 without the cancellation for z < 0.)  Slopes are taken at z clamped to where they are 0 and 1 to fp32's
// last bit, so that no intermediate value overflows; a NaN stays one.
//
// Bound by memory: 16 bytes a load, rows of any alignment.
#pragma once
#include <type_traits>

#include "cascmm_activation.h"
#include "cascmm_norm_kernel.h"

namespace cascmm {

__device__ __forceinline__ float clamped(float z, float most) { return z > most ? most : z < -most ? -most : z; }
// d[e] *= act'(z[e])
template <int N> __device__ __forceinline__ void times_slope(float (&d)[N], const float (&z)[N], int act) {
  if (act == CASCMM_ACT_GELU) {
    // With x = |z|: Phi(-x) = 2^(P(x) - 1) as in gelu_values, phi(x) = exp(-x^2 / 2) / sqrt(2 pi), and the slope is u = Phi(-x) - x phi(x) for z < 0, 1 - u
    // for z > 0.  (x is held down in the product only, where an infinite one would meet phi = 0.)
    float t[N];
#pragma unroll
    for (int e = 0; e < N; ++e) t[e] = kGeluFit[0];
#pragma unroll
    for (int i = 1; i < 10; ++i) {
#pragma unroll
      for (int e = 0; e < N; ++e) t[e] = __builtin_fmaf(t[e], __builtin_fabsf(z[e]), kGeluFit[i]);
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float x = __builtin_fabsf(z[e]);
      const float tail = __builtin_amdgcn_exp2f(__builtin_fmaf(t[e], x, -1.f));
      const float density = __builtin_amdgcn_exp2f(__builtin_fmaf(x * x, -0.5f * kLog2e, -1.3257480647361593f));   // (log2 of 1 / sqrt(2 pi))
      const float u = __builtin_fmaf(-__builtin_fminf(x, 1.0e4f), density, tail);
      d[e] *= z[e] > 0.f ? 1.f - u : u;
    }
  } else if (act == CASCMM_ACT_GELU_TANH) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float x = clamped(z[e], 10.f), q = __builtin_amdgcn_exp2f(-kLog2e * gelu_tanh_twice_u(x)), s = __builtin_amdgcn_rcpf(1.f + q);
      // (1 - s = q s)
      d[e] *= __builtin_fmaf(x * s * (q * s), 1.5957691216057308f * __builtin_fmaf(0.134145f * x, x, 1.f), s);
    }
  } else if (act == CASCMM_ACT_SILU) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float x = clamped(z[e], 80.f), q = __builtin_amdgcn_exp2f(-kLog2e * x), s = __builtin_amdgcn_rcpf(1.f + q);
      d[e] *= s * __builtin_fmaf(x, q * s, 1.f);
    }
  } else if (act == CASCMM_ACT_RELU) {
#pragma unroll
    for (int e = 0; e < N; ++e) d[e] = z[e] <= 0.f ? 0.f : d[e];
  }
}

// dst [rows][cols] = act(src) + residual (NULL: nothing; ldr 0: one row for all).  src may be dst.  A thread takes a chunk of 16 bytes; chunks are
// counted in 32 bits (checked by the host).
template <int IODT, bool TINY>
__global__ __launch_bounds__(256) void cascmm_epilogue_kernel(const void* src, int64_t lds, const void* residual, int64_t ldr, void* dst, int64_t ldd, int cols,
                                                             unsigned per_row, unsigned total, int act) {
  typedef NormRow<IODT, TINY> R;
  typedef typename R::E E;
  typedef typename R::chunk chunk;
  const unsigned i = blockIdx.x * 256u + threadIdx.x;
  if (i >= total) return;
  const unsigned row = i / per_row;
  const int col = (int)(i - row * per_row) * R::VEC;
  const chunk z = R::load_settled((const E*)src + (int64_t)row * lds, col, cols);
  chunk r;
  if (residual) r = R::load_settled((const E*)residual + (int64_t)row * ldr, col, cols);
  float v[R::VEC];
#pragma unroll
  for (int e = 0; e < R::VEC; ++e) v[e] = (float)z[e];
  activate(v, act);
  if (residual) {
#pragma unroll
    for (int e = 0; e < R::VEC; ++e) v[e] += (float)r[e];
  }
  chunk y;
#pragma unroll
  for (int e = 0; e < R::VEC; ++e) y[e] = (E)v[e];
  R::store((E*)dst + (int64_t)row * ldd, col, cols, y);
}

// dz = dy act'(z) (dz NULL: not wanted; act none: z is not read) and, with partials, the workgroup's sums over its rows of dz for its columns at
// partials[blockIdx.y].  LANES lanes side by side on a row, rows gridDim.y workgroups apart, AHEAD of them at a time and the next ones asked for before these are
// looked at; the sums are of dz as it is before it is rounded.
// z and dz are of the elements' type: in 16 bits both are rounded on their way between kernels.  Of the gradients' mean error, 1.45 times that of fp32 z and dz (8192 x
// 640 x 2560 bf16 2.43e-3 for 1.66e-3), dz's rounding makes nearly all, the slope at a rounded z 6e-4.  fp32 dz would want products of two terms, twice their matrix
// work (some 70 us more there); fp32 z 42 MB more written and read, 16 us.
// Measured (graph replay): 8192 x 2560 bf16, gelu, dz 29.5 us (4.3 TB/s; the slope is some 30 instructions an element, 18 us of every SIMD), with dbias, whose
// sums are a second kernel, 34.0; 8192 x 640 fp32 12.9 (4.9 TB/s) and 16.8.
struct SlopeParams {
  const void *dy, *z;
  void* dz;
  float* partials;
  int64_t lddy, ldz, lddz, rows;
  int cols, act;
};
// Workgroup `band` (of columns), `part` (of `parts` that share the rows); lds: kSlopeLds bytes.
constexpr int kSlopeLds = 256 * 16 * 2;
template <int IODT, int LANES, bool TINY>
__device__ __forceinline__ void slope_rows(const SlopeParams& p, int band, int part, int parts, unsigned char* lds) {
  typedef NormRow<IODT, TINY> R;
  typedef typename R::E E;
  typedef typename R::chunk chunk;
  constexpr int VEC = R::VEC, GROUPS = 256 / LANES, AHEAD = 4;
  const void *dy = p.dy, *z = p.z;
  void* dz = p.dz;
  float* partials = p.partials;
  int64_t lddy = p.lddy, ldz = p.ldz, lddz = p.lddz, rows = p.rows;
  int cols = p.cols, act = p.act;
  asm volatile("" : "+s"(dy), "+s"(lddy), "+s"(z), "+s"(ldz), "+s"(dz), "+s"(lddz), "+s"(rows), "+s"(cols), "+s"(act));   // (requested together)
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int col = (band * LANES + lane) * VEC;
  const int64_t stride = (int64_t)parts * GROUPS;
  float sums[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) sums[e] = 0.f;
  struct Rows { chunk d[AHEAD], x[AHEAD]; };
  auto fetch = [&](Rows& to, int64_t row) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int64_t at = row + u * stride;
      if (at >= rows) break;
      to.d[u] = R::load((const E*)dy + at * lddy, col, cols);
      if (act) to.x[u] = R::load((const E*)z + at * ldz, col, cols);
    }
  };
  if (col < cols) {
    Rows next;
    int64_t row = (int64_t)part * GROUPS + (LANES == 64 ? __builtin_amdgcn_readfirstlane(group) : group);
    if (row < rows) fetch(next, row);
    while (row < rows) {
      Rows cur = next;
      const int64_t first = row;
      row += AHEAD * stride;
      if (row < rows) fetch(next, row);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int64_t at = first + u * stride;
        if (at >= rows) break;
        float g[VEC], v[VEC];
        cur.d[u] = R::settle(cur.d[u], col, cols);
        if (act) cur.x[u] = R::settle(cur.x[u], col, cols);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          g[e] = (float)cur.d[u][e];
          v[e] = act ? (float)cur.x[u][e] : 0.f;
        }
        times_slope(g, v, act);
        chunk out;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          sums[e] += g[e];
          out[e] = (E)g[e];
        }
        if (dz) R::store((E*)dz + at * lddz, col, cols, out);
      }
    }
  }
  if (!partials) return;
  static_assert(GROUPS * LANES * VEC * (int)sizeof(float) <= kSlopeLds, "");
  float(*meet)[LANES * VEC] = (float(*)[LANES * VEC])lds;
#pragma unroll
  for (int e = 0; e < VEC; ++e) meet[group][e * LANES + lane] = sums[e];
  __syncthreads();
  for (int i = threadIdx.x; i < LANES * VEC; i += 256) {
    const int64_t c = ((int64_t)band * LANES + i % LANES) * VEC + i / LANES;
    if (c >= cols) continue;
    float s = 0.f;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) s += meet[g][i];
    partials[(int64_t)part * cols + c] = s;
  }
}

template <int IODT, int LANES, bool TINY>
__global__ __launch_bounds__(256) void cascmm_epilogue_backward_kernel(const SlopeParams p) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[kSlopeLds];
  slope_rows<IODT, LANES, TINY>(p, (int)blockIdx.x, (int)blockIdx.y, (int)gridDim.y, lds);
}

// out [cols][rows] = x [rows][cols] transposed; E: an unsigned type of the elements' size.  64 x 64 elements a workgroup through LDS: 16 bytes a load
// along the rows of x and a store along the rows of out.  Rows of the tile are an odd number of dwords apart in LDS, so that the eight (sixteen)
// groups of rows that the lanes of a store read start on banks of their own.
// Measured (graph replay): 8192 x 2560 bf16 13.6 - 16.4 us (5.1 - 6.2 TB/s, part of it from the Infinity Cache), 8192 x 640 fp32 8.1 (5.2 TB/s), 333 x 211 fp16 3.0.
struct TransposeParams {
  const void* x;
  void* out;
  int64_t ldx, ldo;
  int rows, cols;
  unsigned across, tiles;   // tiles side by side over the columns, all of them (0: nothing to do)
};
constexpr int kTransposeLds = 64 * 65 * 4;
template <typename E> __device__ __forceinline__ void transpose_tile(const TransposeParams& p, unsigned at, unsigned char* lds) {
  const E* __restrict__ x = (const E*)p.x;
  E* __restrict__ out = (E*)p.out;
  const int64_t ldx = p.ldx, ldo = p.ldo;
  const int rows = p.rows, cols = p.cols;
  constexpr int VEC = 16 / (int)sizeof(E), PER = 64 / VEC, PITCH = sizeof(E) == 2 ? 66 : 65, DW = 4 / (int)sizeof(E);
  typedef E chunk __attribute__((ext_vector_type(VEC), aligned(sizeof(E))));
  static_assert(64 * PITCH * (int)sizeof(E) <= kTransposeLds, "");
  E* tile = (E*)lds;
  const int r0 = (int)(at / p.across) * 64, c0 = (int)(at % p.across) * 64;
#pragma unroll
  for (int i = threadIdx.x; i < 64 * PER; i += 256) {
    const int r = i / PER, c = i % PER * VEC;
    chunk v;
    if (r0 + r < rows && c0 + c + VEC <= cols) {
      v = *(const chunk*)(x + (int64_t)(r0 + r) * ldx + c0 + c);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = r0 + r < rows && c0 + c + e < cols ? x[(int64_t)(r0 + r) * ldx + c0 + c + e] : (E)0;
    }
    // (dword by dword: the pitch leaves no rows on 16 bytes)
    typedef E pair __attribute__((ext_vector_type(DW)));
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      pair w;
#pragma unroll
      for (int e = 0; e < DW; ++e) w[e] = v[d * DW + e];
      *(pair*)(tile + r * PITCH + c + d * DW) = w;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = threadIdx.x; i < 64 * PER; i += 256) {
    const int c = i / PER, r = i % PER * VEC;
    if (c0 + c >= cols) continue;
    chunk v;
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = tile[(r + e) * PITCH + c];
    E* to = out + (int64_t)(c0 + c) * ldo + r0 + r;
    if (r0 + r + VEC <= rows) {
      *(chunk*)to = v;
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (r0 + r + e < rows) to[e] = v[e];
    }
  }
}
// two of them in one launch
template <typename E> __global__ __launch_bounds__(256) void cascmm_transpose_kernel(const TransposeParams a, const TransposeParams b) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[kTransposeLds];
  if (blockIdx.x < a.tiles) return transpose_tile<E>(a, blockIdx.x, lds);
  transpose_tile<E>(b, blockIdx.x - a.tiles, lds);
}

// Slopes and two transpositions side by side in one launch: what the gradients of a product want before its two products run.  The first workgroups are
// the slopes' (bands x parts of them), then the tiles of the one operand, then the other's.  8192 x 640 x 2560 bf16, gelu, with the finishing kernel: 38 us,
// one launch each 45; without slopes the kernel above, which more of fit on a CU (8192 x 2560 16.4 us, in this one 18.2).
template <int IODT, int LANES, bool TINY>
__global__ __launch_bounds__(256) void cascmm_epilogue_operands_kernel(const SlopeParams p, unsigned bands, unsigned parts, const TransposeParams a, const TransposeParams b) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[kSlopeLds > kTransposeLds ? kSlopeLds : kTransposeLds];
  typedef typename std::conditional<sizeof(typename IoType<IODT>::T) == 4, unsigned, unsigned short>::type E;
  unsigned at = blockIdx.x;
  if (at < bands * parts) return slope_rows<IODT, LANES, TINY>(p, (int)(at % bands), (int)(at / bands), (int)parts, lds);
  at -= bands * parts;
  if (at < a.tiles) return transpose_tile<E>(a, at, lds);
  transpose_tile<E>(b, at - a.tiles, lds);
}

}  // namespace cascmm
