// Activations of an epilogue, in fp32 (the formulas: cascmm_epilogue_kernel.h).
#pragma once
#include "cascmm_common.h"

namespace cascmm {

constexpr float kLog2e = 1.4426950408889634f;
// 1 / (1 + exp(-x))
__device__ __forceinline__ float sigmoid_value(float x) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-kLog2e * x)); }
__device__ __forceinline__ float gelu_tanh_twice_u(float z) { return 1.5957691216057308f * z * __builtin_fmaf(0.044715f * z, z, 1.f); }

// act of several at a time (kinds are uniform: one branch)
template <int N> __device__ __forceinline__ void activate(float (&v)[N], int act) {
  if (act == CASCMM_ACT_GELU) {
    gelu_values(v);
  } else if (act == CASCMM_ACT_GELU_TANH) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] *= sigmoid_value(gelu_tanh_twice_u(v[e]));
  } else if (act == CASCMM_ACT_SILU) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] *= sigmoid_value(v[e]);
  } else if (act == CASCMM_ACT_RELU) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = v[e] < 0.f ? 0.f : v[e];
  }
}

// The epilogue of four adjacent columns z of row m, from column n on: z to preact, act(z) + residual in its place (vec: whole quads of every row).
// Residual and result may not be the same memory: other lanes may have written by then.
template <int IODT>
__device__ __forceinline__ void quad_epilogue(f32x4& s, const void* residual, int64_t ldr, void* preact, int64_t ldp, int act, int m, int n, int N, bool vec) {
  typedef IoType<IODT> Io;
  typedef typename Io::T E;
  typedef E e4 __attribute__((ext_vector_type(4)));
  f32x4 r = {0.f, 0.f, 0.f, 0.f};
  if (residual) {
    const E* src = (const E*)residual + (int64_t)m * ldr + n;
    if (vec) {
      r = __builtin_convertvector(*(const e4*)src, f32x4);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = n + e < N ? Io::load(src + e) : 0.f;
    }
  }
  if (preact) {
    E* dst = (E*)preact + (int64_t)m * ldp + n;
    if (vec) {
      *(e4*)dst = __builtin_convertvector(s, e4);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < N) Io::store(dst + e, s[e]);
    }
  }
  float v[4] = {s[0], s[1], s[2], s[3]};
  activate(v, act);
#pragma unroll
  for (int e = 0; e < 4; ++e) s[e] = v[e] + r[e];
}

}  // namespace cascmm
