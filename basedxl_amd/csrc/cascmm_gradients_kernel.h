// The norm of many tensors taken together, and their scaling by it (gfx950).
//
//   norm = (sum over all elements of |g|^p)^(1/p), p = 1, 2, or max|g|;   factor = min(1, max_norm / (norm + 1e-6));   out = g factor
//
// Sums are fp64 from the first square on: nothing overflows or vanishes between 1e-45 and 3e38, and the norm is good to fp32's last bit whatever
// the number of elements.  The tensors are cut into chunks, one to a workgroup; each chunk's sum goes to a place of its own and the places are added
// in a fixed order, so that the same call gives the same bits.  Results are rounded once, from fp32.  A factor below fp32's normal numbers (gradients of 1e38 and more) would lose its
// bits, or be zero where results are not: it is multiplied in fp64 then.
//
// Bound by memory: the gradients are read for the norm and again to be scaled, 12 bytes an fp32 element with the store.  The tensors' addresses travel in the
// kernels' arguments, as many to a launch as fit: there is no table in memory to be kept, copied or outlived by a recorded graph.
//
// Measured (us among other calls): 786 M fp32 gradients in 400 tensors 1835 (the first pass at 5.9 TB/s, the second at 5.1; a large copy 4.9), 30 M bf16 into fp32 60.5, the 37 thousand
// of 30 small tensors 11.7, two launches of 4 and what the host takes.
#pragma once
#include "cascmm_common.h"

namespace cascmm {

constexpr int kGradTensors = 96;          // of one launch (arguments of 2.7 KB)
constexpr int64_t kGradChunk = 4096;      // elements of a chunk, at least
constexpr int kGradMerged = 2560;         // partial sums that every workgroup of the second pass adds itself
struct GradBatch {
  int64_t chunk;
  double* parts;        // of all chunks of the call
  double* head;         // the factor
  double max_norm;
  float* norm;
  unsigned part0, all_parts;   // the first chunk of this launch; of all launches
  int count, type;      // type: 0 max, 1, 2
  int merged;           // second pass: the partial sums are added by each workgroup
  const void* g[kGradTensors];
  void* out[kGradTensors];
  int64_t n[kGradTensors];
  unsigned first[kGradTensors];        // chunk of this launch that a tensor begins with
  unsigned char dtype[kGradTensors], out_dtype[kGradTensors];
};

template <int DT> struct GradRow {
  typedef typename IoType<DT>::T E;
  static constexpr int VEC = 16 / (int)sizeof(E);
  typedef E chunk __attribute__((ext_vector_type(VEC), aligned(sizeof(E))));   // (elements, not 16 bytes, are aligned)
};

// the tensor that a launch's chunk belongs to: as many begin at or before it
__device__ __forceinline__ int grad_tensor(const GradBatch& b, unsigned at) {
  const int lane = threadIdx.x & 63;
  int found = 0;
#pragma unroll
  for (int i = 0; i < kGradTensors; i += 64) {
    const int t = i + lane;
    found += __builtin_popcountll(__builtin_amdgcn_ballot_w64(t < b.count && t < kGradTensors && b.first[t < kGradTensors ? t : 0] <= at));
  }
  return __builtin_amdgcn_readfirstlane(found - 1);
}

// NaN stays, in either argument
__device__ __forceinline__ double grad_larger(double a, double b) { return b > a || b != b ? (a != a ? a : b) : a; }
__device__ __forceinline__ double grad_join(double a, double b, int type) { return type ? a + b : grad_larger(a, b); }

// a workgroup's values joined in a fixed order, the result in thread 0
template <int NT> __device__ __forceinline__ double grad_meet(double v, int type, double* slots) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = grad_join(v, __shfl_xor(v, off, 64), type);
  if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
  __syncthreads();
  v = slots[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) v = grad_join(v, slots[w], type);
  return v;
}

template <int DT, int TYPE> __device__ __forceinline__ double grad_sum(const void* p, int64_t at, int64_t len) {
  typedef GradRow<DT> R;
  constexpr int VEC = R::VEC, NT = 256, DEEP = 4;
  const typename R::E* src = (const typename R::E*)p + at;
  double acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) acc[e] = 0;
  auto fold = [&](int e, float x) {
    const double d = (double)__builtin_fabsf(x);
    if constexpr (TYPE == 2) acc[e] = __builtin_fma(d, d, acc[e]);
    else acc[e] = grad_join(acc[e], d, TYPE);
  };
  const int64_t chunks = len / VEC;
  int64_t i = threadIdx.x;
  for (; i + (DEEP - 1) * NT < chunks; i += DEEP * NT) {
    typename R::chunk v[DEEP];
#pragma unroll
    for (int u = 0; u < DEEP; ++u) v[u] = *(const typename R::chunk*)(src + (i + u * NT) * VEC);
#pragma unroll
    for (int u = 0; u < DEEP; ++u)
#pragma unroll
      for (int e = 0; e < VEC; ++e) fold(e, (float)v[u][e]);
  }
  for (; i < chunks; i += NT) {
    const typename R::chunk v = *(const typename R::chunk*)(src + i * VEC);
#pragma unroll
    for (int e = 0; e < VEC; ++e) fold(e, (float)v[e]);
  }
  if (threadIdx.x < len - chunks * VEC) fold(0, (float)src[chunks * VEC + threadIdx.x]);
#pragma unroll
  for (int e = 1; e < VEC; ++e) acc[0] = grad_join(acc[0], acc[e], TYPE);
  return acc[0];
}
template <int DT> __device__ __forceinline__ double grad_sum_of(const void* p, int64_t at, int64_t len, int type) {
  return type == 2 ? grad_sum<DT, 2>(p, at, len) : type == 1 ? grad_sum<DT, 1>(p, at, len) : grad_sum<DT, 0>(p, at, len);
}

// the first pass: one chunk's part of the sum (of the maximum)
template <int UNUSED> __global__ __launch_bounds__(256) void cascmm_gradient_parts_kernel(const GradBatch b) {
  __shared__ double slots[4];
  const int t = grad_tensor(b, blockIdx.x);
  const int64_t at = (int64_t)(blockIdx.x - b.first[t]) * b.chunk, left = b.n[t] - at, len = left < b.chunk ? left : b.chunk;
  const int dt = b.dtype[t];
  double v = dt == CASCMM_DT_F32   ? grad_sum_of<CASCMM_DT_F32>(b.g[t], at, len, b.type)
             : dt == CASCMM_DT_F16 ? grad_sum_of<CASCMM_DT_F16>(b.g[t], at, len, b.type)
                                   : grad_sum_of<CASCMM_DT_BF16>(b.g[t], at, len, b.type);
  v = grad_meet<256>(v, b.type, slots);
  if (threadIdx.x == 0) b.parts[b.part0 + blockIdx.x] = v;
}

// norm and factor from all parts, in every thread of a workgroup of NT
template <int NT> __device__ __forceinline__ double grad_factor(const double* parts, unsigned count, int type, double max_norm, double* slots, double& norm) {
  double v = 0;
  for (unsigned i = threadIdx.x; i < count; i += NT) v = grad_join(v, parts[i], type);
  v = grad_meet<NT>(v, type, slots);
  norm = type == 2 ? __builtin_sqrt(v) : v;
  const double f = max_norm / (norm + 1e-6);
  return f > 1.0 ? 1.0 : f;   // (a NaN stays one)
}
template <int UNUSED>
__global__ __launch_bounds__(1024) void cascmm_gradient_norm_kernel(const double* __restrict__ parts, unsigned count, int type, double max_norm, float* norm_out, double* head) {
  __shared__ double slots[16];
  double norm;
  const double f = grad_factor<1024>(parts, count, type, max_norm, slots, norm);
  if (threadIdx.x == 0) {
    *norm_out = (float)norm;
    *head = f;
  }
}

template <int DT, int ODT> __device__ __forceinline__ void grad_scale(const void* p, void* q, int64_t at, int64_t len, float f) {
  typedef GradRow<DT> R;
  typedef typename IoType<ODT>::T O;
  constexpr int VEC = R::VEC, NT = 256, DEEP = 4;
  typedef O ochunk __attribute__((ext_vector_type(VEC), aligned(sizeof(O))));
  const typename R::E* src = (const typename R::E*)p + at;
  O* dst = (O*)q + at;
  auto put = [&](int64_t i, typename R::chunk v) {
    ochunk o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = (O)((float)v[e] * f);
    *(ochunk*)(dst + i * VEC) = o;
  };
  const int64_t chunks = len / VEC;
  int64_t i = threadIdx.x;
  for (; i + (DEEP - 1) * NT < chunks; i += DEEP * NT) {
    typename R::chunk v[DEEP];
#pragma unroll
    for (int u = 0; u < DEEP; ++u) v[u] = *(const typename R::chunk*)(src + (i + u * NT) * VEC);
#pragma unroll
    for (int u = 0; u < DEEP; ++u) put(i + u * NT, v[u]);
  }
  for (; i < chunks; i += NT) put(i, *(const typename R::chunk*)(src + i * VEC));
  if (threadIdx.x < len - chunks * VEC) {
    const int64_t e = chunks * VEC + threadIdx.x;
    dst[e] = (O)((float)src[e] * f);
  }
}

// ... by a factor below fp32's normal numbers: of any types, an element at a time
__device__ __forceinline__ void grad_scale_finely(const GradBatch& b, int t, int64_t at, int64_t len, double f) {
  const int dt = b.dtype[t];
  for (int64_t i = at + threadIdx.x; i < at + len; i += 256) {
    const float g = dt == CASCMM_DT_F32 ? ((const float*)b.g[t])[i] : dt == CASCMM_DT_F16 ? (float)((const _Float16*)b.g[t])[i] : (float)((const __bf16*)b.g[t])[i];
    const float o = (float)((double)g * f);
    if (b.out_dtype[t] == CASCMM_DT_F32) ((float*)b.out[t])[i] = o;
    else if (b.out_dtype[t] == CASCMM_DT_F16) ((_Float16*)b.out[t])[i] = (_Float16)o;
    else ((__bf16*)b.out[t])[i] = (__bf16)o;
  }
}

// the second pass.  Gradients that stay where they are and are not clipped are not touched.
template <int UNUSED> __global__ __launch_bounds__(256) void cascmm_gradient_scale_kernel(const GradBatch b) {
  __shared__ double slots[4];
  const int t = grad_tensor(b, blockIdx.x);
  double factor;
  if (b.merged) {
    double norm;
    factor = grad_factor<256>(b.parts, b.all_parts, b.type, b.max_norm, slots, norm);
    if (b.part0 + blockIdx.x == 0 && threadIdx.x == 0) *b.norm = (float)norm;
  } else {
    factor = *b.head;
  }
  const float f = (float)factor;
  if (f == 1.f && b.out[t] == b.g[t]) return;
  const int64_t at = (int64_t)(blockIdx.x - b.first[t]) * b.chunk, left = b.n[t] - at, len = left < b.chunk ? left : b.chunk;
  if (factor < 0x1p-126) return grad_scale_finely(b, t, at, len, factor);
  const int dt = b.dtype[t], odt = b.out_dtype[t];
  if (dt == CASCMM_DT_F32) grad_scale<CASCMM_DT_F32, CASCMM_DT_F32>(b.g[t], b.out[t], at, len, f);
  else if (dt == CASCMM_DT_F16 && odt == CASCMM_DT_F16) grad_scale<CASCMM_DT_F16, CASCMM_DT_F16>(b.g[t], b.out[t], at, len, f);
  else if (dt == CASCMM_DT_F16) grad_scale<CASCMM_DT_F16, CASCMM_DT_F32>(b.g[t], b.out[t], at, len, f);
  else if (odt == CASCMM_DT_BF16) grad_scale<CASCMM_DT_BF16, CASCMM_DT_BF16>(b.g[t], b.out[t], at, len, f);
  else grad_scale<CASCMM_DT_BF16, CASCMM_DT_F32>(b.g[t], b.out[t], at, len, f);
}

}  // namespace cascmm
