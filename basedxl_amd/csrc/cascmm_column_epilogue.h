// The epilogue of a product (cascmm_epilogue.h) in the stores of the fp32 kernels whose lanes hold a column of a block: z to preact, act(z) + residual.
// A load or store of one register is two whole 128-byte pieces of rows.  The residual of a block is asked for while something else is at hand (the sums
// of the waves, the block before), all its rows at once.
// Every offset is a lane's own, so that rows past the last one and columns past the edge fall beyond the descriptors' ends: loads give zeros, stores are
// dropped.  (Host-checked: a tile's rows span less than 2 GiB in each of the tensors.)
#pragma once
#include "cascmm_activation.h"
#include "cascmm_tile_kernel.h"

namespace cascmm {

// what the launch functions hand to kernels that have parameters of their own
struct EpilogueArgs {
  const void* residual;
  void* preact;
  int64_t ldr, ldp;
  int act;
};
__host__ __device__ inline EpilogueArgs epilogue_args(const GroupParams& p) { return {p.residual, p.preact, p.ldr, p.ldp, p.act}; }

struct ColumnEpilogue {
  i32x4 rr, rp, rc;
  int ldr, ldp, ldc, act;   // (bytes)
  bool res, pre;
  // rows from row0 and columns from col0 on
  __device__ __forceinline__ ColumnEpilogue(const EpilogueArgs& a, float* C, int64_t ldc_, int M, int N, int64_t row0, int col0) {
    res = a.residual != nullptr;
    pre = a.preact != nullptr;
    act = a.act;
    ldr = (int)a.ldr * 4;
    ldp = (int)a.ldp * 4;
    ldc = (int)ldc_ * 4;
    auto rows_of = [&](const void* base, int64_t ld) {
      const int64_t bytes = ((M - 1 - row0) * ld + (N - col0)) * 4;
      return make_rsrc((const float*)base + row0 * ld + col0, bytes < 0 ? 0 : bytes);
    };
    rr = rows_of(a.residual, a.ldr);
    rp = rows_of(a.preact, a.ldp);
    rc = rows_of(C, ldc_);
  }
  // (AUX: the cache policy of the kernel's own stores)
  // Register e of a lane is row `row` + 8 (e / 4) + e % 4 (+ the lane's own `up`), all of column `col` (both relative; inside: it exists)
  static __device__ __forceinline__ int at(int e) { return 8 * (e >> 2) + (e & 3); }
  template <int R> __device__ __forceinline__ void ask(float (&r)[R], int row, int up, int col, bool inside) const {
    if (!res) return;
    const unsigned base = inside ? (unsigned)(up * ldr + col * 4) : 0x7FFFFFFFu;
#pragma unroll
    for (int e = 0; e < R; ++e) r[e] = llvm_raw_buffer_load_f32(rr, (int)(base + (unsigned)((row + at(e)) * ldr)), 0, 0);
  }
  template <int AUX, int R> __device__ __forceinline__ void store(float (&z)[R], const float (&r)[R], int row, int up, int col, bool inside) const {
    if (pre) {
      const unsigned base = inside ? (unsigned)(up * ldp + col * 4) : 0x7FFFFFFFu;
#pragma unroll
      for (int e = 0; e < R; ++e) llvm_raw_buffer_store_f32(z[e], rp, (int)(base + (unsigned)((row + at(e)) * ldp)), 0, AUX);
    }
    activate(z, act);
    if (res) {
#pragma unroll
      for (int e = 0; e < R; ++e) z[e] += r[e];
    }
    const unsigned base = inside ? (unsigned)(up * ldc + col * 4) : 0x7FFFFFFFu;
#pragma unroll
    for (int e = 0; e < R; ++e) llvm_raw_buffer_store_f32(z[e], rc, (int)(base + (unsigned)((row + at(e)) * ldc)), 0, AUX);
  }
};

}  // namespace cascmm
