// Host side of the epilogue of a product, shared by the translation units that launch it.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cascmm {

// y = act(z) + residual behind a product z (cascmm_epilogue_kernel.h); ldr 0: one row for all
struct Epilogue {
  int act;
  const void* residual;
  int64_t ldr;
  void* preact;   // z too (or NULL)
  int64_t ldp;
  int64_t ldc;    // of the result (a Problem's own is what its kernel is chosen for: the product may store z instead)
};
// dst = act(src) + residual as a pass of its own (src may be dst)
int launch_epilogue(const void* src, int64_t lds, const void* residual, int64_t ldr, void* dst, int64_t ldd, int64_t rows, int64_t cols, int act, int dtype,
                    hipStream_t stream);

}  // namespace cascmm
