// The launches of the kernels in cascmm_gated_kernel.h, one translation unit for each element type.
#pragma once
#include <algorithm>

#include "cascmm_gated_kernel.h"

namespace cascmm {

// The lanes of a row and the elements of a lane: sixteen lanes take rows of up to 256 columns, a wave up to 2048 (in the backward pass, which holds the sums beside a
// row, 1536; with four waves on rows of 1025 to 1536 columns 32768 x 1280 bf16 takes 151 us for 112), four of them up to 8192 (backward 6144: beyond, five sums do not fit beside a row); none: longer rows, and rows shorter than 16 bytes
struct GatedShape { int lanes, values; };
inline GatedShape gated_shape(int64_t cols, bool backward, int64_t chunk) {
  const auto fit = [&](int lanes) { return (int)std::min<int64_t>((cols + 8 * lanes - 1) / (8 * lanes) * 8, 1 << 20); };
  if (cols < chunk) return {0, 0};
  if (fit(16) <= 16) return {16, fit(16)};
  if (fit(64) <= (backward ? 24 : 32)) return {64, fit(64)};
  if (fit(256) <= (backward ? 24 : 32)) return {256, fit(256)};
  return {0, 0};
}
// Workgroups of a group: in all four on a CU forward (as layer norm's), backward one, as many as the registers of the longer rows leave room for (32768 x 1280 bf16, gated and
// modulated, with the sums' kernel 112 us; 512 workgroups 121, 768 127, 1024 130; 8 x 1024 x 1280 fp32 57, 61, 67, 70; 32768 x 1024 bf16 85, 86, 97, 93), at least one to a group
inline void gated_parts(int64_t groups, int64_t group_rows, int lanes, bool backward, int& parts, int64_t& part_rows) {
  const int64_t at_a_time = lanes ? 256 / lanes * (backward ? 2 : 1) : 16, most = !lanes ? 512 : !backward ? 1024 : lanes >= 64 ? 256 : 1024;
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>((group_rows + at_a_time - 1) / at_a_time, most / std::max<int64_t>(groups, 1)));
  part_rows = std::max<int64_t>(1, (group_rows + want - 1) / want);
  parts = (int)std::max<int64_t>(1, (group_rows + part_rows - 1) / part_rows);
}

template <int IODT, bool POST, bool RICH> static hipError_t gated_forward_of(const GatedParams& p, unsigned groups, hipStream_t s) {
  hipError_t err = hipSuccess;
  const GatedShape f = gated_shape(p.cols, false, NormRow<IODT>::VEC);
  const dim3 grid(groups * (unsigned)p.parts);
#define GATED_CASE(LPR, NV) \
  case (LPR) * 100 + (NV): CASCMM_LAUNCH(err, (cascmm_gated_norm_kernel<IODT, NV, LPR, POST, RICH>), grid, dim3(256), 0, s, p); break
  switch (f.lanes * 100 + f.values) {
    GATED_CASE(16, 8);
    GATED_CASE(16, 16);
    GATED_CASE(64, 8);
    GATED_CASE(64, 16);
    GATED_CASE(64, 24);
    GATED_CASE(64, 32);
    GATED_CASE(256, 16);
    GATED_CASE(256, 24);
    GATED_CASE(256, 32);
    default: return hipErrorInvalidValue;
  }
#undef GATED_CASE
  return err;
}
template <int IODT, bool POST, bool RICH> static hipError_t gated_backward_of(const GatedParams& p, unsigned groups, hipStream_t s) {
  hipError_t err = hipSuccess;
  const GatedShape f = gated_shape(p.cols, true, NormRow<IODT>::VEC);
  const dim3 grid(groups * (unsigned)p.parts);
#define GATED_CASE(LPR, NV) \
  case (LPR) * 100 + (NV): CASCMM_LAUNCH(err, (cascmm_gated_norm_backward_kernel<IODT, NV, LPR, POST, RICH>), grid, dim3(256), 0, s, p); break
  switch (f.lanes * 100 + f.values) {
    GATED_CASE(16, 8);
    GATED_CASE(16, 16);
    GATED_CASE(64, 8);
    GATED_CASE(64, 16);
    GATED_CASE(64, 24);
    GATED_CASE(256, 8);
    GATED_CASE(256, 16);
    GATED_CASE(256, 24);
    default: return hipErrorInvalidValue;
  }
#undef GATED_CASE
  return err;
}

template <int IODT> hipError_t gated_forward(const GatedParams& p, int64_t groups, bool post, bool rich, hipStream_t s) {
  hipError_t err = hipSuccess;
  if (gated_shape(p.cols, false, NormRow<IODT>::VEC).lanes == 0) {
    const dim3 grid((unsigned)std::min<int64_t>(p.rows, 1 << 20));
    CASCMM_LAUNCH(err, (p.cols < NormRow<IODT>::VEC ? cascmm_gated_norm_wide_kernel<IODT, true> : cascmm_gated_norm_wide_kernel<IODT, false>), grid, dim3(kGatedWide), 0, s, p, post);
    return err;
  }
  if (post) return rich ? gated_forward_of<IODT, true, true>(p, (unsigned)groups, s) : gated_forward_of<IODT, true, false>(p, (unsigned)groups, s);
  return rich ? gated_forward_of<IODT, false, true>(p, (unsigned)groups, s) : gated_forward_of<IODT, false, false>(p, (unsigned)groups, s);
}
template <int IODT> hipError_t gated_backward(const GatedParams& p, int64_t groups, bool post, bool rich, hipStream_t s) {
  hipError_t err = hipSuccess;
  if (gated_shape(p.cols, true, NormRow<IODT>::VEC).lanes == 0) {
    const dim3 grid((unsigned)std::min<int64_t>(p.rows, 1 << 20));
    CASCMM_LAUNCH(err, (p.cols < NormRow<IODT>::VEC ? cascmm_gated_norm_backward_wide_kernel<IODT, true> : cascmm_gated_norm_backward_wide_kernel<IODT, false>), grid, dim3(kGatedWide), 0, s,
                  p, post);
    if (p.partials && err == hipSuccess)
      CASCMM_LAUNCH(err, cascmm_gated_norm_sums_kernel<IODT>, dim3((unsigned)((p.cols + 255) / 256), (unsigned)std::min<int64_t>(groups * p.parts, 4096)), dim3(256), 0, s, p, groups * p.parts, post);
    return err;
  }
  if (post) return rich ? gated_backward_of<IODT, true, true>(p, (unsigned)groups, s) : gated_backward_of<IODT, true, false>(p, (unsigned)groups, s);
  return rich ? gated_backward_of<IODT, false, true>(p, (unsigned)groups, s) : gated_backward_of<IODT, false, false>(p, (unsigned)groups, s);
}
template <int ODT> hipError_t gated_finish(const GatedFinish& p, bool rich, hipStream_t s) {
  hipError_t err = hipSuccess;
  const int64_t turns = (p.groups + 32 / p.share - 1) / (32 / p.share);
  CASCMM_LAUNCH(err, (rich ? cascmm_gated_norm_finish_kernel<ODT, true> : cascmm_gated_norm_finish_kernel<ODT, false>), dim3((unsigned)((p.cols + 31) / 32), p.shared ? 1u : (unsigned)std::max<int64_t>(1, std::min<int64_t>(turns, 4096))), dim3(1024), 0, s, p);
  return err;
}

#define CASCMM_GATED_OF(LINKAGE, DT)                                                                        \
  LINKAGE template hipError_t gated_forward<DT>(const GatedParams&, int64_t, bool, bool, hipStream_t);      \
  LINKAGE template hipError_t gated_backward<DT>(const GatedParams&, int64_t, bool, bool, hipStream_t);     \
  LINKAGE template hipError_t gated_finish<DT>(const GatedFinish&, bool, hipStream_t);

}  // namespace cascmm
