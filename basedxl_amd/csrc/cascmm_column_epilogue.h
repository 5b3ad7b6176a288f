// The epilogue of a product (cascmm_epilogue.h) in the stores of the fp32 kernels whose lanes hold a column of a block: z to preact, act(z) + residual.
// A load or store of one register is two whole 128-byte pieces of rows.  The residual of a block is asked for while something else is at hand (the sums
// of the waves, the block before), all its rows at once.
// Every offset is a lane's own, so that rows past the last one and columns past the edge fall beyond the descriptors' ends: loads give zeros, stores are
// dropped.  (Host-checked: a tile's rows span less than 2 GiB in each of the tensors.)
// Measured (graph replay, us: the product alone / with a residual / with gelu; in brackets the same by a pass behind the product): two bf16 terms 2048 x 1280 x 1280
// prepared 22.9 / 24.7 / 24.8 (res 28.2), 2048 x 5120 x 1280 77 / 80 / 80, 2048 x 1280 x 5120 73 / 86 / 80 (94 / 87; 42 MB of result and of
// residual, no store hides behind another tile's loop), 2 x 1280 x 1280 4.3 / 4.5 / 4.5; three fp16 terms 2048 x 5120 x 1280 168 / 169 / 169.
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
  // (PRE: z may be wanted)
  template <int AUX, bool PRE = true, int R> __device__ __forceinline__ void store(float (&z)[R], const float (&r)[R], int row, int up, int col, bool inside) const {
    if (PRE && pre) {
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

// The store of the LDS-tiled kernels: blocks of permuted columns come in runs of RUN, block b of the tile and lane l31 <-> column 128 (b / 4) + 4 l31 + b % 4, so a
// lane holds RUN adjacent columns of a row; the others are as above.  A quad of rows at a time, the next one's residual asked for before.
// Without z in the kernels of twelve waves, which are not launched for it (tile_keeps_z).
template <class TL>
__device__ __forceinline__ void tile_epilogue(const GroupParams& p, float* C, const float* bias, int m0, int n0, int wm0, int wn0, int l31, int g,
                                              f32x16 (&res)[TL::MT][TL::NTL]) {
  constexpr int NQ = (TL::BNQ == 0) ? 0 : (TL::WN == 1 ? TL::BNQ / 32 : TL::NTL), RUN = (NQ % 4 == 0) ? 4 : 2;
  constexpr bool PRE = tile_keeps_z(TL::NT);
  const EpilogueArgs args = epilogue_args(p);
  const ColumnEpilogue ep(args, C, p.ldc, p.M, p.N, m0 + wm0, n0);
  const bool vec = ((p.N | p.ldc | p.ldr | p.ldp) & 3) == 0 && (((uintptr_t)C | (uintptr_t)p.residual | (uintptr_t)p.preact) & 15) == 0;
  typedef float run_t __attribute__((ext_vector_type(RUN)));
#pragma unroll
  for (int r0 = 0; r0 < NQ; r0 += RUN) {
    const int b = (wn0 >> 5) + r0, col = (b >> 2) * 128 + 4 * l31 + (b & 3);   // (col + i exists or not together with the run where vec)
    float bv[RUN];
#pragma unroll
    for (int i = 0; i < RUN; ++i) bv[i] = bias && n0 + col + i < p.N ? bias[n0 + col + i] : 0.f;
    auto place = [&](int row, int ld, int i) {
      return (int)((n0 + col + i < p.N ? (unsigned)(4 * g * ld + (col + i) * 4) : 0x7FFFFFFFu) + (unsigned)(row * ld));
    };
    auto ask = [&](int k, run_t (&to)[4]) {
      if (!ep.res) return;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = (k >> 2) * 32 + (k & 3) * 8 + e;
        if (vec) {
          if constexpr (RUN == 4) to[e] = llvm_raw_buffer_load_v4f32(ep.rr, place(row, ep.ldr, 0), 0, 0);
          else to[e] = llvm_raw_buffer_load_v2f32(ep.rr, place(row, ep.ldr, 0), 0, 0);
        } else {
#pragma unroll
          for (int i = 0; i < RUN; ++i) to[e][i] = llvm_raw_buffer_load_f32(ep.rr, place(row, ep.ldr, i), 0, 0);
        }
      }
    };
    auto out = [&](const i32x4& to, int ld, int row, const run_t& z) {
      if (vec) {
        if constexpr (RUN == 4) llvm_raw_buffer_store_v4f32(z, to, place(row, ld, 0), 0, kResultStoreAux);
        else llvm_raw_buffer_store_v2f32(z, to, place(row, ld, 0), 0, kResultStoreAux);
      } else {
#pragma unroll
        for (int i = 0; i < RUN; ++i) llvm_raw_buffer_store_f32(z[i], to, place(row, ld, i), 0, kResultStoreAux);
      }
    };
    run_t r[2][4];
    ask(0, r[0]);
#pragma unroll
    for (int k = 0; k < 4 * TL::MT; ++k) {
      const int mi = k >> 2, q = k & 3;
      if (k + 1 < 4 * TL::MT) ask(k + 1, r[(k + 1) & 1]);
      float z[4 * RUN];
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < RUN; ++i) z[e * RUN + i] = res[mi][r0 + i][4 * q + e] + bv[i];
      if (PRE && ep.pre) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          run_t v;
#pragma unroll
          for (int i = 0; i < RUN; ++i) v[i] = z[e * RUN + i];
          out(ep.rp, ep.ldp, mi * 32 + q * 8 + e, v);
        }
      }
      activate(z, ep.act);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        run_t v;
#pragma unroll
        for (int i = 0; i < RUN; ++i) v[i] = z[e * RUN + i];
        if (ep.res) v += r[k & 1][e];
        out(ep.rc, ep.ldc, mi * 32 + q * 8 + e, v);
      }
    }
  }
  if constexpr (NQ < TL::NTL) {
    constexpr int BLOCKS = TL::MT * (TL::NTL - NQ);
    float r[2][16];
    ep.ask(r[0], 0, 4 * g, wn0 + NQ * 32 + l31, n0 + wn0 + NQ * 32 + l31 < p.N);
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      const int ni = NQ + b / TL::MT, mi = b % TL::MT, nx = NQ + (b + 1) / TL::MT, mx = (b + 1) % TL::MT, col = wn0 + ni * 32 + l31;
      if (b + 1 < BLOCKS) ep.ask(r[(b + 1) & 1], mx * 32, 4 * g, wn0 + nx * 32 + l31, n0 + wn0 + nx * 32 + l31 < p.N);
      const float bv = bias && n0 + col < p.N ? bias[n0 + col] : 0.f;
      float z[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) z[e] = res[mi][ni][e] + bv;
      ep.template store<kResultStoreAux, PRE>(z, r[b & 1], mi * 32, 4 * g, col, n0 + col < p.N);
    }
  }
}

}  // namespace cascmm
