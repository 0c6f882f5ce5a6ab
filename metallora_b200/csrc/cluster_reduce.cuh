// Split reduction of a skinny accumulator tile across the CTAs of a cluster,
// shared by the kernels that split their reduction dimension.
#pragma once

#include "ptx.cuh"

namespace mlora {

// Loads this thread's accumulator row (R fp32 columns) from TMEM into `acc`.
template <int R>
__device__ __forceinline__ void load_acc_row(uint32_t taddr_row, float (&acc)[R]) {
#pragma unroll
  for (int c = 0; c < R / 16; ++c) {
    uint32_t r[16];
    tmem_ld_32x32b_x16(taddr_row + c * 16, r);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[c * 16 + i] = __uint_as_float(r[i]);
  }
}

// Cross-CTA split reduction through distributed shared memory.  The S CTAs of
// a cluster computed the same [128 x R] tile over S disjoint ranges of the
// reduction dimension (cluster rank = range index).  Each CTA parks its fp32
// partial in its own shared memory (the TMA stage area, free once the MMAs
// are done), column-major [j][row] so warps touch consecutive words; after a
// cluster barrier CTA c sums its slice of columns [c W, (c+1) W) (W = CP / S)
// of all 128 rows over s = 0..S-1 in that order -- fixed order, so results are
// bitwise reproducible -- and hands pairs of columns to `emit(j, v_j, v_j+1)`.
// A second barrier keeps every CTA resident until its peers have read it.
// Columns go in passes of CP (R > 128: two passes), each read from TMEM at
// `taddr` (this thread's lane) when `have` (zeros otherwise).  Every thread of
// the CTA calls this; only epilogue threads (`epi`) move data.  A cluster may
// hold several such groups of S CTAs side by side: `first` is the cluster rank
// of this group's first CTA, `crank` the rank within the group.
__host__ __device__ constexpr int reduce_cols(int R) { return R <= 128 ? R : 128; }

template <int R, typename Emit>
__device__ __forceinline__ void cluster_reduce(uint32_t taddr, bool have, float* buf, int S,
                                               uint32_t crank, int row_local, bool epi,
                                               Emit&& emit, uint32_t first = 0) {
  constexpr int CP = reduce_cols(R);
#pragma unroll 1
  for (int pass = 0; pass < R / CP; ++pass) {
    if (epi) {
      float acc[CP];
      if (have) {
        load_acc_row<CP>(taddr + pass * CP, acc);
      } else {
#pragma unroll
        for (int j = 0; j < CP; ++j) acc[j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < CP; ++j) buf[j * 128 + row_local] = acc[j];
    }
    cluster_sync();
    if (epi) {
      const int W = CP / S;
      const int j0 = static_cast<int>(crank) * W;
      const uint32_t base = smem_u32(buf) + static_cast<uint32_t>(row_local) * 4u;
      uint32_t peer[8];
#pragma unroll
      for (int s = 0; s < 8; ++s) peer[s] = s < S ? mapa_shared(base, first + static_cast<uint32_t>(s)) : 0u;
#pragma unroll 1
      for (int jj = 0; jj < W; jj += 2) {
        const uint32_t off0 = static_cast<uint32_t>(j0 + jj) * 512u;
        float a[8], b[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          a[s] = s < S ? ld_shared_cluster_f32(peer[s] + off0) : 0.f;
          b[s] = s < S ? ld_shared_cluster_f32(peer[s] + off0 + 512u) : 0.f;
        }
        float v0 = 0.f, v1 = 0.f;
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          v0 += a[s];
          v1 += b[s];
        }
        emit(pass * CP + j0 + jj, v0, v1);
      }
    }
    cluster_sync();
  }
}

}  // namespace mlora
