// Split reduction of a skinny accumulator tile across the CTAs of a cluster,
// shared by the kernels that split their reduction dimension.
#pragma once

#include <type_traits>

#include "ptx.cuh"

namespace mlora {

// Loads this thread's accumulator row (R fp32 columns) from TMEM into `acc`.
template <int R>
__device__ __forceinline__ void load_acc_row(uint32_t taddr_row, float (&acc)[R]) {
  uint32_t r[R / 16][16];
#pragma unroll
  for (int c = 0; c < R / 16; ++c) tmem_ld_32x32b_x16(taddr_row + c * 16, r[c]);
  tmem_ld_wait();
#pragma unroll
  for (int c = 0; c < R / 16; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[c * 16 + i] = __uint_as_float(r[c][i]);
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
// One CTA alone (S = 1) emits straight from its registers, without a barrier.
// Columns go in passes of CP (R > 128: two passes), each read from TMEM at
// `taddr` (this thread's lane) when `have` (zeros otherwise).  Every thread of
// the CTA calls this; only epilogue threads (`epi`) move data.
__host__ __device__ constexpr int reduce_cols(int R) { return R <= 128 ? R : 128; }

// Hands N consecutive column sums from column j to `emit`: all at once to one
// that takes an array, in pairs to one that takes (j, v_j, v_j+1).
template <int N, typename Emit>
__device__ __forceinline__ void emit_columns(Emit& emit, int j, const float (&v)[N]) {
  if constexpr (std::is_invocable<Emit&, int, float, float>::value) {
#pragma unroll
    for (int i = 0; i < N; i += 2) emit(j + i, v[i], v[i + 1]);
  } else {
    emit(j, v);
  }
}

// N consecutive 16-bit values (rounded to nearest) or fp32 values of a row, in
// the widest stores: a sector written in parts costs L2 a pass for each.  `dst`
// is aligned to N values, up to 16 bytes; `wide`: to 32 bytes.
template <typename T, int N>
__device__ __forceinline__ void store_columns(T* dst, const float (&v)[N], bool wide) {
  constexpr int W = N * static_cast<int>(sizeof(T)) / 4;  // 32-bit words
  uint32_t w[W];
#pragma unroll
  for (int i = 0; i < W; ++i) {
    if constexpr (sizeof(T) == 2)
      w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    else
      w[i] = __float_as_uint(v[i]);
  }
  uint32_t* d = reinterpret_cast<uint32_t*>(dst);
  if constexpr (W == 1) {
    *d = w[0];
  } else if constexpr (W == 2) {
    *reinterpret_cast<uint2*>(d) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      if (wide && W % 8 == 0) {
        if (i % 8 == 0) {
          const uint32_t q[8] = {w[i],           w[i + 1],       w[i + 2],       w[i + 3],
                                 w[(i + 4) % W], w[(i + 5) % W], w[(i + 6) % W], w[(i + 7) % W]};
          st_global_32b(d + i, q);
        }
      } else {
        *reinterpret_cast<uint4*>(d + i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
      }
    }
  }
}

// This CTA's slice of the columns: W = CP / S of them from j0, the sums of the
// S peers' values.  Up to 32 loads are in flight before the first sum: each is a
// trip to another SM (with two at a time, 64 columns over two CTAs took 13 us).
template <int CP, int S, typename Emit>
__device__ __forceinline__ void sum_slices(const float* buf, int crank, int row_local,
                                           int j_base, Emit&& emit) {
  constexpr int W = CP / S;
  constexpr int B = W < 32 / S ? W : 32 / S;
  static_assert(W >= 2 && W % B == 0 && B % 2 == 0, "columns come in pairs");
  const int j0 = crank * W;
  const uint32_t base = smem_u32(buf) + static_cast<uint32_t>(row_local) * 4u;
  uint32_t peer[S];
#pragma unroll
  for (int s = 0; s < S; ++s) peer[s] = mapa_shared(base, static_cast<uint32_t>(s));
#pragma unroll 1
  for (int jj = 0; jj < W; jj += B) {
    const uint32_t off = static_cast<uint32_t>(j0 + jj) * 512u;
    float a[B][S];
#pragma unroll
    for (int i = 0; i < B; ++i)
#pragma unroll
      for (int s = 0; s < S; ++s) a[i][s] = ld_shared_cluster_f32(peer[s] + off + i * 512u);
    float v[B];
#pragma unroll
    for (int i = 0; i < B; ++i) {
      v[i] = 0.f;
#pragma unroll
      for (int s = 0; s < S; ++s) v[i] += a[i][s];
    }
    emit_columns(emit, j_base + j0 + jj, v);
  }
}

template <int R, typename Emit>
__device__ __forceinline__ void cluster_reduce(uint32_t taddr, bool have, float* buf, int S,
                                               uint32_t crank, int row_local, bool epi,
                                               Emit&& emit) {
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
      if (S == 1) {  // the whole sum is here
#pragma unroll
        for (int j = 0; j < CP; j += 16) {
          float v[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = 0.f + acc[j + i];
          emit_columns(emit, pass * CP + j, v);
        }
      } else {
#pragma unroll
        for (int j = 0; j < CP; ++j) buf[j * 128 + row_local] = acc[j];
      }
    }
    if (S == 1) continue;
    cluster_sync();
    if (epi) {
      const int c = static_cast<int>(crank);
      if (S == 2)
        sum_slices<CP, 2>(buf, c, row_local, pass * CP, emit);
      else if (S == 4)
        sum_slices<CP, 4>(buf, c, row_local, pass * CP, emit);
      else
        sum_slices<CP, 8>(buf, c, row_local, pass * CP, emit);
    }
    cluster_sync();
  }
}

// The same reduction by pushing: each CTA stores its partial columns into the
// receive buffer of the CTA that sums them, one cluster barrier later every CTA
// sums what it received from its own shared memory, and nothing has to outlive
// that.  Against pulling (cluster_reduce) this saves a barrier and the round
// trips of the loads; it needs `recv` to itself (push_bytes(R)) and the barrier
// arrival of push_begin() at the kernel's start, which tells that a peer's
// shared memory may be written.  Same order of the sums, same bits.  A cluster may
// hold several groups of S CTAs side by side: `first` is the cluster rank of this
// group's first CTA, `crank` the rank within the group.
__host__ __device__ constexpr uint32_t push_bytes(int R) { return reduce_cols(R) * 512u; }

// All threads of the CTA, once, before any work.
__device__ __forceinline__ void push_begin() {
  asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
}

__device__ __forceinline__ void st_shared_cluster_f32(uint32_t cluster_addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_addr), "f"(v) : "memory");
}

// Sends column j of this thread's row to the CTA that owns it: slot [source]
// [column of the slice][row] there.
template <int CP, int S>
__device__ __forceinline__ void push_columns(const float (&acc)[CP], float* recv, uint32_t crank,
                                             uint32_t first, int row_local) {
  constexpr int W = CP / S;
  const uint32_t at = smem_u32(recv) + (crank * W * 128u + static_cast<uint32_t>(row_local)) * 4u;
#pragma unroll
  for (int c = 0; c < S; ++c) {
    const uint32_t dst = mapa_shared(at, first + static_cast<uint32_t>(c));
#pragma unroll
    for (int i = 0; i < W; ++i) st_shared_cluster_f32(dst + i * 512u, acc[c * W + i]);
  }
}

template <int CP, int S, typename Emit>
__device__ __forceinline__ void sum_received(const float* recv, int crank, int row_local, int j_base,
                                             Emit&& emit) {
  constexpr int W = CP / S;
  constexpr int B = W < 16 ? W : 16;
#pragma unroll 1
  for (int jj = 0; jj < W; jj += B) {
    float v[B];
#pragma unroll
    for (int i = 0; i < B; ++i) {
      v[i] = 0.f;
#pragma unroll
      for (int s = 0; s < S; ++s) v[i] += recv[(s * W + jj + i) * 128 + row_local];
    }
    emit_columns(emit, j_base + crank * W + jj, v);
  }
}

template <int R, typename Emit>
__device__ __forceinline__ void cluster_push_reduce(uint32_t taddr, bool have, float* recv, int S,
                                                    uint32_t crank, int row_local, bool epi,
                                                    Emit&& emit, uint32_t first = 0) {
  constexpr int CP = reduce_cols(R);
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");  // push_begin of all CTAs
#pragma unroll 1
  for (int pass = 0; pass < R / CP; ++pass) {
    if (pass > 0) cluster_sync();  // the slots have been summed
    if (epi && S == 1) {
      // (a loop: the code that 16 columns' emit takes comes from memory once)
#pragma unroll 1
      for (int j = 0; j < CP; j += 16) {
        float v[16];
        if (have) {
          load_acc_row<16>(taddr + pass * CP + j, v);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = 0.f + v[i];
        emit_columns(emit, pass * CP + j, v);
      }
    } else if (epi) {
      float acc[CP];
      if (have) {
        load_acc_row<CP>(taddr + pass * CP, acc);
      } else {
#pragma unroll
        for (int j = 0; j < CP; ++j) acc[j] = 0.f;
      }
      if (S == 2) {
        push_columns<CP, 2>(acc, recv, crank, first, row_local);
      } else if (S == 4) {
        push_columns<CP, 4>(acc, recv, crank, first, row_local);
      } else {
        push_columns<CP, 8>(acc, recv, crank, first, row_local);
      }
    }
    if (S == 1) continue;
    cluster_sync();
    if (epi) {
      const int c = static_cast<int>(crank);
      if (S == 2)
        sum_received<CP, 2>(recv, c, row_local, pass * CP, emit);
      else if (S == 4)
        sum_received<CP, 4>(recv, c, row_local, pass * CP, emit);
      else
        sum_received<CP, 8>(recv, c, row_local, pass * CP, emit);
    }
  }
}

}  // namespace mlora
