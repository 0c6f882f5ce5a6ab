// One pass over the activations of a LoRA linear: the rank projection
//
//     s x A^T        (rows [M, R64] for the GEMM, transposed [R, M] for the backward)
//
// on the tensor cores, and from the same shared-memory tiles x's MXFP4 operand
// of the fp4 product and / or its MXINT8 checkpoint (mx.cuh).  HBM-bound: x is
// read once, where separate kernels read it once each.
//
// CTA = 128 tokens x one range of features; the ranges of a token tile are one
// cluster (cluster_push_reduce).  Warp 0 copies [128 x 64] tiles of x and [R x 64]
// tiles of A (TMA ring), warp 1 issues the UMMAs, warps 2-9 quantise: a thread
// owns one block of 32 features, so the block maximum needs no exchange.  A
// stage is free when the UMMAs and all eight warps are done with it.
//
// Roundings.  For the fp4 product the rows come in two 16-bit parts, so that its
// rank term is that of the 32-bit sum to 2^-16 (fp16 2^-22); with one part y's error
// was 1.06 times a correctly rounded y's.  For a dense base's product, and transposed
// for dB, they are one part: y and dB are then the same bits with and without a
// checkpoint, over every base.  dB's own error is 1.4 times a correctly rounded dB's
// (2048 tokens: 0.0024 and 0.0017 over the step's outputs).
//
// Measured under ncu: 16.7 us for 4096 x 4096 with the fp4 operand (floor 6.6), 30
// us for 8192 x 4096 with fp4 operand and checkpoint (118 MB, floor 18).  There
// the quantising warps bound it: about 230 instructions a thread and block, issue
// slots 56 % used by 16 warps an SM.  At a few tokens it is latency: 4 us.
#include <atomic>
#include <type_traits>

#include "cluster_reduce.cuh"
#include "internal.h"
#include "launch.cuh"
#include "mx.cuh"
#include "../../include/metallora_b200.h"

namespace mlora {
namespace {

constexpr int kQuantWarps = 8;
constexpr int kThreads = 64 + 32 * kQuantWarps;
constexpr int kBK = 64;
constexpr uint32_t kXBytes = 128 * kBK * 2;

__host__ __device__ constexpr int ctas_per_sm(int R) { return R <= 64 ? 2 : 1; }
__host__ __device__ constexpr uint32_t stage_bytes(int R) { return kXBytes + R * 128u; }
__host__ __device__ constexpr int num_stages(int R) {
  const uint32_t room = (ctas_per_sm(R) == 2 ? 110u : 220u) * 1024u - push_bytes(R);
  const int n = static_cast<int>(room / stage_bytes(R));
  return n > 8 ? 8 : n;
}
constexpr size_t smem_bytes(int R) {
  return 1024 + num_stages(R) * stage_bytes(R) + push_bytes(R) + 256;
}

struct PrepParams {
  long long M, K;
  int num_kb, splits;
  float scale;
  void* out_rows;
  long long ld_rows;
  int two_parts;  // the row output is followed by what its rounding left, R columns each
  void* out_t;
  long long ld_t;
  uint8_t* q4;       // codes [M, K/2], or nullptr
  uint8_t* q4_atoms;
  long long atoms_k;
  uint8_t* q8;       // codes [M, ld8], or nullptr
  long long ld8;
  int wide8;           // code rows start on 32 bytes
  uint8_t* q8_scales;  // words [ceil(K/128), rows8]
  long long rows8;
  int wide_rows;  // the row output starts on 32 bytes (its rows are 128 apart)
  uint32_t no_max;  // all ones: the bits of no block's maximum
  uint32_t* status;
};

// Grid (token tiles, splits), cluster (1, splits, 1).
template <int R, bool kBF16>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(R))
    mx_prep_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_a,
                   const PrepParams p) {
  using T = typename std::conditional<kBF16, __nv_bfloat16, __half>::type;
  constexpr int S = num_stages(R);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_smem<1024>(smem_raw);
  float* recv = reinterpret_cast<float*>(smem + S * stage_bytes(R));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + S * stage_bytes(R) + push_bytes(R));
  uint64_t* empty_bar = full_bar + S;
  uint64_t* done_bar = empty_bar + S;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done_bar + 1);

  const uint32_t warp = warp_id();
  push_begin();
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) mbar_init(&full_bar[s], 1), mbar_init(&empty_bar[s], 1 + kQuantWarps);
    mbar_init(done_bar, 1);
    fence_mbarrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, tmem_cols(R));
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const int tile = static_cast<int>(blockIdx.x);
  const uint32_t crank = cluster_ctarank();
  const int per = (p.num_kb + p.splits - 1) / p.splits;
  const int kb_begin = static_cast<int>(crank) * per;
  const int kb_end = min(p.num_kb, kb_begin + per);
  const bool has_work = kb_begin < kb_end;

  // Nothing is read, and so nothing written, before the kernel before this one is
  // through.  Each role waits for that itself, so that the limits of its bounded waits
  // count from there: that kernel may be anyone's, and take its time.
  if (warp == 0) {
    if (elect_one()) {
      grid_wait();
      launch_dependents();  // the product may start its set-up and stream its weight
      uint32_t stage = 0, phase = 0;
      bool armed[S];
      uint32_t armed_parity[S];
      for (int s = 0; s < S; ++s) armed[s] = false, armed_parity[s] = 0;
      for (int kb = kb_begin; kb < kb_end; ++kb) {
        if (!mbar_wait(&empty_bar[stage], phase ^ 1u, p.status, kDevTimeoutEmpty)) break;
        uint8_t* st = smem + stage * stage_bytes(R);
        mbar_arrive_expect_tx(&full_bar[stage], stage_bytes(R));
        armed[stage] = true;
        armed_parity[stage] = phase;
        tma_load_2d(st, &tm_x, &full_bar[stage], kb * kBK, tile * 128);
        tma_load_2d(st + kXBytes, &tm_a, &full_bar[stage], kb * kBK, 0);
        if (++stage == S) stage = 0, phase ^= 1u;
      }
      for (int s = 0; s < S; ++s)
        if (armed[s]) mbar_wait(&full_bar[s], armed_parity[s], p.status, kDevTimeoutDrain);
    }
  } else if (warp == 1) {
    if (has_work && elect_one()) {
      grid_wait();
      constexpr uint32_t idesc = make_idesc_f16(128, R, false, false, kBF16);
      uint32_t stage = 0, phase = 0;
      for (int kb = kb_begin; kb < kb_end; ++kb) {
        if (!mbar_wait(&full_bar[stage], phase, p.status, kDevTimeoutFull)) break;
        tc_fence_after();
        const uint32_t sx = smem_u32(smem + stage * stage_bytes(R));
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_f16(tmem, desc_kmajor_sw128(sx, k), desc_kmajor_sw128(sx + kXBytes, k), idesc,
                   (kb != kb_begin || k != 0) ? 1u : 0u);
        umma_commit(&empty_bar[stage]);
        if (++stage == S) stage = 0, phase ^= 1u;
      }
      umma_commit(done_bar);
    }
  } else if (has_work) {
    grid_wait();
    // Lanes 2i, 2i+1: the two blocks of one row's 64 features, 16 rows a warp.  A
    // tile of few tokens leaves warps without rows: they take every second, fourth
    // or eighth k-block instead (one token, K 4096: the pass 5.0 -> 3.9 us).
    const int qw = static_cast<int>(warp) - 2;
    const long long rows = p.M - static_cast<long long>(tile) * 128;
    const int row_warps = rows > 64 ? 8 : (rows > 32 ? 4 : (rows > 16 ? 2 : 1));
    const int turns = kQuantWarps / row_warps, turn = qw / row_warps;
    const int r = (qw % row_warps) * 16 + static_cast<int>(lane_id() >> 1);
    const int b = static_cast<int>(lane_id() & 1u);
    const long long row = static_cast<long long>(tile) * 128 + r;
    const bool live = row < p.M;
    uint8_t* const q4_row = p.q4 + row * (p.K >> 1);
    uint8_t* const q4_atom = p.q4_atoms + (row >> 7) * p.atoms_k * kMxAtomBytes + (r & 31) * 16 +
                             (r >> 5) * 4;
    uint8_t* const q8_row = p.q8 + row * p.ld8;
    uint8_t* const q8_word = p.q8_scales + row * 4;
    uint32_t stage = 0, phase = 0;
    for (int kb = kb_begin; kb < kb_end; ++kb) {
      if (!mbar_wait(&full_bar[stage], phase, p.status, kDevTimeoutFull)) break;
      if (((kb - kb_begin) & (turns - 1)) != turn) {  // another warp's block
        __syncwarp();
        if (lane_id() == 0) mbar_arrive(&empty_bar[stage]);
        if (++stage == S) stage = 0, phase ^= 1u;
        continue;
      }
      uint32_t w[16];
      const uint8_t* src = smem + stage * stage_bytes(R) + r * 128;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 q = *reinterpret_cast<const uint4*>(src + (((4 * b + i) ^ (r & 7)) << 4));
        w[4 * i] = q.x, w[4 * i + 1] = q.y, w[4 * i + 2] = q.z, w[4 * i + 3] = q.w;
      }
      // The stage is free once its words are in registers, and they are once the
      // whole warp's maximum is known: an arrive after the loads alone overtook
      // them (a late load then read the tile copied next; seen in 1 of 8 runs of
      // 4096 x 4096).  So the arrive hangs on that maximum.  It is never all ones, but
      // no_max is a parameter: no compiler can tell, and drop the dependence.
      const uint32_t amax = block_amax<T>(w);
      if (__reduce_max_sync(0xffffffffu, amax) != p.no_max && lane_id() == 0)
        mbar_arrive(&empty_bar[stage]);
      if (++stage == S) stage = 0, phase ^= 1u;

      const int k = kb * kBK + 32 * b;
      const bool in = live && k < p.K;
      if (p.q4 != nullptr) {
        const uint32_t byte = mx_scale_byte_fp4(amax);
        const uint32_t other = __shfl_xor_sync(0xffffffffu, byte, 1);
        if (live && b == 0)
          *reinterpret_cast<uint16_t*>(q4_atom + (kb >> 1) * kMxAtomBytes + (kb & 1) * 2) =
              static_cast<uint16_t>(byte | (other << 8));
        const uint4 c = block_fp4<T>(w, byte);
        if (in) *reinterpret_cast<uint4*>(q4_row + (k >> 1)) = c;
      }
      if (p.q8 != nullptr) {
        const uint32_t byte = mx_scale_byte_int8(amax);
        const uint32_t other = __shfl_xor_sync(0xffffffffu, byte, 1);
        if (live && b == 0) {
          uint16_t* dst = reinterpret_cast<uint16_t*>(q8_word + (kb >> 1) * p.rows8 * 4) + (kb & 1);
          *dst = static_cast<uint16_t>(byte | (other << 8));
          if (kb + 1 == p.num_kb && (kb & 1) == 0) dst[1] = 0;  // the word's blocks past K
        }
        uint4 lo, hi;
        block_int8<T>(w, amax, lo, hi);
        if (in) {
          uint8_t* dst = q8_row + k;
          if (k + 32 <= p.K && p.wide8) {
            const uint32_t v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
            st_global_32b(dst, v);
          } else if (k + 32 <= p.K) {
            *reinterpret_cast<uint4*>(dst) = lo;
            *reinterpret_cast<uint4*>(dst + 16) = hi;
          } else {  // K is a multiple of 8: the row ends between two 8-byte groups
            const uint32_t o[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (k + 8 * i < p.K)
                *reinterpret_cast<uint2*>(dst + 8 * i) = make_uint2(o[2 * i], o[2 * i + 1]);
          }
        }
      }
    }
    __syncwarp();
  }
  const bool epi = warp >= 2 && warp < 6;
  const int row_local = static_cast<int>((warp & 3u) * 32 + lane_id());
  const long long row = static_cast<long long>(tile) * 128 + row_local;
  bool have = false;
  if (warp >= 2 && has_work) {
    have = mbar_wait(done_bar, 0, p.status, kDevTimeoutAccFull);
    tc_fence_after();
  }
  const bool live = epi && row < p.M;
  auto emit = [&](int j, const auto& in) {
    if (!live) return;
    constexpr int C = std::extent<typename std::remove_reference<decltype(in)>::type>::value;
    float v[C];
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] = in[i] * p.scale;
    T* const rows = reinterpret_cast<T*>(p.out_rows) + row * p.ld_rows + j;
    store_columns<T>(rows, v, p.wide_rows != 0);
    if (p.two_parts) {
      float rest[C];
      second_part<T>(v, rest);
      store_columns<T>(rows + R, rest, p.wide_rows != 0);
    }
    if (p.out_t != nullptr) {
      T* dst = reinterpret_cast<T*>(p.out_t) + row + j * p.ld_t;
#pragma unroll
      for (int i = 0; i < C; ++i) dst[i * p.ld_t] = static_cast<T>(v[i]);
    }
  };
  cluster_push_reduce<R>(tmem + ((static_cast<uint32_t>(row_local & ~31)) << 16), have, recv,
                         p.splits, crank, row_local, epi, emit);
  if (live && crank == 0) {  // zero columns past the last part
    T* dst = reinterpret_cast<T*>(p.out_rows) + row * p.ld_rows;
    for (long long j = p.two_parts ? 2 * R : R; j < p.ld_rows; j += 8)
      *reinterpret_cast<uint4*>(dst + j) = make_uint4(0, 0, 0, 0);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols(R));
  }
}

template <int R, bool kBF16>
int launch_typed(const MxPrepArgs& a, cudaStream_t stream) {
  CUtensorMap tx, ta;
  if (!make_tmap_2d_16b(&tx, a.x, a.K, a.M, a.K, kBK, 128) ||
      !make_tmap_2d_16b(&ta, a.a, a.K, a.r, a.K, kBK, R))
    return MLORA_ERR_INVALID_ARG;
  PrepParams p;
  p.M = a.M;
  p.K = a.K;
  p.num_kb = static_cast<int>((a.K + kBK - 1) / kBK);
  p.scale = a.scale;
  p.out_rows = a.out_rows;
  p.ld_rows = a.ld_rows;
  p.two_parts = a.two_parts ? 1 : 0;
  p.out_t = a.out_t;
  p.ld_t = a.ld_t;
  p.q4 = static_cast<uint8_t*>(a.q4);
  p.q4_atoms = static_cast<uint8_t*>(a.q4_atoms);
  p.atoms_k = (a.K + 127) / 128;
  p.q8 = static_cast<uint8_t*>(a.q8);
  p.ld8 = a.ld8;
  p.wide8 = a.ld8 % 32 == 0 && reinterpret_cast<uintptr_t>(a.q8) % 32 == 0;
  p.q8_scales = static_cast<uint8_t*>(a.q8_scales);
  p.rows8 = (a.M + 3) / 4 * 4;
  p.wide_rows = reinterpret_cast<uintptr_t>(a.out_rows) % 32 == 0;
  p.no_max = 0xFFFFFFFFu;
  p.status = device_status_ptr();
  const int64_t tiles = (a.M + 127) / 128;
  // the plain rank projection's split, so that s x A^T has the same bits with and
  // without a checkpoint (up to rank 64 it is also one wave of these CTAs)
  const int splits = rank_splits(a.M, a.K);
  p.splits = splits;
  auto kern = mx_prep_kernel<R, kBF16>;
  static std::atomic<bool> attr_set[64];
  if (int rc = set_max_smem(reinterpret_cast<const void*>(kern), smem_bytes(R), attr_set)) return rc;
  LaunchScope scope(kKindRank, stream);
  return launch_status(
      launch_kernel(kern, dim3(static_cast<unsigned>(tiles), static_cast<unsigned>(splits)), kThreads,
                    smem_bytes(R), stream, 1, static_cast<unsigned>(splits), true, tx, ta, p),
      "mx prep launch");
}

}  // namespace

int launch_mx_prep(const MxPrepArgs& a, cudaStream_t s) {
  if (a.out_rows == nullptr) {
    set_error("rank and quantise pass: the row output is required");
    return MLORA_ERR_INVALID_ARG;
  }
  return with_rank(a.R, [&](auto R) {
    return a.elt == Elt::kBF16 ? launch_typed<R.value, true>(a, s) : launch_typed<R.value, false>(a, s);
  });
}

}  // namespace mlora
