// LoRA weight gradient from an MXINT8 activation checkpoint:
//
//     dA[j, p] = sum_m U[m, j] . x^[m, p]          U = s dy B, x^ the checkpoint
//
// The checkpoint's values are exact in bf16 (mx.cuh), so the codes are turned
// into 16-bit operands inside the kernel and the tensor cores do the sum.  U
// comes as two 16-bit parts, two MMAs into one accumulator: what is left of its
// rounding is 2^-16 (fp16 2^-22, or its subnormal step), and for fp16 the
// rounding of checkpoint values below 2^-24.
// HBM-bound on the codes, half the bytes of a 16-bit x: 8192 x 4096 stream in 7.5
// us (35 MB, 4.7 TB/s), between 1.6 us from U's arrival to the first MMA and 2 us
// of reduction.
//
// CTA = 128 features x one range of tokens; the ranges of a tile are one
// cluster whose partial sums meet through distributed shared memory in fixed
// order (cluster_reduce.cuh).  Warp 0 copies 64-token blocks of codes, scale words
// and U^T (TMA ring), warps 2-9 expand the codes into the swizzled MN-major
// operand, warp 1 issues the UMMAs, warps 2-5 store the tile.
#include <type_traits>

#include "cluster_reduce.cuh"
#include "internal.h"
#include "launch.cuh"
#include "mx.cuh"
#include "../../include/metallora_b200.h"

namespace mlora {
namespace {

constexpr int kConvWarps = 8;
constexpr int kThreads = 64 + 32 * kConvWarps;
constexpr int kBM = 64;                              // tokens per k-block
constexpr uint32_t kCodeBytes = kBM * 128;           // 128 features of 64 tokens
constexpr uint32_t kScaleBytes = kBM * 4;
constexpr uint32_t kOpBytes = kBM * 128 * 2;         // expanded operand, two 64-feature halves
constexpr uint32_t kHalfBytes = kOpBytes / 2;
constexpr int kOps = 2;                              // expanded operands in flight
constexpr int kMaxSplits = 8;

// Pushed sums where their buffer leaves room for the ring; from rank 64 on it
// would take half of it, and the sums are pulled from the stages instead.
__host__ __device__ constexpr bool pushed(int R) { return R <= 32; }
__host__ __device__ constexpr uint32_t recv_bytes(int R) { return pushed(R) ? push_bytes(R) : 0u; }
__host__ __device__ constexpr int ctas_per_sm(int R) { return R <= 64 ? 2 : 1; }
// [R x 64] of both parts of U^T, codes, scale words
__host__ __device__ constexpr uint32_t stage_bytes(int R) { return R * 256u + kCodeBytes + 1024u; }
__host__ __device__ constexpr int num_stages(int R) {
  const uint32_t room =
      (ctas_per_sm(R) == 2 ? 110u : 220u) * 1024u - kOps * kOpBytes - recv_bytes(R);
  return static_cast<int>(room / stage_bytes(R)) > 8 ? 8 : static_cast<int>(room / stage_bytes(R));
}
constexpr size_t smem_bytes(int R) {
  return 1024 + kOps * kOpBytes + num_stages(R) * stage_bytes(R) + recv_bytes(R) + 256;
}

struct MxWgradParams {
  int P, r, num_kb, splits;
  void* out;
  long long ldo;
  int accumulate, out16;
  float clip;
  uint32_t* status;
};

// 1-D grid, cluster (splits, 1, 1): CTA b works on feature tile b / splits over
// token range b % splits (= its cluster rank).
template <int R, bool kBF16>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(R))
    mx_wgrad_kernel(const __grid_constant__ CUtensorMap tm_codes,
                    const __grid_constant__ CUtensorMap tm_scales,
                    const __grid_constant__ CUtensorMap tm_st,
                    const __grid_constant__ CUtensorMap tm_lo, const MxWgradParams p) {
  using T = typename std::conditional<kBF16, __nv_bfloat16, __half>::type;
  constexpr int S = num_stages(R);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_smem<1024>(smem_raw);
  uint8_t* stages = smem + kOps * kOpBytes;
  float* recv = reinterpret_cast<float*>(stages + S * stage_bytes(R));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(stages + S * stage_bytes(R) + recv_bytes(R));
  uint64_t* empty_bar = full_bar + S;
  uint64_t* op_full = empty_bar + S;      // [kOps]
  uint64_t* op_empty = op_full + kOps;    // [kOps]
  uint64_t* done_bar = op_empty + kOps;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done_bar + 1);
  constexpr uint32_t kLoOff = R * 128u;
  constexpr uint32_t kCodeOff = R * 256u;
  constexpr uint32_t kScaleOff = kCodeOff + kCodeBytes;

  const uint32_t warp = warp_id();
  if constexpr (pushed(R)) push_begin();
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) mbar_init(&full_bar[s], 1), mbar_init(&empty_bar[s], 1);
    for (int b = 0; b < kOps; ++b) mbar_init(&op_full[b], kConvWarps), mbar_init(&op_empty[b], 1);
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

  const uint32_t crank = cluster_ctarank();
  const int tile = static_cast<int>(blockIdx.x) / p.splits;
  const int per = (p.num_kb + p.splits - 1) / p.splits;
  const int kb_begin = static_cast<int>(crank) * per;
  const int kb_end = min(p.num_kb, kb_begin + per);
  const bool has_work = kb_begin < kb_end;

  if (warp == 0) {
    if (elect_one()) {
      uint32_t stage = 0, phase = 0;
      bool armed[S];
      uint32_t armed_parity[S];
      for (int s = 0; s < S; ++s) armed[s] = false, armed_parity[s] = 0;
      auto load_codes = [&](int kb, uint8_t* st, uint64_t* bar) {
        mbar_arrive_expect_tx(bar, R * 256u + kCodeBytes + kScaleBytes);
        tma_load_2d(st + kCodeOff, &tm_codes, bar, tile * 128, kb * kBM);
        tma_load_2d(st + kScaleOff, &tm_scales, bar, kb * kBM, tile);
      };
      auto load_u = [&](int kb, uint8_t* st, uint64_t* bar) {
        tma_load_2d(st, &tm_st, bar, kb * kBM, 0);
        tma_load_2d(st + kLoOff, &tm_lo, bar, kb * kBM, 0);
      };
      // U comes from the kernel before this one, the checkpoint does not: a ring
      // of code blocks is on its way before the wait (what wrote it is through:
      // MxWgradArgs::overlap_prev)
      const int ahead = min(S, kb_end - kb_begin);
      for (int i = 0; i < ahead; ++i) {
        load_codes(kb_begin + i, stages + i * stage_bytes(R), &full_bar[i]);
        armed[i] = true;
      }
      grid_wait();
      // the dx GEMM, which reads nothing that this kernel writes, may take the SMs
      // that it frees
      launch_dependents();
      for (int i = 0; i < ahead; ++i)
        load_u(kb_begin + i, stages + i * stage_bytes(R), &full_bar[i]);
      if (ahead == S) phase = 1;
      for (int kb = kb_begin + ahead; kb < kb_end; ++kb) {
        if (!mbar_wait(&empty_bar[stage], phase ^ 1u, p.status, kDevTimeoutEmpty)) break;
        uint8_t* st = stages + stage * stage_bytes(R);
        armed[stage] = true;
        armed_parity[stage] = phase;
        load_codes(kb, st, &full_bar[stage]);
        load_u(kb, st, &full_bar[stage]);
        if (++stage == S) stage = 0, phase ^= 1u;
      }
      for (int s = 0; s < S; ++s)
        if (armed[s]) mbar_wait(&full_bar[s], armed_parity[s], p.status, kDevTimeoutDrain);
    }
  } else if (warp == 1) {
    if (has_work && elect_one()) {
      constexpr uint32_t idesc = make_idesc_f16(128, R, true, false, kBF16);
      uint32_t stage = 0, phase = 0, op = 0, op_phase = 0;
      for (int kb = kb_begin; kb < kb_end; ++kb) {
        if (!mbar_wait(&full_bar[stage], phase, p.status, kDevTimeoutFull)) break;
        if (!mbar_wait(&op_full[op], op_phase, p.status, kDevTimeoutFull)) break;
        tc_fence_after();
        const uint32_t sa = smem_u32(smem + op * kOpBytes);
        const uint32_t sb = smem_u32(stages + stage * stage_bytes(R));
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_f16(tmem, desc_mnmajor_sw128(sa, k, kHalfBytes), desc_kmajor_sw128(sb, k), idesc,
                   (kb != kb_begin || k != 0) ? 1u : 0u);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_f16(tmem, desc_mnmajor_sw128(sa, k, kHalfBytes), desc_kmajor_sw128(sb + kLoOff, k),
                   idesc, 1u);
        umma_commit(&empty_bar[stage]);
        umma_commit(&op_empty[op]);
        if (++stage == S) stage = 0, phase ^= 1u;
        if (++op == kOps) op = 0, op_phase ^= 1u;
      }
      umma_commit(done_bar);
    }
  } else if (has_work) {
    // lane: 16-feature chunk c of token t (and t + 32)
    const int ct = static_cast<int>(threadIdx.x) - 64;
    const int c = ct & 7, t0 = ct >> 3;
    const int half = c >> 2;
    uint32_t stage = 0, phase = 0, op = 0, op_phase = 0;
    for (int kb = kb_begin; kb < kb_end; ++kb) {
      if (!mbar_wait(&full_bar[stage], phase, p.status, kDevTimeoutFull)) break;
      const uint8_t* st = stages + stage * stage_bytes(R);
      uint4 q[2];
      uint32_t byte[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int t = t0 + 32 * i;
        q[i] = *reinterpret_cast<const uint4*>(st + kCodeOff + t * 128 + c * 16);
        byte[i] = st[kScaleOff + t * 4 + (c >> 1)];
      }
      if (!mbar_wait(&op_empty[op], op_phase ^ 1u, p.status, kDevTimeoutEmpty)) break;
      uint8_t* dst = smem + op * kOpBytes + half * kHalfBytes;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int t = t0 + 32 * i;
        uint4 v[2];
        expand16<T>(q[i], byte[i], v[0], v[1]);
        // the two 16-byte chunks of this thread in the 128-byte swizzled row; the
        // halves store theirs in opposite order, so eight lanes hit all banks
        const int c0 = 2 * (c & 3);
        uint8_t* row = dst + t * 128;
        *reinterpret_cast<uint4*>(row + (((c0 + half) ^ (t & 7)) << 4)) = half ? v[1] : v[0];
        *reinterpret_cast<uint4*>(row + (((c0 + 1 - half) ^ (t & 7)) << 4)) = half ? v[0] : v[1];
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane_id() == 0) mbar_arrive(&op_full[op]);
      if (++stage == S) stage = 0, phase ^= 1u;
      if (++op == kOps) op = 0, op_phase ^= 1u;
    }
    __syncwarp();
  }
  const bool epi = warp >= 2 && warp < 6;
  const int row_local = static_cast<int>((warp & 3u) * 32 + lane_id());
  const int prow = tile * 128 + row_local;
  bool have = false;
  if (warp >= 2 && has_work) {
    have = mbar_wait(done_bar, 0, p.status, kDevTimeoutAccFull);
    tc_fence_after();
  }
  const bool live = epi && prow < p.P;
  auto emit = [&](int j, float v0, float v1) {
    if (!live) return;
    float v[2] = {v0, v1};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (j + i >= p.r) continue;
      if (p.clip > 0.f) v[i] = clip_keep_nan(v[i], p.clip);
      const long long at = (j + i) * p.ldo + prow;
      if (p.out16) {
        T* d = reinterpret_cast<T*>(p.out) + at;
        *d = static_cast<T>(p.accumulate ? static_cast<float>(*d) + v[i] : v[i]);
      } else {
        float* d = reinterpret_cast<float*>(p.out) + at;
        *d = p.accumulate ? *d + v[i] : v[i];
      }
    }
  };
  const uint32_t taddr = tmem + ((static_cast<uint32_t>(row_local & ~31)) << 16);
  if constexpr (pushed(R))
    cluster_push_reduce<R>(taddr, have, recv, p.splits, crank, row_local, epi, emit);
  else
    cluster_reduce<R>(taddr, have, reinterpret_cast<float*>(smem), p.splits, crank, row_local, epi,
                      emit);
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols(R));
  }
}

template <int R, bool kBF16>
int launch_typed(const MxWgradArgs& a, cudaStream_t stream) {
  CUtensorMap tc, ts, tu, tl;
  const int64_t m4 = (a.M + 3) / 4 * 4, groups = (a.K + 127) / 128;
  if (!make_tmap_2d(&tc, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.codes, static_cast<uint64_t>(a.K),
                    static_cast<uint64_t>(a.M), static_cast<uint64_t>(a.ld), 128, kBM, false) ||
      // (rows past M, which pad the words, are not read: their bytes are not set)
      !make_tmap_2d(&ts, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, a.scales, static_cast<uint64_t>(a.M),
                    static_cast<uint64_t>(groups), static_cast<uint64_t>(m4) * 4, kBM, 1, false) ||
      !make_tmap_2d_16b(&tu, a.st, a.M, a.R, a.ld_st, kBM, R) ||
      !make_tmap_2d_16b(&tl, a.st_lo, a.M, a.R, a.ld_st, kBM, R))
    return MLORA_ERR_INVALID_ARG;
  MxWgradParams p;
  p.P = static_cast<int>(a.K);
  p.r = static_cast<int>(a.r);
  p.num_kb = static_cast<int>((a.M + kBM - 1) / kBM);
  p.out = a.out;
  p.ldo = a.K;
  p.accumulate = a.accumulate ? 1 : 0;
  p.out16 = a.out16 ? 1 : 0;
  p.clip = a.clip;
  p.status = device_status_ptr();
  // one wave of resident CTAs, at least four k-blocks a split
  const int64_t slots = static_cast<int64_t>(ctas_per_sm(R)) * num_sms();
  int splits = 1;
  while (splits * 2 <= kMaxSplits && splits * 2 * groups <= slots && splits * 8 <= p.num_kb)
    splits *= 2;
  p.splits = splits;
  auto kern = mx_wgrad_kernel<R, kBF16>;
  static std::atomic<bool> attr_set[64];
  if (int rc = set_max_smem(reinterpret_cast<const void*>(kern), smem_bytes(R), attr_set)) return rc;
  LaunchScope scope(kKindWgrad, stream);
  return launch_status(
      launch_kernel(kern, dim3(static_cast<unsigned>(groups * splits)), kThreads, smem_bytes(R),
                    stream, static_cast<unsigned>(splits), 1, a.overlap_prev, tc, ts, tu, tl, p),
      "mx wgrad launch");
}

}  // namespace

int launch_mx_wgrad(const MxWgradArgs& a, cudaStream_t s) {
  return with_rank(a.R, [&](auto R) {
    return a.elt == Elt::kBF16 ? launch_typed<R.value, true>(a, s) : launch_typed<R.value, false>(a, s);
  });
}

}  // namespace mlora
