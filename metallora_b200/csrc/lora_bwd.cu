// The two products of the LoRA backward that read dy, in one launch:
//
//     U  = s dy . B           (rows [M, R64]; transposed [R, M] in two 16-bit parts)
//     dB = dy^T . (s x A^T)   ([N, r])
//
// U reduces over features, dB over tokens, so neither is a by-product of the
// other's pass; but run side by side they read dy at about the same time, so it
// comes from HBM once and from L2 the second time, and one launch's start and
// reduction tail are paid instead of two.  B is read as it lies ([N, r], the
// MMA's MN-major operand): no transposed copy.
//
// U is rounded once for dx (u_rows), as without a checkpoint: dx is the same bits.
// For dA it comes in two parts, since there its rounding would count as much as dA's.
//
// Measured, dy 8192 x 4096, r 16: 17 us, 11 of them streaming (67.8 MB from HBM,
// 152 MB from L2 to the SMs: 13 TB/s, which bounds it), 3 to the first MMA, 2-3 of
// reduction.  The two launches and the transpose it replaces took 31 us.
//
// A CTA owns one 128-row tile of U or of dB and one range of its reduction; the
// ranges of a tile lie in one cluster, and their partial tiles meet through
// distributed shared memory in fixed order (cluster_push_reduce).  The two products
// are split apart from each other, so that all CTAs have about the same number
// of k-blocks.  Warp 0 copies, warp 1 issues the UMMAs, warps 2-5 store.
#include <atomic>
#include <type_traits>

#include "cluster_reduce.cuh"
#include "internal.h"
#include "launch.cuh"
#include "mx.cuh"
#include "../../include/metallora_b200.h"

namespace mlora {
namespace {

constexpr int kThreads = 192;
constexpr int kBK = 64;
constexpr uint32_t kDyBytes = 128 * kBK * 2;   // [128 x 64] of dy
constexpr uint32_t kHalfBytes = 64 * kBK * 2;  // one MN-major box
constexpr int kMaxSplits = 8;

__host__ __device__ constexpr int ctas_per_sm(int R) { return R <= 64 ? 2 : 1; }
__host__ __device__ constexpr uint32_t stage_bytes(int R) { return kDyBytes + R * 128u; }
__host__ __device__ constexpr int num_stages(int R) {
  const uint32_t room = (ctas_per_sm(R) == 2 ? 110u : 220u) * 1024u - push_bytes(R);
  const int n = static_cast<int>(room / stage_bytes(R));
  return n > 8 ? 8 : n;
}
constexpr size_t smem_bytes(int R) {
  return 1024 + num_stages(R) * stage_bytes(R) + push_bytes(R) + 256;
}

// B's tile [64 rows x R columns], R contiguous: one box of R columns in the
// swizzle of its row length (32, 64 or 128 bytes), or boxes of 64 columns.
__host__ __device__ constexpr uint32_t b_row_bytes(int R) { return R >= 64 ? 128u : R * 2u; }
template <int R>
__device__ __forceinline__ uint64_t desc_b(uint32_t saddr, uint32_t k16_step) {
  constexpr uint32_t row = b_row_bytes(R);
  constexpr uint32_t layout = row == 128u ? kLayoutSW128 : (row == 64u ? kLayoutSW64 : kLayoutSW32);
  return make_smem_desc(saddr + k16_step * 16u * row, 64u * row, 8u * row, layout);
}

struct BwdParams {
  long long M, N;
  int r;
  int tiles_u, tiles_db, kb_u, kb_db;
  int splits_u, splits_db;  // ranges a tile (powers of two)
  int ctas_u;               // CTAs of U's tiles, whole clusters; then dB's
  float scale, clip;
  void* u_rows;
  long long ld_rows;
  void* u_t;
  void* u_lo;
  long long ld_t;
  void* db;
  int accumulate, out16;
  int wide;  // dB's rows start on 32 bytes
  int wide_rows;  // the row output starts on 32 bytes (its rows are 128 apart)
  uint32_t* status;
};

// 1-D grid, cluster (max(splits_u, splits_db), 1, 1).  A cluster holds tiles of
// one product only; the last one of each may hold CTAs without a tile.
template <int R, bool kBF16>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(R))
    lora_bwd_kernel(const __grid_constant__ CUtensorMap tm_dy_rows,
                    const __grid_constant__ CUtensorMap tm_dy_cols,
                    const __grid_constant__ CUtensorMap tm_b,
                    const __grid_constant__ CUtensorMap tm_xa, const BwdParams p) {
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
    for (int s = 0; s < S; ++s) mbar_init(&full_bar[s], 1), mbar_init(&empty_bar[s], 1);
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

  const bool is_db = static_cast<int>(blockIdx.x) >= p.ctas_u;
  const int splits = is_db ? p.splits_db : p.splits_u;
  const int id = static_cast<int>(blockIdx.x) - (is_db ? p.ctas_u : 0);
  const int tile = id / splits;
  const uint32_t crank = static_cast<uint32_t>(id % splits);
  const uint32_t first = cluster_ctarank() - crank;
  const int num_kb = is_db ? p.kb_db : p.kb_u;
  const int per = (num_kb + splits - 1) / splits;
  const int kb_begin = static_cast<int>(crank) * per;
  const int kb_end =
      tile < (is_db ? p.tiles_db : p.tiles_u) ? min(num_kb, kb_begin + per) : kb_begin;
  const bool has_work = kb_begin < kb_end;

  // Nothing is read, and so nothing written, before the kernel before this one is
  // through.  Each role waits for that itself, so that the limits of its bounded waits
  // count from there: that kernel may be anyone's, and take its time.
  if (warp == 0) {
    if (elect_one()) {
      grid_wait();
      launch_dependents();  // the dA kernel may start its set-up and stream its codes
      uint32_t stage = 0, phase = 0;
      bool armed[S];
      uint32_t armed_parity[S];
      for (int s = 0; s < S; ++s) armed[s] = false, armed_parity[s] = 0;
      for (int kb = kb_begin; kb < kb_end; ++kb) {
        if (!mbar_wait(&empty_bar[stage], phase ^ 1u, p.status, kDevTimeoutEmpty)) break;
        uint8_t* sa = smem + stage * stage_bytes(R);
        uint8_t* sb = sa + kDyBytes;
        uint64_t* bar = &full_bar[stage];
        mbar_arrive_expect_tx(bar, stage_bytes(R));
        armed[stage] = true;
        armed_parity[stage] = phase;
        if (is_db) {
          tma_load_2d(sa, &tm_dy_cols, bar, tile * 128, kb * kBK);
          tma_load_2d(sa + kHalfBytes, &tm_dy_cols, bar, tile * 128 + 64, kb * kBK);
          tma_load_2d(sb, &tm_xa, bar, kb * kBK, 0);
        } else {
          tma_load_2d(sa, &tm_dy_rows, bar, kb * kBK, tile * 128);
#pragma unroll
          for (int i = 0; i < (R + 63) / 64; ++i)
            tma_load_2d(sb + i * 64 * b_row_bytes(R), &tm_b, bar, i * 64, kb * kBK);
        }
        if (++stage == S) stage = 0, phase ^= 1u;
      }
      for (int s = 0; s < S; ++s)
        if (armed[s]) mbar_wait(&full_bar[s], armed_parity[s], p.status, kDevTimeoutDrain);
    }
  } else if (warp == 1) {
    if (has_work && elect_one()) {
      grid_wait();
      constexpr uint32_t idesc_u = make_idesc_f16(128, R, false, true, kBF16);
      constexpr uint32_t idesc_db = make_idesc_f16(128, R, true, false, kBF16);
      uint32_t stage = 0, phase = 0;
      for (int kb = kb_begin; kb < kb_end; ++kb) {
        if (!mbar_wait(&full_bar[stage], phase, p.status, kDevTimeoutFull)) break;
        tc_fence_after();
        const uint32_t sa = smem_u32(smem + stage * stage_bytes(R));
        const uint32_t sb = sa + kDyBytes;
        if (is_db) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16(tmem, desc_mnmajor_sw128(sa, k, kHalfBytes), desc_kmajor_sw128(sb, k), idesc_db,
                     (kb != kb_begin || k != 0) ? 1u : 0u);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16(tmem, desc_kmajor_sw128(sa, k), desc_b<R>(sb, k), idesc_u,
                     (kb != kb_begin || k != 0) ? 1u : 0u);
        }
        umma_commit(&empty_bar[stage]);
        if (++stage == S) stage = 0, phase ^= 1u;
      }
      umma_commit(done_bar);
    }
  }
  const bool epi = warp >= 2;
  const int row_local = static_cast<int>((warp & 3u) * 32 + lane_id());
  const long long row = static_cast<long long>(tile) * 128 + row_local;
  bool have = false;
  if (epi && has_work) {
    grid_wait();
    have = mbar_wait(done_bar, 0, p.status, kDevTimeoutAccFull);
    tc_fence_after();
  }
  const bool live = epi && row < (is_db ? p.N : p.M);
  auto emit = [&](int j, const auto& in) {
    if (!live) return;
    constexpr int C = std::extent<typename std::remove_reference<decltype(in)>::type>::value;
    float v[C];
    if (!is_db) {
#pragma unroll
      for (int i = 0; i < C; ++i) v[i] = in[i] * p.scale;
      if (p.u_rows != nullptr)
        store_columns<T>(reinterpret_cast<T*>(p.u_rows) + row * p.ld_rows + j, v, p.wide_rows != 0);
      // both parts for dA: with the first alone, U's rounding weighs as much in dA
      // as the rounding of dA itself
      T* hi = reinterpret_cast<T*>(p.u_t) + row + j * p.ld_t;
      T* lo = reinterpret_cast<T*>(p.u_lo) + row + j * p.ld_t;
      float rest[C];
      second_part<T>(v, rest);
#pragma unroll
      for (int i = 0; i < C; ++i) {
        hi[i * p.ld_t] = static_cast<T>(v[i]);
        lo[i * p.ld_t] = static_cast<T>(rest[i]);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < C; ++i)
      v[i] = p.clip > 0.f ? clip_keep_nan(in[i], p.clip) : in[i];
    const long long at = row * p.r + j;
    if (p.accumulate || j + C > p.r) {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        if (j + i >= p.r) continue;
        if (p.out16) {
          T* d = reinterpret_cast<T*>(p.db) + at + i;
          *d = static_cast<T>(p.accumulate ? static_cast<float>(*d) + v[i] : v[i]);
        } else {
          float* d = reinterpret_cast<float*>(p.db) + at + i;
          *d = p.accumulate ? *d + v[i] : v[i];
        }
      }
    } else if (p.out16) {
      store_columns<T>(reinterpret_cast<T*>(p.db) + at, v, p.wide != 0);
    } else {
      store_columns<float>(reinterpret_cast<float*>(p.db) + at, v, p.wide != 0);
    }
  };
  cluster_push_reduce<R>(tmem + ((static_cast<uint32_t>(row_local & ~31)) << 16), have, recv, splits,
                         crank, row_local, epi, emit, first);
  if (live && !is_db && crank == 0 && p.u_rows != nullptr) {  // zero columns past R
    T* dst = reinterpret_cast<T*>(p.u_rows) + row * p.ld_rows;
    for (long long j = R; j < p.ld_rows; j += 8)
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
int launch_typed(const LoraBwdArgs& a, cudaStream_t stream) {
  CUtensorMap tr, tc, tb, tx;
  const CUtensorMapSwizzle sw = b_row_bytes(R) == 128u  ? CU_TENSOR_MAP_SWIZZLE_128B
                                : b_row_bytes(R) == 64u ? CU_TENSOR_MAP_SWIZZLE_64B
                                                        : CU_TENSOR_MAP_SWIZZLE_32B;
  if (!make_tmap_2d_16b(&tr, a.dy, a.N, a.M, a.N, kBK, 128) ||
      !make_tmap_2d_16b(&tc, a.dy, a.N, a.M, a.N, 64, kBK) ||
      !make_tmap_2d_swizzled(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT16, a.b, static_cast<uint64_t>(a.r),
                             static_cast<uint64_t>(a.N), static_cast<uint64_t>(a.r) * 2,
                             R >= 64 ? 64 : R, kBK, sw) ||
      !make_tmap_2d_16b(&tx, a.xa_t, a.M, a.R, a.ld_xa, kBK, R))
    return MLORA_ERR_INVALID_ARG;
  BwdParams p;
  p.M = a.M;
  p.N = a.N;
  p.r = static_cast<int>(a.r);
  p.tiles_db = static_cast<int>((a.N + 127) / 128);
  p.kb_u = static_cast<int>((a.N + kBK - 1) / kBK);
  p.kb_db = static_cast<int>((a.M + kBK - 1) / kBK);
  p.scale = a.scale;
  p.clip = a.clip;
  p.u_rows = a.u_rows;
  p.ld_rows = a.ld_rows;
  p.u_t = a.u_t;
  p.u_lo = a.u_lo;
  p.ld_t = a.ld_t;
  p.db = a.db;
  p.accumulate = a.accumulate ? 1 : 0;
  p.out16 = a.out16 ? 1 : 0;
  p.wide = a.r % 16 == 0 && reinterpret_cast<uintptr_t>(a.db) % 32 == 0;
  p.wide_rows = reinterpret_cast<uintptr_t>(a.u_rows) % 32 == 0;
  p.status = device_status_ptr();
  p.tiles_u = static_cast<int>((a.M + 127) / 128);
  // Halve the longer range while all CTAs stay resident at once (and a range
  // keeps four k-blocks).  8192 x 4096: 128 + 128 CTAs of 32 blocks each; 1001 x
  // 11008: 64 of 22 and 172 of 8.
  const int64_t slots = static_cast<int64_t>(ctas_per_sm(R)) * num_sms();
  int64_t su = 1, sd = 1;
  while (true) {
    const bool can_u = su < kMaxSplits && su * 8 <= p.kb_u &&
                       2 * su * p.tiles_u + sd * p.tiles_db <= slots;
    const bool can_d = sd < kMaxSplits && sd * 8 <= p.kb_db &&
                       su * p.tiles_u + 2 * sd * p.tiles_db <= slots;
    if (can_u && (!can_d || p.kb_u / su >= p.kb_db / sd))
      su *= 2;
    else if (can_d)
      sd *= 2;
    else
      break;
  }
  const int64_t cluster = su > sd ? su : sd;
  p.splits_u = static_cast<int>(su);
  p.splits_db = static_cast<int>(sd);
  p.ctas_u = static_cast<int>((p.tiles_u * su + cluster - 1) / cluster * cluster);
  const int64_t ctas_db = (p.tiles_db * sd + cluster - 1) / cluster * cluster;
  auto kern = lora_bwd_kernel<R, kBF16>;
  static std::atomic<bool> attr_set[64];
  if (int rc = set_max_smem(reinterpret_cast<const void*>(kern), smem_bytes(R), attr_set)) return rc;
  LaunchScope scope(kKindRank, stream);
  return launch_status(
      launch_kernel(kern, dim3(static_cast<unsigned>(p.ctas_u + ctas_db)), kThreads, smem_bytes(R),
                    stream, static_cast<unsigned>(cluster), 1, true, tr, tc, tb, tx, p),
      "lora backward launch");
}

}  // namespace

int launch_lora_bwd(const LoraBwdArgs& a, cudaStream_t s) {
  return with_rank(a.R, [&](auto R) {
    return a.elt == Elt::kBF16 ? launch_typed<R.value, true>(a, s) : launch_typed<R.value, false>(a, s);
  });
}

}  // namespace mlora
