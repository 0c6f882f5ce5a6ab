// LoRA linear over an MXFP4 base on the fp4 tensor cores:
//
//     Y[M, N] = Q4(x) . W4^T  +  X2[M, R] . W2^T        (X2 = s x A^T, W2 = B)
//
// Both factors of the base product are MXFP4 (mx.cuh): tcgen05.mma kind::mxf4
// multiplies code rows and applies the block scales itself, so nothing is
// dequantised.  The rank-r block is appended as 16-bit kind::f16 steps into the
// same TMEM accumulator, as in the dense kernel, so Y is written once.  X2 comes in
// two 16-bit parts: twice the rank steps, which up to rank 32 still fit one k-block
// (16 tokens 4096 -> 4096, rank 16: 7.9 us with one part and with two); from rank 64
// every 64 columns are one more (rank 64: 513 tokens 6848 -> 936 23.7 and 24.0 us, 4096
// tokens 4096 -> 11008 88.2 and 91.9).
//
// A shared-memory row of 128 bytes is 256 codes or 64 16-bit values, so both
// kinds of k-block share one stage layout (128-byte swizzle, K-major) and one
// ring; a main block also carries its scale atoms.
#include <atomic>
#include <string>
#include <type_traits>

#include "cluster_reduce.cuh"
#include "internal.h"
#include "launch.cuh"
#include "mx.cuh"
#include "../../include/metallora_b200.h"

namespace mlora {
namespace {

constexpr int kBK4 = 256;                        // fp4 reduction per main k-block
constexpr int kBK16 = 64;                        // 16-bit reduction per rank k-block
constexpr uint32_t kRowBytes = 128;              // of either
constexpr uint32_t kSfBytes = 2 * kMxAtomBytes;  // scales of 128 rows x 256 features

// X2's two parts take the columns [0, R) and [R, 2R) of its rows, and both meet the
// same W2: the W2 column of the rank block's k-block e, and the W2 step of its step k
// (up to rank 32 both parts lie in one block, and W2 once beside them).
__device__ __forceinline__ int rank_column(int e, int R) { return (e * kBK16) & (R - 1) & ~(kBK16 - 1); }
__device__ __forceinline__ uint32_t rank_step(int k, int R) {
  return static_cast<uint32_t>(R >= kBK16 ? k : k & (R / 16 - 1));
}

// ---------------------------------------------------------------------------
// Few tokens (M <= 128): the weight rows are the MMA's M side (128 a tile) and
// the tokens its N side, so one pass over the weight serves all tokens.
// Bound by latency: one token through 4096 -> 11008 takes 11.0 us with the pass
// before it, of which the weight's 24 MB are 3.7 at the measured bandwidth; a ring
// of weight blocks is loaded while that pass still runs.  The reduction is split
// over the CTAs of a cluster so that about two CTAs per SM stream it, and their
// partial tiles are summed through distributed shared memory in fixed order
// (cluster_push_reduce).
constexpr int kSkinnyThreads = 192;
constexpr int kSkinnyMaxSplits = 8;

__host__ __device__ constexpr uint32_t skinny_stage_bytes(int NT) {
  return (128 + NT) * kRowBytes + 2 * kSfBytes;
}
__host__ __device__ constexpr int skinny_stages(int NT) {
  return static_cast<int>(((NT <= 32 ? 110u : 220u) * 1024u - push_bytes(NT)) /
                          skinny_stage_bytes(NT));
}
constexpr size_t skinny_smem(int NT) {
  return 1024 + skinny_stages(NT) * skinny_stage_bytes(NT) + push_bytes(NT) + 256;
}
// accumulator columns, then two sets of (8 weight, 8 token) scale columns
__host__ __device__ constexpr uint32_t skinny_acc_cols(int NT) { return NT; }
__host__ __device__ constexpr uint32_t skinny_tmem_cols(int NT) { return tmem_cols(NT + 32); }

struct SkinnyParams {
  int M, N, K;
  int num_kb_main, num_kb_extra, R;
  int splits;
  int atoms_k;  // scale atoms along K per 128 rows
  void* d;
  long long ldd;
  uint32_t* status;
};

// Grid (weight tiles, splits), cluster (1, splits, 1).
template <int NT, bool kBF16>
__global__ void __launch_bounds__(kSkinnyThreads, NT <= 32 ? 2 : 1)
    mx_skinny_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                     const __grid_constant__ CUtensorMap tm_ws, const __grid_constant__ CUtensorMap tm_xs,
                     const __grid_constant__ CUtensorMap tm_w2, const __grid_constant__ CUtensorMap tm_x2,
                     const SkinnyParams p) {
  using T = typename std::conditional<kBF16, __nv_bfloat16, __half>::type;
  constexpr int S = skinny_stages(NT);
  constexpr uint32_t kStage = skinny_stage_bytes(NT);
  constexpr uint32_t kXOff = 128 * kRowBytes;
  constexpr uint32_t kWsOff = kXOff + NT * kRowBytes;
  constexpr uint32_t kXsOff = kWsOff + kSfBytes;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_smem<1024>(smem_raw);
  float* recv = reinterpret_cast<float*>(smem + S * kStage);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + S * kStage + push_bytes(NT));
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
    tmem_alloc(tmem_slot, skinny_tmem_cols(NT));
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const int n0 = static_cast<int>(blockIdx.x) * 128;
  const uint32_t crank = cluster_ctarank();
  const int total_kb = p.num_kb_main + p.num_kb_extra;
  const int per = (total_kb + p.splits - 1) / p.splits;
  const int kb_begin = static_cast<int>(crank) * per;
  const int kb_end = min(total_kb, kb_begin + per);
  const bool has_work = kb_begin < kb_end;

  if (warp == 0) {
    if (elect_one()) {
      uint32_t stage = 0, phase = 0;
      bool armed[S];
      uint32_t armed_parity[S];
      for (int s = 0; s < S; ++s) armed[s] = false, armed_parity[s] = 0;
      auto load_weight = [&](int kb, uint8_t* st, uint64_t* bar) {
        if (kb >= p.num_kb_main) {
          mbar_arrive_expect_tx(bar, (128 + NT) * kRowBytes);
          tma_load_2d(st, &tm_w2, bar, rank_column(kb - p.num_kb_main, p.R), n0);
        } else {
          mbar_arrive_expect_tx(bar, kStage);
          tma_load_2d(st, &tm_w, bar, kb * static_cast<int>(kRowBytes), n0);
          tma_load_2d(st + kWsOff, &tm_ws, bar, 0, static_cast<int>(blockIdx.x) * p.atoms_k + 2 * kb);
        }
      };
      auto load_tokens = [&](int kb, uint8_t* st, uint64_t* bar) {
        if (kb >= p.num_kb_main) {
          tma_load_2d(st + kXOff, &tm_x2, bar, (kb - p.num_kb_main) * kBK16, 0);
        } else {
          tma_load_2d(st + kXOff, &tm_x, bar, kb * static_cast<int>(kRowBytes), 0);
          tma_load_2d(st + kXsOff, &tm_xs, bar, 0, 2 * kb);
        }
      };
      // the weight does not come from the kernel before this one, the token
      // operands do: a ring of weight blocks is on its way before the wait (what
      // wrote the weight is through: MxGemmArgs::overlap_prev)
      const int ahead = min(S, kb_end - kb_begin);
      for (int i = 0; i < ahead; ++i) {
        load_weight(kb_begin + i, smem + i * kStage, &full_bar[i]);
        armed[i] = true;
      }
      grid_wait();
      for (int i = 0; i < ahead; ++i) load_tokens(kb_begin + i, smem + i * kStage, &full_bar[i]);
      if (ahead == S) phase = 1;
      stage = ahead == S ? 0u : static_cast<uint32_t>(ahead);
      for (int kb = kb_begin + ahead; kb < kb_end; ++kb) {
        if (!mbar_wait(&empty_bar[stage], phase ^ 1u, p.status, kDevTimeoutEmpty)) break;
        armed[stage] = true;
        armed_parity[stage] = phase;
        load_weight(kb, smem + stage * kStage, &full_bar[stage]);
        load_tokens(kb, smem + stage * kStage, &full_bar[stage]);
        if (++stage == S) stage = 0, phase ^= 1u;
      }
      launch_dependents();
      for (int s = 0; s < S; ++s)
        if (armed[s]) mbar_wait(&full_bar[s], armed_parity[s], p.status, kDevTimeoutDrain);
    }
  } else if (warp == 1) {
    if (has_work && elect_one()) {
      constexpr uint32_t idesc16 = make_idesc_f16(128, NT, false, false, kBF16);
      uint32_t stage = 0, phase = 0;
      for (int kb = kb_begin; kb < kb_end; ++kb) {
        if (!mbar_wait(&full_bar[stage], phase, p.status, kDevTimeoutFull)) break;
        tc_fence_after();
        const uint32_t sw = smem_u32(smem + stage * kStage);
        const uint32_t sx = sw + kXOff;
        const uint32_t first = kb == kb_begin ? 0u : 1u;
        if (kb >= p.num_kb_main) {
          const int nk = min(4, 2 * p.R / 16);
          for (int k = 0; k < nk; ++k)
            umma_f16(tmem, desc_kmajor_sw128(sw, rank_step(k, p.R)), desc_kmajor_sw128(sx, k),
                     idesc16, first | static_cast<uint32_t>(k != 0));
        } else {
          const uint32_t sfa = tmem + skinny_acc_cols(NT) + static_cast<uint32_t>(kb & 1) * 16u;
          const uint32_t sfb = sfa + 8u;
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            tmem_cp_scale_atom(sfa + 4 * a, sw + kWsOff + a * kMxAtomBytes);
            tmem_cp_scale_atom(sfb + 4 * a, sw + kXsOff + a * kMxAtomBytes);
          }
          // codes past K are zero-filled; a step that lies past K entirely would
          // also read scales that belong to other rows, so it is left out
          const int nk = min(4, (p.K - kb * kBK4 + 63) / 64);
          for (int k = 0; k < nk; ++k)
            umma_mxf4(tmem, desc_kmajor_sw128(sw, k), desc_kmajor_sw128(sx, k),
                      make_idesc_mxf4(128, NT, 2u * (k & 1)), sfa + 4 * (k >> 1), sfb + 4 * (k >> 1),
                      first | static_cast<uint32_t>(k != 0));
        }
        umma_commit(&empty_bar[stage]);
        if (++stage == S) stage = 0, phase ^= 1u;
      }
      umma_commit(done_bar);
    }
  }
  const bool epi = warp >= 2;
  const int row_local = static_cast<int>((warp & 3u) * 32 + lane_id());
  const int n = n0 + row_local;
  bool have = false;
  if (epi && has_work) {
    have = mbar_wait(done_bar, 0, p.status, kDevTimeoutAccFull);
    tc_fence_after();
  }
  T* const out = reinterpret_cast<T*>(p.d) + n;
  const bool live = epi && n < p.N;
  auto emit = [&](int j, float v0, float v1) {
    if (!live) return;
    if (j < p.M) out[j * p.ldd] = static_cast<T>(v0);
    if (j + 1 < p.M) out[(j + 1) * p.ldd] = static_cast<T>(v1);
  };
  cluster_push_reduce<NT>(tmem + ((static_cast<uint32_t>(row_local & ~31)) << 16), have, recv,
                          p.splits, crank, row_local, epi, emit);
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, skinny_tmem_cols(NT));
  }
}

// ---------------------------------------------------------------------------
// More tokens: persistent CTA pairs (cta_group::2), one 256 x 256 tile a pair at
// a time, as the dense pair GEMM.  Each CTA stages its own 128 rows of x and of
// W (16 KB each a k-block of 256) and the scale atoms of its x rows and of all
// 256 W rows.
//
// The scales need TMEM next to the accumulator, so the accumulator is not
// double-buffered; eight epilogue warps take it into registers at once and hand
// it back before they convert and store.
//
// Measured, 4096 x 4096 -> 11008, R 64: alone 85 us = 4.4 PFLOP/s at the 1.62 GHz
// that the chip's power cap leaves it (tensor pipe 68 % busy; behind the pass over x,
// whose end it overlaps, the two take 91.9).  A tile takes 12-13 thousand cycles: 9.2
// of MMA (64 fp4 of 128 cycles, 8 bf16), 1.4 of scale copies (they run in the MMAs'
// queue, 15 cycles each), 0.9 until the
// accumulator is free again, 1-2 of waiting for operands (907 MB come from L2; with
// one MMA in four issued, the copies alone took 53 us).  9.3 tiles a pair make nine
// waves and one of half tiles.  Tried and slower: copying a block's scales ahead of
// the MMAs of the block before (107 against 95 us); no effect: raster groups of 1 to 32.
constexpr int kPairStages = 6;
constexpr int kHalf = 128;
constexpr int kPairN = 256;
constexpr uint32_t kPairOpBytes = kHalf * kRowBytes;  // 16 KB
constexpr uint32_t kPairStageBytes = 2 * kPairOpBytes + 3 * kSfBytes;
constexpr int kPairEpiWarps = 8;
constexpr int kPairThreads = 64 + 32 * kPairEpiWarps;
constexpr size_t kPairSmem = 1024 + kPairStages * kPairStageBytes + 256;
constexpr uint32_t kPairTmemCols = 512;  // 256 accumulator, two sets of 8 + 16 scale columns

struct PairParams {
  int M, N, K;
  int num_kb_main, num_kb_extra, R;
  int tiles_m, tiles_n, group_m;
  int whole, num_items;  // tiles of 256 columns, then the others in halves
  int atoms_k;
  int wide;  // rows of d start on 32 bytes (else on 16)
  void* d;
  long long ldd;
  uint32_t* status;
};

// Item -> tile row, first column, width.  Groups of group_m tile rows, tile rows
// fastest inside a group (the dense kernel's order: the tiles in flight cover a
// compact block).
__device__ __forceinline__ void pair_item(const PairParams& p, int item, int& tm, int& n0, int& wide) {
  const int over = item - p.whole;
  const int tile = over < 0 ? item : p.whole + (over >> 1);
  wide = over < 0 ? kPairN : kPairN / 2;
  const int per_group = p.group_m * p.tiles_n;
  const int g = tile / per_group;
  const int rem = tile - g * per_group;
  const int rows = min(p.group_m, p.tiles_m - g * p.group_m);
  tm = g * p.group_m + rem % rows;
  n0 = rem / rows * kPairN + (over >= 0 && (over & 1) != 0 ? kPairN / 2 : 0);
}

template <bool kBF16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    mx_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                   const __grid_constant__ CUtensorMap tm_xs, const __grid_constant__ CUtensorMap tm_ws,
                   const __grid_constant__ CUtensorMap tm_x2, const __grid_constant__ CUtensorMap tm_w2,
                   const PairParams p) {
  using T = typename std::conditional<kBF16, __nv_bfloat16, __half>::type;
  constexpr uint32_t kWOff = kPairOpBytes;
  constexpr uint32_t kXsOff = 2 * kPairOpBytes;
  constexpr uint32_t kWsOff = kXsOff + kSfBytes;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_smem<1024>(smem_raw);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + kPairStages * kPairStageBytes);
  uint64_t* empty_bar = full_bar + kPairStages;
  uint64_t* acc_full = empty_bar + kPairStages;
  uint64_t* acc_empty = acc_full + 1;
  uint64_t* drain_bar = acc_empty + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);

  const uint32_t warp = warp_id();
  const uint32_t lane = lane_id();
  const uint32_t crank = cluster_ctarank();
  const bool lead = crank == 0;
  const int pair = static_cast<int>(blockIdx.x >> 1);
  const int num_pairs = static_cast<int>(gridDim.x >> 1);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) mbar_init(&full_bar[s], 1), mbar_init(&empty_bar[s], 1);
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, 2 * kPairEpiWarps);
    mbar_init(drain_bar, 1);
    fence_mbarrier_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tm_x);
    prefetch_tmap(&tm_w);
    prefetch_tmap(&tm_xs);
    prefetch_tmap(&tm_ws);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, kPairTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();  // both CTAs' barriers initialised and TMEM allocated
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int total_kb = p.num_kb_main + p.num_kb_extra;

  if (warp == 0) {
    if (elect_one()) {
      const uint32_t lead_full = mapa_shared(smem_u32(full_bar), 0);
      uint32_t stage = 0, phase = 0;
      bool armed[kPairStages];
      uint32_t armed_parity[kPairStages];
      for (int s = 0; s < kPairStages; ++s) armed[s] = false, armed_parity[s] = 0;
      bool ok = true;
      // (a row tile past the end lands on rows past the scale table: zeros)
      // (a CTA holds half of an item's columns; of a narrow item's copy, 128 rows
      // too, the second half is not used)
      auto load_w = [&](int kb, int n0, int wide, uint32_t s) {
        uint8_t* st = smem + s * kPairStageBytes;
        const uint32_t bar = lead_full + s * 8u;
        const int row = n0 + static_cast<int>(crank) * (wide / 2);
        if (kb >= p.num_kb_main) {
          tma_load_2d_pair(st + kWOff, &tm_w2, bar, rank_column(kb - p.num_kb_main, p.R), row);
        } else {
          tma_load_2d_pair(st + kWOff, &tm_w, bar, kb * static_cast<int>(kRowBytes), row);
          tma_load_2d_pair(st + kWsOff, &tm_ws, bar, 0, (n0 >> 7) * p.atoms_k + 2 * kb);
          tma_load_2d_pair(st + kWsOff + kSfBytes, &tm_ws, bar, 0,
                           ((n0 >> 7) + 1) * p.atoms_k + 2 * kb);
        }
      };
      auto load_x = [&](int kb, int tm, uint32_t s) {
        uint8_t* st = smem + s * kPairStageBytes;
        const uint32_t bar = lead_full + s * 8u;
        const int m0 = tm * (2 * kHalf) + static_cast<int>(crank) * kHalf;
        if (kb >= p.num_kb_main) {
          tma_load_2d_pair(st, &tm_x2, bar, (kb - p.num_kb_main) * kBK16, m0);
        } else {
          tma_load_2d_pair(st, &tm_x, bar, kb * static_cast<int>(kRowBytes), m0);
          tma_load_2d_pair(st + kXsOff, &tm_xs, bar, 0, (m0 >> 7) * p.atoms_k + 2 * kb);
        }
      };
      auto arm = [&](int kb, uint32_t s, uint32_t parity) {
        if (!lead) return;
        mbar_arrive_expect_tx(&full_bar[s],
                              kb >= p.num_kb_main ? 4 * kPairOpBytes : 2 * kPairStageBytes);
        armed[s] = true;
        armed_parity[s] = parity;
      };
      // W, its scales and W2 do not come from the kernel before this one: the first
      // item's ring of them is on its way before the wait (every pair has an item;
      // what wrote them is through: MxGemmArgs::overlap_prev)
      int tm, n0, wide;
      pair_item(p, pair, tm, n0, wide);
      const int ahead = min(kPairStages, total_kb);
      for (int i = 0; i < ahead; ++i) arm(i, i, 0), load_w(i, n0, wide, i);
      grid_wait();
      for (int i = 0; i < ahead; ++i) load_x(i, tm, i);
      if (ahead == kPairStages) phase = 1;
      stage = ahead == kPairStages ? 0u : static_cast<uint32_t>(ahead);
      for (int item = pair; item < p.num_items && ok; item += num_pairs) {
        pair_item(p, item, tm, n0, wide);
        for (int kb = item == pair ? ahead : 0; kb < total_kb; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1u, p.status, kDevTimeoutEmpty)) {
            ok = false;
            break;
          }
          arm(kb, stage, phase);
          load_x(kb, tm, stage);
          load_w(kb, n0, wide, stage);
          if (++stage == kPairStages) stage = 0, phase ^= 1u;
        }
      }
      for (int s = 0; s < kPairStages; ++s)
        if (armed[s]) mbar_wait(&full_bar[s], armed_parity[s], p.status, kDevTimeoutDrain);
    }
  } else if (warp == 1) {
    if (lead && elect_one()) {
      const uint32_t peer_empty = mapa_shared(smem_u32(empty_bar), 1);
      const uint32_t peer_acc_full = mapa_shared(smem_u32(acc_full), 1);
      uint32_t stage = 0, phase = 0, acc_phase = 0, set = 0;
      bool ok = true;
      for (int item = pair; item < p.num_items && ok; item += num_pairs) {
        const uint32_t wide = item < p.whole ? kPairN : kPairN / 2;
        const uint32_t idesc16 = make_idesc_f16(2 * kHalf, wide, false, false, kBF16);
        const uint32_t idesc4 = make_idesc_mxf4(2 * kHalf, wide, 0);
        if (!mbar_wait(acc_empty, acc_phase ^ 1u, p.status, kDevTimeoutAccEmpty)) break;
        acc_phase ^= 1u;
        tc_fence_after();
        for (int kb = 0; kb < total_kb; ++kb) {
          if (!mbar_wait(&full_bar[stage], phase, p.status, kDevTimeoutFull)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sx = smem_u32(smem + stage * kPairStageBytes);
          const uint32_t sw = sx + kWOff;
          if (kb >= p.num_kb_main) {
            const int nk = min(4, 2 * p.R / 16);
            for (int k = 0; k < nk; ++k)
              umma_f16_pair(tmem, desc_kmajor_sw128(sx, k), desc_kmajor_sw128(sw, rank_step(k, p.R)),
                            idesc16, (kb | k) != 0 ? 1u : 0u);
          } else {
            const uint32_t sfa = tmem + kPairN + set * 32u;
            const uint32_t sfb = sfa + 8u;
            set ^= 1u;
#pragma unroll
            for (int a = 0; a < 2; ++a) {
              tmem_cp_scale_atom_pair(sfa + 4 * a, sx + kXsOff + a * kMxAtomBytes);
              tmem_cp_scale_atom_pair(sfb + 8 * a, sx + kWsOff + a * kMxAtomBytes);
              tmem_cp_scale_atom_pair(sfb + 8 * a + 4, sx + kWsOff + kSfBytes + a * kMxAtomBytes);
            }
            // as in the kernel above: steps that lie past K entirely are left out
            const int nk = min(4, (p.K - kb * kBK4 + 63) / 64);
            for (int k = 0; k < nk; ++k)
              umma_mxf4_pair(tmem, desc_kmajor_sw128(sx, k), desc_kmajor_sw128(sw, k),
                             idesc4 | make_idesc_mxf4(0, 0, 2u * (k & 1)), sfa + 4 * (k >> 1),
                             sfb + 8 * (k >> 1), (kb | k) != 0 ? 1u : 0u);
          }
          umma_commit_pair(smem_u32(&empty_bar[stage]));
          umma_commit_pair(peer_empty + stage * 8u);
          if (++stage == kPairStages) stage = 0, phase ^= 1u;
        }
        if (!ok) break;
        umma_commit_pair(smem_u32(acc_full));
        umma_commit_pair(peer_acc_full);
      }
      umma_commit_pair(smem_u32(drain_bar));
      mbar_wait(drain_bar, 0, p.status, kDevTimeoutDrain);
    }
  } else {
    const uint32_t quarter = warp & 3u;  // TMEM lanes [32 quarter, 32 quarter + 32)
    const int col0 = warp >= 6 ? 128 : 0;
    const uint32_t lead_acc_empty = mapa_shared(smem_u32(acc_empty), 0);
    uint32_t acc_phase = 0;
    for (int item = pair; item < p.num_items; item += num_pairs) {
      int tm, n0, wide;
      pair_item(p, item, tm, n0, wide);
      const int m = tm * (2 * kHalf) + static_cast<int>(crank) * kHalf +
                    static_cast<int>(quarter * 32 + lane);
      n0 += col0;
      if (!mbar_wait(acc_full, acc_phase, p.status, kDevTimeoutAccFull)) break;
      acc_phase ^= 1u;
      __syncwarp();
      tc_fence_after();
      uint32_t r[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        tmem_ld_32x32b_x32(tmem + ((quarter * 32u) << 16) + col0 + c * 32, r[c]);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster_relaxed(lead_acc_empty);
      if (m >= p.M || col0 >= wide) continue;
      T* out = reinterpret_cast<T*>(p.d) + static_cast<long long>(m) * p.ldd + n0;
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int n = c * 32 + q * 16;
          uint32_t v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            v[i] = pack2<T>(__uint_as_float(r[c][q * 16 + 2 * i]),
                            __uint_as_float(r[c][q * 16 + 2 * i + 1]));
          if (p.wide) {
            if (n0 + n < p.N) st_global_32b(out + n, v);
          } else {
            if (n0 + n < p.N)
              *reinterpret_cast<uint4*>(out + n) = make_uint4(v[0], v[1], v[2], v[3]);
            if (n0 + n + 8 < p.N)
              *reinterpret_cast<uint4*>(out + n + 8) = make_uint4(v[4], v[5], v[6], v[7]);
          }
        }
    }
  }

  // After a failure the odd CTA may still have copies in flight that no barrier
  // of its own tracks: give them time to land before the pair exits.
  if (wait_failed(p.status)) {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) {
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // no arrival or copy from the other CTA is still pending
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, kPairTmemCols);
  }
}

// Tensor maps of an fp4 operand: code rows [rows, K/2] and scale atoms.
bool map_codes(CUtensorMap* m, const void* codes, int64_t rows, int64_t K, uint32_t box_rows) {
  return make_tmap_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, codes, static_cast<uint64_t>(K / 2),
                      static_cast<uint64_t>(rows), static_cast<uint64_t>(K / 2), kRowBytes, box_rows,
                      true);
}
bool map_atoms(CUtensorMap* m, const void* atoms, int64_t rows, int64_t K) {
  const uint64_t n = static_cast<uint64_t>(mx_atoms_bytes(rows, K) / kMxAtomBytes);
  return make_tmap_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, atoms, kMxAtomBytes / 4, n, kMxAtomBytes,
                      kMxAtomBytes / 4, 2, false);
}

template <int NT, bool kBF16>
int launch_skinny(const MxGemmArgs& a, cudaStream_t stream) {
  CUtensorMap tw, tx, tws, txs, tw2, tx2;
  if (!map_codes(&tw, a.wq, a.N, a.K, 128) || !map_codes(&tx, a.xq, a.M, a.K, NT) ||
      !map_atoms(&tws, a.ws, a.N, a.K) || !map_atoms(&txs, a.xs, a.M, a.K))
    return MLORA_ERR_INVALID_ARG;
  const int64_t r64 = (2 * a.R + 63) / 64 * 64;
  if (!make_tmap_2d_16b(&tw2, a.w2, a.w2_rows, a.N, a.ldw2, kBK16, 128) ||
      !make_tmap_2d_16b(&tx2, a.x2, r64, a.M, a.ldx2, kBK16, NT))
    return MLORA_ERR_INVALID_ARG;
  SkinnyParams p;
  p.M = static_cast<int>(a.M);
  p.N = static_cast<int>(a.N);
  p.K = static_cast<int>(a.K);
  p.num_kb_main = static_cast<int>((a.K + kBK4 - 1) / kBK4);
  p.R = static_cast<int>(a.R);
  p.num_kb_extra = static_cast<int>((2 * a.R + kBK16 - 1) / kBK16);
  p.atoms_k = static_cast<int>((a.K + 127) / 128);
  p.d = a.d;
  p.ldd = a.ldd;
  p.status = device_status_ptr();
  const int64_t tiles = (a.N + 127) / 128;
  const int64_t slots = (NT <= 32 ? 2 : 1) * static_cast<int64_t>(num_sms());
  int splits = 1;
  while (splits * 2 <= kSkinnyMaxSplits && splits * 2 * tiles <= slots &&
         splits * 4 <= p.num_kb_main + p.num_kb_extra)
    splits *= 2;
  p.splits = splits;
  auto kern = mx_skinny_kernel<NT, kBF16>;
  static std::atomic<bool> attr_set[64];
  if (int rc = set_max_smem(reinterpret_cast<const void*>(kern), skinny_smem(NT), attr_set))
    return rc;
  LaunchScope scope(kKindGemm, stream);
  return launch_status(
      launch_kernel(kern, dim3(static_cast<unsigned>(tiles), static_cast<unsigned>(splits)),
                    kSkinnyThreads, skinny_smem(NT), stream, 1, static_cast<unsigned>(splits),
                    a.overlap_prev, tw, tx, tws, txs, tw2, tx2, p),
      "mx skinny launch");
}

template <bool kBF16>
int launch_pair(const MxGemmArgs& a, cudaStream_t stream) {
  CUtensorMap tx, tw, txs, tws, tx2, tw2;
  if (!map_codes(&tx, a.xq, a.M, a.K, kHalf) || !map_codes(&tw, a.wq, a.N, a.K, kHalf) ||
      !map_atoms(&txs, a.xs, a.M, a.K) || !map_atoms(&tws, a.ws, a.N, a.K))
    return MLORA_ERR_INVALID_ARG;
  const int64_t r64 = (2 * a.R + 63) / 64 * 64;
  if (!make_tmap_2d_16b(&tx2, a.x2, r64, a.M, a.ldx2, kBK16, kHalf) ||
      !make_tmap_2d_16b(&tw2, a.w2, a.w2_rows, a.N, a.ldw2, kBK16, kHalf))
    return MLORA_ERR_INVALID_ARG;
  PairParams p;
  p.M = static_cast<int>(a.M);
  p.N = static_cast<int>(a.N);
  p.K = static_cast<int>(a.K);
  p.num_kb_main = static_cast<int>((a.K + kBK4 - 1) / kBK4);
  p.R = static_cast<int>(a.R);
  p.num_kb_extra = static_cast<int>((2 * a.R + kBK16 - 1) / kBK16);
  p.tiles_m = static_cast<int>((a.M + 2 * kHalf - 1) / (2 * kHalf));
  p.tiles_n = static_cast<int>((a.N + kPairN - 1) / kPairN);
  p.group_m = p.tiles_m < 8 ? p.tiles_m : 8;
  p.atoms_k = static_cast<int>((a.K + 127) / 128);
  p.d = a.d;
  p.ldd = a.ldd;
  // (N and ldd are multiples of 8 and d starts on 16 bytes: the caller's checks)
  p.wide = a.N % 16 == 0 && a.ldd % 16 == 0 && reinterpret_cast<uintptr_t>(a.d) % 32 == 0;
  p.status = device_status_ptr();
  auto kern = mx_pair_kernel<kBF16>;
  static std::atomic<int> max_pairs[64];
  int dev = 0;
  cudaGetDevice(&dev);
  int pairs = dev < 64 ? max_pairs[dev].load(std::memory_order_acquire) : 0;
  if (pairs == 0) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(kPairSmem));
    if (e != cudaSuccess) return launch_status(e, "cudaFuncSetAttribute(mx pair)");
    // clusters that can be resident at once (GPCs may leave an SM unpaired)
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(num_sms() / 2 * 2));
    cfg.blockDim = dim3(kPairThreads);
    cfg.dynamicSmemBytes = kPairSmem;
    if (cudaOccupancyMaxActiveClusters(&pairs, kern, &cfg) != cudaSuccess || pairs <= 0) {
      cudaGetLastError();
      pairs = num_sms() / 2;
    }
    if (dev < 64) max_pairs[dev].store(pairs, std::memory_order_release);
  }
  // The tiles of the last wave go in halves of 128 columns where the pairs left
  // without one can take them (256 tokens 4096 -> 4096: 17.5 us whole, 16.6 in
  // halves; 512 tokens 4096 -> 11008: 25.7 and 24.6).  With more of them than that,
  // some pairs would take two halves, 1.1 of a tile's time.
  const int tiles = p.tiles_m * p.tiles_n, last = tiles % pairs;
  p.whole = 2 * last <= pairs ? tiles - last : tiles;
  p.num_items = p.whole + 2 * (tiles - p.whole);
  const int grid = 2 * (p.num_items < pairs ? p.num_items : pairs);
  LaunchScope scope(kKindGemm, stream);
  return launch_status(launch_kernel(kern, dim3(static_cast<unsigned>(grid)), kPairThreads, kPairSmem,
                                     stream, 0, 0, a.overlap_prev, tx, tw, txs, tws, tx2, tw2, p),
                       "mx pair launch");
}

template <bool kBF16>
int dispatch(const MxGemmArgs& a, cudaStream_t s) {
  if (a.M <= 16) return launch_skinny<16, kBF16>(a, s);
  if (a.M <= 32) return launch_skinny<32, kBF16>(a, s);
  if (a.M <= 64) return launch_skinny<64, kBF16>(a, s);
  if (a.M <= 128) return launch_skinny<128, kBF16>(a, s);
  return launch_pair<kBF16>(a, s);
}

}  // namespace

int launch_mx_gemm(const MxGemmArgs& a, cudaStream_t s) {
  // scale atoms are addressed by a 32-bit tensor-map row
  const int64_t most = (int64_t(1) << 31) * kMxAtomBytes;
  if (mx_atoms_bytes(a.M, a.K) >= most || mx_atoms_bytes(a.N, a.K) >= most) {
    set_error("MXFP4 product: an operand has more than 2^31 blocks of 128 x 128");
    return MLORA_ERR_UNSUPPORTED;
  }
  return a.elt == Elt::kBF16 ? dispatch<true>(a, s) : dispatch<false>(a, s);
}

}  // namespace mlora
