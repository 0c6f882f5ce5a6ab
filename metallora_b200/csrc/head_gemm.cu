// The three products of a vocabulary head, as one persistent tcgen05 kernel over
// CTA pairs:
//
//   logits  l[m, v] = sum_k x[m, k] W[v, k]   (+ X2[m, :] . B[v, :])   both K-major
//   dx      D[k, m] = sum_v W[v, k] g[m, v]   (+ A[:, k] . U[m, :])    W MN-major
//   dW      D[v, k] = sum_m g[m, v] x[m, k]                            both MN-major
//
// and the LoRA linear with dropout, y = x . W^T + drop(X2 . B^T), both K-major.
//
// The logits never go to memory as such.  The epilogue takes, of each row's 128 in half
// a tile, a reference n_t and s_t = sum exp(l) 2^-n_t, and where a gradient is wanted
// writes the exponentials exp(l) 2^-n_t in 16 bits.  Two forms:
//   * bf16 hidden states behind a frozen head: n_t is one whole number for the whole row,
//     the label's logit in units of log 2.  bf16 has the range for it, and a factor of
//     a row of g can be left to the gradient of x: the exponentials are the operand of
//     dx as they are.  A half row whose sum passes 2^90 (logits 60 above the label's)
//     takes a reference of its own; a power of two apart, so that bringing the row to
//     one reference rounds nothing;
//   * else n_t is the half row's largest logit, and the exponentials are fp16 values:
//     11 bits of a number in (0, 1], so that of g, which a pass over them makes, only
//     the rounding to its 16 bits shows.
// The label's own logit is left out (as -inf): it comes in 32 bits from the pass that
// gathers x, since the tensor cores' accumulation rounds toward zero at each of its
// K / 16 steps, which a loss shows as it is.  Of the other logits that cut is given back
// on average: it measured 1.0e-9 K of the value (0.24e-6 at K = 256, 4.0e-6 at 4096,
// 8.4e-6 at 8192; its deviation a tenth to a half of that) for sums that drift or walk
// to where they end, 3.5 (bf16) to 6.3 (fp16) times as much where every product has the
// same sign, nothing where the sums are exact.  A step that adds zeros cuts nothing, so a
// row's features count by the groups of 8 that are not all zero, and beyond the 8192 that
// were measured no more is given back: where nothing was cut a logit is off by 1.0e-9 K of
// itself, 8.2e-6 at most, and where most was by 5.3e-9 K.  (Loss of 512 tokens at 4096
// features against 64 bits 0.7e-7, without 12e-7.)
//
// A (2,1,1) cluster makes a 256 x 256 tile (tcgen05.mma.cta_group::2, M = N = 256,
// K = 16): each CTA stages its own 128 rows of either operand in a 6-stage TMA ring
// and holds its own 128 rows of the fp32 accumulator, two of them in TMEM, so that
// the epilogue of one tile runs beside the main loop of the next.  The roles of the
// warps are those of the LoRA GEMM (tc_gemm.cu).  What is new here:
//   * a tile may have fewer columns (a multiple of 32, which the instruction's time goes
//     by): those of the logits so that whole waves of tiles cover the vocabulary, those of
//     dx, whose columns are the tokens, as many as the counted ones need (412 tokens are
//     two tiles of 224 columns, not two of 256 rows);
//   * the number of counted tokens is read on the device: it bounds the rows of D
//     (logits), its columns (dx) or the reduction (dW), so that tokens that do not count cost
//     nothing and no host waits for their number;
//   * the reduction can be cut into `splits` ranges, each with its own fp32 copy of D
//     (dx of few tokens has few tiles and a reduction over the whole vocabulary);
//     whoever reads D adds the copies in order.
// Bound: the tensor pipe; by HBM (one read of W) below some 250 tokens.
#include <atomic>
#include <string>

#include "internal.h"
#include "launch.cuh"
#include "philox.cuh"
#include "ptx.cuh"
#include "../../include/metallora_b200.h"

namespace mlora {
namespace {

// What a tile becomes: fp32 sums, as they lie or with D's columns as rows; logits by their row's reference or by the half row's
// largest; the LoRA linear with dropout.
enum class Form { kSums, kTransposed, kRowRef, kTop, kDropout };

constexpr int kBK = 64;
constexpr int kHalf = 128;  // rows of either operand per CTA
constexpr int kTile = 2 * kHalf;
constexpr int kStages = 6;
constexpr uint32_t kOpBytes = kHalf * kBK * 2;      // 16 KB
constexpr uint32_t kStageBytes = 2 * kOpBytes;
constexpr uint32_t kMNBoxBytes = 64 * kBK * 2;      // one MN-major TMA box (8 KB)
constexpr int kEpiWarps = 8;  // two for each quarter of the lanes: 128 columns each
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr uint32_t kTmemCols = 512;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRowLimit = 1.2379400392853803e27f;  // 2^90
constexpr size_t kSmemBytes = 1024 + kStages * kStageBytes + 256;

struct HeadGemmParams {
  int M, N;  // of D; at most, where `rows` bounds them
  int num_kb_main, num_kb_extra, R;
  int tile_n;  // columns of a tile (kTransposed: by the counted tokens)
  int splits, group_m;
  const int32_t* rows;  // counted tokens (device), of which those from row0 on are meant
  int row0;
  float* d;
  long long ldd, split_stride;
  int accumulate;
  // logits
  const int32_t* label;  // of row m
  const float* ref;      // of row m: n_t (first form)
  const float* uncut;    // what row m's logits are multiplied by
  uint16_t* e;           // the exponentials (second form: times 2^15), rows ldd apart, or nullptr
  DropoutKey drop;       // of the LoRA term, over [M, N] in a row
  void* d16;             // output of kDropout
  float2* stats;         // (n_t, s_t), second form (m_t, 2^15 s_t), of the t-th half tile at
  long long stats_ld;    // [m * stats_ld + t]
  uint32_t* status;
};

struct Shape {
  int M, N, num_kb, tile_n, tiles_m, tiles_n, num_tiles, units;
};

// kRows: what the counted tokens bound.
enum class Bound { kRows, kColumns, kReduction };

template <Bound kBound>
__device__ __forceinline__ Shape device_shape(const HeadGemmParams& p) {
  Shape s;
  s.M = p.M;
  s.N = p.N;
  s.num_kb = p.num_kb_main;
  s.tile_n = p.tile_n;
  if (p.rows != nullptr) {
    const int n = max(*p.rows - p.row0, 0);
    if (kBound == Bound::kReduction)
      s.num_kb = min(s.num_kb, (n + kBK - 1) / kBK);
    else if (kBound == Bound::kRows)
      s.M = min(s.M, n);
    else
      s.N = min(s.N, n);
  }
  s.tiles_m = (s.M + kTile - 1) / kTile;
  s.tiles_n = (s.N + s.tile_n - 1) / s.tile_n;
  if (kBound == Bound::kColumns && s.tiles_n > 0)  // the same number, as narrow as can be
    s.tile_n = ((s.N + s.tiles_n - 1) / s.tiles_n + 31) / 32 * 32;
  s.num_tiles = s.tiles_m * s.tiles_n;
  s.units = s.num_tiles * p.splits;
  return s;
}

// One unit of work: a tile of D and a range of the reduction.  Tile rows vary
// fastest inside groups of group_m of them, so that the tiles in flight cover a
// compact block of D and share their operands in L2.
struct Unit {
  int tm, tn, split, kb0, kb1, total;
};

__device__ __forceinline__ Unit unit_at(const HeadGemmParams& p, const Shape& s, int u) {
  Unit t;
  // the end of the reduction first: of the weight that the logits have just read, L2
  // still holds that (16 tokens 4096 -> 32000: 50.6 -> 49.4 us)
  t.split = p.splits - 1 - u / s.num_tiles;
  const int tile = u % s.num_tiles;
  const int per_group = p.group_m * s.tiles_n;
  const int g = tile / per_group;
  const int rem = tile - g * per_group;
  const int rows = min(p.group_m, s.tiles_m - g * p.group_m);
  t.tm = g * p.group_m + rem % rows;
  t.tn = rem / rows;
  t.kb0 = static_cast<int>(static_cast<long long>(s.num_kb) * t.split / p.splits);
  t.kb1 = static_cast<int>(static_cast<long long>(s.num_kb) * (t.split + 1) / p.splits);
  t.total = t.kb1 - t.kb0 + (t.split == 0 ? p.num_kb_extra : 0);
  return t;
}

// This thread's half row of the accumulator (128 columns from n0) into D, 32 bytes at a
// time.
__device__ __forceinline__ void store_row_f32(const HeadGemmParams& p, const Shape& s,
                                              const Unit& t, int m, int n0, uint32_t taddr) {
  float* row = p.d + t.split * p.split_stride + static_cast<long long>(m) * p.ldd + n0;
#pragma unroll 1
  for (int c = 0; c < kHalf; c += 32) {
    uint32_t r[32];
    tmem_ld_32x32b_x32(taddr + c, r);
    tmem_ld_wait();
    if (m >= s.M) continue;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (n0 + c + q * 8 >= p.N) continue;
      float* dst = row + c + q * 8;
      uint32_t v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = t.total > 0 ? r[q * 8 + i] : 0u;
      if (p.accumulate) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float4 o = *reinterpret_cast<const float4*>(dst + 4 * h);
          v[4 * h] = __float_as_uint(__uint_as_float(v[4 * h]) + o.x);
          v[4 * h + 1] = __float_as_uint(__uint_as_float(v[4 * h + 1]) + o.y);
          v[4 * h + 2] = __float_as_uint(__uint_as_float(v[4 * h + 2]) + o.z);
          v[4 * h + 3] = __float_as_uint(__uint_as_float(v[4 * h + 3]) + o.w);
        }
      }
      st_global_32b(dst, v);
    }
  }
}

// This thread's row m of the accumulator as a column of the output: D's column n, a
// token, is a row there, and a warp's 32 values of it lie side by side.
__device__ __forceinline__ void store_column_f32(const HeadGemmParams& p, const Shape& s,
                                                 const Unit& t, int m, int n0, uint32_t taddr) {
  const int width = min(s.tile_n / 2, s.N - n0);
  float* dst = p.d + t.split * p.split_stride + static_cast<long long>(n0) * p.ldd + m;
#pragma unroll 1
  for (int c = 0; c < width; c += 32) {
    uint32_t r[32];
    tmem_ld_32x32b_x32(taddr + c, r);
    tmem_ld_wait();
    if (m >= s.M) continue;
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (c + i < width) dst[(c + i) * p.ldd] = __uint_as_float(r[i]);
  }
}

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Logits past the half row or the vocabulary, and the label's, count as -inf (`any`:
// there is a label among the warp's).
__device__ __forceinline__ void mask_logits(uint32_t (&r)[32], int c, int width, int y, bool any) {
  if (!any && c + 32 <= width) return;
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (c + i >= width || c + i == y) r[i] = __float_as_uint(-INFINITY);
}

// First form: this thread's half row of a tile of logits (up to 128 entries from n0).  One
// pass with the row's reference; the largest logit is only looked for where it fails, and
// the half row written again.
template <typename Release>
__device__ __forceinline__ void softmax_row_ref(const HeadGemmParams& p, const Shape& s, int m,
                                                int n0, uint32_t taddr, Release&& release) {
  if (n0 >= p.N) {  // past the vocabulary: no statistics, nothing to write
    release();
    return;
  }
  const bool live = m < s.M;
  const int y = live ? p.label[m] - n0 : -1;
  float n = live ? p.ref[m] : 0.f;
  const int half = s.tile_n / 2, width = min(half, p.N - n0);  // columns that are there
  const bool any = __any_sync(0xffffffffu, static_cast<uint32_t>(y) < static_cast<uint32_t>(width));
  const float log2e = kLog2e * (live ? p.uncut[m] : 1.f);
  uint16_t* const row =
      live && p.e != nullptr ? p.e + static_cast<long long>(m) * p.ldd + n0 : nullptr;
  float sum = 0.f;
  auto exponentials = [&] {
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t r[2][32];
      tmem_ld_32x32b_x32(taddr + h * 64, r[0]);
      tmem_ld_32x32b_x32(taddr + h * 64 + 32, r[1]);
      tmem_ld_wait();
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        mask_logits(r[c], h * 64 + c * 32, width, y, any);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float a = ex2(fmaf(__uint_as_float(r[c][16 * q + 2 * i]), log2e, -n));
            const float b = ex2(fmaf(__uint_as_float(r[c][16 * q + 2 * i + 1]), log2e, -n));
            s0 += a;
            s1 += b;
            v[i] = pack2<__nv_bfloat16>(a, b);
          }
          const int col = h * 64 + c * 32 + q * 16;
          if (row != nullptr && col < half && n0 + col < p.ldd) st_global_32b(row + col, v);
        }
      }
    }
    sum = s0 + s1;
  };
  exponentials();
  const bool over = live && !(sum <= kRowLimit);
  if (__any_sync(0xffffffffu, over)) {
    float top = -INFINITY;
#pragma unroll 1
    for (int c = 0; c < kHalf; c += 32) {
      uint32_t r[32];
      tmem_ld_32x32b_x32(taddr + c, r);
      tmem_ld_wait();
      mask_logits(r, c, width, y, any);
#pragma unroll
      for (int i = 0; i < 32; ++i) top = fmaxf(top, __uint_as_float(r[i]));
    }
    if (over) n = fmaxf(n, ceilf(top * log2e));  // infinite: the sum becomes NaN
    exponentials();
  }
  release();
  if (live) p.stats[static_cast<long long>(m) * p.stats_ld + n0 / half] = make_float2(n, sum);
}

// Second form: all of the half row in registers: largest, exponentials, their sum.  `release` hands the accumulator back
// before the arithmetic, so that the main loop two tiles on does not wait for it.
template <typename Release>
__device__ __forceinline__ void softmax_row(const HeadGemmParams& p, const Shape& s, int m, int n0,
                                            uint32_t taddr, Release&& release) {
  if (n0 >= p.N) {  // past the vocabulary: no statistics, nothing to write
    release();
    return;
  }
  uint32_t r[4][32];
#pragma unroll
  for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(taddr + c * 32, r[c]);
  const bool live = m < s.M;
  const int y = live ? p.label[m] - n0 : -1;
  const float uncut = live ? p.uncut[m] : 1.f;
  const int half = s.tile_n / 2, width = min(half, p.N - n0);  // columns that are there
  tmem_ld_wait();
  release();
  const bool any = __any_sync(0xffffffffu, static_cast<uint32_t>(y) < static_cast<uint32_t>(width));
#pragma unroll
  for (int c = 0; c < 4; ++c) mask_logits(r[c], c * 32, width, y, any);
  float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      t0 = fmaxf(t0, __uint_as_float(r[c][i]));
      t1 = fmaxf(t1, __uint_as_float(r[c][i + 1]));
    }
  const float top = fmaxf(t0, t1);
  const float ref = top == -INFINITY ? 0.f : top;
  const float log2e = kLog2e * uncut;
  float sum0 = 0.f, sum1 = 0.f;
  uint16_t* row = p.e + static_cast<long long>(m) * p.ldd + n0;
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    uint32_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // the difference first: exact near the top, where it counts
      const float a = ex2(fmaf(__uint_as_float(r[c / 2][16 * (c & 1) + 2 * i]) - ref, log2e, 15.f));
      const float b =
          ex2(fmaf(__uint_as_float(r[c / 2][16 * (c & 1) + 2 * i + 1]) - ref, log2e, 15.f));
      sum0 += a;
      sum1 += b;
      v[i] = pack2<__half>(a, b);
    }
    if (live && p.e != nullptr && c * 16 < half && n0 + c * 16 < p.ldd)
      st_global_32b(row + c * 16, v);
  }
  if (live)
    p.stats[static_cast<long long>(m) * p.stats_ld + n0 / half] =
        make_float2(top * uncut, sum0 + sum1);
}

// The LoRA linear with dropout.  The LoRA term has the second accumulator, so that a
// tile's epilogue does not run beside the next one's main loop; but the mask, most of
// its work, needs no accumulator and is made ahead: a bit for each of this thread's 128
// columns from n0, eight to a call of the generator.  (Tiles of 128 columns, two of both
// accumulators in TMEM, moved half as much again from L2 and took 160 us where this
// takes 129: 4096 tokens 4096 -> 4096.)
__device__ __forceinline__ void dropout_bits(const HeadGemmParams& p, const PhiloxKeys& keys, int m,
                                             int n0, uint32_t (&bits)[4]) {
  const int64_t first = (static_cast<int64_t>(m) * p.N + n0) / 8;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    bits[c] = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint64_t at = static_cast<uint64_t>(first + c * 4 + q);
      bits[c] |= kept_bits(philox4x32_10(keys, at, p.drop.call), p.drop.threshold) << (8 * q);
    }
  }
}

template <typename T, typename Release>
__device__ __forceinline__ void dropout_row(const HeadGemmParams& p, const Shape& s, int m, int n0,
                                            uint32_t taddr, const uint32_t (&bits)[4],
                                            Release&& release) {
  T* row = static_cast<T*>(p.d16) + static_cast<long long>(m) * p.ldd + n0;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t base[32], lora[32], out[16];
    tmem_ld_32x32b_x32(taddr + c * 32, base);
    tmem_ld_32x32b_x32(taddr + kTile + c * 32, lora);
    tmem_ld_wait();
    if (c == 3) release();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float z0 = (bits[c] >> (2 * i)) & 1u ? __uint_as_float(lora[2 * i]) : 0.f;
      const float z1 = (bits[c] >> (2 * i + 1)) & 1u ? __uint_as_float(lora[2 * i + 1]) : 0.f;
      out[i] = pack2<T>(__uint_as_float(base[2 * i]) + z0, __uint_as_float(base[2 * i + 1]) + z1);
    }
    if (m >= s.M) continue;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (n0 + c * 32 + q * 8 < p.N)
        *reinterpret_cast<uint4*>(row + c * 32 + q * 8) =
            make_uint4(out[4 * q], out[4 * q + 1], out[4 * q + 2], out[4 * q + 3]);
  }
}

template <bool kXMN, bool kWMN, bool kBF16, Form kForm>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    head_gemm_kernel(const __grid_constant__ CUtensorMap tm_x,
                     const __grid_constant__ CUtensorMap tm_w,
                     const __grid_constant__ CUtensorMap tm_x2,
                     const __grid_constant__ CUtensorMap tm_w2, const HeadGemmParams p) {
  constexpr bool kOneTile = kForm == Form::kDropout;  // both accumulators are a tile's
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_smem<1024>(smem_raw);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + kStages * kStageBytes);
  uint64_t* empty_bar = full_bar + kStages;
  uint64_t* acc_full = empty_bar + kStages;  // [2]
  uint64_t* acc_empty = acc_full + 2;        // [2]
  uint64_t* drain_bar = acc_empty + 2;       // [1]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);

  const uint32_t warp = warp_id();
  const uint32_t lane = lane_id();
  const uint32_t crank = cluster_ctarank();
  const bool lead = crank == 0;
  const int pair = static_cast<int>(blockIdx.x >> 1);
  const int num_pairs = static_cast<int>(gridDim.x >> 1);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * kEpiWarps);
    }
    mbar_init(drain_bar, 1);
    fence_mbarrier_init();
    prefetch_tmap(&tm_x);
    prefetch_tmap(&tm_w);
    if (p.num_kb_extra > 0) {
      prefetch_tmap(&tm_x2);
      prefetch_tmap(&tm_w2);
    }
  }
  __syncwarp();  // the allocation below is a warp-wide instruction
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();  // both CTAs' barriers initialised and TMEM allocated
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  grid_wait();  // every operand but the weight is the kernels' before; in every role
  launch_dependents();
  constexpr Bound kBound = kForm == Form::kTransposed ? Bound::kColumns
                           : kForm == Form::kSums     ? Bound::kReduction
                                                      : Bound::kRows;
  const Shape shape = device_shape<kBound>(p);
  const int half_n = shape.tile_n / 2;

  if (warp == 0) {
    // ------------------------------------------------------------ producer --
    if (elect_one()) {
      const uint32_t lead_full = mapa_shared(smem_u32(full_bar), 0);
      uint32_t stage = 0, phase = 0;
      uint32_t armed_parity[kStages];
      bool armed[kStages];
      for (int s = 0; s < kStages; ++s) armed[s] = false, armed_parity[s] = 0;
      bool ok = true;
      for (int u = pair; u < shape.units && ok; u += num_pairs) {
        const Unit t = unit_at(p, shape, u);
        const int m0 = t.tm * kTile + static_cast<int>(crank) * kHalf;
        const int n0 = t.tn * shape.tile_n + static_cast<int>(crank) * half_n;
        const int main_kb = t.kb1 - t.kb0;
        for (int i = 0; i < t.total; ++i) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1u, p.status, kDevTimeoutEmpty)) {
            ok = false;
            break;
          }
          uint8_t* sx = smem + stage * kStageBytes;
          uint8_t* sw = sx + kOpBytes;
          if (lead) {
            mbar_arrive_expect_tx(&full_bar[stage], 2 * kStageBytes);
            armed[stage] = true;
            armed_parity[stage] = phase;
          }
          const uint32_t bar = lead_full + stage * 8u;
          const bool extra = i >= main_kb;
          const CUtensorMap* mx = extra ? &tm_x2 : &tm_x;
          const CUtensorMap* mw = extra ? &tm_w2 : &tm_w;
          const int k0 = (extra ? i - main_kb : t.kb0 + i) * kBK;
          if constexpr (kXMN) {
            tma_load_2d_pair(sx, mx, bar, m0, k0);
            tma_load_2d_pair(sx + kMNBoxBytes, mx, bar, m0 + 64, k0);
          } else {
            tma_load_2d_pair(sx, mx, bar, k0, m0);
          }
          if constexpr (kWMN) {
            tma_load_2d_pair(sw, mw, bar, n0, k0);
            tma_load_2d_pair(sw + kMNBoxBytes, mw, bar, n0 + 64, k0);
          } else {
            tma_load_2d_pair(sw, mw, bar, k0, n0);
          }
          if (++stage == kStages) stage = 0, phase ^= 1u;
        }
      }
      // Never leave a copy in flight at exit (the even CTA's barriers count
      // both CTAs' bytes).
      for (int s = 0; s < kStages; ++s)
        if (armed[s]) mbar_wait(&full_bar[s], armed_parity[s], p.status, kDevTimeoutDrain);
    }
  } else if (warp == 1) {
    // ------------------------------------------------- MMA (even CTA only) --
    if (lead && elect_one()) {
      const uint32_t idesc =
          make_idesc_f16(kTile, static_cast<uint32_t>(shape.tile_n), kXMN, kWMN, kBF16);
      const uint32_t peer_empty = mapa_shared(smem_u32(empty_bar), 1);
      const uint32_t peer_acc_full = mapa_shared(smem_u32(acc_full), 1);
      uint32_t stage = 0, phase = 0;
      int local = 0;
      bool ok = true;
      for (int u = pair; u < shape.units && ok; u += num_pairs, ++local) {
        const Unit t = unit_at(p, shape, u);
        const int main_kb = t.kb1 - t.kb0;
        const uint32_t buf = kOneTile ? 0 : local & 1;
        const uint32_t use = static_cast<uint32_t>(kOneTile ? local : local >> 1) & 1u;
        if (!mbar_wait(&acc_empty[buf], use ^ 1u, p.status, kDevTimeoutAccEmpty)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + buf * kTile;
        for (int i = 0; i < t.total; ++i) {
          if (!mbar_wait(&full_bar[stage], phase, p.status, kDevTimeoutFull)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sx = smem_u32(smem + stage * kStageBytes);
          const uint32_t sw = sx + kOpBytes;
          int nk = 4;
          if (i >= main_kb) {
            const int rem = p.R - (i - main_kb) * kBK;
            nk = rem >= kBK ? 4 : rem / 16;
          }
          for (int k = 0; k < nk; ++k) {
            const uint64_t ad = kXMN ? desc_mnmajor_sw128(sx, k, kMNBoxBytes)
                                     : desc_kmajor_sw128(sx, k);
            const uint64_t bd = kWMN ? desc_mnmajor_sw128(sw, k, kMNBoxBytes)
                                     : desc_kmajor_sw128(sw, k);
            if (kForm == Form::kDropout && i >= main_kb)  // the LoRA term's own accumulator
              umma_f16_pair(d_tmem + kTile, ad, bd, idesc, i > main_kb || k != 0 ? 1u : 0u);
            else
              umma_f16_pair(d_tmem, ad, bd, idesc, (i | k) != 0 ? 1u : 0u);
          }
          umma_commit_pair(smem_u32(&empty_bar[stage]));
          umma_commit_pair(peer_empty + stage * 8u);
          if (++stage == kStages) stage = 0, phase ^= 1u;
        }
        if (!ok) break;
        umma_commit_pair(smem_u32(&acc_full[buf]));
        umma_commit_pair(peer_acc_full + buf * 8u);
      }
      // Drain: every MMA issued above has completed before TMEM is released.
      umma_commit_pair(smem_u32(drain_bar));
      mbar_wait(drain_bar, 0, p.status, kDevTimeoutDrain);
    }
  } else {
    // ----------------------------------------------------------- epilogue --
    const uint32_t quarter = warp & 3u;  // TMEM lanes [32*quarter, 32*quarter+32)
    const uint32_t half = (warp - 2u) >> 2;  // of the tile's columns
    const uint32_t lead_acc_empty = mapa_shared(smem_u32(acc_empty), 0);
    __shared__ PhiloxKeys keys;  // of the seed in memory, where there is one
    if constexpr (kForm == Form::kDropout) {
      if (threadIdx.x == 64)
        keys = p.drop.seed_dev != nullptr ? philox_keys(static_cast<uint64_t>(*p.drop.seed_dev))
                                          : p.drop.keys;
      named_bar_sync(1, kEpiWarps * 32);
    }
    int local = 0;
    for (int u = pair; u < shape.units; u += num_pairs, ++local) {
      const Unit t = unit_at(p, shape, u);
      const uint32_t buf = kOneTile ? 0 : local & 1;
      const uint32_t use = static_cast<uint32_t>(kOneTile ? local : local >> 1) & 1u;
      const int m = t.tm * kTile + static_cast<int>(crank * kHalf + quarter * 32 + lane);
      const int n0 = t.tn * shape.tile_n + static_cast<int>(half) * half_n;
      uint32_t bits[4];
      if constexpr (kForm == Form::kDropout) dropout_bits(p, keys, m, n0, bits);
      if (!mbar_wait(&acc_full[buf], use, p.status, kDevTimeoutAccFull)) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((quarter * 32u) << 16) + buf * kTile + half * half_n;
      // the arrival orders no memory: only the TMEM loads, complete by then, came before
      auto release = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(lead_acc_empty + buf * 8u);
      };
      if constexpr (kForm == Form::kRowRef)
        softmax_row_ref(p, shape, m, n0, taddr, release);
      else if constexpr (kForm == Form::kTop)
        softmax_row(p, shape, m, n0, taddr, release);
      else if constexpr (kForm == Form::kDropout)
        dropout_row<typename std::conditional<kBF16, __nv_bfloat16, __half>::type>(
            p, shape, m, n0, taddr, bits, release);
      else {
        if constexpr (kForm == Form::kTransposed)
          store_column_f32(p, shape, t, m, n0, taddr);
        else
          store_row_f32(p, shape, t, m, n0, taddr);
        release();
      }
    }
  }

  // After a failure the odd CTA may still have copies in flight that no
  // barrier of its own tracks: give them time to land before the pair exits.
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
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

template <bool kXMN, bool kWMN, bool kBF16, Form kForm>
int launch_typed(const HeadGemmArgs& a, cudaStream_t stream) {
  CUtensorMap tx, tw, tx2, tw2;
  if (kXMN ? !make_tmap_2d_16b(&tx, a.x, a.M, a.K, a.ldx, 64, kBK)
           : !make_tmap_2d_16b(&tx, a.x, a.K, a.M, a.ldx, kBK, kHalf))
    return MLORA_ERR_INVALID_ARG;
  if (kWMN ? !make_tmap_2d_16b(&tw, a.w, a.N, a.K, a.ldw, 64, kBK)
           : !make_tmap_2d_16b(&tw, a.w, a.K, a.N, a.ldw, kBK, kHalf))
    return MLORA_ERR_INVALID_ARG;
  tx2 = tx;
  tw2 = tw;
  if (a.R > 0) {
    const int64_t r64 = (a.R + 63) / 64 * 64;
    if (kXMN ? !make_tmap_2d_16b(&tx2, a.x2, a.M, a.x2_rows, a.ldx2, 64, kBK)
             : !make_tmap_2d_16b(&tx2, a.x2, r64, a.M, a.ldx2, kBK, kHalf))
      return MLORA_ERR_INVALID_ARG;
    if (kWMN ? !make_tmap_2d_16b(&tw2, a.w2, a.N, a.w2_rows, a.ldw2, 64, kBK)
             : !make_tmap_2d_16b(&tw2, a.w2, a.w2_rows, a.N, a.ldw2, kBK, kHalf))
      return MLORA_ERR_INVALID_ARG;
  }
  HeadGemmParams p;
  p.M = static_cast<int>(a.M);
  p.N = static_cast<int>(a.N);
  p.num_kb_main = static_cast<int>((a.K + kBK - 1) / kBK);
  p.R = static_cast<int>(a.R);
  p.num_kb_extra = static_cast<int>((a.R + kBK - 1) / kBK);
  const int tiles_m = static_cast<int>((a.M + kTile - 1) / kTile);
  p.tile_n = a.tile_n;
  const int tiles_n = static_cast<int>((a.N + a.tile_n - 1) / a.tile_n);
  p.splits = a.splits;
  p.group_m = a.group_m < tiles_m ? a.group_m : tiles_m;
  p.rows = a.rows;
  p.row0 = static_cast<int>(a.row0);
  p.d = a.d;
  p.ldd = a.ldd;
  p.split_stride = a.split_stride;
  p.accumulate = a.accumulate ? 1 : 0;
  p.label = a.label;
  p.ref = a.ref;
  if (a.drop != nullptr) p.drop = *a.drop;
  p.d16 = a.d16;
  p.e = static_cast<uint16_t*>(a.e);
  p.stats = static_cast<float2*>(a.stats);
  p.stats_ld = a.stats_ld;
  p.uncut = a.uncut;
  p.status = device_status_ptr();

  auto kern = head_gemm_kernel<kXMN, kWMN, kBF16, kForm>;
  static std::atomic<bool> attr_set[64];
  if (int rc = set_max_smem(reinterpret_cast<const void*>(kern), kSmemBytes, attr_set)) return rc;
  const int64_t units = int64_t{tiles_m} * tiles_n * p.splits;
  const int pairs = head_gemm_pairs();
  const int grid = 2 * static_cast<int>(units < pairs ? units : pairs);
  LaunchScope scope(kKindGemm, stream);
  return launch_status(launch_kernel(kern, dim3(static_cast<unsigned>(grid)), kThreads, kSmemBytes,
                                     stream, 0, 0, true, tx, tw, tx2, tw2, p),
                       "head gemm launch");
}

}  // namespace

int head_gemm_pairs() {
  static std::atomic<int> known[64];
  int dev = 0;
  cudaGetDevice(&dev);
  int n = dev < 64 ? known[dev].load(std::memory_order_acquire) : 0;
  if (n > 0) return n;
  // clusters that can be resident at once (GPCs may leave an SM unpaired)
  const int pairs = num_sms() / 2;
  auto kern = head_gemm_kernel<false, false, true, Form::kTop>;
  static std::atomic<bool> attr_set[64];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  if (set_max_smem(reinterpret_cast<const void*>(kern), kSmemBytes, attr_set) != MLORA_OK ||
      cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    n = pairs;
  }
  if (n > pairs) n = pairs;
  if (dev < 64) known[dev].store(n, std::memory_order_release);
  return n;
}

int launch_head_gemm(const HeadGemmArgs& a, cudaStream_t s) {
  const bool bf16 = a.elt == Elt::kBF16;
  switch (a.product) {
    case HeadProduct::kLogits:
      if (a.ref != nullptr) return launch_typed<false, false, true, Form::kRowRef>(a, s);
      return bf16 ? launch_typed<false, false, true, Form::kTop>(a, s)
                  : launch_typed<false, false, false, Form::kTop>(a, s);
    case HeadProduct::kDx:
      return bf16 ? launch_typed<true, false, true, Form::kTransposed>(a, s)
                  : launch_typed<true, false, false, Form::kTransposed>(a, s);
    case HeadProduct::kDw:
      return bf16 ? launch_typed<true, true, true, Form::kSums>(a, s)
                  : launch_typed<true, true, false, Form::kSums>(a, s);
    case HeadProduct::kLoraDropout:
      return bf16 ? launch_typed<false, false, true, Form::kDropout>(a, s)
                  : launch_typed<false, false, false, Form::kDropout>(a, s);
  }
  return MLORA_ERR_INVALID_ARG;
}

}  // namespace mlora
