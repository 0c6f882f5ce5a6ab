// Embedding lookup with scaling, and the gradient of its table.
//
//   out[t] = c E[i_t],   dE[v] = c * (sum of dy[t] over the tokens with i_t = v)
//
// The sums run over the tokens of an entry in token order, whatever the launch, so the
// gradient is the same bits in every run: tokens are sorted by (entry, token) first.
// Up to 16384 tokens each counts the ones ahead of it, a comparison a pair (up to 512 in
// the CTAs that add them up, for want of a launch); of more,
// blocks of 2048 are sorted in shared memory and each element finds its place by binary
// searches in all the other blocks, a part that grows with the square of the tokens (keys
// are distinct: the token is part of them).  Gradient of 32000x512 in bf16: 8192 tokens
// 29 us, 16384 66, 16385 44, 32768 60, 65536 107, 131072 245.  Runs of equal entries
// in the sorted order are summed by chunks of 16 or 32 tokens, so that an entry that half of
// the batch holds is summed by many CTAs; a run that crosses a chunk's border leaves
// fp32 partial sums, added in chunk order by a last pass.  The rows without tokens are
// zeroed in the same launch as the sums: every row of the gradient is written once.
// Bound: HBM (dy once, the gradient once); for few tokens the chain of launches, which
// start as programmatic dependents of one another.
// An index outside the table gives a zero row, no gradient, and a code in the device
// status word; the padding entry's gradient is zero.
#include <algorithm>
#include <atomic>
#include <string>

#include "internal.h"
#include "launch.cuh"
#include "ptx.cuh"
#include "../../include/metallora_b200.h"

namespace mlora {
namespace {

constexpr int kThreads = 256;
constexpr int kSortThreads = 1024;
constexpr int kSortBlock = 2 * kSortThreads;
constexpr int kJoin = 64;  // threads of a CTA that joins partial sums
constexpr int64_t kPairTokens = 16384;
constexpr int kRankThreads = 512;
constexpr int kRankTokens = 64;  // of a CTA that counts pairs
// Sorted tokens per CTA of the gradient: 32 (gradient of 2000 tokens, 20000x101: 15 us,
// with 64 20 us, 16 13 us; of 16000 tokens, 1000x4095: 126, 118, 137 us); 16 where the
// CTAs sort for themselves (300 tokens, 1000x512: 11.3 us, with 64 18.0, 32 12.9, 8 10.4;
// 512 tokens, 32000x4096: 49, 50, 46, 52; of one entry, 1x64: 17.5, 18.6, 16.5, 22).
constexpr int kChunk = 32, kOwnChunk = 16;
constexpr int kOwnTokens = 512;  // up to which its CTAs sort them themselves
// Up to which the CTA of a run's first token sums the whole run, with nothing to join: a
// launch less, of the host's time too (3 us; 64 tokens, 1000x512, take 5.8 us, with the
// joining pass 6.9; 96 tokens 5.2 and 6.9, 128 6.1 and 8.0).  An entry that is all of the
// batch is one CTA's work then (1x512: 32 tokens 7.0 us and 6.1, 64 12.6 and 6.3, 96 18.2
// and 7.1, 128 23.8 and 7.5), so longer batches are joined: what that costs at 64, twice
// the time at worst, grows with the tokens, what it gains does not.
constexpr int kWholeTokens = 64;
constexpr uint32_t kNone = 0xFFFFFFFFu;  // entry of a token without a gradient

// Columns of a thread that sums rows of no whole 16 bytes, kThreads apart, 16 rows of them
// in flight: the loads of two bytes need many CTAs and few rounds, which the zeroing
// beside them stretches.  Gradient of 3001 tokens, 50257x1001: 31.5 us (one column 33.9,
// four 35.8, the vector path's loop of eight columns and eight rows 47.6); of 8192,
// 32000x4095: 103 (127, 106, 142).
constexpr int kOddCols = 2;

template <typename T>
constexpr int kVec = 16 / static_cast<int>(sizeof(T));

template <typename T>
struct Vec {
  float v[kVec<T>];
};

// A thread's kVec columns of a row: side by side in 16 bytes (`vec`: the rows start on
// 16 bytes and hold a whole number of them), or else `stride` apart, so that a warp's
// accesses are side by side.
struct Cols {
  bool vec;
  int stride;
  int64_t d, D;  // the first one, and the row's length
  __device__ bool any() const { return d < D; }
  __device__ bool has(int j) const { return d + static_cast<int64_t>(j) * stride < D; }
};

template <typename T>
__device__ __forceinline__ Cols thread_cols(int slice, int thread, int threads, bool vec, int64_t D) {
  const int64_t base = static_cast<int64_t>(slice) * threads * kVec<T>;
  return {vec, threads, base + (vec ? thread * kVec<T> : thread), D};
}

// As they are, 16 bytes of them (zeros past the row's end): rows in flight stay small.
template <typename T>
__device__ __forceinline__ uint4 load_raw(const T* row, const Cols& c) {
  if (c.vec) return *reinterpret_cast<const uint4*>(row + c.d);
  uint4 q;
  T* e = reinterpret_cast<T*>(&q);
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i)
    e[i] = c.has(i) ? row[c.d + static_cast<int64_t>(i) * c.stride] : static_cast<T>(0.f);
  return q;
}

template <typename T>
__device__ __forceinline__ void add_raw(Vec<T>& r, const uint4& q) {
  const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i) r.v[i] += static_cast<float>(e[i]);
}

template <typename T>
__device__ __forceinline__ void store_cols(T* row, const Cols& c, const Vec<T>& r, float scale) {
  if (c.vec) {
    uint4 q;
    T* e = reinterpret_cast<T*>(&q);
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) e[i] = static_cast<T>(r.v[i] * scale);
    *reinterpret_cast<uint4*>(row + c.d) = q;
  } else {
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i)
      if (c.has(i)) row[c.d + static_cast<int64_t>(i) * c.stride] = static_cast<T>(r.v[i] * scale);
  }
}

// The same of a row of fp32 partial sums.
template <typename T>
__device__ __forceinline__ void store_partial(float* row, const Cols& c, const Vec<T>& r) {
  if (c.vec) {
#pragma unroll
    for (int i = 0; i < kVec<T>; i += 4)
      *reinterpret_cast<float4*>(row + c.d + i) = make_float4(r.v[i], r.v[i + 1], r.v[i + 2], r.v[i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i)
      if (c.has(i)) row[c.d + static_cast<int64_t>(i) * c.stride] = r.v[i];
  }
}

template <typename T>
__device__ __forceinline__ Vec<T> load_partial(const float* row, const Cols& c) {
  Vec<T> r;
  if (c.vec) {
#pragma unroll
    for (int i = 0; i < kVec<T>; i += 4) {
      const float4 q = *reinterpret_cast<const float4*>(row + c.d + i);
      r.v[i] = q.x, r.v[i + 1] = q.y, r.v[i + 2] = q.z, r.v[i + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i)
      r.v[i] = c.has(i) ? row[c.d + static_cast<int64_t>(i) * c.stride] : 0.f;
  }
  return r;
}

// The 16 bytes that begin `skip` bytes (even, below 16) into two blocks of 16.
__device__ __forceinline__ uint4 shifted(const uint4& a, const uint4& b, uint32_t skip) {
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 6; ++i) w[i] = skip & 8 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = skip & 4 ? w[i + 1] : w[i];
  const uint32_t bits = (skip & 3) * 8;
  return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                    __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}

// A row that fits no 16 bytes, of a 16-bit type: its output's whole 16 bytes from the two
// blocks that they lie in, the ends (and what lies in a block across the table's) by the
// element.  8192 tokens of 4095 fp16 columns take 30 us, by the element 48, 3001 of 1001
// 5.7 and 7.3; fp32, which moves four bytes by the element, would lose on short rows (16000
// of 101 columns 6.8 and 5.8 us) what it wins on long ones (8192 of 4095 50 and 53).
template <typename T>
__device__ __forceinline__ void gather_odd(const T* src, T* dst, int D, float scale, int lane,
                                           int row_threads, uintptr_t begin, uintptr_t end) {
  const int to_block = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(dst) & 15)) & 15);
  const int lead = min(to_block / static_cast<int>(sizeof(T)), D);
  const int blocks = (D - lead) / kVec<T>;
#pragma unroll 2
  for (int j = lane; j < blocks; j += row_threads) {
    const int e = lead + j * kVec<T>;
    const uintptr_t at = reinterpret_cast<uintptr_t>(src + e), block = at & ~uintptr_t{15};
    uint4 q;
    if (block >= begin && block + 32 <= end) {
      const uint4* from = reinterpret_cast<const uint4*>(block);
      q = shifted(from[0], from[1], static_cast<uint32_t>(at & 15));
    } else {
      T* one = reinterpret_cast<T*>(&q);
#pragma unroll
      for (int i = 0; i < kVec<T>; ++i) one[i] = src[e + i];
    }
    Vec<T> r = {};
    add_raw(r, q);
    T* out = reinterpret_cast<T*>(&q);
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) out[i] = static_cast<T>(r.v[i] * scale);
    *reinterpret_cast<uint4*>(dst + e) = q;
  }
  const int tail = lead + blocks * kVec<T>;  // the ends are below 16 bytes each
  for (int j = lane; j < lead + D - tail; j += row_threads) {
    const int e = j < lead ? j : tail + j - lead;
    dst[e] = static_cast<T>(static_cast<float>(src[e]) * scale);
  }
}

// One CTA: 256 / row_threads tokens, row_threads across a row.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    embedding_gather_kernel(const int64_t* idx, const T* table, T* out, int64_t n_tok, int64_t V,
                            int64_t D, float scale, int row_threads, int vec, uint32_t* status) {
  const int lane = static_cast<int>(threadIdx.x) % row_threads;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (kThreads / row_threads) +
                    static_cast<int>(threadIdx.x) / row_threads;
  if (t >= n_tok) return;
  const int64_t v = idx[t];
  const bool ok = v >= 0 && v < V;
  if (!ok && lane == 0) record_status(status, kDevBadIndex);
  const T* src = table + (ok ? v : 0) * D;
  T* dst = out + t * D;
  if constexpr (sizeof(T) == 2) {
    if (vec == 0 && ok) {
      gather_odd(src, dst, static_cast<int>(D), scale, lane, row_threads,
                 reinterpret_cast<uintptr_t>(table), reinterpret_cast<uintptr_t>(table + V * D));
      return;
    }
  }
  for (int slice = 0;; ++slice) {
    const Cols c = thread_cols<T>(slice, lane, row_threads, vec != 0, D);
    if (!c.any()) break;
    Vec<T> r = {};
    if (ok) add_raw(r, load_raw(src, c));
    store_cols(dst, c, r, scale);
  }
}

__device__ __forceinline__ uint64_t make_key(uint32_t entry, int64_t token) {
  return static_cast<uint64_t>(entry) << 32 | static_cast<uint32_t>(token);
}
__device__ __forceinline__ uint32_t entry_of(uint64_t key) { return static_cast<uint32_t>(key >> 32); }

// The entry a token adds to.
__device__ __forceinline__ uint32_t token_entry(int64_t v, int64_t V, int64_t padding,
                                                uint32_t* status) {
  const bool ok = v >= 0 && v < V;
  if (!ok) record_status(status, kDevBadIndex);
  return ok && v != padding ? static_cast<uint32_t>(v) : kNone;
}

// Of the tokens outside token t's own four, those that come before it: smaller entries,
// and its own entry's tokens ahead of it; thread `part` of kPer counts its share.
template <int kPer>
__device__ __forceinline__ int count_ahead(const uint32_t* entries, int padded, int t, int part,
                                           uint32_t mine) {
  int place = 0;
  const int own = t & ~3;
#pragma unroll 4
  for (int i = part * 4; i < own; i += kPer * 4) {
    const uint4 q = *reinterpret_cast<const uint4*>(entries + i);
    place += (q.x <= mine) + (q.y <= mine) + (q.z <= mine) + (q.w <= mine);
  }
  const int after = own / 4 + 1;  // the first four past it that are this thread's
  const int first = after + (part - after % kPer + kPer) % kPer;
#pragma unroll 4
  for (int i = first * 4; i < padded; i += kPer * 4) {
    const uint4 q = *reinterpret_cast<const uint4*>(entries + i);
    place += (q.x < mine) + (q.y < mine) + (q.z < mine) + (q.w < mine);
  }
  return place;
}

// One CTA: the places of 64 tokens, eight threads a token, with every token's entry in
// shared memory.  A token comes after those with a smaller entry, and those before it
// with its own.
__global__ void __launch_bounds__(kRankThreads)
    embedding_rank_kernel(const int64_t* idx, int n_tok, int64_t V, int64_t padding,
                          uint64_t* sorted, uint32_t* status) {
  extern __shared__ __align__(16) uint32_t entries[];  // up to a multiple of 4, the rest above every entry
  constexpr int kPer = kRankThreads / kRankTokens;
  grid_wait();
  launch_dependents();
  const int padded = (n_tok + 3) / 4 * 4;
#pragma unroll 8
  for (int i = threadIdx.x; i < padded; i += kRankThreads)
    entries[i] = i < n_tok ? token_entry(idx[i], V, padding, status) : kNone;
  __syncthreads();
  const int t = static_cast<int>(blockIdx.x) * kRankTokens + static_cast<int>(threadIdx.x) / kPer;
  const int part = static_cast<int>(threadIdx.x) % kPer;
  const uint32_t mine = t < n_tok ? entries[t] : 0;
  int place = t < n_tok ? count_ahead<kPer>(entries, padded, t, part, mine) : 0;
  if (part == 0 && t < n_tok)
    for (int i = t & ~3; i < min((t & ~3) + 4, n_tok); ++i)
      place += i < t ? entries[i] <= mine : entries[i] < mine;
#pragma unroll
  for (int o = kPer / 2; o > 0; o >>= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
  if (part == 0 && t < n_tok) sorted[place] = make_key(mine, t);
}

// Sorts blocks of 2048 keys (entry << 32 | token), a bitonic network in shared memory
// as wide as the block's tokens need; tokens without a gradient sort to the end.
// Steps over less than 64 elements stay within a warp's.
__global__ void __launch_bounds__(kSortThreads)
    embedding_sort_kernel(const int64_t* idx, int64_t n_tok, int64_t V, int64_t padding,
                          uint64_t* keys, uint32_t* status) {
  __shared__ uint64_t s[kSortBlock];
  grid_wait();
  launch_dependents();
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kSortBlock;
  const int n = static_cast<int>(n_tok - base < kSortBlock ? n_tok - base : kSortBlock);
  int width = 64;
  while (width < n) width *= 2;
  for (int i = threadIdx.x; i < width; i += kSortThreads) {
    const int64_t t = base + i;
    // distinct among those without an entry too, for the places they take
    uint64_t key = ~uint64_t{0};
    if (i < n) key = make_key(token_entry(idx[t], V, padding, status), t);
    s[i] = key;
  }
  __syncthreads();
  const int tid = static_cast<int>(threadIdx.x);
  for (int k = 2; k <= width; k <<= 1) {
    for (int j = k >> 1; j > 0; j >>= 1) {
      if (tid < width / 2) {
        const int i = 2 * tid - (tid & (j - 1));
        const uint64_t a = s[i], b = s[i + j];
        if ((a > b) == ((i & k) == 0)) s[i] = b, s[i + j] = a;
      }
      // the next step's pairs: of this warp's 64 elements, or of others
      const int next = j > 1 ? j >> 1 : k;
      if (j >= 64 || next >= 64)
        __syncthreads();
      else
        __syncwarp();
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kSortThreads) keys[base + i] = s[i];
}

// Each key's place among all blocks: its place in its own plus the smaller keys of
// the others, four searches at a time.
__global__ void __launch_bounds__(kThreads)
    embedding_merge_kernel(const uint64_t* keys, int64_t n_tok, uint64_t* sorted) {
  grid_wait();
  launch_dependents();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= n_tok) return;
  const uint64_t key = keys[i];
  const int64_t blocks = (n_tok + kSortBlock - 1) / kSortBlock;
  int64_t place = 0;
  constexpr int kAtOnce = 4;
  for (int64_t b = 0; b < blocks; b += kAtOnce) {
    int lo[kAtOnce], hi[kAtOnce];
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q) {
      const int64_t left = n_tok - (b + q) * kSortBlock;
      lo[q] = 0;
      hi[q] = static_cast<int>(left < 0 ? 0 : left < kSortBlock ? left : kSortBlock);
    }
    for (int step = kSortBlock; step > 0; step >>= 1) {
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {
        if (lo[q] >= hi[q]) continue;
        const int mid = (lo[q] + hi[q]) >> 1;
        if (keys[(b + q) * kSortBlock + mid] < key)
          lo[q] = mid + 1;
        else
          hi[q] = mid;
      }
    }
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q) place += lo[q];
  }
  sorted[place] = key;
}

// Of the 32 entries from v0, sets the bits of those that have tokens; all of a CTA.  The
// first of their tokens is searched with kThreads samples a round, two rounds of dependent
// loads up to 65536 tokens (a binary search by one warp took twelve to fourteen).
__device__ __forceinline__ void mark_entries(const uint64_t* sorted, int64_t n_tok, uint32_t v0,
                                             uint32_t* bits) {
  const int tid = static_cast<int>(threadIdx.x);
  int64_t lo = 0, hi = n_tok;  // the first token of v0 or above is at lo..hi
  while (lo < hi) {
    const int64_t step = (hi - lo + kThreads - 1) / kThreads;
    const int64_t p = lo + tid * step + step - 1;  // a segment's last
    const int below = __syncthreads_count(p < hi && entry_of(sorted[p]) < v0);
    lo += below * step;
    hi = min(hi, lo + step - 1);
  }
  // (v0 + 32 is below kNone)
  const uint32_t e = lo + tid < n_tok ? entry_of(sorted[lo + tid]) : kNone;
  if (e < v0 + 32) atomicOr(bits, 1u << (e - v0));
  if (__syncthreads_count(e < v0 + 32) < kThreads || tid >= 32) return;
  // more tokens than that: a search for each entry
  const uint32_t v = v0 + tid;
  lo += kThreads, hi = n_tok;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (entry_of(sorted[mid]) < v)
      lo = mid + 1;
    else
      hi = mid;
  }
  if (lo < n_tok && entry_of(sorted[lo]) == v) atomicOr(bits, 1u << tid);
}

// CTAs of the first `sum_ctas`: a chunk of sorted tokens, kThreads * kVec columns
// (kThreads * kOddCols without kRows).  A
// run inside the chunk is written to the gradient; one that the border cuts to the
// chunk's partial rows: [0] continues from the chunk before, [1] goes on in the next.
// The others: 32 entries each, those without tokens zeroed.  kOwn (few tokens): no launch
// has sorted them, every CTA does for itself.
// kRows: rows of whole 16 bytes.
// (kOwn needs more registers, and has fewer CTAs.)
template <typename T, bool kOwn, bool kRows>
__global__ void __launch_bounds__(kThreads, kOwn ? 3 : 4)
    embedding_grad_kernel(const int64_t* idx, int64_t padding, uint64_t* sorted, const T* dy,
                          int64_t n_tok, int64_t V, int64_t D, float scale, int sum_ctas, int slices,
                          T* grad, float* partial, uint32_t* status) {
  constexpr int kLen = kOwn ? kOwnChunk : kChunk;
  // the chunk, or the whole order, with a neighbour on either side
  __shared__ uint64_t held[(kOwn ? kOwnTokens : kLen) + 2];
  __shared__ __align__(16) uint32_t entries[kOwn ? kOwnTokens : 4];
  grid_wait();
  launch_dependents();
  if (static_cast<int>(blockIdx.x) >= sum_ctas) {
    const int64_t v0 = static_cast<int64_t>(static_cast<int>(blockIdx.x) - sum_ctas) * 32;
    uint32_t* const has_tokens = reinterpret_cast<uint32_t*>(held);
    if constexpr (kOwn) {
      if (threadIdx.x == 0) *has_tokens = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < static_cast<int>(n_tok); i += kThreads) {
        const int64_t v = idx[i];
        if (v >= v0 && v < v0 + 32 && v < V && v != padding) atomicOr(has_tokens, 1u << (v - v0));
      }
    } else {
      if (threadIdx.x == 0) *has_tokens = 0;
      mark_entries(sorted, n_tok, static_cast<uint32_t>(v0), has_tokens);
    }
    __syncthreads();
    const uint32_t has = *has_tokens;
    const int rows = static_cast<int>(V - v0 < 32 ? V - v0 : 32);
    T* first = grad + v0 * D;
    const int len = static_cast<int>(D), total = rows * len;  // below 2^27
    constexpr int kStep = kThreads * kVec<T>;
    if constexpr (kRows) {
      int row = static_cast<int>(threadIdx.x) * kVec<T> / len;
      int col = static_cast<int>(threadIdx.x) * kVec<T> % len;
      const int step_row = kStep / len, step_col = kStep % len;
      while (row < rows) {
        if (((has >> row) & 1u) == 0)
          *reinterpret_cast<uint4*>(first + row * len + col) = make_uint4(0, 0, 0, 0);
        row += step_row;
        col += step_col;
        if (col >= len) col -= len, ++row;
      }
      return;
    }
    // the rows' elements in whole 16 bytes, from the boundary at or before the first;
    // element e is at `col` of `row` (before the first: at a negative column)
    const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(first) & 15u) / sizeof(T));
    int e = static_cast<int>(threadIdx.x) * kVec<T> - lead;
    int row = e < 0 ? 0 : e / len, col = e - row * len;
    const int step_row = kStep / len, step_col = kStep % len;
    for (; e < total; e += kStep) {
      if (len >= kVec<T> && col >= 0 && e + kVec<T> <= total) {  // of one row or two
        const bool two = col + kVec<T> > len;
        const bool keep0 = (has >> row) & 1u, keep1 = two ? (has >> (row + 1)) & 1u : keep0;
        if (!keep0 && !keep1) {
          *reinterpret_cast<uint4*>(first + e) = make_uint4(0, 0, 0, 0);
        } else if (!keep0 || !keep1) {
          for (int i = keep0 ? len - col : 0; i < (keep1 ? len - col : kVec<T>); ++i)
            first[e + i] = static_cast<T>(0.f);
        }
      } else {
        for (int i = max(e, 0); i < min(e + kVec<T>, total); ++i)
          if (((has >> (i / len)) & 1u) == 0) first[i] = static_cast<T>(0.f);
      }
      row += step_row, col += step_col;
      if (col >= len) col -= len, ++row;
      if (col < 0) col += len, --row;
    }
    return;
  }
  const int64_t chunk = static_cast<int>(blockIdx.x) / slices;
  const int64_t p0 = chunk * kLen;
  int n = static_cast<int>(n_tok - p0 < kLen ? n_tok - p0 : kLen);
  const bool runs = kOwn && n_tok <= kWholeTokens;  // whole ones, of those that begin here
  const uint64_t* const key = held + (kOwn ? p0 : 0);  // of token p at [p - p0 + 1]
  if constexpr (kOwn) {
    const int tokens = static_cast<int>(n_tok), padded = (tokens + 3) / 4 * 4;
    for (int i = threadIdx.x; i < padded; i += kThreads)
      entries[i] = i < tokens ? token_entry(idx[i], V, padding, status) : kNone;
    __syncthreads();
    for (int t = threadIdx.x; t < tokens; t += kThreads) {
      const uint32_t mine = entries[t];
      int place = count_ahead<1>(entries, padded, t, 0, mine);
      for (int i = t & ~3; i < min((t & ~3) + 4, tokens); ++i)
        place += i < t ? entries[i] <= mine : entries[i] < mine;
      held[place + 1] = make_key(mine, t);
    }
    if (threadIdx.x == 0) held[0] = held[tokens + 1] = ~uint64_t{0};
    __syncthreads();
    if (!runs && static_cast<int>(blockIdx.x) % slices == 0)  // for the pass that joins runs
      for (int i = threadIdx.x; i < n; i += kThreads) sorted[p0 + i] = key[i + 1];
  } else {
    if (threadIdx.x < kLen + 2) {
      const int64_t p = p0 + static_cast<int>(threadIdx.x) - 1;
      held[threadIdx.x] = p >= 0 && p < n_tok ? sorted[p] : ~uint64_t{0};
    }
    __syncthreads();
  }
  int begin = 0;
  if (runs) {
    while (begin < n && entry_of(key[begin]) == entry_of(key[begin + 1])) ++begin;
    if (begin == n) return;
    while (p0 + n < n_tok && entry_of(key[n]) == entry_of(key[n + 1])) ++n;
  }
  const int slice = static_cast<int>(blockIdx.x) % slices;
  bool first_run = !runs && entry_of(key[0]) == entry_of(key[1]);  // begun in an earlier chunk
  if constexpr (!kRows) {
    const int64_t d = static_cast<int64_t>(slice) * kThreads * kOddCols + threadIdx.x;
    if (d >= D) return;
    constexpr int kAhead = 16;
    float acc[kOddCols] = {};
    for (int q0 = begin; q0 < n; q0 += kAhead) {
      T row[kAhead][kOddCols];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const bool in = q0 + i < n && entry_of(key[q0 + i + 1]) != kNone;
        const int64_t token = in ? static_cast<uint32_t>(key[q0 + i + 1]) : 0;
        const T* src = dy + token * D + d;
#pragma unroll
        for (int k = 0; k < kOddCols; ++k)
          row[i][k] = in && d + k * kThreads < D ? src[k * kThreads] : static_cast<T>(0.f);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int q = q0 + i;
        if (q >= n) break;
        const uint32_t e = entry_of(key[q + 1]);
        if (e == kNone) return;
#pragma unroll
        for (int k = 0; k < kOddCols; ++k) acc[k] += static_cast<float>(row[i][k]);
        const bool ends = entry_of(key[q + 2]) != e;
        if (!ends && q + 1 < n) continue;
        const bool whole = ends && !first_run;
        T* out = grad + static_cast<int64_t>(e) * D + d;
        float* part = partial + (chunk * 2 + (first_run ? 0 : 1)) * D + d;
#pragma unroll
        for (int k = 0; k < kOddCols; ++k) {
          if (d + k * kThreads >= D) continue;
          if (whole)
            out[k * kThreads] = static_cast<T>(acc[k] * scale);
          else
            part[k * kThreads] = acc[k];
          acc[k] = 0.f;
        }
        first_run = false;
      }
    }
    return;
  }
  const Cols c = thread_cols<T>(slice, static_cast<int>(threadIdx.x), kThreads, true, D);
  if (!c.any()) return;
  constexpr int kAhead = 8;
  Vec<T> acc = {};
  for (int q0 = begin; q0 < n; q0 += kAhead) {
    uint4 row[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (q0 + i < n && entry_of(key[q0 + i + 1]) != kNone)
        row[i] = load_raw(dy + static_cast<int64_t>(static_cast<uint32_t>(key[q0 + i + 1])) * D, c);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int q = q0 + i;
      if (q >= n) break;
      const uint32_t e = entry_of(key[q + 1]);
      if (e == kNone) return;
      add_raw(acc, row[i]);
      const bool ends = entry_of(key[q + 2]) != e;
      if (!ends && q + 1 < n) continue;
      if (ends && !first_run)
        store_cols(grad + static_cast<int64_t>(e) * D, c, acc, scale);
      else
        store_partial(partial + (chunk * 2 + (first_run ? 0 : 1)) * D, c, acc);
      acc = {};
      first_run = false;
    }
  }
}

// One CTA for each chunk whose last run begins in it and goes on in the next: adds
// that run's partial sums in chunk order.
template <typename T>
__global__ void __launch_bounds__(kJoin)
    embedding_join_kernel(const uint64_t* sorted, const float* partial, int len, int64_t n_tok,
                          int64_t D, float scale, int vec, T* grad) {
  grid_wait();
  const int64_t first = blockIdx.x, last = (first + 1) * len - 1;
  if (last + 1 >= n_tok) return;
  const uint32_t e = entry_of(sorted[last]);
  if (e == kNone || entry_of(sorted[last + 1]) != e) return;
  if (first > 0 && entry_of(sorted[first * len - 1]) == e && entry_of(sorted[first * len]) == e)
    return;  // begun before this chunk
  const Cols c = thread_cols<T>(static_cast<int>(blockIdx.y), static_cast<int>(threadIdx.x), kJoin,
                                vec != 0, D);
  if (!c.any()) return;
  Vec<T> acc = load_partial<T>(partial + (first * 2 + 1) * D, c);
  constexpr int kAhead = 4;
  const int64_t chunks = (n_tok + len - 1) / len;
  for (int64_t q = first + 1; q < chunks; q += kAhead) {
    bool goes[kAhead];  // the run reaches chunk q + i
    Vec<T> v[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) goes[i] = q + i < chunks && entry_of(sorted[(q + i) * len]) == e;
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (goes[i]) v[i] = load_partial<T>(partial + (q + i) * 2 * D, c);
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (goes[i])
#pragma unroll
        for (int k = 0; k < kVec<T>; ++k) acc.v[k] += v[i].v[k];
    if (!goes[kAhead - 1]) break;
  }
  store_cols(grad + static_cast<int64_t>(e) * D, c, acc, scale);
}

// ------------------------------------------------------------------- host --

int fail(int code, const std::string& msg) {
  set_error(msg);
  return code;
}

int64_t chunk_len(int64_t n_tok) { return n_tok <= kOwnTokens ? kOwnChunk : kChunk; }
int64_t chunks(int64_t n_tok) { return (n_tok + chunk_len(n_tok) - 1) / chunk_len(n_tok); }
int64_t round_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

int check(int64_t T, int64_t V, int64_t D, int dtype) {
  if (T <= 0 || V <= 0 || D <= 0) return fail(MLORA_ERR_INVALID_ARG, "T, V, D must be positive");
  if (dtype != MLORA_DTYPE_BF16 && dtype != MLORA_DTYPE_F16 && dtype != MLORA_DTYPE_F32)
    return fail(MLORA_ERR_UNSUPPORTED, "dtype must be BF16, F16 or F32");
  if (T > (int64_t{1} << 31) - 256 || V > (int64_t{1} << 31) - 256 || D > (1 << 22))
    return fail(MLORA_ERR_UNSUPPORTED, "shape too large");
  return MLORA_OK;
}

bool elements(const void* p, int dtype) {
  return reinterpret_cast<uintptr_t>(p) % (dtype == MLORA_DTYPE_F32 ? 4 : 2) == 0;
}
bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

template <typename T>
int gather(const int64_t* idx, const void* table, void* out, int64_t n_tok, int64_t V, int64_t D,
           float scale, cudaStream_t s) {
  const int vec = D % kVec<T> == 0 && aligned(table, 16) && aligned(out, 16);
  int row_threads = 8;
  while (row_threads < kThreads && row_threads * kVec<T> < D) row_threads *= 2;
  const int64_t per = kThreads / row_threads;
  LaunchScope scope(kKindElementwise, s);
  embedding_gather_kernel<T><<<static_cast<unsigned>((n_tok + per - 1) / per), kThreads, 0, s>>>(
      idx, static_cast<const T*>(table), static_cast<T*>(out), n_tok, V, D, scale, row_threads, vec,
      device_status_ptr());
  return launch_status(cudaSuccess, "embedding");
}

struct Work {
  uint64_t *keys, *sorted;
  float* partial;
  int64_t bytes;
};

Work plan(void* base, int64_t T, int64_t D) {
  uint8_t* b = static_cast<uint8_t*>(base);
  Work w;
  int64_t off = 0;
  auto take = [&](int64_t bytes) {
    uint8_t* p = b != nullptr ? b + off : nullptr;
    off += round_up(bytes, 256);
    return p;
  };
  w.sorted = reinterpret_cast<uint64_t*>(take(T * 8));
  w.keys = T > kPairTokens ? reinterpret_cast<uint64_t*>(take(T * 8)) : nullptr;
  w.partial = reinterpret_cast<float*>(take(chunks(T) * 2 * D * 4));
  w.bytes = off;
  return w;
}

template <typename T>
int gradient(const int64_t* idx, const void* dy, void* grad, int64_t n_tok, int64_t V, int64_t D,
             float scale, int64_t padding, const Work& w, cudaStream_t s) {
  cudaError_t e = cudaSuccess;
  const bool own = n_tok <= kOwnTokens;
  if (own) {
    // sorted by the sums' own CTAs
  } else if (n_tok <= kPairTokens) {
    static std::atomic<bool> limit_set[64];
    if (int rc = set_max_smem(reinterpret_cast<const void*>(embedding_rank_kernel), kPairTokens * 4,
                              limit_set))
      return rc;
    LaunchScope scope(kKindElementwise, s);
    e = launch_kernel(embedding_rank_kernel,
                      dim3(static_cast<unsigned>((n_tok + kRankTokens - 1) / kRankTokens)), kRankThreads,
                      static_cast<size_t>(n_tok + 3) / 4 * 16, s, 0, 0, true, idx,
                      static_cast<int>(n_tok), V, padding, w.sorted, device_status_ptr());
  } else {
    {
      LaunchScope scope(kKindElementwise, s);
      e = launch_kernel(embedding_sort_kernel,
                        dim3(static_cast<unsigned>((n_tok + kSortBlock - 1) / kSortBlock)),
                        kSortThreads, 0, s, 0, 0, true, idx, n_tok, V, padding, w.keys,
                        device_status_ptr());
    }
    if (e == cudaSuccess) {
      LaunchScope scope(kKindElementwise, s);
      e = launch_kernel(embedding_merge_kernel,
                        dim3(static_cast<unsigned>((n_tok + kThreads - 1) / kThreads)), kThreads, 0, s,
                        0, 0, true, static_cast<const uint64_t*>(w.keys), n_tok, w.sorted);
    }
  }
  const int vec = D % kVec<T> == 0 && aligned(dy, 16) && aligned(grad, 16);
  const int64_t cols = int64_t{kThreads} * (vec ? kVec<T> : kOddCols);
  const int slices = static_cast<int>((D + cols - 1) / cols);
  const int64_t sum_ctas = chunks(n_tok) * slices;
  const int64_t grid = sum_ctas + (V + 31) / 32;
  if (grid > (int64_t{1} << 31) - 1)
    return fail(MLORA_ERR_UNSUPPORTED, "embedding gradient: too many tokens for rows this long");
  if (e == cudaSuccess) {
    LaunchScope scope(kKindElementwise, s);
    auto* kernel = vec ? embedding_grad_kernel<T, false, true> : embedding_grad_kernel<T, false, false>;
    if (own) kernel = vec ? embedding_grad_kernel<T, true, true> : embedding_grad_kernel<T, true, false>;
    e = launch_kernel(kernel,
                      dim3(static_cast<unsigned>(grid)), kThreads, 0, s, 0, 0, true, idx, padding,
                      w.sorted, static_cast<const T*>(dy), n_tok, V, D, scale,
                      static_cast<int>(sum_ctas), slices, static_cast<T*>(grad), w.partial,
                      device_status_ptr());
  }
  if (e == cudaSuccess && n_tok > kWholeTokens) {
    LaunchScope scope(kKindElementwise, s);
    e = launch_kernel(embedding_join_kernel<T>,
                      dim3(static_cast<unsigned>(chunks(n_tok) - 1),
                           static_cast<unsigned>((D + kJoin * kVec<T> - 1) / (kJoin * kVec<T>))),
                      kJoin, 0, s, 0, 0, true, static_cast<const uint64_t*>(w.sorted),
                      static_cast<const float*>(w.partial), static_cast<int>(chunk_len(n_tok)), n_tok, D,
                      scale, vec, static_cast<T*>(grad));
  }
  return launch_status(e, "embedding gradient");
}

}  // namespace
}  // namespace mlora

using namespace mlora;

extern "C" {

int mlora_embedding_forward(const int64_t* idx, const void* table, void* out, int64_t T, int64_t V,
                            int64_t D, float scale, int dtype, void* stream) {
  if (int rc = check(T, V, D, dtype)) return rc;
  if (!idx || !table || !out) return fail(MLORA_ERR_INVALID_ARG, "NULL tensor pointer");
  if (!aligned(idx, 8) || !elements(table, dtype) || !elements(out, dtype))
    return fail(MLORA_ERR_INVALID_ARG, "tensor pointers must be whole elements");
  if (int rc = require_device()) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == MLORA_DTYPE_BF16) return gather<__nv_bfloat16>(idx, table, out, T, V, D, scale, s);
  if (dtype == MLORA_DTYPE_F16) return gather<__half>(idx, table, out, T, V, D, scale, s);
  return gather<float>(idx, table, out, T, V, D, scale, s);
}

size_t mlora_embedding_backward_workspace_bytes(int64_t T, int64_t D) {
  if (check(T, 1, D, MLORA_DTYPE_F32)) return 0;
  return static_cast<size_t>(plan(nullptr, T, D).bytes);
}

int mlora_embedding_backward(const int64_t* idx, const void* dy, void* grad, int64_t T, int64_t V,
                             int64_t D, float scale, int64_t padding_idx, int dtype, void* workspace,
                             size_t workspace_bytes, void* stream) {
  if (int rc = check(T, V, D, dtype)) return rc;
  if (!idx || !dy || !grad) return fail(MLORA_ERR_INVALID_ARG, "NULL tensor pointer");
  if (!aligned(idx, 8) || !elements(dy, dtype) || !elements(grad, dtype))
    return fail(MLORA_ERR_INVALID_ARG, "tensor pointers must be whole elements");
  const Work w = plan(workspace, T, D);
  if (!workspace || !aligned(workspace, 16) || workspace_bytes < static_cast<size_t>(w.bytes))
    return fail(MLORA_ERR_WORKSPACE, "embedding workspace needs " + std::to_string(w.bytes) + " bytes");
  if (int rc = require_device()) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == MLORA_DTYPE_BF16)
    return gradient<__nv_bfloat16>(idx, dy, grad, T, V, D, scale, padding_idx, w, s);
  if (dtype == MLORA_DTYPE_F16)
    return gradient<__half>(idx, dy, grad, T, V, D, scale, padding_idx, w, s);
  return gradient<float>(idx, dy, grad, T, V, D, scale, padding_idx, w, s);
}

}  // extern "C"
