// Embedding lookup with scaling, and the gradient of its table.
//
//   out[t] = c E[i_t],   dE[v] = c * (sum of dy[t] over the tokens with i_t = v)
//
// The sums run over the tokens of an entry in token order, whatever the launch, so the
// gradient is the same bits in every run: tokens are sorted by (entry, token) first.
// Blocks of 2048 are sorted in shared memory, then each element finds its place among
// all of them by binary searches in the other blocks (keys are distinct: the token is
// part of them).  Runs of equal entries in the sorted order are summed by chunks of 32
// tokens, so that an entry that half of the batch holds (padding) is summed by many
// CTAs; a run that crosses a chunk's border leaves fp32 partial sums, added in chunk
// order by a second pass.  Bound: HBM (dy once, the gradient once).
// An index outside the table gives a zero row, no gradient, and a code in the device
// status word; the padding entry's gradient is zero.
#include <algorithm>
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
constexpr int kChunk = 32;  // sorted tokens per CTA of the gradient
constexpr uint64_t kNoEntry = ~uint64_t{0};

template <typename T>
constexpr int kVec = 16 / static_cast<int>(sizeof(T));

template <typename T>
struct Vec {
  float v[kVec<T>];
};

// N elements from p (16-byte aligned where N = kVec<T>), or fewer.
template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* p, bool vec, int64_t left) {
  Vec<T> r;
  if (vec) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) r.v[i] = static_cast<float>(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) r.v[i] = i < left ? static_cast<float>(p[i]) : 0.f;
  }
  return r;
}

template <typename T>
__device__ __forceinline__ void store_vec(T* p, bool vec, int64_t left, const Vec<T>& r, float scale) {
  if (vec) {
    uint4 q;
    T* e = reinterpret_cast<T*>(&q);
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) e[i] = static_cast<T>(r.v[i] * scale);
    *reinterpret_cast<uint4*>(p) = q;
  } else {
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i)
      if (i < left) p[i] = static_cast<T>(r.v[i] * scale);
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
  for (int64_t d = static_cast<int64_t>(lane) * kVec<T>; d < D;
       d += static_cast<int64_t>(row_threads) * kVec<T>) {
    Vec<T> r = {};
    if (ok) r = load_vec(src + d, vec != 0, D - d);
    store_vec(dst + d, vec != 0, D - d, r, scale);
  }
}

// Sorts blocks of 2048 keys (entry << 32 | token), a bitonic network in shared
// memory; tokens without a gradient sort to the end.
__global__ void __launch_bounds__(kSortThreads)
    embedding_sort_kernel(const int64_t* idx, int64_t n_tok, int64_t V, int64_t padding,
                          uint64_t* keys, uint32_t* status) {
  __shared__ uint64_t s[kSortBlock];
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kSortBlock;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = static_cast<int>(threadIdx.x) + h * kSortThreads;
    const int64_t t = base + i;
    uint64_t key = kNoEntry;
    if (t < n_tok) {
      const int64_t v = idx[t];
      if (v < 0 || v >= V)
        record_status(status, kDevBadIndex);
      else if (v != padding)
        key = static_cast<uint64_t>(v) << 32 | static_cast<uint32_t>(t);
      // distinct among those without an entry too, for the places they take
      if (key == kNoEntry) key = uint64_t{0xFFFFFFFFu} << 32 | static_cast<uint32_t>(t);
    }
    s[i] = key;
  }
  for (int k = 2; k <= kSortBlock; k <<= 1) {
    for (int j = k >> 1; j > 0; j >>= 1) {
      __syncthreads();
      const int i = 2 * static_cast<int>(threadIdx.x) - (static_cast<int>(threadIdx.x) & (j - 1));
      const uint64_t a = s[i], b = s[i + j];
      if ((a > b) == ((i & k) == 0)) s[i] = b, s[i + j] = a;
    }
  }
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = static_cast<int>(threadIdx.x) + h * kSortThreads;
    if (base + i < n_tok) keys[base + i] = s[i];
  }
}

// Each key's place among all blocks: its place in its own plus the smaller keys of
// the others.
__global__ void __launch_bounds__(kThreads)
    embedding_merge_kernel(const uint64_t* keys, int64_t n_tok, uint64_t* sorted) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= n_tok) return;
  const uint64_t key = keys[i];
  const int64_t own = i / kSortBlock;
  int64_t place = i - own * kSortBlock;
  for (int64_t b0 = 0; b0 < n_tok; b0 += kSortBlock) {
    if (b0 == own * kSortBlock) continue;
    const int n = static_cast<int>(n_tok - b0 < kSortBlock ? n_tok - b0 : kSortBlock);
    int lo = 0, hi = n;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (keys[b0 + mid] < key)
        lo = mid + 1;
      else
        hi = mid;
    }
    place += lo;
  }
  sorted[place] = key;
}

__device__ __forceinline__ uint32_t entry_of(uint64_t key) { return static_cast<uint32_t>(key >> 32); }

// One CTA: a chunk of 32 sorted tokens, row_threads * kVec columns.  A run inside
// the chunk is written to the gradient; one that the border cuts to the chunk's
// partial rows: [0] continues from the chunk before, [1] goes on in the next.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    embedding_grad_kernel(const uint64_t* sorted, const T* dy, int64_t n_tok, int64_t D, float scale,
                          int vec, T* grad, float* partial) {
  __shared__ uint64_t key[kChunk + 2];  // with a neighbour on either side
  const int64_t p0 = static_cast<int64_t>(blockIdx.x) * kChunk;
  const int n = static_cast<int>(n_tok - p0 < kChunk ? n_tok - p0 : kChunk);
  if (threadIdx.x < kChunk + 2) {
    const int64_t p = p0 + static_cast<int>(threadIdx.x) - 1;
    key[threadIdx.x] = p >= 0 && p < n_tok ? sorted[p] : kNoEntry;
  }
  __syncthreads();
  const int64_t d = (static_cast<int64_t>(blockIdx.y) * kThreads + threadIdx.x) * kVec<T>;
  if (d >= D || entry_of(key[1]) == 0xFFFFFFFFu) return;
  constexpr int kAhead = 8;
  Vec<T> acc = {};
  bool first_run = entry_of(key[0]) == entry_of(key[1]);  // begun in an earlier chunk
  for (int q0 = 0; q0 < n; q0 += kAhead) {
    Vec<T> row[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (q0 + i < n && entry_of(key[q0 + i + 1]) != 0xFFFFFFFFu)
        row[i] = load_vec(dy + static_cast<int64_t>(static_cast<uint32_t>(key[q0 + i + 1])) * D + d,
                          vec != 0, D - d);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int q = q0 + i;
      if (q >= n) break;
      const uint32_t e = entry_of(key[q + 1]);
      if (e == 0xFFFFFFFFu) return;
#pragma unroll
      for (int j = 0; j < kVec<T>; ++j) acc.v[j] += row[i].v[j];
      const bool ends = entry_of(key[q + 2]) != e;
      if (!ends && q + 1 < n) continue;
      if (ends && !first_run) {
        store_vec(grad + static_cast<int64_t>(e) * D + d, vec != 0, D - d, acc, scale);
      } else {
        float* dst = partial + (static_cast<int64_t>(blockIdx.x) * 2 + (first_run ? 0 : 1)) * D + d;
#pragma unroll
        for (int j = 0; j < kVec<T>; ++j)
          if (d + j < D) dst[j] = acc.v[j];
      }
      acc = {};
      first_run = false;
    }
  }
}

// One CTA for each chunk whose last run begins in it and goes on in the next: adds
// that run's partial sums in chunk order.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    embedding_join_kernel(const uint64_t* sorted, const float* partial, int64_t n_tok, int64_t D,
                          float scale, T* grad) {
  const int64_t last = (static_cast<int64_t>(blockIdx.x) + 1) * kChunk - 1;
  if (last + 1 >= n_tok) return;
  const uint32_t e = entry_of(sorted[last]);
  if (e == 0xFFFFFFFFu || entry_of(sorted[last + 1]) != e) return;
  const int64_t p0 = last - kChunk + 1;
  if (p0 > 0 && entry_of(sorted[p0 - 1]) == e) return;  // begun before this chunk
  // the chunk that holds the run's end
  int64_t lo = last + 1, hi = n_tok;  // first position past the run
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (entry_of(sorted[mid]) == e)
      lo = mid + 1;
    else
      hi = mid;
  }
  const int64_t end_chunk = (lo - 1) / kChunk;
  const int64_t d = static_cast<int64_t>(blockIdx.y) * kThreads + threadIdx.x;
  if (d >= D) return;
  float acc = partial[(static_cast<int64_t>(blockIdx.x) * 2 + 1) * D + d];
  constexpr int kAhead = 8;
  for (int64_t c = static_cast<int64_t>(blockIdx.x) + 1; c <= end_chunk; c += kAhead) {
    float v[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) v[i] = c + i <= end_chunk ? partial[(c + i) * 2 * D + d] : 0.f;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) acc += v[i];
  }
  grad[static_cast<int64_t>(e) * D + d] = static_cast<T>(acc * scale);
}

// ------------------------------------------------------------------- host --

int fail(int code, const std::string& msg) {
  set_error(msg);
  return code;
}

int64_t chunks(int64_t n_tok) { return (n_tok + kChunk - 1) / kChunk; }
int64_t round_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

int check(int64_t T, int64_t V, int64_t D, int dtype) {
  if (T <= 0 || V <= 0 || D <= 0) return fail(MLORA_ERR_INVALID_ARG, "T, V, D must be positive");
  if (dtype != MLORA_DTYPE_BF16 && dtype != MLORA_DTYPE_F16 && dtype != MLORA_DTYPE_F32)
    return fail(MLORA_ERR_UNSUPPORTED, "dtype must be BF16, F16 or F32");
  if (T > (int64_t{1} << 31) - 256 || V > (int64_t{1} << 31) - 256 || D > (1 << 23))
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
  const int64_t kb = round_up(T * 8, 256);
  w.keys = reinterpret_cast<uint64_t*>(b);
  w.sorted = T > kSortBlock ? reinterpret_cast<uint64_t*>(b + kb) : w.keys;
  const int64_t off = T > kSortBlock ? 2 * kb : kb;
  w.partial = reinterpret_cast<float*>(b + off);
  w.bytes = off + round_up(chunks(T) * 2 * D * 4, 256);
  return w;
}

template <typename T>
int gradient(const int64_t* idx, const void* dy, void* grad, int64_t n_tok, int64_t V, int64_t D,
             float scale, int64_t padding, const Work& w, cudaStream_t s) {
  cudaError_t e = cudaMemsetAsync(grad, 0, static_cast<size_t>(V * D) * sizeof(T), s);
  if (e != cudaSuccess) return launch_status(e, "embedding gradient");
  {
    LaunchScope scope(kKindElementwise, s);
    embedding_sort_kernel<<<static_cast<unsigned>((n_tok + kSortBlock - 1) / kSortBlock),
                            kSortThreads, 0, s>>>(idx, n_tok, V, padding, w.keys,
                                                  device_status_ptr());
  }
  if (n_tok > kSortBlock) {
    LaunchScope scope(kKindElementwise, s);
    embedding_merge_kernel<<<static_cast<unsigned>((n_tok + kThreads - 1) / kThreads), kThreads, 0,
                             s>>>(w.keys, n_tok, w.sorted);
  }
  const int vec = D % kVec<T> == 0 && aligned(dy, 16) && aligned(grad, 16);
  const int64_t cols = int64_t{kThreads} * kVec<T>;
  const unsigned n = static_cast<unsigned>(chunks(n_tok));
  {
    LaunchScope scope(kKindElementwise, s);
    embedding_grad_kernel<T><<<dim3(n, static_cast<unsigned>((D + cols - 1) / cols)), kThreads, 0, s>>>(
        w.sorted, static_cast<const T*>(dy), n_tok, D, scale, vec, static_cast<T*>(grad), w.partial);
  }
  if (n > 1) {
    LaunchScope scope(kKindElementwise, s);
    embedding_join_kernel<T><<<dim3(n - 1, static_cast<unsigned>((D + kThreads - 1) / kThreads)),
                               kThreads, 0, s>>>(w.sorted, w.partial, n_tok, D, scale,
                                                 static_cast<T*>(grad));
  }
  return launch_status(cudaSuccess, "embedding gradient");
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
