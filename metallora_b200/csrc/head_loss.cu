// Cross entropy of a linear head over a large vocabulary, from the hidden states,
// with its gradient; of [tokens, vocabulary] at most 2 GiB of 16-bit exponentials are
// held at a time, for gradients alone:
//
//   l = x . W^T (+ s (x . A^T) . B^T),   loss_m = log(sum_v exp l[m, v]) - l[m, y_m]
//   g[m, v] = softmax(l[m])[v] - [v = y_m]
//   dx = g . W + s (g . B) . A,  dW = g^T . x,  dB = g^T . (s x A^T),  dA = (s g B)^T . x
//
// Tokens labelled ignore_index have no loss and no gradient: the others are first
// gathered into consecutive rows, and every product runs over those alone (their
// number stays on the device).  Rows go through in pieces that bound the workspace.
// The gradients for a unit upstream gradient are made in the forward, while a piece's
// logits are at hand (a backward that made them would compute the logits again: half
// as many products more behind a frozen head); the backward scales them.
#include <algorithm>
#include <string>

#include "internal.h"
#include "launch.cuh"
#include "ptx.cuh"
#include "../../include/metallora_b200.h"

namespace mlora {
namespace {

constexpr int kScanThreads = 1024;
constexpr int kScanItems = 4;
constexpr int kRowThreads = 256;

// g is kept times this in fp16, so that probabilities down to 2^-20 are normal
// numbers there; a power of two, undone exactly by whoever scales the result.
// |g| <= 1, and 64 |s g B| <= 128 s max|B| is within fp16's range up to s max|B| = 511.
template <typename T>
__host__ __device__ constexpr float grad_unit() { return 1.f; }
template <>
__host__ __device__ constexpr float grad_unit<__half>() { return 64.f; }

struct HeadCount {
  int32_t counted;
  float inv;  // 1 / counted, 0 for none
  uint32_t ticket;  // CTAs that are through with their token's loss
};

__device__ __forceinline__ void set_count(HeadCount* out, int32_t counted) {
  out->counted = counted;
  out->inv = counted > 0 ? 1.f / static_cast<float>(counted) : 0.f;
  out->ticket = 0;
}

// One CTA: numbers the tokens that count in order (many tokens).  slot_of[m] = the token's number
// or -1; row_of[i], label[i] = token i's row and label (row_of = -1 past the last).
__global__ void __launch_bounds__(kScanThreads)
    head_scan_kernel(const int64_t* labels, int64_t M, int64_t V, int64_t ignore_index,
                     int32_t* slot_of, int32_t* row_of, int32_t* label, float* row_loss,
                     HeadCount* out, uint32_t* status) {
  __shared__ int32_t warp_sum[kScanThreads / 32];
  __shared__ int32_t total;
  grid_wait();
  launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int32_t base = 0;
  for (int64_t m0 = 0; m0 < M; m0 += kScanThreads * kScanItems) {
    const int64_t first = m0 + static_cast<int64_t>(threadIdx.x) * kScanItems;
    int32_t y[kScanItems];
    int32_t mine = 0;
#pragma unroll
    for (int i = 0; i < kScanItems; ++i) {
      y[i] = -1;
      if (first + i < M) {
        const int64_t v = labels[first + i];
        if (v != ignore_index) {
          if (v >= 0 && v < V)
            y[i] = static_cast<int32_t>(v);
          else
            record_status(status, kDevBadIndex);
        }
      }
      mine += y[i] >= 0;
    }
    int32_t run = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int32_t t = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += t;
    }
    if (lane == 31) warp_sum[warp] = run;
    __syncthreads();
    if (warp == 0) {
      const int32_t v = warp_sum[lane];
      int32_t w = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int32_t t = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += t;
      }
      warp_sum[lane] = w - v;
      if (lane == 31) total = w;
    }
    __syncthreads();
    int32_t slot = base + warp_sum[warp] + run - mine;
#pragma unroll
    for (int i = 0; i < kScanItems; ++i) {
      if (first + i >= M) break;
      const bool counts = y[i] >= 0;
      slot_of[first + i] = counts ? slot : -1;
      if (counts) {
        row_of[slot] = static_cast<int32_t>(first + i);
        label[slot] = y[i];
        ++slot;
      } else if (row_loss != nullptr) {
        row_loss[first + i] = 0.f;
      }
    }
    base += total;
    __syncthreads();
  }
  for (int64_t i = base + threadIdx.x; i < M; i += kScanThreads) row_of[i] = -1;
  if (threadIdx.x == 0) set_count(out, base);
}

// What the scan leaves of the tokens.
struct Numbers {
  int32_t *slot_of, *row_of, *label;
  HeadCount* count;
};

// xc[i] = x[row_of[i]], zeros past the last counted token (as many as a reduction
// over tokens reads; all of them for the LoRA products, which run over every row);
// and target[i] = the label's logit but for a LoRA term, in 32 bits; ref[i] = it in whole
// units of log 2; and uncut[i] = what gives the row's logits back what the tensor cores'
// accumulation cuts off on average (head_gemm.cu).  One CTA per row of xc, or with kNumber
// per token: each then counts the tokens ahead of its own itself, which up to some
// thousands is faster than a launch that numbers them.
constexpr int kGatherThreads = 128;
constexpr int64_t kNumberTokens = 2048;
constexpr float kCutPerGroup = 8.0e-9f;  // of 8 features
constexpr int kCutGroups = 1024;         // as many as were measured

template <typename T, bool kNumber>
__global__ void __launch_bounds__(kGatherThreads)
    head_gather_kernel(const uint4* x, const uint4* w, const int64_t* labels, int64_t ignore_index,
                       int64_t M, int64_t V, Numbers num, float* row_loss, int64_t K8, int64_t ld8,
                       int zero_all, uint4* xc, float* target, float* ref, float* uncut,
                       uint32_t* status) {
  __shared__ float part[4];
  __shared__ int32_t parts[2][4], groups[4];
  grid_wait();
  launch_dependents();
  int64_t i = blockIdx.x;
  int32_t row = -1, y = 0, counted = 0;
  if constexpr (kNumber) {
    const int64_t m = i;
    int32_t ahead = 0;
    for (int64_t q = threadIdx.x; q < M; q += kGatherThreads) {
      const int64_t v = labels[q];
      const bool counts = v != ignore_index && v >= 0 && v < V;
      ahead += counts && q < m;
      counted += counts;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
      counted += __shfl_xor_sync(0xffffffffu, counted, o);
    }
    if ((threadIdx.x & 31) == 0)
      parts[0][threadIdx.x >> 5] = ahead, parts[1][threadIdx.x >> 5] = counted;
    __syncthreads();
    ahead = parts[0][0] + parts[0][1] + parts[0][2] + parts[0][3];
    counted = parts[1][0] + parts[1][1] + parts[1][2] + parts[1][3];
    const int64_t v = labels[m];
    const bool counts = v != ignore_index && v >= 0 && v < V;
    // the token's number, or among the rest the place behind the counted ones
    i = counts ? ahead : counted + (m - ahead);
    if (counts) row = static_cast<int32_t>(m), y = static_cast<int32_t>(v);
    if (threadIdx.x == 0) {
      if (v != ignore_index && !counts) record_status(status, kDevBadIndex);
      num.slot_of[m] = counts ? ahead : -1;
      num.row_of[i] = row;
      num.label[i] = y;
      if (!counts && row_loss != nullptr) row_loss[m] = 0.f;
      if (m == 0) set_count(num.count, counted);
    }
  } else {
    row = num.row_of[i];
    counted = num.count->counted;
    if (row >= 0) y = num.label[i];
  }
  if (row < 0) {
    if (zero_all || i < (counted + 63) / 64 * 64)
      for (int64_t k = threadIdx.x; k < K8; k += kGatherThreads) xc[i * ld8 + k] = make_uint4(0, 0, 0, 0);
    return;
  }
  const uint4* xr = x + static_cast<int64_t>(row) * K8;
  const uint4* wr = w + static_cast<int64_t>(y) * K8;
  float s = 0.f;
  int32_t nonzero = 0;  // groups of 8 features, of either sign of zero
#pragma unroll 4
  for (int64_t k = threadIdx.x; k < K8; k += kGatherThreads) {
    const uint4 xv = xr[k], wv = wr[k];
    xc[i * ld8 + k] = xv;
    nonzero += ((xv.x | xv.y | xv.z | xv.w) & 0x7fff7fffu) != 0;
    const T* xe = reinterpret_cast<const T*>(&xv);
    const T* we = reinterpret_cast<const T*>(&wv);
#pragma unroll
    for (int j = 0; j < 8; ++j) s = fmaf(static_cast<float>(xe[j]), static_cast<float>(we[j]), s);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    nonzero += __shfl_xor_sync(0xffffffffu, nonzero, o);
  }
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s, groups[threadIdx.x >> 5] = nonzero;
  __syncthreads();
  if (threadIdx.x == 0) {
    const int32_t all = groups[0] + groups[1] + groups[2] + groups[3];
    uncut[i] = 1.f + kCutPerGroup * static_cast<float>(min(all, kCutGroups));
    const float t = part[0] + part[1] + (part[2] + part[3]);
    target[i] = t;
    // in units of log 2, within what leaves room above and below; 0 for no number
    if (ref != nullptr) ref[i] = fabsf(t) < INFINITY ? rintf(t * 1.4426950408889634f) : 0.f;
  }
}

// The loss of the call, once each of the M CTAs has passed here with its token's nll (or
// without one): the last one adds them up in order.  Sum of the counted tokens' losses,
// or their mean (of none: NaN, as 0 / 0 is).
struct LossOut {
  float* loss;  // may be null
  float* nll;
  int64_t M;
  int mean;
};

__device__ __forceinline__ void finish_loss(const LossOut& o, HeadCount* count) {
  if (o.loss == nullptr) return;
  __shared__ bool last;
  __shared__ double part[kRowThreads / 32];
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(&count->ticket, 1u) == static_cast<uint32_t>(o.M - 1);
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  const int32_t counted = count->counted;
  double s = 0.0;
  for (int32_t i = threadIdx.x; i < counted; i += kRowThreads) s += __ldcg(o.nll + i);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < kRowThreads / 32; ++w) s += part[w];
  *o.loss = static_cast<float>(o.mean ? s / counted : s);
}

// W2 of the logits: [B 0 | B 0], R columns each, for the two parts of s x A^T.
__global__ void __launch_bounds__(256)
    head_stack_kernel(const uint16_t* b, int64_t V, int r, int R, uint16_t* b2) {
  const int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (e >= V * R) return;
  const int64_t v = e / R;
  const int j = static_cast<int>(e - v * R);
  const uint16_t x = j < r ? b[v * r + j] : uint16_t{0};
  b2[v * 2 * R + j] = x;
  b2[v * 2 * R + R + j] = x;
}

__device__ __forceinline__ void join_max_sum(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2);
  // two empty parts (or rows of -infinity): nothing to scale by
  const float ref = top == -INFINITY ? 0.f : top;
  s = s * expf(m - ref) + s2 * expf(m2 - ref);
  m = top;
}

// The loss of a token from gap = m - l_y and s, where s exp(m) is the sum over the other
// entries, and u = s exp(gap): log(1 + u), by way of the larger of the two terms.
__device__ __forceinline__ float row_loss_of(float gap, float s, float u) {
  return gap < 0.f || s == 0.f ? log1pf(u) : gap + logf(s + expf(-gap));
}

// Summand j of the label's LoRA term: both parts of (s x A^T)[j] times B[y][j].
template <typename T>
__device__ __forceinline__ float lora_term(const T* xa, const T* b, int32_t y, int j, int r, int R) {
  return (static_cast<float>(xa[j]) + static_cast<float>(xa[R + j])) *
         static_cast<float>(b[static_cast<int64_t>(y) * r + j]);
}

// An infinite logit has no softmax, the label's neither.
__device__ __forceinline__ float gap_of(float gap, float ly) { return ly == INFINITY ? NAN : gap; }

// After the logits with one reference a row: one CTA per counted token of the piece.
// Its loss; the exponentials become its row of g but for a factor row_scale (left to
// the gradient of x) by setting the label's to -S, S the sum of the others.  Only a row
// with more than one reference is rewritten, by powers of two.
__global__ void __launch_bounds__(kRowThreads)
    head_ref_kernel(const float2* stats, int cols, int64_t V, int64_t ld, int64_t row0, Numbers num,
                    const float* target, float* row_loss, LossOut out, __nv_bfloat16* eg, float* rest,
                    float* row_scale) {
  __shared__ float sn[kRowThreads / 32], sl[kRowThreads / 32], ss[kRowThreads / 32];
  grid_wait();
  launch_dependents();
  const int64_t i = blockIdx.x;
  const int64_t slot = row0 + i;
  if (slot >= num.count->counted) {
    finish_loss(out, num.count);
    return;
  }
  const int tiles = static_cast<int>((V + cols - 1) / cols);
  const float2* st = stats + i * tiles;
  float top = -INFINITY, low = INFINITY;
  for (int t = threadIdx.x; t < tiles; t += kRowThreads) {
    const float n = st[t].x;
    top = fmaxf(top, n);
    low = fminf(low, n);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
  }
  if ((threadIdx.x & 31) == 0) sn[threadIdx.x >> 5] = top, sl[threadIdx.x >> 5] = low;
  __syncthreads();
  for (int w = 0; w < kRowThreads / 32; ++w) top = fmaxf(top, sn[w]), low = fminf(low, sl[w]);
  float s = 0.f;
  for (int t = threadIdx.x; t < tiles; t += kRowThreads) {
    const float2 q = st[t];
    s += q.x == top ? q.y : q.y * exp2f(q.x - top);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) ss[threadIdx.x >> 5] = s;
  __syncthreads();
  s = ss[0];
  for (int w = 1; w < kRowThreads / 32; ++w) s += ss[w];
  if (eg != nullptr && low != top) {
    __nv_bfloat16* row = eg + i * ld;
    for (int64_t v = threadIdx.x; v < V; v += kRowThreads) {
      const float n = st[static_cast<int>(v) / cols].x;
      if (n != top) row[v] = __float2bfloat16_rn(__bfloat162float(row[v]) * exp2f(n - top));
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    // top log 2 - l_y, log 2 in two parts (the first of 13 bits: its product is exact)
    const float ly = target[slot];
    const float gap = gap_of(fmaf(top, 0.693115234375f, -ly) + top * 3.19461832987e-05f, ly);
    const float u = s * expf(gap);
    const float loss = row_loss_of(gap, s, u);
    out.nll[slot] = loss;
    if (row_loss != nullptr) row_loss[num.row_of[slot]] = loss;
    if (eg != nullptr) {
      // 1 / (S + exp(l_y) 2^-top)
      row_scale[slot] = u < 1.f ? expf(gap) / (1.f + u) : 1.f / (s + expf(-gap));
      const __nv_bfloat16 gy = __float2bfloat16_rn(-s);
      eg[i * ld + num.label[slot]] = gy;
      rest[slot] = -s - __bfloat162float(gy);
    }
  }
  finish_loss(out, num.count);
}

constexpr int kHalfTile = 128;

// After the logits with a reference for each 128: one CTA per counted token of the piece.
// Its loss, and its row of g in place of the exponentials,
// e[v] -> g[v] = 2^-15 e[v] exp(m_t - lse).  With the sum S exp(m) over
// the other entries and u = S exp(m - l_y), the loss is log(1 + u) and
// g[y] = -u / (1 + u), without cancellation for a token that is nearly certain.
// What rounding g[y], the largest part, left over goes to `rest` (0 for tokens that do not
// count), which every gradient adds back: dx times W[y], U times B[y], rows y of dW and dB
// times x and s x A^T.  Bound: HBM, 4 bytes a logit.
template <typename T>
__global__ void __launch_bounds__(kRowThreads)
    head_row_kernel(const float2* stats, int64_t V, int64_t ld, int64_t row0, Numbers num,
                    const float* target, const T* xa, const T* b, int64_t xa_ld, int r, int R,
                    float* row_loss, LossOut out, void* eg, float* rest, float* row_scale,
                    int zero_all) {
  extern __shared__ float factor[];  // of each tile of logits
  __shared__ float sm[kRowThreads / 32], ss[kRowThreads / 32], sx[kRowThreads / 32];
  grid_wait();
  launch_dependents();
  const int64_t i = blockIdx.x;
  const int64_t slot = row0 + i;
  const int32_t counted = num.count->counted;
  uint4* row = static_cast<uint4*>(eg) + i * (ld / 8);
  if (slot >= counted) {
    if (eg != nullptr && (zero_all || slot < (counted + 63) / 64 * 64))
      for (int64_t v = threadIdx.x; v < ld / 8; v += kRowThreads) row[v] = make_uint4(0, 0, 0, 0);
    if (eg != nullptr && threadIdx.x == 0) rest[slot] = 0.f;
    finish_loss(out, num.count);
    return;
  }
  const int32_t y = num.label[slot];
  const int tiles = static_cast<int>((V + kHalfTile - 1) / kHalfTile);
  float m = -INFINITY, s = 0.f, extra = 0.f;
  for (int t = threadIdx.x; t < tiles; t += kRowThreads) {
    const float2 q = stats[i * tiles + t];
    factor[t] = q.x;
    join_max_sum(m, s, q.x, q.y * (1.f / 32768.f));
  }
  for (int j = threadIdx.x; j < r; j += kRowThreads) extra += lora_term(xa + slot * xa_ld, b, y, j, r, R);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    join_max_sum(m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
    extra += __shfl_xor_sync(0xffffffffu, extra, o);
  }
  if ((threadIdx.x & 31) == 0)
    sm[threadIdx.x >> 5] = m, ss[threadIdx.x >> 5] = s, sx[threadIdx.x >> 5] = extra;
  __syncthreads();
  m = sm[0], s = ss[0], extra = sx[0];
  for (int w = 1; w < kRowThreads / 32; ++w) {
    join_max_sum(m, s, sm[w], ss[w]);
    extra += sx[w];
  }
  const float ly = target[slot] + extra;
  const float gap = gap_of(m - ly, ly);
  const float u = s * expf(gap);
  const float loss = row_loss_of(gap, s, u);
  if (threadIdx.x == 0) {
    out.nll[slot] = loss;
    if (row_loss != nullptr) row_loss[num.row_of[slot]] = loss;
  }
  finish_loss(out, num.count);
  if (eg == nullptr) return;
  constexpr float unit = grad_unit<T>();
  const float lse = loss + ly;
  __syncthreads();
  for (int t = threadIdx.x; t < tiles; t += kRowThreads)
    factor[t] = factor[t] == -INFINITY ? 0.f : expf(factor[t] - lse) * (unit / 32768.f);
  __syncthreads();
  // -u / (1 + u), and -1 where u has no number
  const float gy = -unit * (gap < 60.f ? u / (1.f + u) : 1.f);
  if (threadIdx.x == 0) {
    rest[slot] = gy - static_cast<float>(static_cast<T>(gy));
    row_scale[slot] = 1.f / unit;
  }
  const int n8 = static_cast<int>((V + 7) / 8);
  constexpr int kAhead = 4;  // 16 bytes each in flight
  for (int q0 = threadIdx.x; q0 < n8; q0 += kAhead * kRowThreads) {
    uint4 v[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
      if (q0 + a * kRowThreads < n8) v[a] = row[q0 + a * kRowThreads];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int q = q0 + a * kRowThreads;
      if (q >= n8) break;
      const float f = factor[q * 8 / kHalfTile];
      const __half2* e = reinterpret_cast<const __half2*>(&v[a]);
      float o[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 p = __half22float2(e[j]);
        o[2 * j] = p.x * f;
        o[2 * j + 1] = p.y * f;
      }
      if (q == y >> 3) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j == (y & 7)) o[j] = gy;
      }
      row[q] = make_uint4(pack2<T>(o[0], o[1]), pack2<T>(o[2], o[3]), pack2<T>(o[4], o[5]),
                          pack2<T>(o[6], o[7]));
    }
  }
}

// What rounding g[y] left over, for the rows of dW and dB, by ranges of kRestTokens counted
// tokens, which bounds the search for tokens of one label and the work of a CTA.
//
// First each token's place in its range by (label, token), by counting: order[place] = the
// token, run[token] = (its label's first place, how many tokens that has, how many of them
// are ahead, the label).  A warp a token, all labels in shared memory.
constexpr int kRestTokens = 4096;
constexpr int kRunThreads = 32;

__global__ void __launch_bounds__(kRowThreads)
    head_runs_kernel(Numbers num, int32_t* order, int4* run) {
  __shared__ __align__(16) int32_t label[kRestTokens];
  grid_wait();
  launch_dependents();
  constexpr int kTokens = kRowThreads / kRunThreads;  // of a CTA, all of one range
  static_assert(kRestTokens % kTokens == 0, "ranges of whole CTAs");
  const int64_t cta_first = static_cast<int64_t>(blockIdx.x) * kTokens;
  const int64_t first = cta_first / kRestTokens * kRestTokens;
  const int64_t counted = num.count->counted;
  if (cta_first >= counted) return;
  const int tokens = static_cast<int>(min(counted - first, static_cast<int64_t>(kRestTokens)));
  const int own = static_cast<int>(cta_first - first) + static_cast<int>(threadIdx.x) / kRunThreads;
  const int padded = (tokens + 3) / 4 * 4;
#pragma unroll 8
  for (int i = threadIdx.x; i < padded; i += kRowThreads)
    label[i] = i < tokens ? num.label[first + i] : INT32_MAX;  // (behind every label)
  __syncthreads();
  const int32_t y = own < tokens ? label[own] : 0;
  int less = 0, ahead = 0, same = 0;
#pragma unroll 4
  for (int i = static_cast<int>(threadIdx.x) % kRunThreads * 4; i < padded; i += kRunThreads * 4) {
    const int4 q = *reinterpret_cast<const int4*>(label + i);
    less += (q.x < y) + (q.y < y) + (q.z < y) + (q.w < y);
    const int equal = (q.x == y) + (q.y == y) + (q.z == y) + (q.w == y);
    same += equal;
    if (i + 3 < own)
      ahead += equal;
    else if (i < own)
      ahead += (q.x == y) + (i + 1 < own && q.y == y) + (i + 2 < own && q.z == y);
  }
#pragma unroll
  for (int o = kRunThreads / 2; o > 0; o >>= 1) {
    less += __shfl_xor_sync(0xffffffffu, less, o);
    ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
    same += __shfl_xor_sync(0xffffffffu, same, o);
  }
  if (threadIdx.x % kRunThreads != 0 || own >= tokens) return;
  order[first + less + ahead] = own;
  run[first + own] = make_int4(less, same, ahead, y);
}

// Then, a launch for each range in order, out[y] += the sum of rest[i] src[i] over the
// tokens i of label y: row y of dW and dB would show all of it where y has few tokens (with
// one, up to the half step that rounding the row adds again).  src rows have `cols` columns
// and, with `second`, their second part that far behind.  A CTA per token and 2048 columns:
// of a label's CTAs the first one sums its tokens, or, where they are many, the first 16
// do, 128 columns each and their tokens in 16 groups of threads; in a fixed order either way.
// Bound: HBM, a row of dW read and written for each label: 60 us of 8192 tokens and 4096
// features, where the call takes 3.6 ms (a label that all of them have: 305 us); their
// places take 14 us.  What it is for: dW from two tokens is off by 0.0017 of itself,
// without it by 0.0031.
constexpr int kRestCols = 8 * kRowThreads;
constexpr int kRestMany = 16;  // and the groups

template <typename T>
__global__ void __launch_bounds__(kRowThreads, 4)
    head_rest_kernel(const HeadCount* count, int64_t first, const int32_t* order, const int4* run,
                     const float* rest, const T* src, int64_t ld, int second, int64_t cols, float* out) {
  __shared__ float4 sums[2 * kRowThreads];
  grid_wait();
  launch_dependents();
  const int own = static_cast<int>(blockIdx.x);  // of the tokens from `first` on
  if (first + own >= count->counted) return;
  const int4 r = run[first + own];
  const int n = r.y;
  const int tid = static_cast<int>(threadIdx.x);
  const int groups = n < kRestMany ? 1 : kRestMany;
  const int lanes = kRowThreads / groups, group = tid / lanes;
  const int64_t first_col = static_cast<int64_t>(blockIdx.y) * kRestCols;
  const int64_t width = min(cols - first_col, static_cast<int64_t>(kRestCols));
  if (r.z >= groups || r.z * lanes * 8 >= width) return;
  const int c = r.z * lanes * 8 + (tid - group * lanes) * 8;  // of `width` columns
  float4* const row =
      reinterpret_cast<float4*>(out + static_cast<int64_t>(r.w) * cols + first_col + c);
  const bool writes = group == 0 && c < width;
  float4 was[2];
  if (writes) was[0] = row[0], was[1] = row[1];
  float acc[8] = {};
  for (int part = 0; c < width && part <= second; part += second > 0 ? second : 1) {
    const T* const from = src + first * ld + part + first_col + c;
    constexpr int kAhead = 4;
    for (int i0 = group; i0 < n; i0 += groups * kAhead) {
      uint4 q[kAhead];
      float left[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const int i = i0 + a * groups;
        left[a] = 0.f;
        if (i < n) {
          const int64_t token = n == 1 ? own : order[first + r.x + i];
          q[a] = *reinterpret_cast<const uint4*>(from + token * ld);
          left[a] = rest[first + token];
        }
      }
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        if (i0 + a * groups >= n) break;
        const T* e = reinterpret_cast<const T*>(&q[a]);
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] = fmaf(left[a], static_cast<float>(e[k]), acc[k]);
      }
    }
  }
  if (groups > 1) {
    sums[2 * tid] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    sums[2 * tid + 1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
    __syncthreads();
    for (int g = 1; writes && g < groups; ++g) {
      const float4 a = sums[2 * (tid + g * lanes)], b = sums[2 * (tid + g * lanes) + 1];
      acc[0] += a.x, acc[1] += a.y, acc[2] += a.z, acc[3] += a.w;
      acc[4] += b.x, acc[5] += b.y, acc[6] += b.z, acc[7] += b.w;
    }
  }
  if (!writes) return;
  row[0] = make_float4(was[0].x + acc[0], was[0].y + acc[1], was[0].z + acc[2], was[0].w + acc[3]);
  row[1] = make_float4(was[1].x + acc[4], was[1].y + acc[5], was[1].z + acc[6], was[1].w + acc[7]);
}

// dx[row] = grad row_scale[slot] (sum over splits of part[split][slot] + rest[slot] W[y]);
// zeros for tokens that do not count.
template <typename T>
__global__ void __launch_bounds__(256)
    head_dx_kernel(const float* part, int64_t split_stride, int splits, const int32_t* slot_of,
                   const int32_t* label, const float* rest, const float* row_scale, const T* w,
                   const HeadCount* count, const float* grad, int per_row, int mean, int64_t K, T* dx) {
  const int64_t row = blockIdx.x;
  const int64_t k = (static_cast<int64_t>(blockIdx.y) * 256 + threadIdx.x) * 8;
  if (k >= K) return;
  const int32_t slot = slot_of[row];
  float v[8] = {};
  if (slot >= 0) {
    const float* src = part + static_cast<int64_t>(slot) * K + k;
    for (int s = 0; s < splits; ++s, src += split_stride) {
      const float4 a = *reinterpret_cast<const float4*>(src);
      const float4 b = *reinterpret_cast<const float4*>(src + 4);
      v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w;
      v[4] += b.x, v[5] += b.y, v[6] += b.z, v[7] += b.w;
    }
    const float scale = grad[per_row ? row : 0] * (mean ? count->inv : 1.f) * row_scale[slot];
    const float left = rest[slot];
    const uint4 wv = *reinterpret_cast<const uint4*>(w + static_cast<int64_t>(label[slot]) * K + k);
    const T* we = reinterpret_cast<const T*>(&wv);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = scale * fmaf(left, static_cast<float>(we[i]), v[i]);
  }
  uint4 o;
  o.x = pack2<T>(v[0], v[1]);
  o.y = pack2<T>(v[2], v[3]);
  o.z = pack2<T>(v[4], v[5]);
  o.w = pack2<T>(v[6], v[7]);
  *reinterpret_cast<uint4*>(dx + row * K + k) = o;
}

template <typename O>
__device__ __forceinline__ void store8(O* dst, const float (&v)[8]) {
  if constexpr (sizeof(O) == 2) {
    *reinterpret_cast<uint4*>(dst) = make_uint4(pack2<O>(v[0], v[1]), pack2<O>(v[2], v[3]),
                                                pack2<O>(v[4], v[5]), pack2<O>(v[6], v[7]));
  } else {
    reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}

// out (+)= grad / unit * src, n a multiple of 8; a gradient of a weight.  (Where no
// token counted, src is zero and so is the result, whatever grad is.)
template <typename O>
__global__ void __launch_bounds__(256)
    head_scale_kernel(const float* src, int64_t n8, const HeadCount* count, const float* grad,
                      int mean, float inv_unit, int accumulate, O* out) {
  const float scale = count->counted > 0 ? *grad * (mean ? count->inv : 1.f) * inv_unit : 0.f;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n8;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    const float4 a = reinterpret_cast<const float4*>(src)[2 * i];
    const float4 b = reinterpret_cast<const float4*>(src)[2 * i + 1];
    float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = scale == 0.f ? 0.f : v[j] * scale;
      if (accumulate) v[j] += static_cast<float>(out[i * 8 + j]);
    }
    store8(out + i * 8, v);
  }
}

// ------------------------------------------------------------------- host --

int fail(int code, const std::string& msg) {
  set_error(msg);
  return code;
}

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
int64_t round_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

struct Carve {
  uint8_t* base;
  int64_t off = 0;
  explicit Carve(void* b) : base(static_cast<uint8_t*>(b)) {}
  template <typename T>
  T* take(int64_t n) {
    off = round_up(off, 256);
    T* p = base != nullptr ? reinterpret_cast<T*>(base + off) : nullptr;
    off += n * static_cast<int64_t>(sizeof(T));
    return p;
  }
};

struct Dims {
  int64_t M, K, V, r;
  int grads;
  bool bf16;
  // one reference a row: g's factor per row, and what rounding its label's entry left
  // over, go to dx (for a LoRA head, whose dA and dB would want both too, it gained 1.4 %
  // and took their error from 0.0019 to 0.0026)
  bool by_row() const { return bf16 && r == 0 && !want(MLORA_HEAD_GRAD_W); }
  bool lora() const { return r > 0; }
  bool want(int g) const { return (grads & g) != 0; }
  int64_t R() const {
    int64_t v = 16;
    while (v < r) v *= 2;
    return v;
  }
  int64_t R64() const { return round_up(R(), 64); }
  int64_t ld_xa() const { return round_up(2 * R(), 64); }  // two parts of s x A^T
  // of a row of e and g, and of the gathered x: whole 128-byte lines, since a TMA box
  // row that crosses a line costs two requests (x of 1032 features and the weight's
  // rows both off the lines: 870 cycles for a 256 x 256 x 64 step that takes 512)
  int64_t ld() const { return round_up(V, 64); }
  int64_t ldx() const { return round_up(K, 64); }
  int64_t tiles(int cols) const { return (V + cols / 2 - 1) / (cols / 2); }  // half tiles
};

// Columns of a tile of logits with one reference a row (else 256, whose halves the
// softmax pass finds by a shift): 256, or the multiple of 32 from 192 on that makes the
// waves of tiles over the CTA pairs take at least a twelfth less together.  412 tokens
// 4096 -> 32000: 4 waves of 256 columns take 101 us, 4 of 224 95 us; narrower tiles
// move more per product, and 55 waves took a tenth longer for a nominal gain.
int logit_cols(const Dims& d, int64_t rows) {
  if (!d.by_row()) return 256;
  const int64_t pairs = num_sms() / 2, tiles_m = (rows + 255) / 256;
  auto time = [&](int64_t n) { return (tiles_m * ((d.V + n - 1) / n) + pairs - 1) / pairs * n; };
  int best = 256;
  for (int n = 224; n >= 192; n -= 32)
    if (time(n) * 12 <= time(256) * 11 && (best == 256 || time(n) < time(best))) best = n;
  return best;
}

// Ranges of the vocabulary that dx is summed over: enough for the tiles of few tokens
// to occupy every CTA pair, against the copies that the backward then reads.  The rule
// takes the count with the least time for whole waves of tiles (a 256 x 256 x 64 step
// takes 0.29 us) plus writing and reading the copies.
int dx_splits(const Dims& d) {
  const int64_t tiles = (d.M + 255) / 256 * ((d.K + 255) / 256);
  const int64_t kbs = (d.V + 63) / 64;
  const int64_t pairs = num_sms() / 2;
  int best = 1;
  double best_us = 0;
  for (int s = 1; s <= 32 && s <= kbs; ++s) {
    const double waves = static_cast<double>((tiles * s + pairs - 1) / pairs);
    const double us = waves * static_cast<double>((kbs + s - 1) / s) * 0.29 +
                      static_cast<double>(s) * d.M * d.K * 8 / 6.0e6;
    if (s == 1 || us < best_us) best = s, best_us = us;
  }
  return best;
}

// What the backward takes.
struct State {
  HeadCount* count;
  int32_t *slot_of, *label;
  float *rest, *row_scale, *dx, *da, *db, *dw;
  int splits;
  int64_t bytes;
};

State plan_state(void* base, const Dims& d) {
  State s{};
  Carve c(base);
  s.splits = dx_splits(d);
  s.count = c.take<HeadCount>(1);
  s.slot_of = c.take<int32_t>(d.M);
  s.label = c.take<int32_t>(d.M);
  s.rest = c.take<float>(d.M);
  s.row_scale = c.take<float>(d.M);
  if (d.want(MLORA_HEAD_GRAD_X)) s.dx = c.take<float>(s.splits * d.M * d.K);
  if (d.want(MLORA_HEAD_GRAD_AB)) {
    s.da = c.take<float>(d.r * d.K);
    s.db = c.take<float>(d.V * d.r);
  }
  if (d.want(MLORA_HEAD_GRAD_W)) s.dw = c.take<float>(d.V * d.K);
  s.bytes = round_up(c.off, 256);
  return s;
}

struct Work {
  int32_t *row_of, *order;
  int4* run;
  float* nll;
  float *target, *ref, *uncut;
  void *xc, *xa_rows, *xa_t, *xa_lo, *b2, *bt, *u_rows, *u_t, *u_lo, *eg;
  float2* stats;
  int64_t piece;  // rows that go through at a time
  int cols;       // of a tile of logits
  int64_t tiles;  // half tiles: what shares a reference
  int64_t bytes;
};

Work plan_work(void* base, const Dims& d) {
  Work w{};
  Carve c(base);
  // pieces of two gigabytes of exponentials (or 256 rows), equal up to the tile
  const int64_t per_row = d.grads ? d.ld() * 2 : d.tiles(192) * 8;
  const int64_t most = std::max<int64_t>(int64_t{2048} << 20, 256 * per_row) / per_row / 256 * 256;
  const int64_t n = (d.M + most - 1) / most;
  w.piece = std::min(d.M, round_up((d.M + n - 1) / n, 256));
  w.cols = logit_cols(d, w.piece);
  w.tiles = d.tiles(w.cols);
  w.row_of = c.take<int32_t>(d.M);
  if (d.grads & (MLORA_HEAD_GRAD_W | MLORA_HEAD_GRAD_AB)) {
    w.order = c.take<int32_t>(d.M);
    w.run = c.take<int4>(d.M);
  }
  w.nll = c.take<float>(d.M);
  w.target = c.take<float>(d.M);
  w.ref = c.take<float>(d.M);
  w.uncut = c.take<float>(d.M);
  w.xc = c.take<uint16_t>(d.M * d.ldx());
  if (d.lora()) {
    w.xa_rows = c.take<uint16_t>(d.M * d.ld_xa());
    w.b2 = c.take<uint16_t>(d.V * 2 * d.R());
    if (d.grads) {
      w.xa_t = c.take<uint16_t>(d.R() * round_up(d.M, 8));
      w.xa_lo = c.take<uint16_t>(d.R() * round_up(d.M, 8));
      w.bt = c.take<uint16_t>(d.R() * d.V);
      w.u_rows = c.take<uint16_t>(w.piece * d.R64());
      w.u_t = c.take<uint16_t>(d.R() * round_up(w.piece, 8));
      w.u_lo = c.take<uint16_t>(d.R() * round_up(w.piece, 8));
    }
  }
  w.stats = c.take<float2>(w.tiles * w.piece);
  if (d.grads) w.eg = c.take<uint16_t>(w.piece * d.ld());
  w.bytes = round_up(c.off, 256);
  return w;
}

int check_dims(const Dims& d, int dtype) {
  if (d.M <= 0 || d.K <= 0 || d.V <= 0) return fail(MLORA_ERR_INVALID_ARG, "M, K, V must be positive");
  if (dtype != MLORA_DTYPE_BF16 && dtype != MLORA_DTYPE_F16)
    return fail(MLORA_ERR_UNSUPPORTED, "the linear cross entropy takes BF16 or F16");
  if (d.grads & ~(MLORA_HEAD_GRAD_X | MLORA_HEAD_GRAD_W | MLORA_HEAD_GRAD_AB))
    return fail(MLORA_ERR_INVALID_ARG, "unknown gradient flags");
  if (d.r < 0 || d.r > 256) return fail(MLORA_ERR_INVALID_ARG, "rank must be in [0, 256]");
  if ((d.grads & MLORA_HEAD_GRAD_AB) && d.r == 0)
    return fail(MLORA_ERR_INVALID_ARG, "gradients of A and B need a rank");
  if (d.K % 8 || d.r % 8)
    return fail(MLORA_ERR_UNSUPPORTED, "K and r must be multiples of 8 (16-byte rows)");
  if (d.lora() && d.V % 8)
    return fail(MLORA_ERR_UNSUPPORTED, "a LoRA head needs V % 8 == 0 (16-byte rows of B^T)");
  if (d.M > (int64_t{1} << 31) - 256 || d.K > (1 << 24) || d.V > (1 << 20))
    return fail(MLORA_ERR_UNSUPPORTED, "shape too large");
  return MLORA_OK;
}

template <typename T>
int forward(const void* x, const void* w, const void* a, const void* b, const int64_t* labels,
            float* loss, float* row_loss, const State& st, const Work& ws, const Dims& d,
            float alpha, int64_t ignore_index, bool mean, cudaStream_t s) {
  const Elt elt = std::is_same<T, __half>::value ? Elt::kF16 : Elt::kBF16;
  const int64_t M = d.M, K = d.K, V = d.V, ld = d.ld(), ldx = d.ldx();
  const int zero_all = d.lora() ? 1 : 0;
  const bool by_row = d.by_row();
  int rc;
  const Numbers num{st.slot_of, ws.row_of, st.label, st.count};
  const LossOut out{loss, ws.nll, M, mean ? 1 : 0};
  const bool number = M <= kNumberTokens;
  // every kernel here waits for the one before it and then lets the next one start
  cudaError_t e = cudaSuccess;
  if (!number) {
    LaunchScope scope(kKindElementwise, s);
    e = launch_kernel(head_scan_kernel, dim3(1), kScanThreads, 0, s, 0, 0, true, labels, M, V,
                      ignore_index, st.slot_of, ws.row_of, st.label, row_loss, st.count,
                      device_status_ptr());
  }
  if (e == cudaSuccess) {
    LaunchScope scope(kKindElementwise, s);
    e = launch_kernel(number ? head_gather_kernel<T, true> : head_gather_kernel<T, false>,
                      dim3(static_cast<unsigned>(M)), kGatherThreads, 0, s, 0, 0, true,
                      static_cast<const uint4*>(x), static_cast<const uint4*>(w), labels, ignore_index, M,
                      V, num, row_loss, K / 8, ldx / 8, zero_all, static_cast<uint4*>(ws.xc), ws.target,
                      by_row ? ws.ref : nullptr, ws.uncut, device_status_ptr());
  }
  if ((rc = launch_status(e, "linear cross entropy: gather"))) return rc;
  RankArgs ra;
  if (d.lora()) {
    ra.x = ws.xc;
    ra.l = a;
    ra.M = M;
    ra.K = K;
    ra.r = d.r;
    ra.R = d.R();
    ra.ldx = ldx;
    ra.ldl = K;
    ra.scale = alpha / static_cast<float>(d.r);
    ra.out_rows = ws.xa_rows;
    ra.ld_rows = d.ld_xa();
    ra.two_rows = true;
    ra.out_t = ws.xa_t;
    ra.out_t_lo = ws.xa_lo;
    ra.ld_t = round_up(M, 8);
    ra.splits = rank_splits(M, K);
    ra.elt = elt;
    if ((rc = launch_rank(ra, s))) return rc;
    {
      LaunchScope scope(kKindElementwise, s);
      head_stack_kernel<<<static_cast<unsigned>((V * d.R() + 255) / 256), 256, 0, s>>>(
          static_cast<const uint16_t*>(b), V, static_cast<int>(d.r), static_cast<int>(d.R()),
          static_cast<uint16_t*>(ws.b2));
    }
    if (d.grads && (rc = launch_transpose_pad(b, V, d.r, d.r, ws.bt, d.R(), elt, s))) return rc;
  }
  for (int64_t row0 = 0; row0 < M; row0 += ws.piece) {
    const int64_t rows = std::min(ws.piece, M - row0);
    const T* xc = static_cast<const T*>(ws.xc) + row0 * ldx;
    HeadGemmArgs l;
    l.product = HeadProduct::kLogits;
    l.x = xc;
    l.w = w;
    l.M = rows;
    l.N = V;
    l.K = K;
    l.ldx = ldx;
    l.ldw = K;
    l.ldd = ld;
    l.rows = &st.count->counted;
    l.row0 = row0;
    l.label = st.label + row0;
    l.e = ws.eg;
    l.stats = ws.stats;
    l.stats_ld = ws.tiles;
    l.tile_n = ws.cols;
    l.uncut = ws.uncut + row0;
    l.ref = by_row ? ws.ref + row0 : nullptr;
    l.elt = elt;
    if (d.lora()) {
      l.x2 = static_cast<const T*>(ws.xa_rows) + row0 * d.ld_xa();
      l.w2 = ws.b2;
      l.R = 2 * d.R();
      l.w2_rows = 2 * d.R();
      l.ldx2 = d.ld_xa();
      l.ldw2 = 2 * d.R();
    }
    if ((rc = launch_head_gemm(l, s))) return rc;
    {
      LaunchScope scope(kKindElementwise, s);
      const dim3 grid(static_cast<unsigned>(rows));
      if (by_row)
        e = launch_kernel(head_ref_kernel, grid, kRowThreads, 0, s, 0, 0, true,
                          static_cast<const float2*>(ws.stats), ws.cols / 2, V, ld, row0, num,
                          static_cast<const float*>(ws.target), row_loss, out,
                          static_cast<__nv_bfloat16*>(ws.eg), st.rest, st.row_scale);
      else
        e = launch_kernel(head_row_kernel<T>, grid, kRowThreads, static_cast<size_t>(ws.tiles) * 4, s, 0,
                          0, true, static_cast<const float2*>(ws.stats), V, ld, row0, num,
                          static_cast<const float*>(ws.target), static_cast<const T*>(ws.xa_rows),
                          static_cast<const T*>(b), d.ld_xa(), static_cast<int>(d.r),
                          static_cast<int>(d.R()), row_loss, out, ws.eg, st.rest, st.row_scale, zero_all);
      if ((rc = launch_status(e, "linear cross entropy: rows"))) return rc;
    }
    if (d.lora() && d.grads) {
      // U = s g B.  It enters dx in one 16-bit part, of a term that is small beside g W
      // (rank 16 to 64: dx is off by 0.0017 to 0.0018 of itself, rounded 0.0017), and dA,
      // which has nothing else, in two (one: 0.0026)
      RankArgs ru = ra;
      ru.x = ws.eg;
      ru.l = ws.bt;
      ru.M = rows;
      ru.K = V;
      ru.r = d.R();
      ru.ldx = ld;
      ru.ldl = V;
      ru.out_rows = ws.u_rows;
      ru.ld_rows = d.R64();
      ru.two_rows = false;
      ru.out_t = ws.u_t;
      ru.out_t_lo = ws.u_lo;
      ru.ld_t = round_up(ws.piece, 8);
      ru.add_weight = st.rest + row0;
      ru.add_row = st.label + row0;
      ru.add = b;
      ru.add_cols = d.r;
      ru.splits = rank_splits(rows, V);
      if ((rc = launch_rank(ru, s))) return rc;
      if (d.want(MLORA_HEAD_GRAD_AB)) {
        WgradArgs g[2];
        g[0].big = ws.eg;
        g[0].st = static_cast<const T*>(ws.xa_t) + row0;
        g[0].st_lo = static_cast<const T*>(ws.xa_lo) + row0;
        g[0].ld_st = round_up(M, 8);
        g[0].M = rows;
        g[0].P = V;
        g[0].r = d.r;
        g[0].R = d.R();
        g[0].ldb = ld;
        g[0].out = st.db;
        g[0].ldo = d.r;
        g[0].transposed = false;
        g[0].accumulate = row0 > 0;
        g[0].clip = 0.f;
        g[0].splits = wgrad_splits(rows, std::max(V, K), 2);
        g[0].elt = elt;
        g[1] = g[0];
        g[1].big = xc;
        g[1].st = ws.u_t;
        g[1].st_lo = ws.u_lo;
        g[1].ld_st = round_up(ws.piece, 8);
        g[1].P = K;
        g[1].ldb = ldx;
        g[1].out = st.da;
        g[1].ldo = K;
        g[1].transposed = true;
        if ((rc = launch_wgrad(g, 2, s))) return rc;
      }
    }
    if (d.want(MLORA_HEAD_GRAD_X)) {
      HeadGemmArgs q;
      q.product = HeadProduct::kDx;
      q.x = w;
      q.w = ws.eg;
      q.d = st.dx + row0 * K;
      q.M = K;
      q.N = rows;
      q.K = V;
      q.ldx = K;
      q.ldw = ld;
      q.ldd = K;
      q.split_stride = M * K;
      q.splits = st.splits;
      q.rows = &st.count->counted;
      q.row0 = row0;
      q.elt = elt;
      if (d.lora()) {
        q.x2 = a;
        q.w2 = ws.u_rows;
        q.R = d.R();
        q.x2_rows = d.r;
        q.w2_rows = d.R64();
        q.ldx2 = K;
        q.ldw2 = d.R64();
      }
      if ((rc = launch_head_gemm(q, s))) return rc;
    }
    if (d.want(MLORA_HEAD_GRAD_W)) {
      HeadGemmArgs q;
      q.product = HeadProduct::kDw;
      q.x = ws.eg;
      q.w = xc;
      q.d = st.dw;
      q.M = V;
      q.N = K;
      q.K = rows;
      q.ldx = ld;
      q.ldw = ldx;
      q.ldd = K;
      q.rows = &st.count->counted;
      q.row0 = row0;
      q.group_m = 1;
      q.accumulate = row0 > 0;
      q.elt = elt;
      if ((rc = launch_head_gemm(q, s))) return rc;
    }
  }
  auto add_rest = [&](int64_t first, const void* src, int64_t ld_src, int second, int64_t cols,
                      float* out_rows) {
    LaunchScope scope(kKindElementwise, s);
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(M - first, kRestTokens)),
                    static_cast<unsigned>((cols + kRestCols - 1) / kRestCols));
    return launch_kernel(head_rest_kernel<T>, grid, kRowThreads, 0, s, 0, 0, true,
                         static_cast<const HeadCount*>(st.count), first,
                         static_cast<const int32_t*>(ws.order), static_cast<const int4*>(ws.run),
                         static_cast<const float*>(st.rest), static_cast<const T*>(src), ld_src, second,
                         cols, out_rows);
  };
  const bool dw = d.want(MLORA_HEAD_GRAD_W), db = d.want(MLORA_HEAD_GRAD_AB);
  if (dw || db) {
    LaunchScope scope(kKindElementwise, s);
    const int64_t per = kRowThreads / kRunThreads;
    e = launch_kernel(head_runs_kernel, dim3(static_cast<unsigned>((M + per - 1) / per)), kRowThreads, 0,
                      s, 0, 0, true, num, ws.order, ws.run);
  }
  for (int64_t first = 0; (dw || db) && first < M; first += kRestTokens) {
    if (e == cudaSuccess && dw) e = add_rest(first, ws.xc, ldx, 0, K, st.dw);
    if (e == cudaSuccess && db)
      e = add_rest(first, ws.xa_rows, d.ld_xa(), static_cast<int>(d.R()), d.r, st.db);
    if ((rc = launch_status(e, "linear cross entropy: rest of the labels' entries"))) return rc;
  }
  return MLORA_OK;
}

int launch_scale(const float* src, int64_t n, const State& st, const float* grad, bool mean,
                 float inv_unit, bool accumulate, void* out, int dtype, cudaStream_t s) {
  const int64_t n8 = n / 8;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>((n8 + 255) / 256, num_sms() * 16));
  LaunchScope scope(kKindElementwise, s);
  const int m = mean ? 1 : 0, acc = accumulate ? 1 : 0;
  if (dtype == MLORA_DTYPE_BF16)
    head_scale_kernel<<<grid, 256, 0, s>>>(src, n8, st.count, grad, m, inv_unit, acc,
                                           static_cast<__nv_bfloat16*>(out));
  else if (dtype == MLORA_DTYPE_F16)
    head_scale_kernel<<<grid, 256, 0, s>>>(src, n8, st.count, grad, m, inv_unit, acc,
                                           static_cast<__half*>(out));
  else
    head_scale_kernel<<<grid, 256, 0, s>>>(src, n8, st.count, grad, m, inv_unit, acc,
                                           static_cast<float*>(out));
  return launch_status(cudaSuccess, "linear cross entropy: weight gradient");
}

template <typename T>
int backward(const State& st, const Dims& d, const void* w, const float* grad, bool per_row,
             bool mean, void* dx, cudaStream_t s) {
  LaunchScope scope(kKindElementwise, s);
  const dim3 grid(static_cast<unsigned>(d.M), static_cast<unsigned>((d.K / 8 + 255) / 256));
  head_dx_kernel<T><<<grid, 256, 0, s>>>(st.dx, d.M * d.K, st.splits, st.slot_of, st.label, st.rest,
                                         st.row_scale, static_cast<const T*>(w), st.count, grad, per_row ? 1 : 0,
                                         mean ? 1 : 0, d.K, static_cast<T*>(dx));
  return launch_status(cudaSuccess, "linear cross entropy: dx");
}

}  // namespace
}  // namespace mlora

using namespace mlora;

extern "C" {

size_t mlora_linear_cross_entropy_state_bytes(int64_t M, int64_t K, int64_t V, int64_t r, int dtype,
                                              int grads) {
  const Dims d{M, K, V, r, grads, dtype == MLORA_DTYPE_BF16};
  if (check_dims(d, dtype)) return 0;
  return static_cast<size_t>(plan_state(nullptr, d).bytes);
}

size_t mlora_linear_cross_entropy_workspace_bytes(int64_t M, int64_t K, int64_t V, int64_t r,
                                                  int dtype, int grads) {
  const Dims d{M, K, V, r, grads, dtype == MLORA_DTYPE_BF16};
  if (check_dims(d, dtype)) return 0;
  return static_cast<size_t>(plan_work(nullptr, d).bytes);
}

int mlora_linear_cross_entropy(const void* x, const void* w, const void* a, const void* b,
                               const int64_t* labels, float* loss, float* row_loss, void* state,
                               size_t state_bytes, int64_t M, int64_t K, int64_t V, int64_t r,
                               float alpha, int64_t ignore_index, int mean, int dtype, int grads,
                               void* workspace, size_t workspace_bytes, void* stream) {
  const Dims d{M, K, V, r, grads, dtype == MLORA_DTYPE_BF16};
  if (int rc = check_dims(d, dtype)) return rc;
  if (!x || !w || !labels || !state || (!loss && !row_loss) || (r > 0 && (!a || !b)))
    return fail(MLORA_ERR_INVALID_ARG, "NULL tensor pointer");
  if (!aligned(x, 16) || !aligned(w, 16) || !aligned(a, 16) || !aligned(b, 16) ||
      !aligned(labels, 8) || !aligned(loss, 4) || !aligned(row_loss, 4))
    return fail(MLORA_ERR_INVALID_ARG,
                "tensor pointers must be 16-byte aligned, labels and losses whole elements");
  const State st = plan_state(state, d);
  if (!aligned(state, 256) || state_bytes < static_cast<size_t>(st.bytes))
    return fail(MLORA_ERR_WORKSPACE, "the state needs " + std::to_string(st.bytes) +
                                         " bytes on a 256-byte boundary");
  const Work ws = plan_work(workspace, d);
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < static_cast<size_t>(ws.bytes))
    return fail(MLORA_ERR_WORKSPACE, "the workspace needs " + std::to_string(ws.bytes) +
                                         " bytes on a 256-byte boundary");
  if (int rc = require_device()) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == MLORA_DTYPE_BF16
             ? forward<__nv_bfloat16>(x, w, a, b, labels, loss, row_loss, st, ws, d, alpha,
                                      ignore_index, mean != 0, s)
             : forward<__half>(x, w, a, b, labels, loss, row_loss, st, ws, d, alpha, ignore_index,
                               mean != 0, s);
}

int mlora_linear_cross_entropy_backward(const void* state, size_t state_bytes, const float* grad,
                                        int per_row, int mean, const void* w, void* dx, void* da,
                                        void* db, int ab_dtype, int accumulate_ab, void* dw,
                                        int64_t M, int64_t K, int64_t V, int64_t r, int dtype,
                                        int grads, void* stream) {
  const Dims d{M, K, V, r, grads, dtype == MLORA_DTYPE_BF16};
  if (int rc = check_dims(d, dtype)) return rc;
  if (!state || !grad || !w) return fail(MLORA_ERR_INVALID_ARG, "NULL tensor pointer");
  if (d.want(MLORA_HEAD_GRAD_X) != (dx != nullptr) || d.want(MLORA_HEAD_GRAD_AB) != (da != nullptr) ||
      d.want(MLORA_HEAD_GRAD_AB) != (db != nullptr) || d.want(MLORA_HEAD_GRAD_W) != (dw != nullptr))
    return fail(MLORA_ERR_INVALID_ARG, "the gradients asked for are those the forward made");
  if (!aligned(w, 16) || !aligned(dx, 16) || !aligned(da, 16) || !aligned(db, 16) ||
      !aligned(dw, 16) || !aligned(grad, 4))
    return fail(MLORA_ERR_INVALID_ARG, "tensor pointers must be 16-byte aligned");
  if (ab_dtype != MLORA_DTYPE_BF16 && ab_dtype != MLORA_DTYPE_F16 && ab_dtype != MLORA_DTYPE_F32)
    return fail(MLORA_ERR_UNSUPPORTED, "gradients of A and B are BF16, F16 or F32");
  if (per_row && (grads & ~MLORA_HEAD_GRAD_X))
    return fail(MLORA_ERR_UNSUPPORTED, "a gradient per token reaches x alone");
  const State st = plan_state(const_cast<void*>(state), d);
  if (!aligned(state, 256) || state_bytes < static_cast<size_t>(st.bytes))
    return fail(MLORA_ERR_WORKSPACE, "the state is smaller than the forward's");
  if (int rc = require_device()) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf16 = dtype == MLORA_DTYPE_BF16, avg = mean != 0;
  const float inv_unit = 1.f / (bf16 ? grad_unit<__nv_bfloat16>() : grad_unit<__half>());
  int rc = MLORA_OK;
  if (da != nullptr) {
    rc = launch_scale(st.da, r * K, st, grad, avg, inv_unit, accumulate_ab != 0, da, ab_dtype, s);
    if (rc == MLORA_OK)
      rc = launch_scale(st.db, V * r, st, grad, avg, inv_unit, accumulate_ab != 0, db, ab_dtype, s);
  }
  if (rc == MLORA_OK && dx != nullptr)
    rc = bf16 ? backward<__nv_bfloat16>(st, d, w, grad, per_row != 0, avg, dx, s)
              : backward<__half>(st, d, w, grad, per_row != 0, avg, dx, s);
  if (rc == MLORA_OK && dw != nullptr)
    rc = launch_scale(st.dw, V * K, st, grad, avg, inv_unit, false, dw, dtype, s);
  return rc;
}

}  // extern "C"
