// Dropout whose mask is never stored: out = kept ? x * 65536 / (65536 - t) : 0, kept
// where the element's 16 bits (philox.cuh) are at least t.  The backward is the same
// call on dy.  Eight elements share one generator call, so that its ~90 integer
// instructions per thread hide behind the 16 (fp32: 32) bytes in and out; bound: HBM.
#include <string>

#include "internal.h"
#include "launch.cuh"
#include "philox.cuh"
#include "ptx.cuh"
#include "../../include/metallora_b200.h"

namespace mlora {
namespace {

constexpr int kThreads = 128;

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(e[i]);
  } else {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]),
                                              pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
  } else {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}

// x and out may be the same; `vec`: both start on 16 bytes.  Two blocks of eight a
// thread, loaded ahead of the generator's calls, which run interleaved.
template <typename T, bool kDevSeed>
__global__ void __launch_bounds__(kThreads)
    dropout_kernel(const T* x, T* out, int64_t n, int vec, float scale, DropoutKey key) {
  constexpr int kBlocks = 2;
  PhiloxKeys own;
  if constexpr (kDevSeed) own = philox_keys(static_cast<uint64_t>(*key.seed_dev));
  const PhiloxKeys& keys = kDevSeed ? own : key.keys;
  const int64_t whole = vec != 0 ? n / 8 : 0;  // blocks that go in vectors
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kThreads * kBlocks + threadIdx.x;
  float v[kBlocks][8];
#pragma unroll
  for (int j = 0; j < kBlocks; ++j) {
    const int64_t b = first + j * kThreads;
    if (b < whole) load8(x + b * 8, v[j]);
  }
#pragma unroll
  for (int j = 0; j < kBlocks; ++j) {
    const int64_t b = first + j * kThreads, e = b * 8;
    if (e >= n) break;
    const uint4 words = philox4x32_10(keys, static_cast<uint64_t>(b), key.call);
    if (b < whole) {
      dropout8(v[j], words, key.threshold, scale);
      store8(out + e, v[j]);
    } else {
      const int m = static_cast<int>(n - e < 8 ? n - e : 8);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = i < m ? static_cast<float>(x[e + i]) : 0.f;
      dropout8(v[j], words, key.threshold, scale);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < m) out[e + i] = static_cast<T>(v[j][i]);
    }
  }
}

}  // namespace

int launch_dropout(const void* x, void* out, int64_t n, int dtype, const DropoutKey& key,
                   bool scaled, cudaStream_t s) {
  const float scale = scaled ? dropout_scale(key.threshold) : 1.f;
  const int64_t ctas = (n + 16 * kThreads - 1) / (16 * kThreads);
  if (ctas > (int64_t{1} << 31) - 1) {
    set_error("dropout: too many elements");
    return MLORA_ERR_UNSUPPORTED;
  }
  const unsigned grid = static_cast<unsigned>(ctas);
  const int vec = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
  LaunchScope scope(kKindElementwise, s);
  auto run = [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    if (key.seed_dev != nullptr)
      dropout_kernel<T, true><<<grid, kThreads, 0, s>>>(static_cast<const T*>(x), static_cast<T*>(out), n,
                                                        vec, scale, key);
    else
      dropout_kernel<T, false><<<grid, kThreads, 0, s>>>(static_cast<const T*>(x),
                                                         static_cast<T*>(out), n, vec, scale, key);
  };
  if (dtype == MLORA_DTYPE_BF16)
    run(static_cast<__nv_bfloat16*>(nullptr));
  else if (dtype == MLORA_DTYPE_F16)
    run(static_cast<__half*>(nullptr));
  else
    run(static_cast<float*>(nullptr));
  return launch_status(cudaSuccess, "dropout");
}

}  // namespace mlora

using namespace mlora;

extern "C" int mlora_dropout(const void* x, void* out, int64_t n, int threshold, int scaled,
                             uint64_t seed, const int64_t* seed_dev, uint64_t call, int dtype,
                             void* stream) {
  auto fail = [](int code, const char* msg) {
    set_error(msg);
    return code;
  };
  if (n <= 0) return fail(MLORA_ERR_INVALID_ARG, "n must be positive");
  if (threshold < 0 || threshold > 65536)
    return fail(MLORA_ERR_INVALID_ARG, "threshold must be in [0, 65536]");
  if (dtype != MLORA_DTYPE_BF16 && dtype != MLORA_DTYPE_F16 && dtype != MLORA_DTYPE_F32)
    return fail(MLORA_ERR_UNSUPPORTED, "dtype must be BF16, F16 or F32");
  if (!x || !out) return fail(MLORA_ERR_INVALID_ARG, "NULL tensor pointer");
  const uintptr_t size = dtype == MLORA_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(x) % size || reinterpret_cast<uintptr_t>(out) % size ||
      reinterpret_cast<uintptr_t>(seed_dev) % 8)
    return fail(MLORA_ERR_INVALID_ARG, "pointers must be whole elements");
  if (int rc = require_device()) return rc;
  const DropoutKey key = dropout_key(seed, seed_dev, call, threshold);
  return launch_dropout(x, out, n, dtype, key, scaled != 0, static_cast<cudaStream_t>(stream));
}
