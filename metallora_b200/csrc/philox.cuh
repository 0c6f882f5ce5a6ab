// Philox4x32-10, the counter-based generator of Salmon, Moraes, Dror and Shaw,
// "Parallel Random Numbers: As Easy as 1, 2, 3" (SC 2011): four 32-bit words for a
// 64-bit key and a 128-bit counter, with no state, so that any thread makes the
// numbers of any element, and the backward those of the forward.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace mlora {

// The key of each round.
struct PhiloxKeys {
  uint32_t k0[10], k1[10];
};

__host__ __device__ inline PhiloxKeys philox_keys(uint64_t seed) {
  PhiloxKeys k;
  uint32_t a = static_cast<uint32_t>(seed), b = static_cast<uint32_t>(seed >> 32);
  for (int r = 0; r < 10; ++r) {
    k.k0[r] = a;
    k.k1[r] = b;
    a += 0x9E3779B9u;
    b += 0xBB67AE85u;
  }
  return k;
}

struct DropoutKey {
  PhiloxKeys keys;          // of the seed: made on the host, read as constants
  const int64_t* seed_dev;  // where not null, the seed (read by the kernel, so that
                            // a replayed graph follows it)
  uint64_t call;            // which use of the seed this is
  uint32_t threshold;       // of 65536: elements whose 16 bits are below it are dropped
};

inline DropoutKey dropout_key(uint64_t seed, const int64_t* seed_dev, uint64_t call, int threshold) {
  return {philox_keys(seed), seed_dev, call, static_cast<uint32_t>(threshold)};
}

__device__ __forceinline__ uint4 philox4x32_10(const PhiloxKeys& k, uint64_t block, uint64_t call) {
  uint4 c = make_uint4(static_cast<uint32_t>(block), static_cast<uint32_t>(block >> 32),
                       static_cast<uint32_t>(call), static_cast<uint32_t>(call >> 32));
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = static_cast<uint64_t>(0xD2511F53u) * c.x;
    const uint64_t p1 = static_cast<uint64_t>(0xCD9E8D57u) * c.z;
    c = make_uint4(static_cast<uint32_t>(p1 >> 32) ^ c.y ^ k.k0[r], static_cast<uint32_t>(p1),
                   static_cast<uint32_t>(p0 >> 32) ^ c.w ^ k.k1[r], static_cast<uint32_t>(p0));
  }
  return c;
}

// Multiplies the 8 elements of a block (elements 8 block .. 8 block + 7 of the
// tensor in row-major order) by 0 or `scale`; a dropped element is 0 whatever it
// was.  Element e takes half-word e % 8 of the block's words, the low half first.
__device__ __forceinline__ void dropout8(float (&v)[8], const uint4& words, uint32_t threshold,
                                         float scale) {
  const uint32_t w[4] = {words.x, words.y, words.z, words.w};
  if (threshold >= 65536u) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
    return;
  }
  // a half-word is at least t where the word with it on top is at least t on top
  const uint32_t top = threshold << 16;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = (i & 1) != 0 ? w[i >> 1] : w[i >> 1] << 16;
    v[i] = u >= top ? v[i] * scale : 0.f;
  }
}

// Which of the 8 are kept, a bit each.
__device__ __forceinline__ uint32_t kept_bits(const uint4& words, uint32_t threshold) {
  const uint32_t w[4] = {words.x, words.y, words.z, words.w};
  const uint32_t top = threshold << 16;
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = (i & 1) != 0 ? w[i >> 1] : w[i >> 1] << 16;
    bits |= u >= top ? 1u << i : 0u;
  }
  return threshold >= 65536u ? 0u : bits;
}

__host__ __device__ inline float dropout_scale(uint32_t threshold) {
  return threshold >= 65536u ? 0.f : 65536.f / static_cast<float>(65536u - threshold);
}

}  // namespace mlora
