// Microscaled block formats (device side): one power-of-two scale X = 2^E for
// 32 consecutive features of a row, held as the byte E + 127 (255 = NaN).
//
//   MXFP4 : E = max(floor(log2 amax) - 2, -127), code = e2m1(x / X) rounded to
//           nearest even on {0, .5, 1, 1.5, 2, 3, 4, 6}, saturating at 6;
//           two codes a byte, the even feature in the low nibble.
//   MXINT8: E = max(floor(log2 amax), -127), code = clamp(rint(64 x / X), +-127),
//           value = code / 64 * X.
// amax = 0 gives byte 0 and codes 0; a block holding an infinity or a NaN gives
// byte 255 and codes 0, so all its values read back as NaN.
//
// Every step is exact except the rounding to the code: X is a power of two, so
// x / X only moves the exponent, and a value (at most 8 significant bits) is
// exact in bf16.  In fp16 it is exact too while X >= 2^-18; below that the
// smallest values round to fp16's subnormal grid.
#pragma once

#include <stdint.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "ptx.cuh"
#include "quant.cuh"

namespace mlora {

constexpr int kMxBlock = 32;

// The scale byte of a block from the bits of max|x| (integer maximum of the
// absolute values' bits, which orders NaN above infinity above the finite).
__device__ __forceinline__ uint32_t mx_scale_byte_fp4(uint32_t amax_bits) {
  const uint32_t f = amax_bits >> 23;  // biased exponent; 0 for zero and subnormals
  return f == 255u ? 255u : (f > 2u ? f - 2u : 0u);
}
__device__ __forceinline__ uint32_t mx_scale_byte_int8(uint32_t amax_bits) {
  return amax_bits >> 23;
}

// 1 / X for a scale byte (0 for the NaN byte, whose codes are 0).
__device__ __forceinline__ float mx_inv_scale(uint32_t byte) {
  if (byte == 255u) return 0.f;
  return __uint_as_float(byte == 254u ? 0x00400000u : (254u - byte) << 23);
}
// X for a scale byte (NaN for 255).
__device__ __forceinline__ float mx_scale(uint32_t byte) {
  if (byte == 255u) return __uint_as_float(0x7FC00000u);
  return __uint_as_float(byte == 0u ? 0x00400000u : byte << 23);
}

// Eight e2m1 codes, v[0] in the lowest nibble.
__device__ __forceinline__ uint32_t mx_pack_e2m1(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t"
      ".reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t"
      "}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// The four pairs of e2m1 values of eight codes (exact in f16).
__device__ __forceinline__ void mx_unpack_e2m1(uint32_t w, float (&v)[8]) {
  uint32_t h[4];
  asm("{\n\t"
      ".reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t"
      "}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// Four int8 codes of values already divided by X / 64 and clamped to +-127:
// adding 1.5 * 2^23 rounds to the nearest integer (ties to even) and leaves
// its two's complement in the low byte.
__device__ __forceinline__ uint32_t mx_pack_int8(float a, float b, float c, float d) {
  constexpr float kMagic = 12582912.f;
  const uint32_t ua = __float_as_uint(__fadd_rn(a, kMagic)), ub = __float_as_uint(__fadd_rn(b, kMagic));
  const uint32_t uc = __float_as_uint(__fadd_rn(c, kMagic)), ud = __float_as_uint(__fadd_rn(d, kMagic));
  return __byte_perm(__byte_perm(ua, ub, 0x0040u), __byte_perm(uc, ud, 0x0040u), 0x5410u);
}

// ------------------------------------------------------- a block of a thread --
// 32 consecutive 16-bit values (16 words) or 16 codes held by one thread: packed
// fp32 pairs, two or three instructions a value.

// The bits of max|x| (as fp32) of the 32 16-bit values in w; a NaN among them
// gives a NaN.  Four running maxima keep the chain short.
template <typename T>
__device__ __forceinline__ uint32_t block_amax(const uint32_t (&w)[16]) {
  using T2 = typename std::conditional<std::is_same<T, __nv_bfloat16>::value, __nv_bfloat162,
                                       __half2>::type;
  T2 m[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = __habs2(*reinterpret_cast<const T2*>(&w[i]));
#pragma unroll
  for (int i = 4; i < 16; ++i)
    m[i & 3] = __hmax2_nan(m[i & 3], __habs2(*reinterpret_cast<const T2*>(&w[i])));
  m[0] = __hmax2_nan(__hmax2_nan(m[0], m[1]), __hmax2_nan(m[2], m[3]));
  const float2 f = std::is_same<T, __nv_bfloat16>::value
                       ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&m[0]))
                       : __half22float2(*reinterpret_cast<const __half2*>(&m[0]));
  return max(__float_as_uint(f.x), __float_as_uint(f.y)) & 0x7FFFFFFFu;
}

// The two values of a word as packed fp32.
template <typename T>
__device__ __forceinline__ uint64_t widen2(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    return (static_cast<uint64_t>(w & 0xFFFF0000u) << 32) | (w << 16);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return f2_pack(f.x, f.y);
  }
}

__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

// What rounding to T left of N values: the second of two 16-bit parts.  An infinite
// first part (an overflow too) has none: inf and -inf would add up to NaN.
template <typename T, int N>
__device__ __forceinline__ void second_part(const float (&v)[N], float (&rest)[N]) {
  uint64_t seen = 0;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const uint64_t d = f2_sub(f2_pack(v[i], v[i + 1]), widen2<T>(pack2<T>(v[i], v[i + 1])));
    seen = f2_fma(d, 0, seen);  // stays 0 unless one is an infinity or a NaN
    rest[i] = f2_lo(d);
    rest[i + 1] = f2_hi(d);
  }
  if (f2_lo(seen) != 0.f || f2_hi(seen) != 0.f) {
#pragma unroll
    for (int i = 0; i < N; ++i) rest[i] = isfinite(rest[i]) ? rest[i] : 0.f;
  }
}

// The 32 e2m1 codes of a block with this scale byte.
template <typename T>
__device__ __forceinline__ uint4 block_fp4(const uint32_t (&w)[16], uint32_t byte) {
  const float inv = mx_inv_scale(byte);
  const uint64_t ii = f2_pack(inv, inv);
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float v[8];
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const uint64_t p = f2_mul(widen2<T>(w[4 * i + h]), ii);
      v[2 * h] = f2_lo(p);
      v[2 * h + 1] = f2_hi(p);
    }
    o[i] = mx_pack_e2m1(v);
  }
  return byte == 255u ? make_uint4(0, 0, 0, 0) : make_uint4(o[0], o[1], o[2], o[3]);
}

// 32 int8 codes; inv64 = 64 / X.  The product is exact, so the fused add of
// 1.5 * 2^23 is the one rounding; its low 16 bits are the code.  Only a block
// whose maximum is at least 127.5 / 64 X (`high`) can reach 128 and is clamped.
template <typename T>
__device__ __forceinline__ void block_int8_scaled(const uint32_t (&w)[16], float inv64, bool high,
                                                  uint4& lo, uint4& hi) {
  const uint64_t ii = f2_pack(inv64, inv64);
  const uint64_t mm = f2_pack(12582912.f, 12582912.f);
  uint32_t h[16], o[8];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint64_t p = f2_fma(widen2<T>(w[i]), ii, mm);
    h[i] = __byte_perm(static_cast<uint32_t>(p), static_cast<uint32_t>(p >> 32), 0x5410u);
  }
  if (high) {
#pragma unroll
    for (int i = 0; i < 16; ++i) h[i] = __vmaxs2(__vmins2(h[i], 0x007F007Fu), 0xFF81FF81u);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = __byte_perm(h[2 * i], h[2 * i + 1], 0x6420u);
  lo = make_uint4(o[0], o[1], o[2], o[3]);
  hi = make_uint4(o[4], o[5], o[6], o[7]);
}

// The 32 int8 codes of a block with this maximum.
template <typename T>
__device__ __forceinline__ void block_int8(const uint32_t (&w)[16], uint32_t amax_bits, uint4& lo,
                                           uint4& hi) {
  const uint32_t byte = mx_scale_byte_int8(amax_bits);
  const bool high = (amax_bits & 0x7FFFFFu) >= 0x7F0000u;  // (subnormals are below it as values)
  if (byte >= 6u) {
    block_int8_scaled<T>(w, mx_inv_scale(byte) * 64.f, high, lo, hi);
  } else {
    // 64 / X is past fp32's range: X = 2^(byte - 127) is moved up by 2^8 together
    // with the values (exact: they are below 2^-120)
    uint32_t u[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint64_t v = f2_mul(widen2<T>(w[i]), f2_pack(256.f, 256.f));
      u[i] = pack2<__nv_bfloat16>(f2_lo(v), f2_hi(v));
    }
    block_int8_scaled<__nv_bfloat16>(u, mx_inv_scale(byte + 8u) * 64.f, true, lo, hi);
  }
  if (byte == 255u) lo = hi = make_uint4(0, 0, 0, 0);  // 0 * inf made NaN of them
}

// Sixteen MXINT8 codes times X / 64, in T (rounded to nearest where fp16 is
// subnormal, else exact).  The byte with
// its sign bit flipped is u = code + 128; placed in the mantissa of
// 2^(23+k) (2^k = X / 64) it makes 2^k (2^23 + u), and subtracting
// 2^k (2^23 + 128) leaves code * 2^k exactly.
template <typename T>
__device__ __forceinline__ void expand16(const uint4& q, uint32_t byte, uint4& lo, uint4& hi) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  uint32_t o[8];
  if (byte <= 237u) {
    const uint32_t magic = (byte + 17u) << 23;
    const float c = __uint_as_float(magic | 0x80u);
    const uint64_t cc = f2_pack(c, c);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = w[i] ^ 0x80808080u;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t a = __byte_perm(u, magic, 0x7640u | (2 * h));
        const uint32_t b = __byte_perm(u, magic, 0x7640u | (2 * h + 1));
        const uint64_t v = f2_sub((static_cast<uint64_t>(b) << 32) | a, cc);
        o[2 * i + h] = pack2<T>(f2_lo(v), f2_hi(v));
      }
    }
  } else {  // exponents the mantissa form cannot hold, and the NaN byte
    const float X = mx_scale(byte);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float a = static_cast<float>(static_cast<int8_t>(w[i] >> (16 * h))) * (1.f / 64.f);
        const float b = static_cast<float>(static_cast<int8_t>(w[i] >> (16 * h + 8))) * (1.f / 64.f);
        o[2 * i + h] = pack2<T>(__fmul_rn(a, X), __fmul_rn(b, X));
      }
  }
  lo = make_uint4(o[0], o[1], o[2], o[3]);
  hi = make_uint4(o[4], o[5], o[6], o[7]);
}

// --------------------------------------------------- fp4 tensor-core product --
// tcgen05.mma kind::mxf4 (K = 64 codes a step): A and B are K-major code rows in
// shared memory; their scale bytes sit in TMEM.  The scale bytes of 128 rows x
// 128 features form one 512-byte atom: byte (row % 32) * 16 + (row / 32) * 4 +
// (block % 4), which one tcgen05.cp spreads over 4 TMEM columns (lane = row %
// 32, column = row / 32, repeated in the four lane quarters).  A K step reads
// two of a column's four bytes, picked by the scale id (0 or 2) of the
// instruction descriptor.
constexpr uint32_t kMxAtomBytes = 512;

// [4,6) B scale id; [7,10) a format, [10,12) b format (1 = e2m1); [17,23) N >> 3;
// [23] scale type (1 = power of two); [27,29) M >> 7; [29,31) A scale id.
__host__ __device__ constexpr uint32_t make_idesc_mxf4(uint32_t M, uint32_t N, uint32_t sf_id) {
  return (sf_id << 4) | (1u << 7) | (1u << 10) | ((N >> 3) << 17) | (1u << 23) | ((M >> 7) << 27) |
         (sf_id << 29);
}

__device__ __forceinline__ void umma_mxf4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                          uint32_t idesc, uint32_t sfa_tmem, uint32_t sfb_tmem,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], "
      "p;\n\t"
      "}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa_tmem), "r"(sfb_tmem), "r"(accumulate)
      : "memory");
}

// One scale atom from shared memory (16-byte aligned) to 4 TMEM columns.
// tcgen05.cp and tcgen05.mma of one thread execute in issue order.
__device__ __forceinline__ void tmem_cp_scale_atom(uint32_t taddr, uint32_t saddr) {
  const uint64_t desc = make_smem_desc(saddr, 16u, 128u, kLayoutNone);
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc)
               : "memory");
}

// The same over a CTA pair (issued by the even CTA): the M side's scales in each
// CTA are its own 128 rows', the N side's those of all N columns.
__device__ __forceinline__ void umma_mxf4_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                               uint32_t idesc, uint32_t sfa_tmem,
                                               uint32_t sfb_tmem, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], "
      "p;\n\t"
      "}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa_tmem), "r"(sfb_tmem), "r"(accumulate)
      : "memory");
}

// Each CTA of the pair copies the atom at this offset of its own shared memory.
__device__ __forceinline__ void tmem_cp_scale_atom_pair(uint32_t taddr, uint32_t saddr) {
  const uint64_t desc = make_smem_desc(saddr, 16u, 128u, kLayoutNone);
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc)
               : "memory");
}

}  // namespace mlora
