// Quantisers and dequantisers of the microscaled block formats (mx.cuh):
// MXFP4 weights and GEMM operands, MXINT8 activation checkpoints.
//
// HBM-bound: x is read once, codes and scales are written once (and the reverse).
// Rows of whole blocks of 16-bit values: a thread owns blocks (64 bytes, moved as
// 32-byte sectors), the maximum needs no exchange, and the codes come from packed
// pairs.  Other rows (a tail block, odd strides, fp32): a warp owns up to 1024
// features of a row, 8 a lane and step, so four lanes share a block.
//
// Measured: 8192 x 4096 bf16 to MXINT8 and back 30.5 us = 201 MB at 6.6 TB/s, the
// measured copy rate; 11008 x 4096 to MXFP4 (with the product's table) and back
// 38 us = 231 MB at 6.1 TB/s.  The eight-a-lane form, taken for whole blocks too,
// needs 42.4 and 48.5 us: twice the instructions, half the bytes a load.
#include "internal.h"
#include "launch.cuh"
#include "mx.cuh"
#include "../../include/metallora_b200.h"

namespace mlora {
namespace {

constexpr int kMxThreads = 256;
constexpr int kMxWarps = kMxThreads / 32;
constexpr int kMxSteps = 4;
constexpr int kMxSeg = kMxSteps * 256;  // features of a row per warp

// Eight consecutive elements of a row starting at k (zeros past K).
template <typename T, bool kVec>
__device__ __forceinline__ void load8(const T* row, int64_t k, int64_t K, float (&v)[8]) {
  if constexpr (kVec) {
    if (k < K) {
      if constexpr (sizeof(T) == 2) {
        const uint4 q = __ldg(reinterpret_cast<const uint4*>(row + k));
        const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(e[i]);
      } else {
        const float4 q0 = __ldg(reinterpret_cast<const float4*>(row + k));
        const float4 q1 = __ldg(reinterpret_cast<const float4*>(row + k) + 1);
        v[0] = q0.x, v[1] = q0.y, v[2] = q0.z, v[3] = q0.w;
        v[4] = q1.x, v[5] = q1.y, v[6] = q1.z, v[7] = q1.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < K ? static_cast<float>(row[k + i]) : 0.f;
  }
}

// Writes the scale bytes of the four blocks of 128 features starting at k
// (one word, first block in the low byte).
__device__ __forceinline__ void store_scales(const MxScales& sc, int64_t row, int64_t k,
                                             uint32_t word) {
  const int64_t g = k >> 7;
  if (sc.layout == kMxPlain) {
    uint8_t* dst = sc.data + row * sc.blocks + 4 * g;
    if ((sc.blocks & 3) == 0) {
      *reinterpret_cast<uint32_t*>(dst) = word;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (4 * g + i < sc.blocks) dst[i] = static_cast<uint8_t>(word >> (8 * i));
    }
  } else {
    reinterpret_cast<uint32_t*>(sc.data)[g * sc.rows + row] = word;
  }
}

// Thread t of a CTA owns blocks t, t + 256 of the CTA's 512.
constexpr int kOwn = 2;

__device__ __forceinline__ uint8_t* scale_of(const MxScales& sc, uint32_t block, uint32_t per_row) {
  if (sc.layout == kMxPlain) return sc.data + block;
  const uint32_t row = block / per_row, b = block - row * per_row;
  return sc.data + (static_cast<int64_t>(b >> 2) * sc.rows + row) * 4 + (b & 3u);
}

// Plain loads, which stay behind grid_wait(): the block kernels start while the
// kernel that writes their input may still run, so it is not read-only for their
// whole life, as the read-only path (ld.global.nc, __ldg) wants.
__device__ __forceinline__ void ld_global_32b(const void* p, uint32_t* v) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]),
                 "=r"(v[6]), "=r"(v[7])
               : "l"(p)
               : "memory");
}
__device__ __forceinline__ uint4 ld_global_16b(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}
__device__ __forceinline__ uint32_t ld_global_byte(const void* p) {
  uint32_t v;
  asm volatile("ld.global.u8 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// x, codes: [blocks] of 32 values, without gaps between the rows.
template <int kBits, typename T>
__global__ void __launch_bounds__(kMxThreads)
    mx_quantize_blocks_kernel(const T* x, uint32_t blocks, uint32_t per_row, uint8_t* codes,
                              const MxScales sc, uint8_t* atoms) {
  grid_wait();
  launch_dependents();
  const uint32_t b0 = blockIdx.x * (kMxThreads * kOwn) + threadIdx.x;
  uint32_t w[kOwn][16];
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const uint32_t b = b0 + i * kMxThreads;
    if (b >= blocks) continue;
    ld_global_32b(x + static_cast<int64_t>(b) * 32, w[i]);
    ld_global_32b(x + static_cast<int64_t>(b) * 32 + 16, w[i] + 8);
  }
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const uint32_t b = b0 + i * kMxThreads;
    if (b >= blocks) continue;
    const uint32_t amax = block_amax<T>(w[i]);
    const uint32_t byte = kBits == 4 ? mx_scale_byte_fp4(amax) : mx_scale_byte_int8(amax);
    *scale_of(sc, b, per_row) = static_cast<uint8_t>(byte);
    if (kBits == 4 && atoms != nullptr) {  // rows of whole atoms
      const uint32_t row = b / per_row, k = b - row * per_row;
      atoms[(static_cast<int64_t>(row >> 7) * (per_row >> 2) + (k >> 2)) * kMxAtomBytes +
            (row & 31u) * 16 + ((row >> 5) & 3u) * 4 + (k & 3u)] = static_cast<uint8_t>(byte);
    }
    if constexpr (kBits == 4) {
      reinterpret_cast<uint4*>(codes)[b] = block_fp4<T>(w[i], byte);
    } else {
      uint4 lo, hi;
      block_int8<T>(w[i], amax, lo, hi);
      const uint32_t v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      st_global_32b(codes + static_cast<int64_t>(b) * 32, v);
    }
  }
}

template <int kBits, typename O>
__global__ void __launch_bounds__(kMxThreads)
    mx_dequantize_blocks_kernel(const uint8_t* codes, const MxScales sc, uint32_t blocks,
                                uint32_t per_row, O* out) {
  grid_wait();
  launch_dependents();
  const uint32_t b0 = blockIdx.x * (kMxThreads * kOwn) + threadIdx.x;
  uint32_t c[kOwn][kBits], byte[kOwn];
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const uint32_t b = b0 + i * kMxThreads;
    if (b >= blocks) continue;
    byte[i] = ld_global_byte(scale_of(sc, b, per_row));
    if constexpr (kBits == 4) {
      const uint4 q = ld_global_16b(codes + static_cast<int64_t>(b) * 16);
      c[i][0] = q.x, c[i][1] = q.y, c[i][2] = q.z, c[i][3] = q.w;
    } else {
      ld_global_32b(codes + static_cast<int64_t>(b) * 32, c[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const uint32_t b = b0 + i * kMxThreads;
    if (b >= blocks) continue;
    O* dst = out + static_cast<int64_t>(b) * 32;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t v[8];
      if constexpr (kBits == 4) {
        const float X = mx_scale(byte[i]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float u[8];
          mx_unpack_e2m1(c[i][2 * h + j], u);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            v[4 * j + k] = pack2<O>(__fmul_rn(u[2 * k], X), __fmul_rn(u[2 * k + 1], X));
        }
      } else {
        uint4 lo, hi;
        expand16<O>(make_uint4(c[i][4 * h], c[i][4 * h + 1], c[i][4 * h + 2], c[i][4 * h + 3]),
                    byte[i], lo, hi);
        v[0] = lo.x, v[1] = lo.y, v[2] = lo.z, v[3] = lo.w;
        v[4] = hi.x, v[5] = hi.y, v[6] = hi.z, v[7] = hi.w;
      }
      st_global_32b(dst + 16 * h, v);
    }
  }
}

template <int kBits, typename T, bool kVec>
__global__ void __launch_bounds__(kMxThreads)
    mx_quantize_kernel(const T* __restrict__ x, int64_t M, int64_t K, uint8_t* __restrict__ codes,
                       int64_t ld, const MxScales sc) {
  const int lane = static_cast<int>(lane_id());
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kMxWarps + warp_id();
  if (row >= M) return;
  const T* xr = x + row * K;
  uint8_t* cr = codes + row * ld;
  const int64_t k0 = static_cast<int64_t>(blockIdx.y) * kMxSeg + lane * 8;
  float v[kMxSteps][8];
#pragma unroll
  for (int s = 0; s < kMxSteps; ++s) load8<T, kVec>(xr, k0 + s * 256, K, v[s]);
#pragma unroll
  for (int s = 0; s < kMxSteps; ++s) {
    const int64_t k = k0 + s * 256;
    if (k - lane * 8 >= K) break;  // the same for all lanes
    uint32_t am = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) am = max(am, __float_as_uint(v[s][i]) & 0x7FFFFFFFu);
    am = max(am, __shfl_xor_sync(0xffffffffu, am, 1));
    am = max(am, __shfl_xor_sync(0xffffffffu, am, 2));
    const uint32_t byte = kBits == 4 ? mx_scale_byte_fp4(am) : mx_scale_byte_int8(am);
    uint32_t word = byte << (8 * ((lane >> 2) & 3));
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    word |= __shfl_xor_sync(0xffffffffu, word, 8);
    if ((lane & 15) == 0 && k < K) store_scales(sc, row, k, word);
    const float inv = mx_inv_scale(byte);
    const bool dead = byte == 255u;  // 0 * inf would be NaN: the codes are 0
    float u[8];
    if constexpr (kBits == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] = dead ? 0.f : __fmul_rn(v[s][i], inv);
      const uint32_t c = mx_pack_e2m1(u);
      if constexpr (kVec) {
        if (k < K) *reinterpret_cast<uint32_t*>(cr + (k >> 1)) = c;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (k + 2 * i < K) cr[(k >> 1) + i] = static_cast<uint8_t>(c >> (8 * i));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float q = __fmul_rn(__fmul_rn(v[s][i], inv), 64.f);
        u[i] = dead ? 0.f : fminf(fmaxf(q, -127.f), 127.f);
      }
      const uint32_t c0 = mx_pack_int8(u[0], u[1], u[2], u[3]);
      const uint32_t c1 = mx_pack_int8(u[4], u[5], u[6], u[7]);
      if constexpr (kVec) {
        if (k < K) *reinterpret_cast<uint2*>(cr + k) = make_uint2(c0, c1);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (k + i < K) cr[k + i] = static_cast<uint8_t>((i < 4 ? c0 : c1) >> (8 * (i & 3)));
      }
    }
  }
}

__device__ __forceinline__ uint32_t load_scale(const MxScales& sc, int64_t row, int64_t block) {
  if (sc.layout == kMxPlain) return __ldg(sc.data + row * sc.blocks + block);
  return __ldg(sc.data + ((block >> 2) * sc.rows + row) * 4 + (block & 3));
}

template <typename O>
__device__ __forceinline__ O mx_out(float v) {
  if constexpr (sizeof(O) == 4)
    return v;
  else
    return static_cast<O>(v);  // round to nearest even
}

template <int kBits, typename O, bool kVec>
__global__ void __launch_bounds__(kMxThreads)
    mx_dequantize_kernel(const uint8_t* __restrict__ codes, int64_t ld, const MxScales sc,
                         int64_t M, int64_t K, O* __restrict__ out) {
  const int lane = static_cast<int>(lane_id());
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kMxWarps + warp_id();
  if (row >= M) return;
  const uint8_t* cr = codes + row * ld;
  O* orow = out + row * K;
  const int64_t k0 = static_cast<int64_t>(blockIdx.y) * kMxSeg + lane * 8;
  uint32_t c0[kMxSteps], c1[kMxSteps], byte[kMxSteps];
#pragma unroll
  for (int s = 0; s < kMxSteps; ++s) {
    const int64_t k = k0 + s * 256;
    c0[s] = c1[s] = byte[s] = 0;
    if (k >= K) continue;
    byte[s] = load_scale(sc, row, k >> 5);
    if constexpr (kVec) {
      if constexpr (kBits == 4) {
        c0[s] = __ldg(reinterpret_cast<const uint32_t*>(cr + (k >> 1)));
      } else {
        const uint2 q = __ldg(reinterpret_cast<const uint2*>(cr + k));
        c0[s] = q.x, c1[s] = q.y;
      }
    } else if constexpr (kBits == 4) {
      for (int i = 0; i < 4; ++i)
        if (k + 2 * i < K) c0[s] |= static_cast<uint32_t>(cr[(k >> 1) + i]) << (8 * i);
    } else {
      for (int i = 0; i < 8; ++i)
        if (k + i < K) (i < 4 ? c0[s] : c1[s]) |= static_cast<uint32_t>(cr[k + i]) << (8 * (i & 3));
    }
  }
#pragma unroll
  for (int s = 0; s < kMxSteps; ++s) {
    const int64_t k = k0 + s * 256;
    if (k >= K) break;
    const float X = mx_scale(byte[s]);
    float v[8];
    if constexpr (kBits == 4) {
      mx_unpack_e2m1(c0[s], v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[i] = static_cast<float>(static_cast<int8_t>((i < 4 ? c0[s] : c1[s]) >> (8 * (i & 3)))) *
               (1.f / 64.f);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], X);
    if constexpr (kVec) {
      if constexpr (sizeof(O) == 4) {
        reinterpret_cast<float4*>(orow + k)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(orow + k)[1] = make_float4(v[4], v[5], v[6], v[7]);
      } else {
        *reinterpret_cast<uint4*>(orow + k) = make_uint4(pack2<O>(v[0], v[1]), pack2<O>(v[2], v[3]),
                                                         pack2<O>(v[4], v[5]), pack2<O>(v[6], v[7]));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k + i < K) orow[k + i] = mx_out<O>(v[i]);
    }
  }
}

// Plain scale bytes [rows, blocks] -> the fp4 product's atoms (rows rounded up
// to 128, features to 128; the padding is 0, a finite scale of codes that are 0).
__global__ void mx_prepare_scales_kernel(const uint8_t* __restrict__ src, int64_t rows,
                                         int64_t blocks, int64_t groups, int64_t words,
                                         uint32_t* __restrict__ dst) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= words) return;
  // word i of the atoms: [row tile][group][row % 32][row / 32 % 4]
  const int64_t atom = i >> 7;
  const int in = static_cast<int>(i & 127);
  const int64_t g = atom % groups;
  const int64_t row = (atom / groups) * 128 + (in & 3) * 32 + (in >> 2);
  uint32_t word = 0;
  if (row < rows)
    for (int b = 0; b < 4; ++b)
      if (4 * g + b < blocks) word |= static_cast<uint32_t>(src[row * blocks + 4 * g + b]) << (8 * b);
  dst[i] = word;
}

int mx_grid(int64_t M, int64_t K, dim3* grid) {
  const int64_t gx = (M + kMxWarps - 1) / kMxWarps, gy = (K + kMxSeg - 1) / kMxSeg;
  if (gx > (int64_t(1) << 31) - 1 || gy > 65535) {
    set_error("microscaled format: too many rows or features");
    return MLORA_ERR_UNSUPPORTED;
  }
  *grid = dim3(static_cast<unsigned>(gx), static_cast<unsigned>(gy));
  return MLORA_OK;
}

int launched(const char* what) { return launch_status(cudaSuccess, what); }

// A block kernel, as a programmatic dependent of the kernel before it.
template <typename... P, typename... A>
int launch_blocks(const char* what, void (*kern)(P...), unsigned grid, cudaStream_t s, const A&... args) {
  return launch_status(launch_kernel(kern, dim3(grid), kMxThreads, 0, s, 0, 0, true, args...), what);
}

bool aligned(const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

template <typename T>
void run_quantize(int bits, bool vec, dim3 grid, const void* x, int64_t M, int64_t K, void* codes,
                  int64_t ld, const MxScales& sc, cudaStream_t s) {
  const T* xt = static_cast<const T*>(x);
  auto* c = static_cast<uint8_t*>(codes);
  if (bits == 4)
    vec ? mx_quantize_kernel<4, T, true><<<grid, kMxThreads, 0, s>>>(xt, M, K, c, ld, sc)
        : mx_quantize_kernel<4, T, false><<<grid, kMxThreads, 0, s>>>(xt, M, K, c, ld, sc);
  else
    vec ? mx_quantize_kernel<8, T, true><<<grid, kMxThreads, 0, s>>>(xt, M, K, c, ld, sc)
        : mx_quantize_kernel<8, T, false><<<grid, kMxThreads, 0, s>>>(xt, M, K, c, ld, sc);
}

template <typename O>
void run_dequantize(int bits, bool vec, dim3 grid, const void* codes, int64_t ld,
                    const MxScales& sc, int64_t M, int64_t K, void* out, cudaStream_t s) {
  const auto* c = static_cast<const uint8_t*>(codes);
  O* o = static_cast<O*>(out);
  if (bits == 4)
    vec ? mx_dequantize_kernel<4, O, true><<<grid, kMxThreads, 0, s>>>(c, ld, sc, M, K, o)
        : mx_dequantize_kernel<4, O, false><<<grid, kMxThreads, 0, s>>>(c, ld, sc, M, K, o);
  else
    vec ? mx_dequantize_kernel<8, O, true><<<grid, kMxThreads, 0, s>>>(c, ld, sc, M, K, o)
        : mx_dequantize_kernel<8, O, false><<<grid, kMxThreads, 0, s>>>(c, ld, sc, M, K, o);
}

// Whether rows of K 16-bit values at `wide` and codes `code_bytes` apart go block
// by block: whole blocks without gaps, sectors aligned, 32-bit block numbers.  A
// checkpoint's scale words hold four blocks, so its rows hold whole words.
bool whole_blocks(const void* wide, int dtype, const void* codes, int64_t ld, int64_t code_bytes,
                  const MxScales& sc, int64_t M, int64_t K) {
  return dtype != MLORA_DTYPE_F32 && K % (sc.layout == kMxPlain ? 32 : 128) == 0 &&
         ld == code_bytes && aligned(wide, 32) && aligned(codes, 32) &&
         M * (K / kMxBlock) < (int64_t(1) << 31);
}

}  // namespace

int launch_mx_quantize(int bits, const void* x, int dtype, int64_t M, int64_t K, void* codes,
                       int64_t ld, const MxScales& sc, cudaStream_t s, void* atoms,
                       bool* atoms_made) {
  if (whole_blocks(x, dtype, codes, ld, K * bits / 8, sc, M, K)) {
    const auto blocks = static_cast<uint32_t>(M * (K / kMxBlock));
    const auto per_row = static_cast<uint32_t>(K / kMxBlock);
    const unsigned grid = (blocks + kMxThreads * kOwn - 1) / (kMxThreads * kOwn);
    auto* c = static_cast<uint8_t*>(codes);
    // (a group that is not whole would leave padding bytes of its atoms unset)
    auto* t = K % 128 == 0 ? static_cast<uint8_t*>(atoms) : nullptr;
    if (atoms_made != nullptr) *atoms_made = t != nullptr;
    LaunchScope scope(kKindQuant, s);
    auto run = [&](auto type) {
      using T = decltype(type);
      return launch_blocks("mx quantize",
                           bits == 4 ? mx_quantize_blocks_kernel<4, T> : mx_quantize_blocks_kernel<8, T>,
                           grid, s, static_cast<const T*>(x), blocks, per_row, c, sc, t);
    };
    return dtype == MLORA_DTYPE_BF16 ? run(__nv_bfloat16()) : run(__half());
  }
  if (atoms_made != nullptr) *atoms_made = false;
  dim3 grid;
  if (int rc = mx_grid(M, K, &grid)) return rc;
  // whole 8-feature groups, 16-byte loads, 4- (fp4) or 8-byte (int8) stores
  const uintptr_t st = bits == 4 ? 4 : 8;
  const bool vec = K % 8 == 0 && aligned(x, 16) && aligned(codes, st) && ld % static_cast<int64_t>(st) == 0;
  LaunchScope scope(kKindQuant, s);
  if (dtype == MLORA_DTYPE_BF16)
    run_quantize<__nv_bfloat16>(bits, vec, grid, x, M, K, codes, ld, sc, s);
  else if (dtype == MLORA_DTYPE_F16)
    run_quantize<__half>(bits, vec, grid, x, M, K, codes, ld, sc, s);
  else
    run_quantize<float>(bits, vec, grid, x, M, K, codes, ld, sc, s);
  return launched("mx quantize");
}

int launch_mx_dequantize(int bits, const void* codes, int64_t ld, const MxScales& sc, int64_t M,
                         int64_t K, void* out, int out_dtype, cudaStream_t s) {
  if (whole_blocks(out, out_dtype, codes, ld, K * bits / 8, sc, M, K)) {
    const auto blocks = static_cast<uint32_t>(M * (K / kMxBlock));
    const auto per_row = static_cast<uint32_t>(K / kMxBlock);
    const unsigned grid = (blocks + kMxThreads * kOwn - 1) / (kMxThreads * kOwn);
    const auto* c = static_cast<const uint8_t*>(codes);
    LaunchScope scope(kKindQuant, s);
    auto run = [&](auto type) {
      using O = decltype(type);
      return launch_blocks("mx dequantize",
                           bits == 4 ? mx_dequantize_blocks_kernel<4, O> : mx_dequantize_blocks_kernel<8, O>,
                           grid, s, c, sc, blocks, per_row, static_cast<O*>(out));
    };
    return out_dtype == MLORA_DTYPE_BF16 ? run(__nv_bfloat16()) : run(__half());
  }
  dim3 grid;
  if (int rc = mx_grid(M, K, &grid)) return rc;
  const uintptr_t st = bits == 4 ? 4 : 8;
  const bool vec = K % 8 == 0 && aligned(out, 16) && aligned(codes, st) && ld % static_cast<int64_t>(st) == 0;
  LaunchScope scope(kKindQuant, s);
  if (out_dtype == MLORA_DTYPE_BF16)
    run_dequantize<__nv_bfloat16>(bits, vec, grid, codes, ld, sc, M, K, out, s);
  else if (out_dtype == MLORA_DTYPE_F16)
    run_dequantize<__half>(bits, vec, grid, codes, ld, sc, M, K, out, s);
  else
    run_dequantize<float>(bits, vec, grid, codes, ld, sc, M, K, out, s);
  return launched("mx dequantize");
}

int launch_mx_prepare_scales(const void* scales, int64_t rows, int64_t K, void* atoms,
                             cudaStream_t s) {
  const int64_t blocks = (K + kMxBlock - 1) / kMxBlock, groups = (blocks + 3) / 4;
  const int64_t words = (rows + 127) / 128 * groups * 128;
  const int64_t grid = (words + 255) / 256;
  if (grid > (int64_t(1) << 31) - 1) {
    set_error("mx prepare scales: too many blocks");
    return MLORA_ERR_UNSUPPORTED;
  }
  LaunchScope scope(kKindElementwise, s);
  mx_prepare_scales_kernel<<<static_cast<unsigned>(grid), 256, 0, s>>>(
      static_cast<const uint8_t*>(scales), rows, blocks, groups, words,
      static_cast<uint32_t*>(atoms));
  return launched("mx prepare scales");
}

}  // namespace mlora
