// Launch helpers of the kernels that take a padded rank, run in clusters or start
// as programmatic dependents.
#pragma once

#include <cuda_runtime.h>

#include <string>
#include <type_traits>

#include "internal.h"
#include "../../include/metallora_b200.h"

namespace mlora {

// TMEM columns to allocate for n: a power of two, at least 32.
__host__ __device__ constexpr uint32_t tmem_cols(int n) {
  uint32_t c = 32;
  while (c < static_cast<uint32_t>(n)) c *= 2;
  return c;
}

inline int launch_status(cudaError_t e, const char* what) {
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e == cudaSuccess) return MLORA_OK;
  set_error(std::string(what) + ": " + cudaGetErrorString(e));
  return MLORA_ERR_CUDA;
}

// Launches kern with clusters of (cx, cy, 1) CTAs (0, 0: as the kernel says), where
// `overlap_prev` as a programmatic dependent of the kernel before it on the stream.
template <typename... P, typename... A>
cudaError_t launch_kernel(void (*kern)(P...), dim3 grid, int threads, size_t smem, cudaStream_t s,
                          unsigned cx, unsigned cy, bool overlap_prev, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if (cx != 0) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cx;
    attr[n].val.clusterDim.y = cy;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (overlap_prev) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

// Calls f with the padded rank R as a constant (f(std::integral_constant<int, R>())).
template <typename F>
int with_rank(int64_t R, F&& f) {
  switch (R) {
    case 16: return f(std::integral_constant<int, 16>());
    case 32: return f(std::integral_constant<int, 32>());
    case 64: return f(std::integral_constant<int, 64>());
    case 128: return f(std::integral_constant<int, 128>());
    case 256: return f(std::integral_constant<int, 256>());
    default: set_error("unsupported padded rank"); return MLORA_ERR_UNSUPPORTED;
  }
}

}  // namespace mlora
