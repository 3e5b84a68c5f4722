// Host helper: an ordinary launch that reports its own error.  (After `kernel<<<...>>>` only cudaGetLastError tells, and that may be what a
// failed call before this one left behind.)
#pragma once
#include <cuda_runtime.h>

namespace bshmem {

template <typename... P, typename... A>
static inline cudaError_t launch_kernel(void (*kernel)(P...), dim3 grid, dim3 block, cudaStream_t stream, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = stream;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace bshmem
