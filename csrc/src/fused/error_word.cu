// The word that kernels of this library set when they gave up on a wait, one per GPU, for callers that keep none of their own.
#include <cuda_runtime.h>

#include <mutex>

#include "../../include/bshmem/fused.h"

namespace bshmem {

// Zeroed memory of the current device.  The call may come in the middle of a stream capture: the memory belongs to no graph, and its zeroing is no
// part of one (each replay would take errors back).  So this thread's calls are not held against a capture, and the stream is its own.
static int* zeroed_word() {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) return nullptr;
  void* word = nullptr;
  cudaStream_t stream = nullptr;
  bool ok = cudaMalloc(&word, sizeof(int)) == cudaSuccess && cudaStreamCreateWithFlags(&stream, cudaStreamNonBlocking) == cudaSuccess &&
            cudaMemsetAsync(word, 0, sizeof(int), stream) == cudaSuccess && cudaStreamSynchronize(stream) == cudaSuccess;
  if (stream) cudaStreamDestroy(stream);
  if (!ok && word) cudaFree(word);
  cudaThreadExchangeStreamCaptureMode(&mode);
  return ok ? (int*)word : nullptr;
}

}  // namespace bshmem

extern "C" int* bshmem_fused_error_word(int device) {
  static std::mutex mutex;
  static int* words[64];
  if (device < 0 || device >= 64) return nullptr;
  std::lock_guard<std::mutex> lock(mutex);
  int current = 0;
  if (!words[device] && cudaGetDevice(&current) == cudaSuccess && cudaSetDevice(device) == cudaSuccess) {
    words[device] = bshmem::zeroed_word();
    cudaSetDevice(current);
  }
  return words[device];
}
