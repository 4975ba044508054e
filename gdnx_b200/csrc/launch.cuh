// Launches whose set-up overlaps the kernel before them on the stream (programmatic dependent
// launch).  A kernel launched so calls `dependents_may_start` as soon as it likes (its successor
// is then set up beside it) and `wait_for_earlier` before it touches memory, which returns when
// every kernel before it has ended and its writes are visible.
#pragma once

#include <atomic>
#include <cuda_runtime.h>

namespace gdnx {

// The current device's number of SMs (148 where it cannot be asked).
inline int sm_count() {
  static std::atomic<int> sms[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) {
    cudaGetLastError();
    return 148;
  }
  int n = sms[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
      cudaGetLastError();
      return 148;
    }
    sms[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

__device__ __forceinline__ void dependents_may_start() { asm volatile("griddepcontrol.launch_dependents;"); }
__device__ __forceinline__ void wait_for_earlier() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... P, typename... A>
cudaError_t launch_early(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

}  // namespace gdnx
