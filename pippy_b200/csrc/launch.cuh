// Host: kernel attributes, which belong to a kernel on one device.
#pragma once
#include <cuda_runtime.h>

#include <atomic>

namespace pb {

constexpr int kMaxDevices = 64;

// Allows `kKernel` to be launched with `kBytes` of dynamic shared memory on the current device.  Asked of the runtime once
// per kernel and device; two threads that come first together ask twice, with the same value.
template <auto kKernel, int kBytes>
cudaError_t allow_smem() {
  static std::atomic<bool> allowed[kMaxDevices];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const bool known = dev >= 0 && dev < kMaxDevices;
  if (known && allowed[dev].load(std::memory_order_relaxed)) return cudaSuccess;
  e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kKernel), cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
  if (e == cudaSuccess && known) allowed[dev].store(true, std::memory_order_relaxed);
  return e;
}

// A launch whose blocks may take their places as the blocks of the launch before them leave, once all of these have called
// let_next_start().  Such a kernel calls after_previous() before it touches memory that earlier launches wrote or read
// (or, where its own memory and the one before it are apart, before it ends: a launch counts as complete without it).
template <class... P, class... A>
cudaError_t launch_chained(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, A&&... args) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid, cfg.blockDim = block, cfg.dynamicSmemBytes = smem, cfg.stream = stream;
  cfg.attrs = &attr, cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

#ifdef __CUDACC__
// Waits until the launches that this one was chained to are complete and their writes visible.
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Called by every block, at its start if need be.  What keeps a launch from running ahead of the one before the last: a launch
// that was chained itself ends after the one before it, because a thread of each of its blocks calls after_previous() at some point
// (packed_dq_kernel only before it ends, since its memory and that of the launch before are apart); and the launch after it
// waits for its end in after_previous().
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
#endif

}  // namespace pb
