// Kernel launches inside one call: the kernels of a call run back to back on one stream and each depends on the one
// before it. A programmatic dependent launch lets the next kernel's blocks start while the last ones of the current
// kernel drain; pdl_wait() is where a kernel first touches what the kernels before it wrote (it returns when they have
// completed and their writes are visible), pdl_trigger() lets the next one be scheduled. In the sparse attention's path the
// trigger stands at a kernel's end: given at its start, blocks of the next kernel sat in slots that the current one still needed
// (a [1,24,4608,128] call took 207 us, 195 without dependent launches, 188 like this). The rotation and the bookkeeping of pages
// give it right behind their own wait: their calls of a step are one block, or a few short ones, and what comes next starts up
// under them. Either is right, since every kernel waits before it touches what another one writes. Without the launch attribute
// both are no-ops.
// No block leaves a kernel in front of pdl_wait() by a return: if all of them did, the kernel would end before the one it
// depends on, and what follows on the stream (the next user of the workspace) waits for this one only.
// A kernel with a pdl_wait() takes no `const T* __restrict__`: that promises data which nothing writes while the kernel runs,
// so that loads may go through the non-coherent path and in front of the wait, and the kernel before it still writes.
#pragma once
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

namespace sparge {

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... KArgs, typename... Args>
inline cudaError_t launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, bool dependent, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
  if (e != cudaSuccess) cudaGetLastError();   // reported by the caller's status: the next check of this thread is not about it
  return e;
}

// Function attributes are per device and outlive the call: set once for each (kernel, device).
inline bool kernel_attributes(const void* kern, int smem, std::atomic<uint64_t>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_acquire) & bit)) return true;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return false;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) != cudaSuccess)
    return false;
  if (dev < 64) done.fetch_or(bit, std::memory_order_release);
  return true;
}

// Multiprocessors of the current device.
inline int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
  if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
  return n;
}

}  // namespace sparge
