// Launches that start while the one before them in the stream ends; the kernel waits for that itself, before it reads or writes anything that another one may have.
#pragma once
#include <atomic>

#include "gguf_common.cuh"

namespace b200gguf {

// cluster: CTAs along x that form one (1: none).
template <typename... P, typename... A>
inline int launch_dependent(void (*kernel)(P...), dim3 grid, unsigned threads, size_t shared, unsigned cluster, cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? RC_OK : RC_LAUNCH;
}

// Lets a kernel have `shared` bytes of dynamic shared memory, once a device (`done` is the kernel's own).
template <typename K> inline int allow_shared(K kernel, size_t shared, std::atomic<uint64_t>& done) {
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return RC_LAUNCH;
  if ((done.load(std::memory_order_acquire) >> dev & 1) == 0) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(shared)) != cudaSuccess) return RC_LAUNCH;
    done.fetch_or(uint64_t(1) << dev, std::memory_order_release);
  }
  return RC_OK;
}

#ifdef __CUDACC__
__device__ __forceinline__ void wait_for_launch_before() {
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
}
#endif

}  // namespace b200gguf
