// Launching the group norm and state space kernels (host side).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "conv_internal.h"

namespace fdnn {

// Programmatic stream serialization as for the other kernels: the set-up of this launch overlaps the tail of the one
// before it; every kernel waits for that one before it touches memory.  `cluster`: CTAs per cluster along x.
template <typename... P, typename... A>
cudaError_t launch_seq(void (*kernel)(P...), dim3 grid, int threads, int smem, int cluster, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(unsigned(threads), 1, 1);
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (launch_overlap_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = unsigned(cluster);
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = unsigned(n);
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

// Opts a kernel in to `bytes` of dynamic shared memory, once per device (`done`: a bit per device ordinal).
template <typename K>
cudaError_t allow_smem(K* kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if ((done.load(std::memory_order_acquire) & bit) != 0) return cudaSuccess;
  e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

// Clusters of `cluster` blocks that run at once on an idle device; 0 if that cannot be had.  `known`: what each device has answered for this
// kernel, shared memory and cluster, one more than it, so that it is asked once.
struct ClusterCounts {
  std::atomic<int> of_device[64];
};
template <typename K>
int clusters_at_once(K* kernel, int threads, size_t smem, int cluster, ClusterCounts& known) {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  std::atomic<int>* place = dev >= 0 && dev < 64 ? &known.of_device[dev] : nullptr;
  if (place != nullptr && (n = place->load(std::memory_order_relaxed)) > 0) return n - 1;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(cluster);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(cluster));
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, reinterpret_cast<const void*>(kernel), &cfg) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  if (place != nullptr) place->store(n + 1, std::memory_order_relaxed);
  return n;
}

}  // namespace fdnn
