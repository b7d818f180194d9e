// How many thread-block clusters run at once.
#pragma once

#include <algorithm>
#include <atomic>

#include "common.cuh"

namespace dyn {

// Clusters of `size` blocks that the current device runs at once: a cluster stays within a part of the device whose SMs the size
// rarely divides (at a block per SM 74 clusters of 2, 22 of 6, 15 of 7 to 9, 11 of 10, 7 of 11 to 16). 0: a size of more than
// eight cannot be launched. The kernel must have been opted into SMEM bytes before. Found once per device and kernel.
template <auto KERNEL, int THREADS, int SMEM>
int clusters_at_once(int dev, int size) {
  static std::atomic<int> kept[16][17];
  std::atomic<int>* const slot = dev < 16 ? &kept[dev][size] : nullptr;
  int n = slot ? slot->load(std::memory_order_relaxed) : 0;
  if (n) return n;
  const void* const kernel = reinterpret_cast<const void*>(KERNEL);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(size * 64)), cfg.blockDim = dim3(THREADS), cfg.dynamicSmemBytes = SMEM;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)size, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr, cfg.numAttrs = 1;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();
    if (size > 8) return 0;  // sizes up to eight can be launched everywhere
    n = std::max(1, sm_count() / size);
  }
  if (slot) slot->store(n, std::memory_order_relaxed);
  return n;
}

// The largest size of 1 .. most (16 at the most) of which `clusters` run at once; 1 where none lets them.
template <auto KERNEL, int THREADS, int SMEM>
int blocks_per_cluster(int64_t clusters, int64_t most) {
  int dev = 0, size = (int)std::min<int64_t>(most, 16);
  if (cudaGetDevice(&dev) != cudaSuccess) return 1;
  while (size > 1 && clusters > clusters_at_once<KERNEL, THREADS, SMEM>(dev, size)) size--;
  return std::max(1, size);
}

}  // namespace dyn
