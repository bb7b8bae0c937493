// Launches of the single operators' kernels: as programmatic dependents, in
// clusters, and how many CTAs the device holds at once.
#pragma once

#include <algorithm>
#include <utility>

#include "launch_limits.h"
#include "runtime.h"

namespace iec {

// Lets `Kernel` use `bytes` of dynamic shared memory, and clusters of 16.
template <auto Kernel>
void allow_smem(Device& dev, size_t bytes) {
  static SmemLimit limit;
  limit.raise(dev.ordinal(), bytes, [](size_t most, bool first) {
    if (first) IEC_CUDA(cudaFuncSetAttribute(Kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    IEC_CUDA(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
  });
}

inline cudaLaunchConfig_t ops_config(dim3 grid, int threads, size_t smem, int cluster, cudaStream_t s,
                                     cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {(unsigned)cluster, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cfg;
}

// launch_pdl (runtime.h) in clusters of `cluster` CTAs along x.
template <class... KArgs, class... Args>
void launch_ops(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t s,
                Args&&... args) {
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = ops_config(grid, threads, smem, cluster, s, attr);
  IEC_CUDA(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...));
}

// CTAs of `Kernel` that the device holds at once, in clusters of `cluster`,
// with `smem` rounded up to 16 KB; 0 where such a cluster has no room (large
// ones may not: the callers go on to smaller ones).
template <auto Kernel>
int resident_ctas(Device& dev, int threads, size_t smem, int cluster) {
  static Residency found;
  return found.get(dev.ordinal(), cluster, smem, [&] {
    const size_t rounded = std::max(smem, std::min<size_t>((smem / Residency::STEP + 1) * Residency::STEP, 227 * 1024 - 2048));
    allow_smem<Kernel>(dev, rounded);
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg =
        ops_config(dim3((unsigned)(4096 / cluster * cluster)), threads, rounded, cluster, nullptr, attr);
    int n = 0;
    if (cluster > 1) {
      cfg.attrs = attr + 1;
      cfg.numAttrs = 1;
      IEC_CUDA(cudaOccupancyMaxActiveClusters(&n, Kernel, &cfg));
    } else {
      IEC_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, Kernel, threads, rounded));
      n *= dev.sms();
    }
    return n * cluster;
  });
}

}  // namespace iec
