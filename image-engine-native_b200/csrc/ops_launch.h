// Launches of the single operators' kernels: as programmatic dependents, in
// clusters, and how many CTAs the device holds at once.
#pragma once

#include <algorithm>
#include <utility>

#include "runtime.h"

namespace iec {

// Lets `Kernel` use `bytes` of dynamic shared memory, and clusters of 16.
template <auto Kernel>
void allow_smem(Device& dev, size_t bytes) {
  static size_t most[64] = {};
  size_t& m = most[dev.ordinal() & 63];
  if (m == 0) IEC_CUDA(cudaFuncSetAttribute(Kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  if (bytes > m) IEC_CUDA(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  m = std::max(m, std::max(bytes, (size_t)1));
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

// CTAs of `Kernel` (allow_smem called) that the device holds at once, in
// clusters of `cluster`; looked up once per cluster size and 16 KB of shared
// memory.
template <auto Kernel>
int resident_ctas(Device& dev, int threads, size_t smem, int cluster) {
  static int found[64][17][16] = {};
  int& f = found[dev.ordinal() & 63][cluster][std::min<size_t>(15, smem >> 14)];
  if (f == 0) {
    const size_t rounded = std::min<size_t>(((smem >> 14) + 1) << 14, 227 * 1024 - 2048);
    allow_smem<Kernel>(dev, std::max(smem, rounded));
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg = ops_config(dim3((unsigned)(4096 / cluster * cluster)), threads, std::max(smem, rounded),
                                        cluster, nullptr, attr);
    int n = 0;
    if (cluster > 1) {
      cfg.attrs = attr + 1;
      cfg.numAttrs = 1;
      IEC_CUDA(cudaOccupancyMaxActiveClusters(&n, Kernel, &cfg));
    } else {
      IEC_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, Kernel, threads, std::max(smem, rounded)));
      n *= dev.sms();
    }
    if (n < 1) throw Error(ERR_GPU, "no room for a cluster of CTAs");
    f = n * cluster;
  }
  return f;
}

}  // namespace iec
