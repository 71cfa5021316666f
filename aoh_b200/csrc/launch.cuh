// Kernel launches as programmatic dependents.
#pragma once

#include <cuda_runtime.h>

#include "internal.h"

namespace aoh {

// Launch whose grid may start while the kernel before it in the stream ends:
// every thread of it that reads or writes what that kernel may touch calls
// griddep_wait() first.  cluster: CTAs in x, or 1.
template <class F, class... A>
int launch_dependent(F kernel, dim3 grid, int cluster, int threads, size_t smem, cudaStream_t st, const char* what,
                     A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cuda_check(cudaLaunchKernelEx(&cfg, kernel, args...), what);
}

// The larger of two cluster sizes of which the current device can hold one: clusters
// of 16 are not portable, and need a GPC with as many SMs for CTAs that fill one each.
// smem: the most dynamic shared memory that the kernel is launched with.
template <class F>
int larger_cluster(F kernel, int large, int portable, int threads, size_t smem, const char* what, int* cluster) {
  int rc = cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), what);
  if (rc) return rc;
  rc = cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), what);
  if (rc) return rc;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)large;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)large);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int n = 0;
  rc = cuda_check(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg), what);
  if (rc) return rc;
  *cluster = n > 0 ? large : portable;
  return AOH_OK;
}

}  // namespace aoh
