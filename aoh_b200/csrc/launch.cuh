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

}  // namespace aoh
