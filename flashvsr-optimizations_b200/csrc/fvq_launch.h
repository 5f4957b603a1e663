// fvq_launch.h -- launches of the block operators' kernels.
//
// They follow one another in a block, each a few microseconds long at a few rows, so every one
// is launched as a programmatic dependent of the kernel before it.  All but the streaming norm,
// which lost by it, let the next one start setting up (grid_launch_dependents).  Each waits for the
// previous one to complete (grid_dependency_wait) before any of its threads reads or writes global
// memory; the product of one or two rows sends L2 prefetches of W ahead of that wait, which read
// nothing.  A kernel may so be running while another writes what it is going to read: it reads
// with ordinary loads, never through the read-only path (__ldg, ld.global.nc, __restrict__),
// whose lines nothing promises to refresh inside a running kernel.
#pragma once

#include <cuda_runtime.h>

#include <utility>

namespace fvq {

// cluster: CTAs per cluster along x (0: none).
template <class... Params, class... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t st,
                             int cluster, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

}  // namespace fvq
