// fa4d_launch.cuh — launches that start before the kernel ahead of them in the stream is through
// (programmatic dependent launch), for kernels of a few microseconds.
//
// A kernel launched by launch_chained may run up to pdl_wait() while the one ahead is still at
// work; pdl_wait() returns when that one is complete and its writes are visible, so everything
// that touches global memory comes after it, and no load is of the kind (__ldg, ld.global.nc) that
// asks for data that stay as they are for the whole kernel, its time before the wait included: the
// kernel ahead may write them, and the compiler may move such a load above the wait.
// pdl_launch() lets the kernel behind start (up to its own wait) once every CTA of this grid has
// called it or ended.  After an ordinary kernel, or in front of one, both mean nothing and the
// stream's order holds as always.
#pragma once

#include <cuda_runtime.h>

namespace fa4d {

__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// `cluster`: CTAs per cluster along x.
template <typename... Params, typename... Args>
cudaError_t launch_chained(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t s,
                           Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

}  // namespace fa4d
