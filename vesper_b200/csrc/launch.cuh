// Launches with attributes: thread-block clusters, and programmatic dependent launch, in which a kernel
// may be brought onto the SMs while the one before it on the stream is still finishing. Such a kernel
// calls grid_wait() before it touches global memory; what it does before that (barriers, tensor memory,
// index arithmetic) then costs no time of its own. grid_release() lets the next kernel come early too.
#pragma once
#include "common.cuh"

namespace vb {

// every earlier kernel of the stream has ended and its writes are visible
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename K, typename... P>
int launch_early(const char* what, K kernel, dim3 grid, int threads, int smem, int cluster, cudaStream_t st, P... args) {
  if (smem > 32 * 1024)  // with the kernel's static arrays this may pass the 48 KB a launch has by default
    VB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), what);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) {
    cudaGetLastError();  // reported here, not again by the next launch's check
    set_error("%s: launch failed: %s", what, cudaGetErrorString(e));
    return VB_ERR_CUDA;
  }
  count_launch();
  return VB_OK;
}

}  // namespace vb
