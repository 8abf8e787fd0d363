#pragma once

// Shared by the expert-layer kernels: their limits, and a launch that may overlap the end of the kernel before it.

#include <cuda_runtime.h>

#include <cstddef>

namespace kl::capi {

constexpr int kMaxExperts = 1024;
constexpr int kMaxTopK = 32;

// Dynamic shared memory: what each of these kernels may have beside its static arrays (up to 16 KB) without asking, and the
// most that one takes (the plan of 1024 experts).
constexpr size_t kPlainSmem = 32 * 1024;
constexpr size_t kMostSmem = 128 * 1024;

inline cudaError_t launch_dependent(cudaStream_t stream, dim3 grid, int threads, size_t smem, int cluster, void const* kernel,
                                    void** args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = grid;
  cfg.blockDim = dim3(unsigned(threads), 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  if (smem > kPlainSmem) {
    // Always to the most: a limit of this call's own would undercut a larger call that another thread is about to launch.
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kMostSmem));
    if (e != cudaSuccess) return e;
  }
  return cudaLaunchKernelExC(&cfg, kernel, args);
}

}  // namespace kl::capi
