// Launches with programmatic dependent launch: a kernel's blocks may be set up while the stream's
// previous kernel still runs, and wait in grid_dependency_wait() until that one has completed and
// its writes are visible.  Back to back this saves some 2 us of the 3 us between kernels (a
// kernel of 3 us every 3.8 us instead of every 6.1).
//
// Every kernel launched this way calls grid_dependency_wait() in every thread before that thread
// touches global memory, and allow_dependents() after it: a kernel that starts early behind it
// then knows that everything before the two of them has completed.  Such a kernel reads its inputs
// by plain loads: a load through the read-only path promises data that nobody writes while the
// kernel runs, which is not so before the wait, and the compiler need not keep it behind the wait.
// So no read-only intrinsic and no restrict-qualified pointer, from which the compiler infers one.
//
// The wait costs a block time of its own even when there is nothing to wait for: a grid of
// thousands of short blocks loses more than it gains (quantising 20161 x 5120 before a product of
// 64 columns, 12600 blocks: 91 us launched this way, 82 plainly), so grids of more than
// kOverlapBlocks blocks per SM are launched plainly, and the wait returns at once.
#pragma once
#include <cuda_runtime.h>
#include <c10/cuda/CUDAException.h>
#include <utility>

#include "tma_host.h"

namespace osp {

__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void allow_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

constexpr int kOverlapBlocks = 10;

// `cluster` blocks along x form a cluster where it is above 1.
template <typename... P, typename... A>
inline void launch_kernel(void (*kern)(P...), dim3 grid, int threads, int smem, int cluster, cudaStream_t stream,
                          A&&... a) {
  if (smem > 48 * 1024) smem_opt_in(reinterpret_cast<const void*>(kern), smem);
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  int dev = 0;
  C10_CUDA_CHECK(cudaGetDevice(&dev));
  attr[0].val.programmaticStreamSerializationAllowed =
      (long)grid.x * grid.y <= (long)kOverlapBlocks * num_sms(dev) ? 1 : 0;
  cfg.numAttrs = 1;
  if (cluster > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, std::forward<A>(a)...));
}

}  // namespace osp
