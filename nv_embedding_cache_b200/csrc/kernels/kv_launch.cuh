// Launches of the paged cache's kernels, each overlapping the end of whatever runs before it on the stream
// (programmatic dependent launch): blocks may be in place before that is done, and wait for it before they touch
// memory.  Worth 1 to 2 us a call (attention of 9 short sequences 28.1 -> 26.6 us, of 131072 rows 102 -> 100).
#pragma once

#include <utility>

#include "../common.hpp"

namespace nve_b200 {

// Waits until everything before this grid on its stream is complete and visible.  Every block of every kernel calls it
// before it ends, so a grid never ends before the one it was launched behind.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Lets the next grid's blocks come in as soon as every block of this one has said so (or ended).  Called after
// grid_wait: what the next grid reads before its own wait is then complete as well, unless this grid writes it.
__device__ __forceinline__ void grid_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// cluster: CTAs of a thread-block cluster, 1 for none
template <typename... Params, typename... Args>
void launch_overlapped(void (*kernel)(Params...), int64_t grid, int block, size_t smem, unsigned cluster, cudaStream_t stream,
                       Args&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(static_cast<unsigned>(block));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2]{};
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = cluster;
  attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  NVE_B200_CUDA(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...));
}

}  // namespace nve_b200
