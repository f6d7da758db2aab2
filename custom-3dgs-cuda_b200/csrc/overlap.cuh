// Kernels that overlap at their ends (programmatic dependent launch). A kernel launched so may start
// before the one in front of it in the stream has ended; it waits for that one's end before it
// touches memory that the other may write or still read, which hides the launch and its set-up
// (1 to 2 us between small kernels). Such a kernel does not read through the read-only path (ld.global.nc,
// __ldg, const __restrict__), which is for data that nobody writes while the kernel lives. A kernel that lets the next one start early only gives up the
// room on the SMs: the next one still waits.
#pragma once

#include <cuda_runtime.h>

namespace gs {

__device__ __forceinline__ void let_next_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void wait_for_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Launches a kernel that may start before the previous one in the stream has ended, in clusters of
// `cluster` CTAs.
template <typename... Params, typename... Args>
cudaError_t launch_overlapped_clusters(void (*kernel)(Params...), dim3 grid, dim3 cluster,
                                       unsigned threads, size_t shared, cudaStream_t stream,
                                       const Args&... args) {
  cudaLaunchAttribute attributes[2] = {};
  attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[0].val.programmaticStreamSerializationAllowed = 1;
  attributes[1].id = cudaLaunchAttributeClusterDimension;
  attributes[1].val.clusterDim = {cluster.x, cluster.y, cluster.z};
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = shared;
  config.stream = stream;
  config.attrs = attributes;
  config.numAttrs = cluster.x * cluster.y * cluster.z > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&config, kernel, Params(args)...);
}
template <typename... Params, typename... Args>
cudaError_t launch_overlapped(void (*kernel)(Params...), dim3 grid, unsigned threads,
                              size_t shared, cudaStream_t stream, const Args&... args) {
  return launch_overlapped_clusters(kernel, grid, dim3(1), threads, shared, stream, args...);
}

}  // namespace gs
