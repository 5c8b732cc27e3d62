// pdl.cuh -- programmatic dependent launch: a kernel's blocks are brought up while
// the kernel before it on the stream drains.
//
// Every kernel launched with launch_dependent calls dependent_wait() before it
// touches global memory: from there on the preceding kernel is complete and its
// writes are visible.  (That kernel has itself waited for its own predecessor, so
// completion carries along the stream.)  Behind other work -- copies, library
// kernels -- the launch is an ordinary one.
#pragma once
#include <cuda_runtime.h>

#include <utility>

namespace velo {

__device__ __forceinline__ void dependent_wait() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// cluster > 1: thread-block clusters of that many blocks along x.
template <typename... Params, typename... Args>
inline cudaError_t launch_dependent(void (*kernel)(Params...), dim3 grid, int threads, int smem, int cluster,
                                    cudaStream_t s, Args&&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

}  // namespace velo
