// pdl.cuh -- launches whose start overlaps the end of the kernel before them in the stream
// (programmatic dependent launch). A kernel launched so sets itself up, then calls pdl_wait()
// before it touches any memory that another kernel may write or read: the wait returns when
// every kernel before it has finished and its writes are visible. pdl_release() lets the next
// kernel start its own set-up; it orders nothing.
// Such a kernel is resident while the one before it still writes, so nothing that it reads is
// constant over its lifetime: no read-only loads (ld.global.nc), neither by name nor through
// `const ... __restrict__` parameters, which would also let the compiler move a load above the wait.
#pragma once

#include "common.cuh"

namespace k3 {

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// `cluster` CTAs a cluster (1: none)
template <typename... P, typename... A>
inline int launch_pdl(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t s, int cluster, A &&...args)
{
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
    const int st = launch_status();
    return e != cudaSuccess ? cuda_status(e) : st;
}

}  // namespace k3
