// Launches that may begin beside the end of the kernel before them in the stream.
#pragma once
#include <cuda_runtime.h>

#include <cstddef>

namespace gmm {

// On the device: until the kernel before has ended and its writes are there, which comes before any access to memory; and leave for the
// next kernel to begin, once every block has called it.
__device__ __forceinline__ void dependent_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void dependent_release() { asm volatile("griddepcontrol.launch_dependents;"); }

template <typename... P, typename... A>
cudaError_t launch_dependent(void (*kernel)(P...), dim3 blocks, unsigned threads, size_t smem, int cluster, cudaStream_t stream, const A &...args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = blocks;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace gmm
