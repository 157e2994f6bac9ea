// launch.cuh -- programmatic dependent launch for kernels that follow one another on a stream.
//
// A kernel's own start (barriers, TMEM, descriptors, its blocks' launch) overlaps the end of the kernel
// before it. Norm, ffn1, quantiser, ffn2 in a CUDA graph on B200, without and with: 16 tokens 17.6 / 15.4 us,
// 1560 tokens 58.6 / 55.9 us; 4680 x 4608 x 1536 products back to back 29.2 / 27.9 us.
#pragma once

#include <cuda_runtime.h>

#include <utility>

namespace ss {

// Waits until the grids before this one on the stream are complete and their memory is visible. Every
// thread of a kernel started by launch_after() calls it before it touches global memory, and such a
// kernel reads nothing through the non-coherent path (ld.global.nc, const __restrict__): its inputs may
// still be written while it already runs.
__device__ __forceinline__ void wait_for_earlier() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Lets the next such kernel on the stream set itself up once every block of this one has got here.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename K, typename... A>
static cudaError_t launch_after(K kernel, unsigned blocks, unsigned threads, size_t smem, cudaStream_t st, unsigned cluster,
                                const A &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
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
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace ss
