// Kernel launches with programmatic stream serialization: the kernel may be put on the SMs while the one before
// it in the stream still runs.  Every kernel launched this way waits (griddep_wait) for the end of the kernel
// before it, in all its CTAs, ahead of its first access to memory that anything else in the stream may write
// or read; so what it follows, and what follows it, see the order of the stream.  Launched one after the
// other, a product's set-up (barriers, tensor memory, tensor maps) is off the critical path.
// The last kernel of a call does not let the next kernel start before its end: the planner and the decode kernel
// read router logits ahead of their wait, and a product may have written them.  The quantiser and the loss, whose
// outputs no kernel reads ahead of its wait, let the next one start once their own wait is over.
#pragma once
#include <cuda_runtime.h>

namespace moe {

template <class K, class... A>
cudaError_t launch_after(K kernel, int grid, int threads, int smem, int cluster, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
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
    cfg.numAttrs = cluster > 0 ? 2 : 1;  // 0: no cluster, or the kernel's own
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace moe
