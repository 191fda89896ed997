// Kernel launches with programmatic stream serialization: the kernel may be put on the SMs while the one before
// it in the stream still runs.  Launched one after the other, a product's set-up (barriers, tensor memory, tensor
// maps) is off the critical path.  The rules that keep the order of the stream:
//
// * Every kernel launched this way waits (griddep_wait) for the end of the kernel before it, in all its CTAs, before it
//   writes to global memory and before it reads what that kernel writes.  As the kernel before did the same, all
//   earlier ones have then ended too.
// * Three kernels read ahead of that wait what older kernels wrote:
//     f8_scatter_kernel       the tokens              behind f8_plan_kernel
//     f8_few_kernel<kF8Down>  groups, down weights    behind f8_few_kernel<kF8GateUp>
//     f8_combine_kernel       slots, weights w, out   behind the down product
//   A kernel starts when every CTA of the one before it has let it (griddep_launch_dependents) or ended.  The plan and
//   the gate / up product let it after their own wait, so the caller's kernels (and the grouping, for the gate / up
//   product) have ended and their writes are performed by then; the down product lets its successor start at once, but
//   has itself started behind that point.  The wait that makes those writes visible was another grid's, so
//   these reads go past L1, whose lines might be older, to L2 (ld.cg, TMA), where nothing older is left.
// * No kernel launched this way uses non-coherent loads (__ldg, ld.global.nc, const __restrict__ pointers): its operands
//   may be written while it is on the SMs already, and the compiler may move such loads ahead of the wait.
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
