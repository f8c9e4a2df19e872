// dw_launch.h -- launches as a programmatic dependent of the previous kernel on the
// backend's stream.  The kernel's blocks may start while that kernel finishes; they
// touch no global memory before pdl_wait(), which returns once it has completed and
// its writes are visible.  Each block then calls pdl_trigger(): not before pdl_wait()
// (kernels waiting in a row would fill the SMs: quantise and dequantise of 1000 x 1010
// f32 took 18 instead of 9 us), and after any tcgen05.alloc (a dependent block that
// took tensor memory first would wait for a kernel that waits for it).  What such a kernel
// reads may be written during its own life, so it reads by ordinary loads: no __ldg and no
// `const T *__restrict__`, whose loads may be moved above the wait and past coherence.
#pragma once

#include <cstdlib>

#include "dw_internal.h"

namespace dw {

#ifdef __CUDACC__
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
#endif

// DW_PDL=0: tuning switch, plain stream order.
inline bool pdl_enabled() {
    static const bool on = !(getenv("DW_PDL") && atoi(getenv("DW_PDL")) == 0);
    return on;
}

// cluster: CTAs of a cluster along x (0: the kernel's own).
template <typename... P, typename... A>
dw_status launch_dependent(dw_backend *be, const char *what, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem,
                           unsigned cluster, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = be->stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster, attr[n].val.clusterDim.y = 1, attr[n].val.clusterDim.z = 1;
        n++;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    dw_status st = dw_cuda_check(be, cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...), what);
    return st != DW_OK ? st : dw_after_launch(be, what);
}

}  // namespace dw
