// How this library launches a kernel, shared by its translation units.
#pragma once

#include <cuda_runtime.h>

#include <utility>

namespace lnsb {
namespace {

inline int status_of(cudaError_t e) { return e == cudaSuccess ? 0 : (int) e; }
inline int launch_status() { return status_of(cudaGetLastError()); }

// Programmatic dependent launch.  Every kernel of this library is launched
// with programmatic stream serialisation and begins with pdl_entry(): it
// waits there for the grid before it in the stream to complete (and its
// writes to be visible) before touching any data, then lets the grid after
// it launch.  The next kernel's launch and block scheduling so overlap this
// kernel's run instead of following its last block -- in a decode step of
// ~1,000 dependent launches that latency is a visible share.  A kernel
// launched without the attribute (torch's, say) is ordered as usual.
#ifndef LNSB_PDL
#define LNSB_PDL 1
#endif
__device__ __forceinline__ void pdl_entry() {
#if LNSB_PDL
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" :::);
#endif
}
template <typename... KArgs, typename... Args>
void launch_k(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args &&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = LNSB_PDL;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    (void) cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);   // an error stays in cudaGetLastError
}

}  // namespace
}  // namespace lnsb
