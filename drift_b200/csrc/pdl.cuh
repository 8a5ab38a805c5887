// pdl.cuh — programmatic dependent launch: a kernel may be set up on the SMs while
// the one before it on the stream still runs, and waits for that one's results
// itself. Every kernel launched with launch_pdl calls pdl_wait() in every thread
// before its first access to global memory (so that a chain of them is ordered:
// the wait returns once the kernel before has ended, which had waited in turn)
// and pdl_trigger() to let the next one be set up. They read global
// memory with plain loads: one marked as read-only for the kernel's life may be
// moved before the wait. Cast and product of 64 x 2048 x 2048 take 6.4 us in a row
// for it, 7.9 without.
#pragma once

#include <cuda_runtime.h>

namespace drift {

__device__ __forceinline__ void pdl_wait() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void pdl_trigger() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// `cluster`: CTAs a cluster, 0 where the kernel has its own or none.
template <class... P, class... A>
inline int launch_pdl(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem,
                      cudaStream_t st, unsigned cluster, const A &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    if (cluster) {
        at[1].id = cudaLaunchAttributeClusterDimension;
        at[1].val.clusterDim.x = cluster;
        at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
        cfg.numAttrs = 2;
    }
    return cudaLaunchKernelEx(&cfg, kernel, P(args)...) == cudaSuccess ? 0 : 3;
}

// Sets a kernel's dynamic shared memory once a process and device, not once a call.
template <class K>
inline bool allow_smem(K kernel, int bytes, unsigned long long &done) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return false;
    const unsigned long long bit = 1ULL << (dev & 63);
    if (__atomic_load_n(&done, __ATOMIC_ACQUIRE) & bit) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) !=
        cudaSuccess)
        return false;
    __atomic_fetch_or(&done, bit, __ATOMIC_RELEASE);
    return true;
}

}  // namespace drift
