// Internal: what the launchers of the library's kernels share.
#ifndef SAL_LAUNCH_H
#define SAL_LAUNCH_H

#include <cuda_runtime.h>

#include <atomic>

#include "sal_lutgemm.h"

// Lets `kernel` be launched with all the dynamic shared memory that the current device gives a block.  The limit belongs to the (kernel,
// device) pair and is set once, to its largest value: one that followed the launches' needs could be lowered by a thread with a smaller
// launch between another thread's look at it and its launch.  `done` is the kernel's own, per device ordinal.
template <typename Kernel>
cudaError_t sal_allow_shared_memory(Kernel *kernel, std::atomic<bool> (&done)[64]) {
    int dev = 0, most = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (done[dev].load(std::memory_order_acquire)) return cudaSuccess;
    cudaFuncAttributes attr;
    if ((e = cudaFuncGetAttributes(&attr, kernel)) != cudaSuccess) return e;
    if ((e = cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev)) != cudaSuccess) return e;
    if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most - (int)attr.sharedSizeBytes)) != cudaSuccess) return e;
    done[dev].store(true, std::memory_order_release);
    return cudaSuccess;
}

// The decode-step helpers are launched with the programmatic-stream-serialization attribute: their kernels begin with
// griddepcontrol.launch_dependents and griddepcontrol.wait.
template <typename... KArgs, typename... Args>
int sal_launch_pdl(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, void *stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = reinterpret_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...) == cudaSuccess ? SAL_OK : SAL_E_LAUNCH;
}

#endif
