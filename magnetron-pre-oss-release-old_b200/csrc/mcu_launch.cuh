// Programmatic dependent launches, device and host side.  Everything has internal linkage.
#ifndef MCU_LAUNCH_CUH
#define MCU_LAUNCH_CUH
#include <cuda_runtime.h>
#include <utility>

namespace {

// Programmatic dependent launch: a kernel launched so may be scheduled while its
// predecessor on the stream finishes; it waits for the previous
// grid's completion (and memory) before it touches memory, and lets its own dependents be
// scheduled at once.  Both are no-ops for a kernel launched without the attribute.
__device__ __forceinline__ void pdl_begin() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
}

// A kernel launched as a programmatic dependent of the previous kernel on the stream (it waits in the
// kernel, pdl_begin, before touching memory).
template <typename... KArgs, typename... Args>
cudaError_t launch_dep(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                       Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

// Lets a kernel use more than 48 KB of dynamic shared memory: asked for once per kernel and device.
template <typename K>
cudaError_t allow_smem(K kern, int bytes, bool (&done)[64]) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev < 64 && done[dev])) return e;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 64) done[dev] = true;
    return e;
}

}  // namespace
#endif
