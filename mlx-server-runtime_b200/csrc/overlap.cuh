// Helpers of the decoder-layer kernels: the launch-overlap instructions and launch,
// packed pairs of 16-bit elements.
#pragma once

#include "common.cuh"
#include "launch.h"

namespace mlxq {

__device__ __forceinline__ void pdl_launch_dependents() {
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
}
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t u) {
    return make_float2(Elem<T>::lo(u), Elem<T>::hi(u));
}

template <typename T>
__device__ __forceinline__ uint16_t bits16(T v) {
    return *reinterpret_cast<const uint16_t*>(&v);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    return static_cast<uint32_t>(bits16(Elem<T>::from_f(a))) |
           (static_cast<uint32_t>(bits16(Elem<T>::from_f(b))) << 16);
}

template <typename T>
__device__ __forceinline__ float round_t(float v) {
    return Elem<T>::to_f(Elem<T>::from_f(v));
}

// Launch with the overlap attribute when asked; the kernel's carveout is set to the
// whole shared-memory capacity once per device (see ensure_smem_attr).
inline cudaError_t launch_ex(const void* func, PerDevice& cache, dim3 grid, dim3 block, size_t smem,
                             cudaStream_t st, bool overlap, void** args) {
    int dev = 0;
    cudaError_t e = current_device(&dev);
    if (e != cudaSuccess) return e;
    e = ensure_smem_attr(func, cache, dev, smem > 0 ? static_cast<int>(smem) : 1);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = overlap ? attr : nullptr;
    cfg.numAttrs = overlap ? 1 : 0;
    return cudaLaunchKernelExC(&cfg, func, args);
}

}  // namespace mlxq
