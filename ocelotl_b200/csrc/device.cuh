// device.cuh -- small device helpers shared by the decode-step kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace ocl {

// Programmatic dependent launch: every thread of a kernel launched with it waits
// here before its first read or write of memory that another kernel uses, so a
// kernel's own completion implies that of all kernels before it.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <class... KArgs, class... Args>
cudaError_t launch_kernel(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, bool pdl, cudaStream_t s,
                          const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// float -> 16-bit cache element, round to nearest even
__device__ __forceinline__ uint32_t pack16(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack16(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack16(uint32_t w, __nv_bfloat16) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack16(uint32_t w, __half) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// Key of a greedy pick: the largest value wins, among equals the smallest index.
__device__ __forceinline__ unsigned long long greedy_key(float v, uint32_t idx) {
    uint32_t b = __float_as_uint(v == 0.0f ? 0.0f : v);  // -0.0 -> +0.0
    b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);       // monotone in v
    return ((unsigned long long)b << 32) | (unsigned long long)(0xFFFFFFFFu - idx);
}

}  // namespace ocl
