// lrs_ops.cuh — what the stateless operators (draws, 8-bit quantisation, the head's product)
// share: element types, wide loads of unaligned rows, and errors of calls without a context.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/llamars_sampler.h"

// Sets lrs_last_error(NULL) of this thread and returns `code`.
int lrs_call_error(int code, const char* fmt, ...);

namespace lrs {

// A launch's result as a status.  The runtime's last error is not asked: it may be that of an earlier call of this
// thread; what a failed launch left there is taken away, since it is reported here.
inline int launched(const char* what, cudaError_t e) {
    if (e == cudaSuccess) return LRS_OK;
    cudaGetLastError();
    return lrs_call_error(LRS_E_CUDA, "%s: launch failed: %s", what, cudaGetErrorString(e));
}

template <typename... P, typename... A>
int launch_kernel(const char* what, void (*kernel)(P...), unsigned grid, unsigned block, size_t smem, cudaStream_t s,
                  const A&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid), cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem, cfg.stream = s;
    return launched(what, cudaLaunchKernelEx(&cfg, kernel, args...));
}

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float(float v) { return v; }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }

// The elements of 16 bytes as floats.
__device__ __forceinline__ void unpack(const uint4& v, float (&x)[4], const float*) {
    x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void unpack(const uint4& v, float (&x)[8], const __nv_bfloat16*) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(u[i] << 16);
        x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ void unpack(const uint4& v, float (&x)[8], const __half*) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        __half2 h;
        *reinterpret_cast<uint32_t*>(&h) = u[i];
        const float2 f = __half22float2(h);
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
}

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

}  // namespace lrs
