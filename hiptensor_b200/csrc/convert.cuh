// f32, f16 and bf16 elements as f32 numbers and back, rounded once to the nearest.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace htb
{
    namespace
    {
        __device__ __forceinline__ float widen(float v)
        {
            return v;
        }
        __device__ __forceinline__ float widen(__half v)
        {
            return __half2float(v);
        }
        __device__ __forceinline__ float widen(__nv_bfloat16 v)
        {
            return __bfloat162float(v);
        }
        template <typename T>
        __device__ __forceinline__ T narrow(float v);
        template <>
        __device__ __forceinline__ float narrow<float>(float v)
        {
            return v;
        }
        template <>
        __device__ __forceinline__ __half narrow<__half>(float v)
        {
            return __float2half_rn(v);
        }
        template <>
        __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v)
        {
            return __float2bfloat16_rn(v);
        }
    } // namespace
} // namespace htb
