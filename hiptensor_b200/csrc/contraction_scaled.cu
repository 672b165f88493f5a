// Block-scaled 8-bit contraction: D[m, n] = alpha * sum over blocks of 128 of k of
// scaleA * scaleB * sum_k A[m, k] B[n, k], + beta * C[m, n]; operands e4m3 / e5m2, sums in f32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "kernels.hpp"
#include "scaled.hpp"

namespace htb
{
    namespace
    {
        __device__ __forceinline__ float widen8(unsigned char v, bool e5m2)
        {
            return __half2float(__half(__nv_cvt_fp8_to_halfraw(v, e5m2 ? __NV_E5M2 : __NV_E4M3)));
        }
        template <typename TD>
        __device__ __forceinline__ TD narrow(float v);
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

        // Any strides and extents: 64 x 64 tiles, 16 x 16 threads with 4 x 4 results each, byte loads into shared memory as
        // f32, FMA. A block's products are summed by themselves and scaled once.
        template <typename TD>
        __global__ void __launch_bounds__(256) scaled_simt_kernel(const unsigned char* __restrict__ A, const float* __restrict__ sA,
                                                                  const unsigned char* __restrict__ B, const float* __restrict__ sB,
                                                                  const TD* C, TD* D, float alpha, float beta, const __grid_constant__ ScaledPlan p)
        {
            constexpr int    kStep = 32;
            __shared__ float a[kStep][65], b[kStep][65];
            const int64_t    m0 = int64_t(blockIdx.x) * 64, n0 = int64_t(blockIdx.y) * 64;
            const int        tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
            const bool       aWide = p.typeA == CUDA_R_8F_E5M2, bWide = p.typeB == CUDA_R_8F_E5M2;
            float            sum[4][4] = {};
            for(int64_t k0 = 0; k0 < p.K; k0 += kScaleBlock)
            {
                float part[4][4] = {};
                for(int64_t k1 = k0; k1 < min(k0 + kScaleBlock, p.K); k1 += kStep)
                {
                    for(int i = threadIdx.x; i < 64 * kStep; i += 256)
                    {
                        // neighbouring threads along the contiguous mode
                        const int     ra = p.aK == 1 ? i / kStep : i % 64, ka = p.aK == 1 ? i % kStep : i / 64;
                        const int     rb = p.bK == 1 ? i / kStep : i % 64, kb = p.bK == 1 ? i % kStep : i / 64;
                        const int64_t m = m0 + ra, n = n0 + rb;
                        a[ka][ra] = (m < p.M && k1 + ka < p.K) ? widen8(A[m * p.aM + (k1 + ka) * p.aK], aWide) : 0.f;
                        b[kb][rb] = (n < p.N && k1 + kb < p.K) ? widen8(B[n * p.bN + (k1 + kb) * p.bK], bWide) : 0.f;
                    }
                    __syncthreads();
#pragma unroll 8
                    for(int k = 0; k < kStep; k++)
                    {
                        float x[4], y[4];
#pragma unroll
                        for(int i = 0; i < 4; i++)
                        {
                            x[i] = a[k][ty + 16 * i];
                            y[i] = b[k][tx + 16 * i];
                        }
#pragma unroll
                        for(int i = 0; i < 4; i++)
#pragma unroll
                            for(int j = 0; j < 4; j++)
                                part[i][j] = fmaf(x[i], y[j], part[i][j]);
                    }
                    __syncthreads();
                }
                const int64_t kb = k0 / kScaleBlock;
                float         x[4], y[4];
#pragma unroll
                for(int i = 0; i < 4; i++)
                {
                    const int64_t m = m0 + ty + 16 * i, n = n0 + tx + 16 * i;
                    x[i] = m < p.M ? sA[(m / p.blockM) * p.saM + kb * p.saK] : 0.f;
                    y[i] = n < p.N ? sB[(n / p.blockN) * p.sbN + kb * p.sbK] : 0.f;
                }
#pragma unroll
                for(int i = 0; i < 4; i++)
#pragma unroll
                    for(int j = 0; j < 4; j++)
                        sum[i][j] = fmaf(part[i][j] * x[i], y[j], sum[i][j]);
            }
#pragma unroll
            for(int i = 0; i < 4; i++)
#pragma unroll
                for(int j = 0; j < 4; j++)
                {
                    const int64_t m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
                    if(m >= p.M || n >= p.N)
                        continue;
                    const int64_t at = m * p.dM + n * p.dN;
                    const float   v  = alpha * sum[i][j];
                    D[at]            = narrow<TD>(C ? fmaf(beta, widen(C[at]), v) : v);
                }
        }

        template <typename TD>
        cudaError_t launchTyped(const ScaledPlan& p, float alpha, const void* A, const float* sA, const void* B, const float* sB,
                                float beta, const void* C, void* D, cudaStream_t stream)
        {
            const int64_t gx = (p.M + 63) / 64, gy = (p.N + 63) / 64;
            if(gx > 0x7fffffffll || gy > 65535)
                return cudaErrorInvalidConfiguration;
            scaled_simt_kernel<TD><<<dim3(unsigned(gx), unsigned(gy)), 256, 0, stream>>>(
                (const unsigned char*)A, sA, (const unsigned char*)B, sB, (const TD*)C, (TD*)D, alpha, beta, p);
            const cudaError_t e = cudaGetLastError();
            if(e == cudaSuccess)
                noteLaunch("scaled_simt");
            return e;
        }
    } // namespace

    cudaError_t launchScaled(const ScaledPlan& p, float alpha, const void* A, const float* scaleA, const void* B,
                             const float* scaleB, float beta, const void* C, void* D, int smCount, int* deviceStatus,
                             cudaStream_t stream)
    {
        (void)smCount;
        (void)deviceStatus;
        switch(p.typeD)
        {
        case CUDA_R_32F: return launchTyped<float>(p, alpha, A, scaleA, B, scaleB, beta, C, D, stream);
        case CUDA_R_16F: return launchTyped<__half>(p, alpha, A, scaleA, B, scaleB, beta, C, D, stream);
        case CUDA_R_16BF: return launchTyped<__nv_bfloat16>(p, alpha, A, scaleA, B, scaleB, beta, C, D, stream);
        }
        return cudaErrorNotSupported;
    }
} // namespace htb
