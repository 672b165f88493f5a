// Kernels of the linear cross entropy around the library's contractions.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "cross_entropy.hpp"
#include "kernels.hpp"

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

        __device__ __forceinline__ int64_t rowOffset(const TokenRows& r, int64_t row)
        {
            int64_t off = 0;
            for(int i = r.nt - 1; i >= 0; i--)
            {
                const int64_t q = i ? row / r.ext[i] : 0;
                off += (row - q * r.ext[i]) * r.stride[i];
                row = q;
            }
            return off;
        }
        __device__ __forceinline__ bool counts(int64_t target, int64_t ignore, int64_t V)
        {
            return target != ignore && target >= 0 && target < V;
        }

        template <typename T>
        __global__ void pack_rows_kernel(const T* __restrict__ X, const __grid_constant__ TokenRows rows, int64_t count, int64_t cols, int64_t ld,
                                         T* __restrict__ X2, const int64_t* __restrict__ targets, int64_t ignore, int64_t V)
        {
            for(int64_t r = blockIdx.x; r < count; r += gridDim.x)
            {
                const bool    live = !targets || counts(targets[r], ignore, V);
                const T*      src  = X + rowOffset(rows, r);
                for(int64_t c = threadIdx.x; c < ld; c += blockDim.x)
                    X2[r * ld + c] = (live && c < cols) ? src[c * rows.elem] : narrow<T>(0.f);
            }
        }

        // one block per token
        __global__ void __launch_bounds__(256) softmax_piece_kernel(const float* __restrict__ z, int64_t ldz, int64_t T, int64_t v0, int64_t count,
                                                                    const int64_t* __restrict__ targets, float* state)
        {
            __shared__ float part[8];
            for(int64_t t = blockIdx.x; t < T; t += gridDim.x)
            {
                const float* row = z + t * ldz;
                float        m   = -INFINITY;
                for(int64_t v = threadIdx.x; v < count; v += 256)
                {
                    const float x = row[v];
                    m             = (x > m || x != x) ? x : m; // a NaN stays
                }
                for(int s = 16; s; s >>= 1)
                {
                    const float o = __shfl_xor_sync(0xffffffffu, m, s);
                    m             = (o > m || o != o) ? o : m;
                }
                __syncthreads();
                if((threadIdx.x & 31) == 0)
                    part[threadIdx.x >> 5] = m;
                __syncthreads();
                for(int i = 0; i < 8; i++)
                    m = (part[i] > m || part[i] != part[i]) ? part[i] : m;
                const float ref = fabsf(m) == INFINITY ? 0.f : m;
                float       sum = 0.f;
                for(int64_t v = threadIdx.x; v < count; v += 256)
                    sum += expf(row[v] - ref);
                for(int s = 16; s; s >>= 1)
                    sum += __shfl_xor_sync(0xffffffffu, sum, s);
                __syncthreads();
                if((threadIdx.x & 31) == 0)
                    part[threadIdx.x >> 5] = sum;
                __syncthreads();
                if(threadIdx.x == 0)
                {
                    sum = 0.f;
                    for(int i = 0; i < 8; i++)
                        sum += part[i];
                    const int64_t target = targets[t];
                    if(target >= v0 && target < v0 + count)
                        state[2 * T + t] = row[target - v0];
                    if(v0)
                    {
                        const float m1 = state[t], s1 = state[T + t];
                        const float top = (m1 > m || m1 != m1) ? m1 : m;
                        const float r2  = fabsf(top) == INFINITY ? 0.f : top;
                        // each sum was taken relative to its own reference
                        const float f1 = fabsf(m1) == INFINITY ? 0.f : m1;
                        sum            = s1 * expf(f1 - r2) + sum * expf(ref - r2);
                        m              = top;
                    }
                    state[t]     = m;
                    state[T + t] = sum;
                }
            }
        }

        __global__ void loss_finish_kernel(const float* __restrict__ state, int64_t T, int64_t V, int64_t ignore,
                                           const int64_t* __restrict__ targets, float* loss, float* lse, int* status)
        {
            const int64_t t = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
            if(t >= T)
                return;
            const float   m = state[t], ref = fabsf(m) == INFINITY ? 0.f : m;
            const float   l = ref + logf(state[T + t]);
            const int64_t target = targets[t];
            lse[t] = l;
            if(target == ignore)
                loss[t] = 0.f;
            else if(target < 0 || target >= V)
            {
                loss[t] = __int_as_float(0x7fc00000);
                atomicExch_system(status, kStatusBadTarget);
            }
            else
                loss[t] = l - state[2 * T + t];
        }

        __global__ void __launch_bounds__(1024) gradient_scale_kernel(const float* __restrict__ g, float alpha, int64_t T, float* scale)
        {
            __shared__ float part[32];
            float            m = 0.f;
            for(int64_t t = threadIdx.x; t < T; t += 1024)
                m = fmaxf(m, fabsf(g[t] * alpha));
            for(int s = 16; s; s >>= 1)
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
            if((threadIdx.x & 31) == 0)
                part[threadIdx.x >> 5] = m;
            __syncthreads();
            if(threadIdx.x == 0)
            {
                for(int i = 0; i < 32; i++)
                    m = fmaxf(m, part[i]);
                int e = 15; // m < 2^e: the factor 2^(15 - e) keeps |P| below 2^15
                if(m > 0.f && m < INFINITY)
                    frexpf(m, &e);
                e        = max(e, -100);
                scale[0] = ldexpf(1.f, 15 - e);
                scale[1] = ldexpf(1.f, e - 15);
            }
        }

        template <typename TP>
        __global__ void probabilities_kernel(const float* z, int64_t ldz, int64_t T, int64_t v0, int64_t count, int64_t V, int64_t ignore,
                                             const int64_t* __restrict__ targets, const float* __restrict__ lse, const float* __restrict__ g,
                                             float alpha, const float* __restrict__ scale, TP* P, int64_t ldp, int* status)
        {
            for(int64_t t = blockIdx.x; t < T; t += gridDim.x)
            {
                const int64_t target = targets[t];
                const bool    live   = counts(target, ignore, V);
                const float   l = lse[t], f = g[t] * alpha * (scale ? scale[0] : 1.f);
                if(!live && target != ignore && threadIdx.x == 0)
                    atomicExch_system(status, kStatusBadTarget);
                for(int64_t v = threadIdx.x; v < count; v += blockDim.x)
                {
                    float p = expf(z[t * ldz + v] - l);
                    if(v0 + v == target)
                        p -= 1.f;
                    P[t * ldp + v] = narrow<TP>(live ? p * f : 0.f);
                }
            }
        }

        template <typename T>
        __global__ void store_rows_kernel(const float* __restrict__ X, int64_t ldx, int64_t count, int64_t cols, const float* __restrict__ scale,
                                          T* __restrict__ Y, const __grid_constant__ TokenRows rows)
        {
            const float f = scale ? scale[1] : 1.f;
            for(int64_t r = blockIdx.x; r < count; r += gridDim.x)
            {
                T* dst = Y + rowOffset(rows, r);
                for(int64_t c = threadIdx.x; c < cols; c += blockDim.x)
                    dst[c * rows.elem] = narrow<T>(X ? X[r * ldx + c] * f : 0.f);
            }
        }

        int rowGrid(int64_t rows)
        {
            return int(std::min<int64_t>(rows, 148 * 64));
        }
        cudaError_t noted(const char* name)
        {
            const cudaError_t e = cudaGetLastError();
            if(e == cudaSuccess)
                noteLaunch(name);
            return e;
        }
    } // namespace

    cudaError_t launchPackRows(int type, const void* X, const TokenRows& rows, int64_t count, int64_t cols, int64_t ld, void* X2,
                               const int64_t* targets, int64_t ignore, int64_t V, cudaStream_t stream)
    {
        const int grid = rowGrid(count);
        if(type == CUDA_R_32F)
            pack_rows_kernel<float><<<grid, 256, 0, stream>>>((const float*)X, rows, count, cols, ld, (float*)X2, targets, ignore, V);
        else if(type == CUDA_R_16F)
            pack_rows_kernel<__half><<<grid, 256, 0, stream>>>((const __half*)X, rows, count, cols, ld, (__half*)X2, targets, ignore, V);
        else
            pack_rows_kernel<__nv_bfloat16>
                <<<grid, 256, 0, stream>>>((const __nv_bfloat16*)X, rows, count, cols, ld, (__nv_bfloat16*)X2, targets, ignore, V);
        return noted("cross_entropy_pack");
    }

    cudaError_t launchSoftmaxPiece(const float* z, int64_t ldz, int64_t T, int64_t v0, int64_t count, const int64_t* targets, float* state,
                                   cudaStream_t stream)
    {
        softmax_piece_kernel<<<rowGrid(T), 256, 0, stream>>>(z, ldz, T, v0, count, targets, state);
        return noted("cross_entropy_softmax");
    }

    cudaError_t launchLossFinish(const float* state, int64_t T, int64_t V, int64_t ignore, const int64_t* targets, float* loss, float* lse,
                                 int* deviceStatus, cudaStream_t stream)
    {
        loss_finish_kernel<<<unsigned((T + 255) / 256), 256, 0, stream>>>(state, T, V, ignore, targets, loss, lse, deviceStatus);
        return noted("cross_entropy_loss");
    }

    cudaError_t launchGradientScale(const float* g, float alpha, int64_t T, float* scale, cudaStream_t stream)
    {
        gradient_scale_kernel<<<1, 1024, 0, stream>>>(g, alpha, T, scale);
        return noted("cross_entropy_scale");
    }

    cudaError_t launchProbabilities(int type, const float* z, int64_t ldz, int64_t T, int64_t v0, int64_t count, int64_t V, int64_t ignore,
                                    const int64_t* targets, const float* lse, const float* g, float alpha, const float* scale, void* P,
                                    int64_t ldp, int* deviceStatus, cudaStream_t stream)
    {
        const int grid = rowGrid(T);
        if(type == CUDA_R_32F)
            probabilities_kernel<float><<<grid, 256, 0, stream>>>(z, ldz, T, v0, count, V, ignore, targets, lse, g, alpha, scale, (float*)P,
                                                                  ldp, deviceStatus);
        else if(type == CUDA_R_16F)
            probabilities_kernel<__half><<<grid, 256, 0, stream>>>(z, ldz, T, v0, count, V, ignore, targets, lse, g, alpha, scale,
                                                                   (__half*)P, ldp, deviceStatus);
        else
            probabilities_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(z, ldz, T, v0, count, V, ignore, targets, lse, g, alpha, scale,
                                                                          (__nv_bfloat16*)P, ldp, deviceStatus);
        return noted("cross_entropy_probabilities");
    }

    cudaError_t launchStoreRows(int type, const float* X, int64_t ldx, int64_t count, int64_t cols, const float* scale, void* Y,
                                const TokenRows& rows, cudaStream_t stream)
    {
        const int grid = rowGrid(count);
        if(type == CUDA_R_32F)
            store_rows_kernel<float><<<grid, 256, 0, stream>>>(X, ldx, count, cols, scale, (float*)Y, rows);
        else if(type == CUDA_R_16F)
            store_rows_kernel<__half><<<grid, 256, 0, stream>>>(X, ldx, count, cols, scale, (__half*)Y, rows);
        else
            store_rows_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(X, ldx, count, cols, scale, (__nv_bfloat16*)Y, rows);
        return noted("cross_entropy_store");
    }
} // namespace htb
