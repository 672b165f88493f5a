// The gradient of a few tokens in one pass over W, and the loss of a few tokens of f32 and unaligned heads. A few tokens are
// bound by the bytes of W and dW; the tensor-core path reads W twice and P once more, after copying what no TMA load can read.
// Here a block takes a few classes at a time: its threads hold the columns, multiply their parts of the classes' rows with
// all tokens (H is in shared memory), add the parts up over the block, make the probabilities, and use them while the rows
// are still in the first-level cache: a class's row of dW is written once, and dH's sums over the block's classes stay in
// shared memory until the end, when a second kernel adds the blocks up in a fixed order. All sums and P are f32.
//
// One token x 32000 x 1024 f32: gradient 51 us (5.2 TB/s; by the tensor cores 242), loss 33 (123); 8 tokens 103 (247) and 64
// (126): instructions, no longer bytes. 2 tokens x 128000 x 4096 bf16: gradient 433 us (4.8 TB/s; 664).
#include <algorithm>

#include "common.hpp"
#include "cross_entropy_device.cuh"
#include "kernels.hpp"

namespace htb
{
    namespace
    {
        constexpr int kFewThreads = 256;

        struct FewArgs
        {
            const void*    H;
            const void*    W;
            TokenRows      rows; // of H
            int64_t        T, V, wV;
            int64_t        units; // of a row: 16 bytes, two elements or one
            const int64_t* targets;
            int64_t        ignore;
            float          alpha;
            int*           status;
            // loss: (maximum, sum of exponentials) of a block's classes, [block][T]; target logits
            float2* part;
            float*  targetLogit;
            // gradient
            const float *lse, *g;
            void*        dW; // rows wV apart; null: not wanted
            float*       dH; // [block][T][ldh]; null: not wanted
            int64_t      ldh;
        };

        // Adds K values up over the 32 lanes: halves are exchanged, so that each step moves half as many. The sum number
        // lane / (32 / K) is returned.
        template <int K>
        __device__ __forceinline__ float sumOverLanes(float (&v)[K], int lane)
        {
            int off = 16;
#pragma unroll
            for(int n = K / 2; n >= 1; n /= 2)
            {
                const bool upper = lane & off;
#pragma unroll
                for(int i = 0; i < n; i++)
                {
                    const float send = upper ? v[i] : v[i + n], keep = upper ? v[i + n] : v[i];
                    v[i] = keep + __shfl_xor_sync(0xffffffffu, send, off);
                }
                off /= 2;
            }
            float sum = v[0];
            for(; off; off /= 2)
                sum += __shfl_xor_sync(0xffffffffu, sum, off);
            return sum;
        }

        // E elements that a thread holds of a row: 16 bytes, two or one
        template <typename T, int E>
        struct alignas(E * sizeof(T)) Unit
        {
            T e[E];
        };

        // NT: tokens, rounded up; R classes at a time
        template <typename T, int E, int NT, int R, bool GRADIENT>
        __global__ void __launch_bounds__(kFewThreads, 2) few_tokens_kernel(const __grid_constant__ FewArgs a)
        {
            using U            = Unit<T, E>;
            constexpr int K    = NT * R;
            constexpr int Q    = E >= 4 ? 4 : E, PLANES = E / Q; // a unit's f32 sums lie as PLANES words of up to 16 bytes
            using F            = Unit<float, Q>;
            static_assert(K <= 32);
            extern __shared__ __align__(16) unsigned char smem[];
            __shared__ float red[2][kFewThreads / 32][K], probability[kFewThreads / 32][K];
            const int tid = int(threadIdx.x), lane = tid & 31, warp = tid >> 5, warps = int(blockDim.x) >> 5, threads = int(blockDim.x);
            const int units = int(a.units);
            U*        h     = reinterpret_cast<U*>(smem); // [NT][units]
            F*        dh    = reinterpret_cast<F*>(smem + (NT * units * sizeof(U) + 15) / 16 * 16); // [NT][PLANES][units]

            // every lane makes one of the batch's results: class lane / NT, token lane % NT
            const int  t = lane % NT, r = (lane / NT) % R;
            bool       live = t < a.T;
            int64_t    y = -1;
            float      lse = 0.f, g = 0.f;
            if(live)
            {
                y = a.targets[t];
                if(GRADIENT)
                {
                    live = counts(y, a.ignore, a.V);
                    if(live)
                        lse = a.lse[t], g = a.g[t] * a.alpha;
                    else if(y != a.ignore && blockIdx.x == 0 && tid < NT)
                        atomicExch_system(a.status, kStatusBadTarget);
                }
            }
            const uint32_t lives = __ballot_sync(0xffffffffu, live);
            for(int i = 0; i < NT; i++)
            {
                // rows of ignored tokens become zeros: what lies there must not reach dW through 0 * NaN
                const T* src = static_cast<const T*>(a.H) + (i < a.T ? rowOffset(a.rows, i) : 0);
                for(int64_t d = tid; d < int64_t(units) * E; d += threads)
                    reinterpret_cast<T*>(h + int64_t(i) * units)[d] = (lives >> i & 1) ? src[d * a.rows.elem] : narrow<T>(0.f);
                if(GRADIENT)
                    for(int64_t d = tid; d < int64_t(units) * E; d += threads)
                        reinterpret_cast<float*>(dh + int64_t(i) * PLANES * units)[d] = 0.f;
            }
            __syncthreads();

            float m = -INFINITY, s = 0.f;
            int   turn = 0;
            for(int64_t v0 = int64_t(blockIdx.x) * R; v0 < a.V; v0 += int64_t(gridDim.x) * R, turn ^= 1)
            {
                const T* row[R]; // classes past the last are read as the last and count for nothing
#pragma unroll
                for(int i = 0; i < R; i++)
                    row[i] = static_cast<const T*>(a.W) + min(v0 + i, a.V - 1) * a.wV;
                const int64_t next = int64_t(gridDim.x) * R;
                float         z[K];
#pragma unroll
                for(int i = 0; i < K; i++)
                    z[i] = 0.f;
                for(int u = tid; u < units; u += threads)
                {
                    U w[R];
#pragma unroll
                    for(int i = 0; i < R; i++)
                        w[i] = *reinterpret_cast<const U*>(row[i] + int64_t(u) * E);
                    // the next classes' rows are asked for now: a line by one lane
                    if((u * int(sizeof(U))) % 128 < int(sizeof(U)))
#pragma unroll
                        for(int i = 0; i < R; i++)
                            if(v0 + next + i < a.V)
                                asm volatile("prefetch.global.L2 [%0];" ::"l"(row[i] + next * a.wV + int64_t(u) * E));
#pragma unroll
                    for(int j = 0; j < NT; j++)
                    {
                        const U x = h[j * units + u];
#pragma unroll
                        for(int e = 0; e < E; e++)
#pragma unroll
                            for(int i = 0; i < R; i++)
                                z[i * NT + j] = fmaf(widen(w[i].e[e]), widen(x.e[e]), z[i * NT + j]);
                    }
                }
                const float sum = sumOverLanes<K>(z, lane);
                if(lane % (32 / K) == 0)
                    red[turn][warp][lane / (32 / K)] = sum;
                __syncthreads(); // of two buffers: the other one's readers have passed here
                const int64_t v = v0 + r;
                auto          logit = [&]() {
                    float x = 0.f;
                    for(int i = 0; i < warps; i++)
                        x += red[turn][i][lane % K];
                    return x * a.alpha;
                };
                if constexpr(!GRADIENT)
                {
                    if(warp == 0 && v < a.V) // the other warps go on to the next classes
                    {
                        const float x = logit();
                        joinSums(m, s, x, exp2f(x - reference(x))); // 1, or what an infinity stands for
                        if(v == y && live)
                            a.targetLogit[t] = x;
                    }
                }
                else
                {
                    if(lane < K)
                        probability[warp][lane] = live && v < a.V ? (expf(logit() - lse) - (v == y ? 1.f : 0.f)) * g : 0.f;
                    __syncwarp();
                    float p[K];
#pragma unroll
                    for(int i = 0; i < K; i++)
                        p[i] = probability[warp][i];
                    for(int u = tid; u < units; u += threads)
                    {
                        U w[R];
#pragma unroll
                        for(int i = 0; i < R; i++)
                            w[i] = *reinterpret_cast<const U*>(row[i] + int64_t(u) * E);
                        if(a.dH)
                        {
#pragma unroll
                            for(int j = 0; j < NT; j++)
#pragma unroll
                                for(int q = 0; q < PLANES; q++)
                                {
                                    F f = dh[(j * PLANES + q) * units + u];
#pragma unroll
                                    for(int e = 0; e < Q; e++)
#pragma unroll
                                        for(int i = 0; i < R; i++)
                                            f.e[e] = fmaf(p[i * NT + j], widen(w[i].e[q * Q + e]), f.e[e]);
                                    dh[(j * PLANES + q) * units + u] = f;
                                }
                        }
                        if(a.dW)
                        {
                            U x[NT];
#pragma unroll
                            for(int j = 0; j < NT; j++)
                                x[j] = h[j * units + u];
#pragma unroll
                            for(int i = 0; i < R; i++)
                                if(v0 + i < a.V)
                                {
                                    U o;
#pragma unroll
                                    for(int e = 0; e < E; e++)
                                    {
                                        float f = 0.f;
#pragma unroll
                                        for(int j = 0; j < NT; j++)
                                            f = fmaf(p[i * NT + j], widen(x[j].e[e]), f);
                                        o.e[e] = narrow<T>(f);
                                    }
                                    *reinterpret_cast<U*>(static_cast<T*>(a.dW) + (v0 + i) * a.wV + int64_t(u) * E) = o;
                                }
                        }
                    }
                }
            }
            if constexpr(!GRADIENT)
            {
                if(warp == 0)
                {
#pragma unroll
                    for(int off = NT; off < K; off *= 2) // the classes of a batch
                    {
                        const float m2 = __shfl_xor_sync(0xffffffffu, m, off), s2 = __shfl_xor_sync(0xffffffffu, s, off);
                        joinSums(m, s, m2, s2);
                    }
                    if(lane < NT && t < a.T)
                        a.part[int64_t(blockIdx.x) * a.T + t] = make_float2(m, s);
                }
            }
            else if(a.dH)
            {
                for(int j = 0; j < int(a.T); j++)
                    for(int q = 0; q < PLANES; q++)
                        for(int u = tid; u < units; u += threads)
                            *reinterpret_cast<F*>(a.dH + (int64_t(blockIdx.x) * a.T + j) * a.ldh + int64_t(u) * E + q * Q)
                                = dh[(j * PLANES + q) * units + u];
            }
        }

        // dH[token, column] = the blocks' sums, added in a fixed order; a warp takes every 32nd block
        template <typename T>
        __global__ void __launch_bounds__(1024) few_hidden_kernel(const float* __restrict__ part, int parts, int64_t T_, int64_t D, int64_t ldh,
                                                                  T* __restrict__ dH, const __grid_constant__ TokenRows rows,
                                                                  const int64_t* __restrict__ targets, int64_t ignore, int64_t V)
        {
            __shared__ float sums[32][33];
            const int        lane = int(threadIdx.x) & 31, warp = int(threadIdx.x) >> 5;
            const int64_t    d = int64_t(blockIdx.x) * 32 + lane, t = blockIdx.y;
            float            s = 0.f;
            if(d < D)
            {
#pragma unroll 8
                for(int i = warp; i < parts; i += 32)
                    s += part[(int64_t(i) * T_ + t) * ldh + d];
            }
            sums[lane][warp] = s;
            __syncthreads();
            s = sums[warp][lane];
            for(int off = 16; off; off /= 2)
                s += __shfl_xor_sync(0xffffffffu, s, off);
            const int64_t c = int64_t(blockIdx.x) * 32 + warp;
            if(lane == 0 && c < D) // an ignored token's is 0, whatever W holds
                dH[rowOffset(rows, t) + c * rows.elem] = narrow<T>(counts(targets[t], ignore, V) ? s : 0.f);
        }

        template <typename T, int E, int NT, int R>
        cudaError_t launchForm(const FewShape& f, const FewArgs& a, bool gradient, cudaStream_t stream)
        {
            const auto kernel = gradient ? few_tokens_kernel<T, E, NT, R, true> : few_tokens_kernel<T, E, NT, R, false>;
            if(cudaError_t e = ensureDynamicSmem(reinterpret_cast<const void*>(kernel), f.smem); e != cudaSuccess)
                return e;
            kernel<<<unsigned(f.blocks), unsigned(f.threads), size_t(f.smem), stream>>>(a);
            noteLaunch(gradient ? "cross_entropy_few_gradient" : "cross_entropy_few");
            return cudaGetLastError();
        }
        template <typename T, int E>
        cudaError_t launchTokens(const FewShape& f, const FewArgs& a, bool gradient, cudaStream_t stream)
        {
            switch(f.tokens)
            {
            case 1: return launchForm<T, E, 1, 8>(f, a, gradient, stream);
            case 2: return launchForm<T, E, 2, 8>(f, a, gradient, stream);
            case 4: return launchForm<T, E, 4, 8>(f, a, gradient, stream);
            default: return launchForm<T, E, 8, 4>(f, a, gradient, stream);
            }
        }
        template <typename T>
        cudaError_t launchUnits(const FewShape& f, const FewArgs& a, bool gradient, cudaStream_t stream)
        {
            constexpr int E = 16 / int(sizeof(T));
            return f.unit == E ? launchTokens<T, E>(f, a, gradient, stream)
                               : (f.unit == 2 ? launchTokens<T, 2>(f, a, gradient, stream) : launchTokens<T, 1>(f, a, gradient, stream));
        }
        cudaError_t launchFew(const FewShape& f, int type, const FewArgs& a, bool gradient, cudaStream_t stream)
        {
            return type == CUDA_R_32F ? launchUnits<float>(f, a, gradient, stream)
                                      : (type == CUDA_R_16F ? launchUnits<__half>(f, a, gradient, stream) : launchUnits<__nv_bfloat16>(f, a, gradient, stream));
        }
        FewArgs argsOf(const CrossEntropyPlan& p, const FewShape& f, const void* H, const TokenRows& rows, const void* W, const int64_t* targets,
                       float alpha, int* status)
        {
            FewArgs a{};
            a.H = H, a.W = W, a.rows = rows;
            a.T = p.T, a.V = p.V, a.wV = p.wV;
            a.units   = f.units;
            a.targets = targets, a.ignore = p.ignore, a.alpha = alpha, a.status = status;
            return a;
        }
    } // namespace

    cudaError_t launchFewLoss(const CrossEntropyPlan& p, const FewShape& f, const void* H, const TokenRows& rows, const void* W, const int64_t* targets,
                              float alpha, void* part, float* state, int* status, cudaStream_t stream)
    {
        FewArgs a     = argsOf(p, f, H, rows, W, targets, alpha, status);
        a.part        = static_cast<float2*>(part);
        a.targetLogit = state + 2 * p.T;
        return launchFew(f, p.type, a, false, stream);
    }

    cudaError_t launchFewGradient(const CrossEntropyPlan& p, const FewShape& f, const void* H, const TokenRows& rows, const void* W,
                                  const int64_t* targets, const float* lse, const float* g, float alpha, float* part, void* dH, void* dW, int* status,
                                  cudaStream_t stream)
    {
        FewArgs a = argsOf(p, f, H, rows, W, targets, alpha, status);
        a.lse = lse, a.g = g;
        a.dW  = dW;
        a.dH  = dH ? part : nullptr;
        a.ldh = f.ldh;
        if(cudaError_t e = launchFew(f, p.type, a, true, stream); e != cudaSuccess || !dH)
            return e;
        const dim3 grid(unsigned((p.D + 31) / 32), unsigned(p.T));
        if(p.type == CUDA_R_32F)
            few_hidden_kernel<float><<<grid, 1024, 0, stream>>>(part, f.blocks, p.T, p.D, f.ldh, (float*)dH, rows, targets, p.ignore, p.V);
        else if(p.type == CUDA_R_16F)
            few_hidden_kernel<__half><<<grid, 1024, 0, stream>>>(part, f.blocks, p.T, p.D, f.ldh, (__half*)dH, rows, targets, p.ignore, p.V);
        else
            few_hidden_kernel<__nv_bfloat16><<<grid, 1024, 0, stream>>>(part, f.blocks, p.T, p.D, f.ldh, (__nv_bfloat16*)dH, rows, targets, p.ignore, p.V);
        noteLaunch("cross_entropy_few_hidden");
        return cudaGetLastError();
    }
} // namespace htb
