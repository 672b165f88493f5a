// Block quantisation: f16 / bf16 / f32 -> e4m3 / e5m2 with one f32 scale for each block of 128 elements of a mode, or of
// 128 x 128 elements of two modes, in any order of the result's modes (a permutation in the same pass).
//
//   a = max(max |A| over the block, 2^-100)   S = q / q' with q = a, q' = 448 (e4m3) or 57344 (e5m2), rounded to f32
//   R = q' / a rounded to f32                 Q = the 8-bit number nearest to A * R, ties to even
//
// The floor keeps R finite: a block of zeros gets the scale of the floor and quantises to zeros. A block that holds a NaN
// gets the scale NaN; one that holds an infinity the scale infinity: either way all of it is NaN once multiplied out.
//
// ONE rounding. A * R rounded to f32 and then to 8 bits would round twice: an f32 product can land exactly on the border
// between two 8-bit numbers although the product itself lies beside it. The product is therefore rounded to f32 "to odd":
// truncated, and its last bit set when the truncation was not exact. A number rounded to odd at 24 bits rounds to 4 bits or
// fewer as the number itself does.
//
// Bound by memory: each element is read once and written once. 16384 x 8192 bf16 in blocks along rows takes 76 to 80 us (5.1 to 5.4
// TB/s; at the copy rate it would be 62), other blocks and orders of that size 85 to 101 (4.0 to 4.8: about ten instructions
// an element), f32 137 (4.9); 8192 x 4096 f32 in other blocks and orders 36 to 37 (4.5 to 4.7). Smaller tensors have fewer
// tiles in flight: 5001 x 4104 bf16 in blocks along columns, turned, 19 us (3.2 TB/s). One token of 4096 takes 2.7 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

#include "kernels.hpp"
#include "scaled.hpp"

namespace htb
{
    namespace
    {
        constexpr int   kTile    = 128; // columns of a tile; rows too unless the blocks are rows and the order is kept
        constexpr int   kThreads = 256; // 16 threads along a row of the tile, eight columns each, times 16 groups of rows
        constexpr float kFloor   = 7.88860905221011805411728565282787e-31f; // 2^-100

        __device__ __forceinline__ float maxNan(float a, float b)
        {
            float r;
            asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
            return r;
        }
        // Eight elements as they lie in memory: four words of 16-bit pairs, or eight f32 words.
        template <typename T>
        struct Eight
        {
            static constexpr int W = int(sizeof(T)) * 2;
            uint32_t             w[W];

            __device__ __forceinline__ float2 pair(int j) const // elements 2 j, 2 j + 1
            {
                if constexpr(sizeof(T) == 4)
                    return make_float2(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1]));
                else if constexpr(std::is_same<T, __nv_bfloat16>::value)
                    return make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
                else
                    return __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
            }
            __device__ __forceinline__ float at(int j) const
            {
                const float2 f = pair(j >> 1);
                return (j & 1) ? f.y : f.x;
            }
            // the largest magnitude (NaN if there is one): 16-bit numbers two in an instruction
            __device__ __forceinline__ float top() const
            {
                if constexpr(sizeof(T) == 4)
                {
                    float m = fabsf(__uint_as_float(w[0]));
#pragma unroll
                    for(int j = 1; j < 8; j++)
                        m = maxNan(m, fabsf(__uint_as_float(w[j])));
                    return m;
                }
                else
                {
                    using T2 = typename std::conditional<std::is_same<T, __nv_bfloat16>::value, __nv_bfloat162, __half2>::type;
                    T2 m     = __habs2(*reinterpret_cast<const T2*>(&w[0]));
#pragma unroll
                    for(int j = 1; j < 4; j++)
                        m = __hmax2_nan(m, __habs2(*reinterpret_cast<const T2*>(&w[j])));
                    return maxNan(__low2float(m), __high2float(m));
                }
            }
            // the same for each of the eight columns over N rows
            template <int N>
            static __device__ __forceinline__ void tops(const Eight (&v)[N], float (&m)[8])
            {
                if constexpr(sizeof(T) == 4)
                {
#pragma unroll
                    for(int j = 0; j < 8; j++)
                    {
                        m[j] = fabsf(v[0].at(j));
#pragma unroll
                        for(int i = 1; i < N; i++)
                            m[j] = maxNan(m[j], fabsf(v[i].at(j)));
                    }
                }
                else
                {
                    using T2 = typename std::conditional<std::is_same<T, __nv_bfloat16>::value, __nv_bfloat162, __half2>::type;
#pragma unroll
                    for(int j = 0; j < 4; j++)
                    {
                        T2 t = __habs2(*reinterpret_cast<const T2*>(&v[0].w[j]));
#pragma unroll
                        for(int i = 1; i < N; i++)
                            t = __hmax2_nan(t, __habs2(*reinterpret_cast<const T2*>(&v[i].w[j])));
                        m[2 * j]     = __low2float(t);
                        m[2 * j + 1] = __high2float(t);
                    }
                }
            }
        };
        // 16 bytes of elements `stride` apart, zeros from element n on. Out of line: the tiles at the edges take it, and unrolled
        // into every row of a tile it cost the registers that keep loads in flight.
        template <typename T>
        __device__ __noinline__ uint4 gather(const T* src, int n, int64_t stride)
        {
            constexpr int N = 16 / int(sizeof(T));
            __align__(16) T e[N];
#pragma unroll
            for(int j = 0; j < N; j++)
                e[j] = j < n ? src[j * stride] : T(0.f);
            return *reinterpret_cast<const uint4*>(e);
        }
        __device__ __noinline__ void scatter(unsigned char* dst, uint2 w, int n, int64_t stride)
        {
            for(int j = 0; j < n; j++)
                dst[j * stride] = (unsigned char)((j < 4 ? w.x : w.y) >> (8 * (j & 3)));
        }

        // a * r rounded to odd. Exact products matter only where they lie on a border between two 8-bit numbers, which has at most
        // five significant bits: r is then one of at most five bits itself (r = border / a is a 24-bit number only if a's odd
        // part divides the border's). For a 16-bit a and such an r the product is exact; for any other r the last bit may
        // always be set. So the bit depends on r alone: bitFor(r). An f32 a takes the remainder.
        __device__ __forceinline__ uint32_t bitFor(float r)
        {
            return (__float_as_uint(r) & 0x7ffffu) ? 1u : 0u;
        }
        template <typename T>
        __device__ __forceinline__ float mulOdd(float a, float r, uint32_t bit)
        {
            const float p = __fmul_rz(a, r);
            if constexpr(sizeof(T) == 2)
                return __uint_as_float(__float_as_uint(p) | bit);
            else
                return __fmaf_rn(a, r, -p) != 0.f ? __uint_as_float(__float_as_uint(p) | 1u) : p;
        }
        template <bool E5M2>
        __device__ __forceinline__ uint32_t pair8(float lo, float hi)
        {
            return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, E5M2 ? __NV_E5M2 : __NV_E4M3);
        }

        struct QuantArgs
        {
            QuantPlan p;
            int64_t   tilesR, tilesC;
            int       vecStore; // the result's runs are aligned: 8- and 16-byte stores
        };

        enum BlockForm : int
        {
            BLOCK_ROW  = 0, // 1 x 128
            BLOCK_COL  = 1, // 128 x 1
            BLOCK_BOTH = 2 // 128 x 128
        };

        __host__ __device__ constexpr int rowsPerThread(int form, bool trans, int size)
        {
            return (form == BLOCK_ROW && !trans && size == 4) ? 4 : 8;
        }
        // resident blocks that the registers are limited for: 32 or 64 of a thread's hold elements
        __host__ __device__ constexpr int blocksPerSm(int form, bool trans, int size)
        {
            return (form == BLOCK_ROW && !trans) ? 4 : (size == 2 ? 3 : 2);
        }

        // One tile of P * 16 rows and 128 columns at a time. Thread (tx, ty) holds columns tx * 8 .. + 7 of rows
        // ty * P .. + P - 1 in registers, so A is read once (and as it is: 16-bit elements take half the registers, which is
        // what keeps enough loads in flight); a row's maximum is a shuffle over 16 lanes, a column's goes
        // through shared memory. VEC: rows of A are read as 16-byte words. TRANS: the result is contiguous along A's
        // rows' mode: the bytes pass through shared memory, 8 rows at a time, in units of 8 bytes whose place in a column
        // is XORed with the thread's tx so that the 16 threads of a row write to 16 different pairs of banks.
        template <typename T, int FORM, bool TRANS, bool VEC, bool E5M2>
        __global__ void __launch_bounds__(kThreads, blocksPerSm(FORM, TRANS, sizeof(T)))
            block_quantize_kernel(const T* __restrict__ A, unsigned char* __restrict__ Q, float* __restrict__ S, const __grid_constant__ QuantArgs a)
        {
            constexpr int   P    = rowsPerThread(FORM, TRANS, sizeof(T));
            constexpr float kMax = E5M2 ? 57344.f : 448.f;
            const QuantPlan& p   = a.p;
            const int        tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
            __shared__ float part[FORM == BLOCK_ROW ? 1 : (FORM == BLOCK_COL ? 16 * kTile : 16)];
            __shared__ __align__(16) unsigned char turn[TRANS ? kTile * kTile : 16];

            // tiles by the grid's three dimensions (decoding a running number takes longer than the rest)
#pragma unroll 1
            for(int64_t b = blockIdx.z; b < p.batch; b += gridDim.z)
#pragma unroll 1
            for(int64_t tc = blockIdx.y; tc < a.tilesC; tc += gridDim.y)
#pragma unroll 1
            for(int64_t tr = blockIdx.x; tr < a.tilesR; tr += gridDim.x)
            {
                const int64_t r0 = tr * (16 * P) + ty * P, c0 = tc * kTile + tx * 8;
                const int     nr = int(min(int64_t(P), p.rows - r0)), nc = int(min(int64_t(8), p.cols - c0)); // may be negative
                const T*      src = A + b * p.aB + r0 * p.aR + c0 * p.aC;
                Eight<T>      v[P];
#pragma unroll
                for(int i = 0; i < P; i++, src += p.aR)
                {
                    constexpr int N = 16 / int(sizeof(T));
#pragma unroll
                    for(int w = 0; w < Eight<T>::W / 4; w++) // 16-byte words
                    {
                        uint4 q = make_uint4(0, 0, 0, 0);
                        if(VEC && i < nr && nc == 8)
                            q = __ldg(reinterpret_cast<const uint4*>(src) + w);
                        else if(i < nr && nc > w * N)
                            q = gather<T>(src + w * N * p.aC, nc - w * N, p.aC);
                        v[i].w[4 * w] = q.x, v[i].w[4 * w + 1] = q.y, v[i].w[4 * w + 2] = q.z, v[i].w[4 * w + 3] = q.w;
                    }
                }

                // factors of the thread's elements: one per row, one per column, or one
                float scale[FORM == BLOCK_ROW ? P : (FORM == BLOCK_COL ? 8 : 1)];
                if constexpr(FORM == BLOCK_ROW)
                {
                    // the 16 lanes of a row share its divisions: lane i < P makes the factor of row i, lane P + i its scale
                    float mine = 0.f;
#pragma unroll
                    for(int i = 0; i < P; i++)
                    {
                        float m = maxNan(kFloor, v[i].top());
#pragma unroll
                        for(int s = 8; s >= 1; s >>= 1)
                            m = maxNan(m, __shfl_xor_sync(0xffffffffu, m, s));
                        if((tx & (P - 1)) == i)
                            mine = m;
                    }
                    const float d = tx < P ? __fdiv_rn(kMax, mine) : __fdiv_rn(mine, kMax);
#pragma unroll
                    for(int i = 0; i < P; i++)
                        scale[i] = __shfl_sync(0xffffffffu, d, int(threadIdx.x & 16) + i);
                    if(tx >= P && tx < 2 * P && tx - P < nr)
                        S[b * p.sB + (r0 + tx - P) * p.sR + tc * p.sC] = d;
                }
                else if constexpr(FORM == BLOCK_COL)
                {
                    float m[8];
                    Eight<T>::template tops<P>(v, m);
#pragma unroll
                    for(int j = 0; j < 8; j++)
                        m[j] = maxNan(m[j], kFloor);
                    __syncthreads(); // the maxima of the tile before have been read
#pragma unroll
                    for(int j = 0; j < 8; j += 4)
                        *reinterpret_cast<float4*>(&part[ty * kTile + tx * 8 + j]) = make_float4(m[j], m[j + 1], m[j + 2], m[j + 3]);
                    __syncthreads();
                    if(threadIdx.x < kTile)
                    {
                        float top = part[threadIdx.x];
#pragma unroll
                        for(int g = 1; g < 16; g++)
                            top = maxNan(top, part[g * kTile + threadIdx.x]);
                        const int64_t c = tc * kTile + threadIdx.x;
                        if(c < p.cols)
                            S[b * p.sB + tr * p.sR + c * p.sC] = __fdiv_rn(top, kMax);
                        part[threadIdx.x] = __fdiv_rn(kMax, top);
                    }
                    __syncthreads();
#pragma unroll
                    for(int j = 0; j < 8; j++)
                        scale[j] = part[tx * 8 + j];
                }
                else
                {
                    float m = kFloor;
#pragma unroll
                    for(int i = 0; i < P; i++)
                        m = maxNan(m, v[i].top());
#pragma unroll
                    for(int s = 16; s >= 1; s >>= 1)
                        m = maxNan(m, __shfl_xor_sync(0xffffffffu, m, s));
                    __syncthreads();
                    if((threadIdx.x & 31) == 0)
                        part[threadIdx.x >> 5] = m;
                    __syncthreads();
#pragma unroll
                    for(int g = 0; g < kThreads / 32; g++)
                        m = maxNan(m, part[g]);
                    scale[0] = __fdiv_rn(kMax, m);
                    if(threadIdx.x == 0)
                        S[b * p.sB + tr * p.sR + tc * p.sC] = __fdiv_rn(m, kMax);
                }
                auto     factor = [&](int i, int j) { return scale[FORM == BLOCK_ROW ? i : (FORM == BLOCK_COL ? j : 0)]; };
                uint32_t bits[FORM == BLOCK_ROW ? P : (FORM == BLOCK_COL ? 8 : 1)];
#pragma unroll
                for(int k = 0; k < int(sizeof(bits) / 4); k++)
                    bits[k] = bitFor(scale[k]);
                auto odd = [&](float x, int i, int j) {
                    return mulOdd<T>(x, factor(i, j), bits[FORM == BLOCK_ROW ? i : (FORM == BLOCK_COL ? j : 0)]);
                };

                if constexpr(!TRANS)
                {
                    unsigned char* dst = Q + b * p.qB + r0 * p.qR + c0 * p.qC;
#pragma unroll
                    for(int i = 0; i < P; i++, dst += p.qR)
                    {
                        if(i >= nr || nc <= 0)
                            continue;
                        uint32_t w[4];
#pragma unroll
                        for(int j = 0; j < 4; j++)
                        {
                            const float2 f = v[i].pair(j);
                            w[j]           = pair8<E5M2>(odd(f.x, i, 2 * j), odd(f.y, i, 2 * j + 1));
                        }
                        const uint2 bytes = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
                        if(a.vecStore && nc == 8)
                            *reinterpret_cast<uint2*>(dst) = bytes;
                        else
                            scatter(dst, bytes, nc, p.qC);
                    }
                }
                else
                {
                    __syncthreads(); // the tile before has been written out
#pragma unroll
                    for(int j = 0; j < 8; j++)
                    {
                        uint32_t w[4];
#pragma unroll
                        for(int i = 0; i < 4; i++)
                            w[i] = pair8<E5M2>(odd(v[2 * i].at(j), 2 * i, j), odd(v[2 * i + 1].at(j), 2 * i + 1, j));
                        *reinterpret_cast<uint2*>(&turn[(tx * 8 + j) * kTile + ((ty ^ tx) << 3)])
                            = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
                    }
                    __syncthreads();
                    // eight threads write the 128 rows of a column, 16 bytes each
                    const int     unit = int(threadIdx.x & 7) * 2;
                    const int64_t row  = tr * kTile + unit * 8;
                    const int     left = int(min(int64_t(16), p.rows - row));
#pragma unroll
                    for(int k = 0; k < kTile / 32; k++)
                    {
                        const int     col = k * 32 + int(threadIdx.x >> 3);
                        const int64_t c   = tc * kTile + col;
                        if(c >= p.cols || left <= 0)
                            continue;
                        const int x = col >> 3;
                        uint4     w = *reinterpret_cast<const uint4*>(&turn[col * kTile + (((unit ^ x) & ~1) << 3)]);
                        if(x & 1)
                            w = make_uint4(w.z, w.w, w.x, w.y);
                        unsigned char* dst = Q + b * p.qB + c * p.qC + row * p.qR;
                        if(a.vecStore && left == 16)
                            *reinterpret_cast<uint4*>(dst) = w;
                        else
                        {
                            scatter(dst, make_uint2(w.x, w.y), min(left, 8), p.qR);
                            scatter(dst + 8 * p.qR, make_uint2(w.z, w.w), left - 8, p.qR);
                        }
                    }
                }
            }
        }

        template <typename T, int FORM, bool TRANS>
        cudaError_t launchForm(const QuantArgs& a, bool vec, dim3 grid, const void* A, void* Q, float* S, cudaStream_t stream)
        {
            const bool e5m2 = a.p.typeQ == CUDA_R_8F_E5M2;
            auto       kernel = vec ? (e5m2 ? block_quantize_kernel<T, FORM, TRANS, true, true> : block_quantize_kernel<T, FORM, TRANS, true, false>)
                                    : (e5m2 ? block_quantize_kernel<T, FORM, TRANS, false, true>
                                            : block_quantize_kernel<T, FORM, TRANS, false, false>);
            kernel<<<grid, kThreads, 0, stream>>>((const T*)A, (unsigned char*)Q, S, a);
            const cudaError_t e = cudaGetLastError();
            if(e == cudaSuccess)
                noteLaunch("block_quantize");
            return e;
        }

        template <typename T>
        cudaError_t launchTyped(const QuantPlan& p, const void* A, void* Q, float* S, cudaStream_t stream)
        {
            const int  form  = p.blockR > 1 ? (p.blockC > 1 ? BLOCK_BOTH : BLOCK_COL) : BLOCK_ROW;
            const bool trans = p.qR == 1 && p.qC != 1; // else along the columns, or along neither
            // 16-byte loads: rows contiguous, and every row starts at a multiple of 16 bytes
            const int64_t words = 16 / int64_t(sizeof(T));
            const bool    vec   = p.aC == 1 && p.aR % words == 0 && p.aB % words == 0 && (uintptr_t(A) & 15) == 0;
            const int64_t unit  = trans ? 16 : 8;
            QuantArgs     a;
            a.p        = p;
            const int64_t tileRows = 16 * rowsPerThread(form, trans, sizeof(T));
            a.tilesR               = (p.rows + tileRows - 1) / tileRows;
            a.tilesC               = (p.cols + kTile - 1) / kTile;
            a.vecStore = (trans ? p.qR : p.qC) == 1 && (trans ? p.qC : p.qR) % unit == 0 && p.qB % unit == 0 && uintptr_t(Q) % unit == 0;
            const dim3 grid(unsigned(std::min<int64_t>(a.tilesR, 0x7fffffff)), unsigned(std::min<int64_t>(a.tilesC, 65535)),
                            unsigned(std::min<int64_t>(p.batch, 65535)));
            if(form == BLOCK_ROW)
                return trans ? launchForm<T, BLOCK_ROW, true>(a, vec, grid, A, Q, S, stream)
                             : launchForm<T, BLOCK_ROW, false>(a, vec, grid, A, Q, S, stream);
            if(form == BLOCK_COL)
                return trans ? launchForm<T, BLOCK_COL, true>(a, vec, grid, A, Q, S, stream)
                             : launchForm<T, BLOCK_COL, false>(a, vec, grid, A, Q, S, stream);
            return trans ? launchForm<T, BLOCK_BOTH, true>(a, vec, grid, A, Q, S, stream)
                         : launchForm<T, BLOCK_BOTH, false>(a, vec, grid, A, Q, S, stream);
        }
    } // namespace

    cudaError_t launchQuantize(const QuantPlan& p, const void* A, void* Q, float* S, cudaStream_t stream)
    {
        switch(p.typeA)
        {
        case CUDA_R_32F: return launchTyped<float>(p, A, Q, S, stream);
        case CUDA_R_16F: return launchTyped<__half>(p, A, Q, S, stream);
        case CUDA_R_16BF: return launchTyped<__nv_bfloat16>(p, A, Q, S, stream);
        }
        return cudaErrorNotSupported;
    }
} // namespace htb
