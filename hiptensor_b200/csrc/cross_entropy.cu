// Kernels of the linear cross entropy around the library's contractions.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "accumulate.cuh"
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
                                         T* __restrict__ X2, const int64_t* __restrict__ targets, int64_t ignore, int64_t V, int* status, bool twice)
        {
            for(int64_t r = blockIdx.x; r < count; r += gridDim.x)
            {
                const bool    live = !targets || counts(targets[r], ignore, V);
                const T*      src  = X + rowOffset(rows, r);
                if(!live && targets[r] != ignore && threadIdx.x == 0)
                    atomicExch_system(status, kStatusBadTarget);
                for(int64_t c = threadIdx.x; c < ld; c += blockDim.x)
                {
                    const T x      = (live && c < cols) ? src[c * rows.elem] : narrow<T>(0.f);
                    X2[r * ld + c] = x;
                    if(twice)
                        X2[(count + r) * ld + c] = x;
                }
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

        __global__ void probabilities_kernel(float* z, int64_t ldz, int64_t T, int64_t v0, int64_t count, int64_t V, int64_t ignore,
                                             const int64_t* __restrict__ targets, const float* __restrict__ lse, const float* __restrict__ g,
                                             float alpha)
        {
            for(int64_t t = blockIdx.x; t < T; t += gridDim.x)
            {
                const int64_t target = targets[t];
                const bool    live   = counts(target, ignore, V);
                const float   l = lse[t], f = g[t] * alpha;
                for(int64_t v = threadIdx.x; v < count; v += blockDim.x)
                {
                    float p = expf(z[t * ldz + v] - l);
                    if(v0 + v == target)
                        p -= 1.f;
                    z[t * ldz + v] = live ? p * f : 0.f;
                }
            }
        }

        template <typename T>
        __global__ void store_rows_kernel(const float* __restrict__ X, int64_t ldx, int64_t count, int64_t cols, const float* __restrict__ scale,
                                          T* __restrict__ Y, const __grid_constant__ TokenRows rows, const __grid_constant__ TargetRest rest, int parts)
        {
            const float f = scale ? scale[1] : 1.f;
            for(int64_t r = blockIdx.x; r < count; r += gridDim.x)
            {
                T*       dst = Y + rowOffset(rows, r);
                const T* w   = nullptr; // the target's row of W, times what rounding took from its entry of P
                float    e   = 0.f;
                if(rest.rest)
                {
                    const int64_t target = rest.targets[r];
                    if(counts(target, rest.ignore, rest.V))
                    {
                        w = static_cast<const T*>(rest.W) + target * rest.wV;
                        e = rest.rest[r];
                    }
                }
                for(int64_t c = threadIdx.x; c < cols; c += blockDim.x)
                {
                    float x = 0.f;
                    for(int i = 0; i < parts; i++)
                        x += X[(int64_t(i) * count + r) * ldx + c];
                    if(w)
                        x = fmaf(e, widen(w[c * rest.wD]), x);
                    dst[c * rows.elem] = narrow<T>(x * f);
                }
            }
        }

        // ------------------------------------------------------------------ f16 / bf16: logits that stay on the chip
        constexpr float kLog2e = 1.4426950408889634f;

        __device__ __forceinline__ float maxNan(float a, float b)
        {
            float r;
            asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
            return r;
        }
        // the value that exponents are taken relative to: 0 where a maximum is infinite
        __device__ __forceinline__ float reference(float m)
        {
            return fabsf(m) == INFINITY ? 0.f : m;
        }

        struct HeadArgs
        {
            int64_t        T, n, v0, V; // tokens; classes of this piece, its first class, all classes
            int64_t        ignore;
            const int64_t* targets;
            float          alpha;
            // forward: partial (maximum, sum) of 128 classes each, [classes][T], in powers of two; target logits
            float2* part;
            float*  targetLogit;
            // gradient
            const float *lse, *g, *scale;
            float*       rest; // what rounding took from the target's entry of P
            CUtensorMap  mapP, mapLow;
        };

        // Common to both: the sums of a chunk of up to 1024 elements are added to the running ones with rounding (the
        // accumulation inside a chunk truncates; sums over 4096 elements in one chunk were short by 3.6e-6 of their value).
        template <int TN>
        struct HeadSums
        {
            static constexpr int COLS = TN / 2;
            uint64_t             acc[COLS / 2];

            template <class Release>
            __device__ __forceinline__ void addSums(uint32_t taddr, bool first, Release release)
            {
                constexpr int CL = COLS < 32 ? COLS : 32;
                uint32_t      v0[CL], v1[CL];
                auto          put = [&](const uint32_t(&v)[CL], int c) {
#pragma unroll
                    for(int j = 0; j < CL; j += 2)
                        acc[(c + j) / 2] = first ? pack2(v[j], v[j + 1]) : add2(pack2(v[j], v[j + 1]), acc[(c + j) / 2]);
                };
                tmemLoad<CL>(taddr, v0);
                if constexpr(CL < COLS)
                    tmemLoad<CL>(taddr + CL, v1);
#pragma unroll
                for(int c = 0; c < COLS; c += 2 * CL)
                {
                    tmemWait();
                    if(c + 2 * CL >= COLS)
                        release();
                    put(v0, c);
                    if(c + 2 * CL < COLS)
                        tmemLoad<CL>(taddr + c + 2 * CL, v0);
                    if(c + CL < COLS)
                        put(v1, c + CL);
                    if(c + 3 * CL < COLS)
                        tmemLoad<CL>(taddr + c + 3 * CL, v1);
                }
            }
            // sum j of this thread, j not known when compiling
            __device__ __forceinline__ float at(int j) const
            {
                float r = 0.f;
#pragma unroll
                for(int i = 0; i < COLS / 2; i++)
                {
                    const float2 f = unpack2(acc[i]);
                    r              = j == 2 * i ? f.x : (j == 2 * i + 1 ? f.y : r);
                }
                return r;
            }
        };

        // Loss: one pass over a tile's logits in registers, maximum then sum of powers of two; what leaves the SM are two
        // floats for 128 logits.
        struct LossEpi : HeadSums<256>
        {
            using Args                 = HeadArgs;
            using Sums                 = HeadSums<256>;
            static constexpr int kSide = 0;
            static constexpr bool kSplit = false;
            static constexpr int ROOM  = 0; // shared memory behind the stages
            const Args&          a;

            __device__ LossEpi(const Args& args, int, int, unsigned char*)
                : a(args)
            {
            }
            __device__ __forceinline__ void begin() {}
            template <class Release>
            __device__ __forceinline__ void add(uint32_t taddr, bool first, Release release)
            {
                Sums::addSums(taddr, first, release);
            }
            __device__ __forceinline__ void end(int64_t row, int64_t col)
            {
                if(row >= a.T || col >= a.n)
                    return;
                const int64_t t = a.targets[row] - a.v0 - col;
                if(t >= 0 && t < COLS && col + t < a.n)
                    a.targetLogit[row] = Sums::at(int(t)) * a.alpha;
                const float    c  = a.alpha * kLog2e;
                const uint64_t c2 = pack2(c, c);
                float          m  = -INFINITY;
                const int      n  = int(min(int64_t(COLS), a.n - col));
#pragma unroll
                for(int i = 0; i < COLS / 2; i++)
                {
                    acc[i]         = mul2(acc[i], c2);
                    const float2 f = unpack2(acc[i]);
                    if(n == COLS)
                        m = maxNan(maxNan(f.x, f.y), m);
                    else
                    {
                        const float x = 2 * i < n ? f.x : -INFINITY, y = 2 * i + 1 < n ? f.y : -INFINITY;
                        acc[i]        = pack2(x, y);
                        m             = maxNan(maxNan(x, y), m);
                    }
                }
                const float    ref  = reference(m);
                const uint64_t less = pack2(-ref, -ref);
                uint64_t       sum[4] = {0, 0, 0, 0}; // sums of a quarter each: short chains, and rounding errors of short sums
#pragma unroll
                for(int i = 0; i < COLS / 2; i++)
                {
                    const float2 f = unpack2(add2(acc[i], less));
                    sum[i & 3]     = add2(sum[i & 3], pack2(exp2f(f.x), exp2f(f.y)));
                }
                const float2 s = unpack2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])));
                a.part[(col / COLS) * a.T + row] = make_float2(m, s.x + s.y);
            }
            __device__ __forceinline__ void leave() {}
        };

        // Gradient: P = (exp(z - lse) - [class is the target]) * g * alpha, rounded to the operands' type for the two products
        // that follow (the products' sums are f32; a rounding of 2^-9 or 2^-12 of each entry is about what the rounding of
        // the results to the same type costs). The target's entry outweighs the others: what its rounding takes is kept and
        // added to dH in f32.
        // PARTS = 2: P as a sum of two numbers of the type, what rounding took from every entry goes to mapLow.
        template <typename TP, int PARTS>
        struct ProbabilityEpi : HeadSums<256>
        {
            using Args                 = HeadArgs;
            using Sums                 = HeadSums<256>;
            static constexpr int kSide = 0;
            static constexpr bool kSplit = false;
            static constexpr int ROUND = 64; // columns of a slot: rows of 128 bytes
            static constexpr int SLOTS = 1;
            static constexpr int ROOM  = 8 * SLOTS * 4096;
            const Args&          a;
            const int            lane;
            const uint32_t       slot;
            int                  stores;

            __device__ ProbabilityEpi(const Args& args, int w, int l, unsigned char* smem)
                : a(args)
                , lane(l)
                , slot(smemAddr(smem) + uint32_t(w * SLOTS * 4096))
                , stores(0)
            {
            }
            __device__ __forceinline__ void begin() {}
            template <class Release>
            __device__ __forceinline__ void add(uint32_t taddr, bool first, Release release)
            {
                Sums::addSums(taddr, first, release);
            }
            __device__ __forceinline__ void end(int64_t row, int64_t col)
            {
                int64_t target = -1;
                float   l = 0.f, f = 0.f;
                bool    live = false;
                if(row < a.T)
                {
                    target = a.targets[row];
                    live   = counts(target, a.ignore, a.V);
                    if(live)
                    {
                        l = a.lse[row] * kLog2e;
                        f = a.g[row] * a.alpha * (a.scale ? a.scale[0] : 1.f);
                    }
                }
                const float    c  = a.alpha * kLog2e;
                const uint64_t c2 = pack2(c, c), l2 = pack2(-l, -l);
                const int64_t  t = live ? target - a.v0 - col : -1;
                if(t >= 0 && t < COLS)
                {
                    const float x = unpack2(fma2(pack2(Sums::at(int(t)), 0.f), c2, l2)).x;
                    const float p = (exp2f(x) - 1.f) * f;
                    a.rest[row]   = p - widen(narrow<TP>(p));
                }
#pragma unroll 1
                for(int low = 0; low < PARTS; low++)
#pragma unroll
                    for(int r = 0; r < COLS; r += ROUND)
                    {
                        const uint32_t at = slot + uint32_t((stores % SLOTS) * 4096);
                        if(lane == 0)
                            asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(SLOTS - 1) : "memory"); // the slot's last store has read it
                        __syncwarp();
                        stores++;
#pragma unroll
                        for(int u = 0; u < ROUND / 8; u++)
                        {
                            uint32_t q[4];
#pragma unroll
                            for(int j = 0; j < 4; j++)
                            {
                                const int    k = r + 8 * u + 2 * j;
                                const float2 x = unpack2(fma2(acc[k / 2], c2, l2));
                                float        p0 = exp2f(x.x), p1 = exp2f(x.y);
                                if(t == k)
                                    p0 -= 1.f;
                                if(t == k + 1)
                                    p1 -= 1.f;
                                p0 = live ? p0 * f : 0.f;
                                p1 = live ? p1 * f : 0.f;
                                TP lo = narrow<TP>(p0), hi = narrow<TP>(p1);
                                if(low)
                                {
                                    lo = narrow<TP>(p0 - widen(lo));
                                    hi = narrow<TP>(p1 - widen(hi));
                                }
                                q[j] = uint32_t(reinterpret_cast<const unsigned short&>(lo))
                                       | (uint32_t(reinterpret_cast<const unsigned short&>(hi)) << 16);
                            }
                            // 16-byte units permuted as the map's swizzle has them
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + uint32_t(lane * 128 + ((u ^ (lane & 7)) << 4))), "r"(q[0]), "r"(q[1]), "r"(q[2]), "r"(q[3])
                                         : "memory");
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if(lane == 0)
                        {
                            // a block that begins outside P has nothing to store (one that ends outside is clipped)
                            if(row < a.T && col + r < a.n)
                                asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(low ? &a.mapLow : &a.mapP),
                                             "r"(at), "r"(int(col + r)), "r"(int(row))
                                             : "memory");
                            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                        }
                    }
            }
            __device__ __forceinline__ void leave()
            {
                if(lane == 0)
                    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            }
        };

        // dW = P^T H of a piece: the sums (times scale[1]) rounded once, out by bulk stores while the next tile is summed.
        struct WeightArgs
        {
            int64_t      rows, cols;
            const float* scale;
            CUtensorMap  mapD;
        };
        template <typename TD>
        struct WeightEpi : HeadSums<256>
        {
            using Args                   = WeightArgs;
            static constexpr int  kSide  = 0;
            static constexpr bool kSplit = false;
            static constexpr int  SLOTS  = 1;
            static constexpr int  ROOM   = 8 * SLOTS * 4096;
            const Args&           a;
            const int             lane;
            const uint32_t        slot;
            int                   stores;

            __device__ WeightEpi(const Args& args, int w, int l, unsigned char* smem)
                : a(args)
                , lane(l)
                , slot(smemAddr(smem) + uint32_t(w * SLOTS * 4096))
                , stores(0)
            {
            }
            __device__ __forceinline__ void begin() {}
            template <class Release>
            __device__ __forceinline__ void add(uint32_t taddr, bool first, Release release)
            {
                addSums(taddr, first, release);
            }
            __device__ __forceinline__ void end(int64_t row, int64_t col)
            {
                const float    f  = a.scale ? a.scale[1] : 1.f;
                const uint64_t f2 = pack2(f, f);
#pragma unroll
                for(int r = 0; r < COLS; r += 64)
                {
                    const uint32_t at = slot + uint32_t((stores % SLOTS) * 4096);
                    if(lane == 0)
                        asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(SLOTS - 1) : "memory"); // the slot's last store has read it
                    __syncwarp();
                    stores++;
#pragma unroll
                    for(int u = 0; u < 8; u++)
                    {
                        uint32_t q[4];
#pragma unroll
                        for(int j = 0; j < 4; j++)
                        {
                            const float2 x = unpack2(mul2(acc[(r + 8 * u + 2 * j) / 2], f2));
                            const TD     lo = narrow<TD>(x.x), hi = narrow<TD>(x.y);
                            q[j] = uint32_t(reinterpret_cast<const unsigned short&>(lo)) | (uint32_t(reinterpret_cast<const unsigned short&>(hi)) << 16);
                        }
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + uint32_t(lane * 128 + ((u ^ (lane & 7)) << 4))),
                                     "r"(q[0]), "r"(q[1]), "r"(q[2]), "r"(q[3])
                                     : "memory");
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if(lane == 0)
                    {
                        if(row < a.rows && col + r < a.cols)
                            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(&a.mapD), "r"(at),
                                         "r"(int(col + r)), "r"(int(row))
                                         : "memory");
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                }
            }
            __device__ __forceinline__ void leave()
            {
                if(lane == 0)
                    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            }
        };

        // dH = P W over parts of the classes: f32 sums of every part, [part][T][ld]
        struct HiddenArgs
        {
            int64_t T, ld;
            int     tiles; // of 128 tokens: tile rows of a part
            float*  out;
            int     add; // to what the pieces before left there
        };
        struct HiddenEpi : HeadSums<256>
        {
            using Args                   = HiddenArgs;
            static constexpr int  kSide  = 0;
            static constexpr bool kSplit = false;
            static constexpr int  ROOM   = 0;
            const Args&           a;

            __device__ HiddenEpi(const Args& args, int, int, unsigned char*)
                : a(args)
            {
            }
            __device__ __forceinline__ void begin() {}
            template <class Release>
            __device__ __forceinline__ void add(uint32_t taddr, bool first, Release release)
            {
                addSums(taddr, first, release);
            }
            __device__ __forceinline__ void end(int64_t row, int64_t col)
            {
                const int64_t tile = row >> 7, part = tile / a.tiles;
                const int64_t t    = row - part * a.tiles * 128;
                if(t >= a.T)
                    return;
                float* out = a.out + (part * a.T + t) * a.ld + col; // ld is a multiple of eight
#pragma unroll
                for(int j = 0; j < COLS; j += 4)
                    if(col + j < a.ld)
                    {
                        const float2 x = unpack2(acc[j / 2]), y = unpack2(acc[j / 2 + 1]);
                        float4       v = make_float4(x.x, x.y, y.x, y.y);
                        if(a.add)
                        {
                            const float4 o = *reinterpret_cast<const float4*>(out + j);
                            v = make_float4(v.x + o.x, v.y + o.y, v.z + o.z, v.w + o.w);
                        }
                        *reinterpret_cast<float4*>(out + j) = v;
                    }
            }
            __device__ __forceinline__ void leave() {}
        };

        // Joins the partial maxima and sums of a piece, 32 tokens a block, a slice of the classes a warp (in the order of the
        // classes, so results are the same every time), with what the pieces before left; after the last piece the results.
        constexpr int kJoinWarps = 16;
        __global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(const float2* __restrict__ part, int64_t groups, int64_t T, float* state,
                                                                       bool first, bool last, int64_t V, int64_t ignore,
                                                                       const int64_t* __restrict__ targets, float* loss, float* lse, int* status)
        {
            __shared__ float2 mine[kJoinWarps][32];
            const int         lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
            const int64_t     t = int64_t(blockIdx.x) * 32 + lane;
            float             m = -INFINITY, s = 0.f;
            auto              join = [](float& m, float& s, float m2, float s2) {
                const float top = maxNan(m, m2), ref = reference(top);
                s = s * exp2f(reference(m) - ref) + s2 * exp2f(reference(m2) - ref);
                m = top;
            };
            if(t < T)
            {
                int64_t i = warp;
                for(; i + 3 * kJoinWarps < groups; i += 4 * kJoinWarps)
                {
                    float2 p[4]; // four loads on their way
#pragma unroll
                    for(int j = 0; j < 4; j++)
                        p[j] = part[(i + j * kJoinWarps) * T + t];
#pragma unroll
                    for(int j = 0; j < 4; j++)
                        join(m, s, p[j].x, p[j].y);
                }
                for(; i < groups; i += kJoinWarps)
                {
                    const float2 p = part[i * T + t];
                    join(m, s, p.x, p.y);
                }
            }
            mine[warp][lane] = make_float2(m, s);
            __syncthreads();
            if(warp != 0 || t >= T)
                return;
            for(int w = 1; w < kJoinWarps; w++)
                join(m, s, mine[w][lane].x, mine[w][lane].y);
            if(!first)
                join(m, s, state[t], state[T + t]);
            if(!last)
            {
                state[t]     = m;
                state[T + t] = s;
                return;
            }
            const float   l = (reference(m) + log2f(s)) * 0.6931471805599453f;
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

        bool encodeMatrix(PFN_encodeTiled encode, CUtensorMap* map, const void* base, int64_t cols, int64_t rows, int64_t ld, int boxCols, int boxRows,
                          CUtensorMapSwizzle swizzle)
        {
            cuuint64_t gdim[2] = {cuuint64_t(cols), cuuint64_t(rows)}, gstr[1] = {rows > 1 ? cuuint64_t(ld) * 2 : cuuint64_t((cols + 7) / 8 * 16)};
            cuuint32_t bx[2] = {cuuint32_t(boxCols), cuuint32_t(boxRows)}, estr[2] = {1, 1};
            return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(base), gdim, gstr, bx, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE)
                   == CUDA_SUCCESS;
        }

        template <class Epi, bool PAIR, int TN, bool XMN, bool YMN>
        cudaError_t launchAccumulate(const CUtensorMap& mapX, const CUtensorMap& mapY, const AccArgs& a, const typename Epi::Args& ea, int smCount,
                                     cudaStream_t stream, const char* name)
        {
            auto                     kernel = accumulate_kernel<Epi, PAIR, TN, false, XMN, YMN>;
            static const cudaError_t regs   = accCheckRegs((const void*)kernel, TN);
            if(regs != cudaSuccess)
                return regs;
            const size_t smem = size_t(a.stageBytes) + 1024 + Epi::ROOM;
            if(cudaError_t e = ensureDynamicSmem((const void*)kernel, int(smem)))
                return e;
            const int           csize = PAIR ? 2 : 1;
            cudaLaunchConfig_t  cfg{};
            cudaLaunchAttribute attr[2];
            attr[0].id                                         = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x                           = unsigned(csize);
            attr[0].val.clusterDim.y                           = 1;
            attr[0].val.clusterDim.z                           = 1;
            attr[1].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr[1].val.programmaticStreamSerializationAllowed = 1;
            cfg.gridDim          = dim3(unsigned(csize * std::min<int64_t>(int64_t(a.tilesM) * a.tilesN, (smCount > 0 ? smCount : 148) / csize)));
            cfg.blockDim         = dim3(kAccThreads);
            cfg.dynamicSmemBytes = smem;
            cfg.stream           = stream;
            cfg.attrs            = attr;
            cfg.numAttrs         = 2;
            cudaError_t e        = cudaLaunchKernelEx(&cfg, kernel, mapX, mapY, a, ea);
            if(e == cudaSuccess)
                noteLaunch(name);
            return e;
        }

        template <class Epi, bool PAIR>
        cudaError_t launchHeadForm(const HeadProduct& h, HeadArgs& ea, int smCount, int* status, cudaStream_t stream, const char* name)
        {
            PFN_encodeTiled encode = tensorMapEncoder();
            if(!encode)
                return cudaErrorNotSupported;
            constexpr int rows = PAIR ? 256 : 128, TN = 256;
            const int     xRows = PAIR ? 128 : int(std::min<int64_t>(128, (h.T + 7) / 8 * 8)); // no more rows of H than there are tokens
            const uint32_t stage = (uint32_t(xRows) + (PAIR ? 128u : uint32_t(TN))) * 128u, behind = uint32_t(128 - xRows) * 128u;
            CUtensorMap mapX, mapY;
            if(!encodeMatrix(encode, &mapX, h.H, h.D, h.T, h.ldh, 64, xRows, CU_TENSOR_MAP_SWIZZLE_128B)
               || !encodeMatrix(encode, &mapY, h.W, h.D, h.n, h.ldw, 64, PAIR ? 128 : TN, CU_TENSOR_MAP_SWIZZLE_128B))
                return cudaErrorNotSupported;
            AccArgs        a{};
            a.tilesM     = int((h.T + rows - 1) / rows);
            a.tilesN     = int((h.n + TN - 1) / TN);
            a.kBlocks    = int((h.D + 63) / 64);
            a.chunk      = 16;
            a.kElems     = 64;
            a.ksplit     = 1;
            a.groupM     = int(std::max<int64_t>(1, std::min<int64_t>(a.tilesM, (int64_t(32) << 20) / (rows * h.D * 2))));
            a.xRows      = xRows;
            // Waits and commits between MMAs cost the issuing thread several hundred cycles: two K blocks a stage (1024 cycles
            // of MMAs) where three stages of them fit
            const int room = 226 * 1024 - 1024 - Epi::ROOM - int(behind);
            a.sub          = room / int(2 * stage) >= 3 ? 2 : 1;
            a.kParts       = 1;
            a.stages       = std::min<int>(kAccMaxStages, room / int(stage * a.sub));
            a.stageBytes = (uint32_t(a.stages * a.sub) * stage + behind + 1023) / 1024 * 1024;
            a.idesc      = (1u << 4) | (h.type == CUDA_R_16BF ? (1u << 7) | (1u << 10) : 0u) | (uint32_t(TN >> 3) << 17) | (uint32_t(rows >> 4) << 24);
            a.status     = status;
            a.statusCode = kStatusSoftmax;
            return launchAccumulate<Epi, PAIR, TN, false, false>(mapX, mapY, a, ea, smCount, stream, name);
        }
        // Up to 128 tokens the classes' rows are the traffic and a tile of 128 tokens is enough: 128 x 256 tiles of one CTA each.
        // (1 token, 32000 x 4096: 56 us; tiles of 128 classes 60, of 64 94, of 32 146: a K block costs the same however narrow.)
        // Beyond, 256 x 256 tiles of CTA pairs.
        bool narrowHead(int64_t T)
        {
            return T <= 128;
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

    // How many parts of the classes dH's products run in, side by side: tiles of 128 x 256 of [T, D] alone would leave SMs idle
    // when there are few tokens. About one unit for every SM, each of at least 1024 classes. 0: many tokens, the general
    // contraction has enough tiles.
    int hiddenParts(int64_t T, int64_t D, int64_t piece)
    {
        if(T > 384)
            return 0;
        const int64_t tiles = (D + 255) / 256 * ((T + 127) / 128);
        return int(std::max<int64_t>(1, std::min<int64_t>((148 + tiles / 2) / tiles, piece / 1024)));
    }

    cudaError_t launchHiddenGradient(int type, const void* P, int64_t ldp, const void* W, int64_t ldw, int64_t T, int64_t n, int64_t D, int parts,
                                     float* out, int64_t ldo, bool add, int smCount, int* status, cudaStream_t stream)
    {
        PFN_encodeTiled encode = tensorMapEncoder();
        HiddenArgs      ea{};
        const int       tiles = int((T + 127) / 128), xRows = int(std::min<int64_t>(128, (T + 7) / 8 * 8));
        ea.T = T, ea.ld = ldo, ea.tiles = tiles, ea.out = out, ea.add = add;
        CUtensorMap mapX, mapY;
        if(!encode || !encodeMatrix(encode, &mapX, P, n, T, ldp, 64, xRows, CU_TENSOR_MAP_SWIZZLE_128B)
           || !encodeMatrix(encode, &mapY, W, D, n, ldw, 64, 64, CU_TENSOR_MAP_SWIZZLE_128B))
            return cudaErrorNotSupported;
        const uint32_t block = (uint32_t(xRows) + 256u) * 128u, behind = uint32_t(128 - xRows) * 128u;
        const int      room  = 226 * 1024 - 1024 - int(behind);
        parts                = int(std::min<int64_t>(parts, (n + 63) / 64)); // a short last piece: every part has something to add
        AccArgs a{};
        a.tilesM     = parts * tiles;
        a.tilesN     = int((D + 255) / 256);
        a.kBlocks    = int((n + 63) / 64);
        a.chunk      = 16;
        a.sub        = room / int(2 * block) >= 3 ? 2 : 1;
        a.kParts     = parts;
        a.kElems     = 64;
        a.xRows      = xRows;
        a.ksplit     = 1;
        a.groupM     = a.tilesM;
        a.stages     = std::min<int>(kAccMaxStages, room / int(block * a.sub));
        a.stageBytes = (uint32_t(a.stages * a.sub) * block + behind + 1023) / 1024 * 1024;
        a.idesc      = (1u << 4) | (type == CUDA_R_16BF ? (1u << 7) | (1u << 10) : 0u) | (1u << 16) | (uint32_t(256 >> 3) << 17)
                  | (uint32_t(128 >> 4) << 24); // Y transposed
        a.status     = status;
        a.statusCode = kStatusSoftmax;
        return launchAccumulate<HiddenEpi, false, 256, false, true>(mapX, mapY, a, ea, smCount, stream, "cross_entropy_hidden");
    }

    cudaError_t launchWeightGradient(int type, const void* P, int64_t ldp, const void* H, int64_t ldh, int64_t K, int64_t n, int64_t D,
                                     const float* scale, void* dW, int64_t ldw, int smCount, int* status, cudaStream_t stream)
    {
        PFN_encodeTiled encode = tensorMapEncoder();
        WeightArgs      ea{};
        ea.rows = n, ea.cols = D, ea.scale = scale;
        CUtensorMap mapX, mapY;
        if(!encode || !encodeMatrix(encode, &mapX, P, n, K, ldp, 64, 64, CU_TENSOR_MAP_SWIZZLE_128B)
           || !encodeMatrix(encode, &mapY, H, D, K, ldh, 64, 64, CU_TENSOR_MAP_SWIZZLE_128B)
           || !encodeMatrix(encode, &ea.mapD, dW, D, n, ldw, 64, 32, CU_TENSOR_MAP_SWIZZLE_128B))
            return cudaErrorNotSupported;
        AccArgs a{};
        a.tilesM     = int((n + 255) / 256);
        a.tilesN     = int((D + 255) / 256);
        a.kBlocks    = int((K + 63) / 64);
        a.chunk      = 16;
        a.kElems     = 64;
        a.xRows      = 128;
        a.ksplit     = 1;
        a.groupM     = int(std::max<int64_t>(1, std::min<int64_t>(a.tilesM, (int64_t(32) << 20) / (256 * K * 2))));
        a.sub        = 2;
        a.kParts     = 1;
        a.stages     = int((226 * 1024 - 1024 - WeightEpi<__half>::ROOM) / 65536);
        a.stageBytes = uint32_t(a.stages) * 65536u;
        // f32 sums, both operands transposed (contiguous along their rows)
        a.idesc = (1u << 4) | (type == CUDA_R_16BF ? (1u << 7) | (1u << 10) : 0u) | (1u << 15) | (1u << 16) | (uint32_t(256 >> 3) << 17)
                  | (uint32_t(256 >> 4) << 24);
        a.status     = status;
        a.statusCode = kStatusSoftmax;
        return type == CUDA_R_16F ? launchAccumulate<WeightEpi<__half>, true, 256, true, true>(mapX, mapY, a, ea, smCount, stream, "cross_entropy_weight")
                                  : launchAccumulate<WeightEpi<__nv_bfloat16>, true, 256, true, true>(mapX, mapY, a, ea, smCount, stream, "cross_entropy_weight");
    }

    // A row of dW is a sum over the tokens of which the class's own ones outweigh the others: over few tokens the rounding of
    // P does not average out (up to 1.5 times the rounding of dW itself). P is then handed over as two numbers, which
    // doubles a short sum that is bound by the bytes of dW all the same.
    bool splitProbabilities(int64_t T)
    {
        return T <= 64;
    }

    cudaError_t launchHeadLoss(const HeadProduct& h, int64_t v0, const int64_t* targets, float alpha, void* part, float* state, int smCount,
                               int* status, cudaStream_t stream)
    {
        HeadArgs ea{};
        ea.T = h.T, ea.n = h.n, ea.v0 = v0;
        ea.targets     = targets;
        ea.alpha       = alpha;
        ea.part        = static_cast<float2*>(part);
        ea.targetLogit = state + 2 * h.T;
        return narrowHead(h.T) ? launchHeadForm<LossEpi, false>(h, ea, smCount, status, stream, "cross_entropy_head")
                               : launchHeadForm<LossEpi, true>(h, ea, smCount, status, stream, "cross_entropy_head_pair");
    }

    cudaError_t launchLossJoin(const void* part, int64_t n, int64_t T, float* state, bool first, bool last, int64_t V, int64_t ignore,
                               const int64_t* targets, float* loss, float* lse, int* status, cudaStream_t stream)
    {
        const int group = kHeadGroup;
        join_kernel<<<unsigned((T + 31) / 32), 32 * kJoinWarps, 0, stream>>>(static_cast<const float2*>(part), (n + group - 1) / group, T, state, first,
                                                                            last, V, ignore, targets, loss, lse, status);
        return noted("cross_entropy_join");
    }

    cudaError_t launchHeadGradient(const HeadProduct& h, int64_t v0, int64_t V, int64_t ignore, const int64_t* targets, const float* lse,
                                   const float* g, float alpha, const float* scale, void* P, int64_t ldp, float* rest, int smCount, int* status,
                                   cudaStream_t stream)
    {
        HeadArgs ea{};
        ea.T = h.T, ea.n = h.n, ea.v0 = v0, ea.V = V, ea.ignore = ignore;
        ea.targets = targets, ea.alpha = alpha, ea.lse = lse, ea.g = g, ea.scale = scale, ea.rest = rest;
        PFN_encodeTiled encode = tensorMapEncoder();
        const bool      two    = splitProbabilities(h.T), half = h.type == CUDA_R_16F;
        if(!encode || !encodeMatrix(encode, &ea.mapP, P, h.n, h.T, ldp, 64, 32, CU_TENSOR_MAP_SWIZZLE_128B)
           || !encodeMatrix(encode, &ea.mapLow, static_cast<const char*>(P) + (two ? h.T * ldp * 2 : 0), h.n, h.T, ldp, 64, 32, CU_TENSOR_MAP_SWIZZLE_128B))
            return cudaErrorNotSupported;
        const char* name = "cross_entropy_head_gradient";
        if(two)
            return half ? launchHeadForm<ProbabilityEpi<__half, 2>, false>(h, ea, smCount, status, stream, name)
                        : launchHeadForm<ProbabilityEpi<__nv_bfloat16, 2>, false>(h, ea, smCount, status, stream, name);
        if(narrowHead(h.T))
            return half ? launchHeadForm<ProbabilityEpi<__half, 1>, false>(h, ea, smCount, status, stream, name)
                        : launchHeadForm<ProbabilityEpi<__nv_bfloat16, 1>, false>(h, ea, smCount, status, stream, name);
        return half ? launchHeadForm<ProbabilityEpi<__half, 1>, true>(h, ea, smCount, status, stream, "cross_entropy_head_gradient_pair")
                    : launchHeadForm<ProbabilityEpi<__nv_bfloat16, 1>, true>(h, ea, smCount, status, stream, "cross_entropy_head_gradient_pair");
    }

    cudaError_t launchPackRows(int type, const void* X, const TokenRows& rows, int64_t count, int64_t cols, int64_t ld, void* X2,
                               const int64_t* targets, int64_t ignore, int64_t V, int* status, bool twice, cudaStream_t stream)
    {
        const int grid = rowGrid(count);
        if(type == CUDA_R_32F)
            pack_rows_kernel<float><<<grid, 256, 0, stream>>>((const float*)X, rows, count, cols, ld, (float*)X2, targets, ignore, V, status, twice);
        else if(type == CUDA_R_16F)
            pack_rows_kernel<__half><<<grid, 256, 0, stream>>>((const __half*)X, rows, count, cols, ld, (__half*)X2, targets, ignore, V, status, twice);
        else
            pack_rows_kernel<__nv_bfloat16>
                <<<grid, 256, 0, stream>>>((const __nv_bfloat16*)X, rows, count, cols, ld, (__nv_bfloat16*)X2, targets, ignore, V, status, twice);
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

    cudaError_t launchProbabilities(float* z, int64_t ldz, int64_t T, int64_t v0, int64_t count, int64_t V, int64_t ignore,
                                    const int64_t* targets, const float* lse, const float* g, float alpha, cudaStream_t stream)
    {
        probabilities_kernel<<<rowGrid(T), 256, 0, stream>>>(z, ldz, T, v0, count, V, ignore, targets, lse, g, alpha);
        return noted("cross_entropy_probabilities");
    }

    cudaError_t launchStoreRows(int type, const float* X, int64_t ldx, int64_t count, int64_t cols, const float* scale, void* Y,
                                const TokenRows& rows, const TargetRest& rest, int parts, cudaStream_t stream)
    {
        const int grid = rowGrid(count);
        if(type == CUDA_R_32F)
            store_rows_kernel<float><<<grid, 256, 0, stream>>>(X, ldx, count, cols, scale, (float*)Y, rows, rest, parts);
        else if(type == CUDA_R_16F)
            store_rows_kernel<__half><<<grid, 256, 0, stream>>>(X, ldx, count, cols, scale, (__half*)Y, rows, rest, parts);
        else
            store_rows_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(X, ldx, count, cols, scale, (__nv_bfloat16*)Y, rows, rest, parts);
        return noted("cross_entropy_store");
    }
} // namespace htb
