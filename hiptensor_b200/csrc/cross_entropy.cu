// Kernels of the linear cross entropy and its gradient. All products run on the shared pipeline of accumulate.cuh; logits and
// probabilities are made in the epilogue of the product that needs them. f32 operands are sums of three bf16 numbers each, of
// whose nine products the six that matter are added (at most 2^-24 of a product is left out, 2^-27 in the mean): the rate is a sixth of bf16's, as with the
// TF32 split of the f32 contraction, and everything else is shared.
//
// Many tokens are bound by the tensor cores under the power limit: 8192 tokens x 128000 classes x 4096 bf16, loss 6.6 to 6.8 ms
// (1.26 to 1.30 PFLOP/s; a plain library product of that size runs at 1.39 sustained; 5.7 after a pause), 4096 tokens' gradient 10.3
// to 10.9 ms (1.18 to 1.25). Few tokens are bound by the bytes of W: 1 token x 32000 x 4096, loss 56 us (4.7 TB/s); 8 tokens'
// gradient 230 us (W read twice, dW written). Gradients of fewer tokens run in one pass over W (cross_entropy_few.cu).
// f32: 1024 x 32000 x 1024, loss 370 to 480 us (by where the copies lie in memory), gradient 1.1 ms (185 TFLOP/s, 0.7 of a sixth
// of bf16's rate). A W whose classes are contiguous ([d, v]) is copied and its gradient stored element by element: 1024 x 32000 x
// 1024 bf16 takes 196 us for the loss and 673 for the gradient, 73 and 201 as [v, d].
#include <algorithm>

#include "accumulate.cuh"
#include "cross_entropy.hpp"
#include "cross_entropy_device.cuh"
#include "kernels.hpp"

namespace htb
{
    namespace
    {
        // Rows of a strided tensor as packed rows of ld 16-bit elements, eight elements a thread. SPLIT: f32 numbers as three bf16
        // ones, x = h + m + l, [3][rows][ld] (an infinity or NaN stays in h; a number that would round to an infinity,
        // as f32's lowest value would, is truncated in h).
        template <typename T, bool SPLIT>
        __global__ void pack_rows_kernel(const T* __restrict__ X, const __grid_constant__ TokenRows rows, int64_t count, int64_t total, int64_t cols,
                                         int64_t ld, unsigned short* __restrict__ X2, const int64_t* __restrict__ targets, int64_t ignore,
                                         int64_t V, int* __restrict__ classes, int* status, bool vec)
        {
            for(int64_t c = (int64_t(blockIdx.y) * blockDim.x + threadIdx.x) * 8; c < ld; c += int64_t(gridDim.y) * blockDim.x * 8)
            for(int64_t r = int64_t(blockIdx.x) * blockDim.y + threadIdx.y; r < total; r += int64_t(gridDim.x) * blockDim.y)
            {
                bool live = r < count;
                if(live && targets)
                {
                    const int64_t target = targets[r];
                    live                 = counts(target, ignore, V);
                    if(!live && target != ignore && c == 0)
                        atomicExch_system(status, kStatusBadTarget);
                    if(classes && c == 0)
                        classes[r] = live ? int(target) : -1;
                }
                T x[8];
                if(live && vec && c + 8 <= cols)
                {
                    const uint4* src = reinterpret_cast<const uint4*>(X + rowOffset(rows, r) + c);
#pragma unroll
                    for(int w = 0; w < int(sizeof(T)) / 2; w++)
                        reinterpret_cast<uint4*>(x)[w] = __ldg(src + w);
                }
                else
                {
                    const T* src = X + (live ? rowOffset(rows, r) + c * rows.elem : 0);
#pragma unroll
                    for(int j = 0; j < 8; j++)
                        x[j] = (live && c + j < cols) ? src[j * rows.elem] : narrow<T>(0.f);
                }
                if constexpr(!SPLIT)
                    *reinterpret_cast<uint4*>(X2 + r * ld + c) = *reinterpret_cast<const uint4*>(x);
                else
                {
                    __nv_bfloat16 part[3][8];
                    bool          odd = false;
#pragma unroll
                    for(int j = 0; j < 8; j++)
                    {
                        float left = x[j];
#pragma unroll
                        for(int k = 0; k < 3; k++)
                        {
                            part[k][j] = narrow<__nv_bfloat16>(left);
                            left -= widen(part[k][j]);
                        }
                        odd = odd || !(fabsf(widen(part[0][j])) < INFINITY);
                    }
                    if(odd)
                    {
#pragma unroll
                        for(int j = 0; j < 8; j++)
                        {
                            if(fabsf(widen(part[0][j])) < INFINITY)
                                continue;
                            const bool finite = fabsf(x[j]) < INFINITY;
                            if(finite)
                                part[0][j] = __float2bfloat16_rz(x[j]);
                            const float left = finite ? x[j] - widen(part[0][j]) : 0.f;
                            part[1][j] = narrow<__nv_bfloat16>(left);
                            part[2][j] = narrow<__nv_bfloat16>(left - widen(part[1][j]));
                        }
                    }
#pragma unroll
                    for(int k = 0; k < 3; k++)
                        *reinterpret_cast<uint4*>(X2 + (k * total + r) * ld + c) = *reinterpret_cast<const uint4*>(part[k]);
                }
            }
        }

        // The lists of tokens of 32 classes a block: each of its warps searches an eighth of the tokens, 16 a lane and round, in an
        // order that is always the same, and the warps' lists are linked in the order of the warps. Classes whose list is full
        // are no longer looked for, so that a frequent one (a token's turn takes about 50 instructions) does not outlast the products.
        // 4 bytes a token for 32 classes, out of L2: 1024 tokens x 32000 classes 5 us, 65536 x 8000 22 us.
        constexpr int kListWarps = 8;
        __global__ void __launch_bounds__(32 * kListWarps) token_lists_kernel(const __grid_constant__ TokenLists lists, int64_t T, int64_t V)
        {
            __shared__ int firsts[kListWarps][32], lasts[kListWarps][32], counts[kListWarps][32];
            const int      lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
            const int64_t  v0   = int64_t(blockIdx.x) * 32, share = ((T + kListWarps - 1) / kListWarps + 511) / 512 * 512;
            const int64_t  begin = warp * share, end = min(begin + share, T);
            const int      base  = int(v0);
            int            first = -1, last = -1, count = 0;
            uint32_t       open  = v0 + 32 <= V ? 0xffffffffu : (1u << (V - v0)) - 1;
            int4           next[4];
            auto           load = [&](int64_t t0) {
#pragma unroll
                for(int j = 0; j < 4; j++)
                {
                    const int64_t t = t0 + j * 128 + lane * 4; // (the buffer is of whole words)
                    next[j]         = t < end ? *reinterpret_cast<const int4*>(lists.classes + t) : make_int4(-1, -1, -1, -1);
                }
            };
            load(begin);
            for(int64_t t0 = begin; t0 < end && open; t0 += 512)
            {
                int      c[16];
                uint32_t hits = 0; // token t0 + 128 j + 4 lane + k is number 4 j + k
#pragma unroll
                for(int j = 0; j < 16; j++)
                {
                    const int4& q = next[j / 4];
                    c[j]          = (j % 4 == 0 ? q.x : (j % 4 == 1 ? q.y : (j % 4 == 2 ? q.z : q.w))) - base;
                    if(uint32_t(c[j]) < 32u && (open >> c[j] & 1) && t0 + j / 4 * 128 + lane * 4 + j % 4 < end)
                        hits |= 1u << j;
                }
                load(t0 + 512);
                for(uint32_t lanes; (lanes = __ballot_sync(0xffffffffu, hits != 0)) != 0;)
                {
                    // the first lane's first token and its class
                    const int bit = __ffs(int(hits)) - 1, from = __ffs(int(lanes)) - 1;
                    int       its = c[0];
#pragma unroll
                    for(int j = 1; j < 16; j++)
                        its = bit == j ? c[j] : its;
                    const int number = __shfl_sync(0xffffffffu, bit, from), token = int(t0) + number / 4 * 128 + from * 4 + number % 4;
                    if(lane == from)
                        hits &= hits - 1;
                    if(__shfl_sync(0xffffffffu, its, from) == lane && count < kListed)
                    {
                        if(count++ == 0)
                            first = token;
                        else
                            lists.next[last] = token;
                        last = token;
                    }
                }
                open &= __ballot_sync(0xffffffffu, count < kListed);
            }
            firsts[warp][lane] = first, lasts[warp][lane] = last, counts[warp][lane] = count;
            __syncthreads();
            if(warp != 0 || v0 + lane >= V)
                return;
            for(int w = 1; w < kListWarps && count < kListed; w++)
                if(counts[w][lane])
                {
                    if(count)
                        lists.next[last] = firsts[w][lane];
                    else
                        first = firsts[w][lane];
                    last = lasts[w][lane];
                    count += counts[w][lane];
                }
            if(count)
                lists.next[last] = -1;
            lists.first[v0 + lane] = first;
        }

        // Only tokens whose row of P is not zero have a say, and of these only finite factors: one that is not makes its own row
        // (and dW) what it is, and the others' rows need their power of two all the same.
        __global__ void __launch_bounds__(1024) gradient_scale_kernel(const float* __restrict__ g, float alpha, int64_t T,
                                                                      const int64_t* __restrict__ targets, int64_t ignore, int64_t V, float* scale)
        {
            __shared__ float part[32];
            float            m = 0.f;
            for(int64_t t = threadIdx.x; t < T; t += 1024)
            {
                const float f = fabsf(g[t] * alpha);
                if(f < INFINITY && counts(targets[t], ignore, V))
                    m = fmaxf(m, f);
            }
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
                if(m > 0.f)
                    frexpf(m, &e);
                e        = max(e, -100);
                scale[0] = ldexpf(1.f, 15 - e);
                scale[1] = ldexpf(1.f, e - 15);
            }
        }

        // Y[row r, c] = (sum of the parts' X[r, c] + rest[r] * W[target of r, c]) * scale[1]; four columns a thread. A token that does
        // not count gets zeros, whatever W holds: its row of P is 0, but 0 times an infinity in W is NaN.
        template <typename T>
        __global__ void store_rows_kernel(const float* __restrict__ X, int64_t ldx, int64_t count, int64_t cols, const float* __restrict__ scale,
                                          T* __restrict__ Y, const __grid_constant__ TokenRows rows, const __grid_constant__ TargetRest rest, int parts,
                                          int64_t partRows, bool vec)
        {
            const float f = scale ? scale[1] : 1.f;
            for(int64_t c = (int64_t(blockIdx.y) * blockDim.x + threadIdx.x) * 4; c < cols; c += int64_t(gridDim.y) * blockDim.x * 4)
            for(int64_t r = int64_t(blockIdx.x) * blockDim.y + threadIdx.y; r < count; r += int64_t(gridDim.x) * blockDim.y)
            {
                const int64_t target = rest.targets ? rest.targets[r] : 0;
                const bool    live   = !rest.targets || counts(target, rest.ignore, rest.V);
                float4        x      = make_float4(0.f, 0.f, 0.f, 0.f);
                for(int i = 0; i < parts; i++)
                {
                    const float4 v = *reinterpret_cast<const float4*>(X + (int64_t(i) * partRows + r) * ldx + c); // ldx is a multiple of eight
                    x = make_float4(x.x + v.x, x.y + v.y, x.z + v.z, x.w + v.w);
                }
                float y[4] = {live ? x.x : 0.f, live ? x.y : 0.f, live ? x.z : 0.f, live ? x.w : 0.f};
                if(rest.rest && live)
                {
                    const T*    w = static_cast<const T*>(rest.W) + target * rest.wV + c * rest.wD;
                    const float e = rest.rest[r];
#pragma unroll
                    for(int j = 0; j < 4; j++)
                        if(c + j < cols)
                            y[j] = fmaf(e, widen(w[j * rest.wD]), y[j]);
                }
                T* dst = Y + rowOffset(rows, r) + c * rows.elem;
                if(vec && c + 4 <= cols)
                {
                    struct alignas(4 * sizeof(T)) Four
                    {
                        T e[4];
                    } o;
#pragma unroll
                    for(int j = 0; j < 4; j++)
                        o.e[j] = narrow<T>(y[j] * f);
                    *reinterpret_cast<Four*>(dst) = o;
                }
                else
                {
#pragma unroll
                    for(int j = 0; j < 4; j++)
                        if(c + j < cols)
                            dst[j * rows.elem] = narrow<T>(y[j] * f);
                }
            }
        }

        // threads along a row and rows side by side for kernels of `units` threads a row
        struct RowShape
        {
            dim3 grid, block;
        };
        RowShape rowShape(int64_t rows, int64_t units)
        {
            unsigned tx = 8;
            while(tx < 256 && tx < units)
                tx *= 2;
            const unsigned ty = 256 / tx;
            return RowShape{dim3(unsigned(std::min<int64_t>((rows + ty - 1) / ty, 1 << 20)), unsigned(std::min<int64_t>((units + tx - 1) / tx, 65535))),
                            dim3(tx, ty)};
        }
        // every row of a strided tensor starts at a multiple of `unit` elements
        bool rowsAligned(const TokenRows& rows, const void* base, int64_t unit, int64_t size)
        {
            bool ok = rows.elem == 1 && uintptr_t(base) % uintptr_t(unit * size) == 0;
            for(int i = 0; i < rows.nt; i++)
                ok = ok && rows.stride[i] % unit == 0;
            return ok;
        }

        // ------------------------------------------------------------------ logits that stay on the chip
        struct HeadArgs
        {
            int64_t        T, n, v0, V; // tokens; classes of this piece, its first class, all classes
            int64_t        ignore;
            const int64_t* targets;
            float          alpha;
            // loss: partial (maximum, sum of exponentials relative to it) of 128 classes each, [classes][T]; target logits
            float2* part;
            float*  targetLogit;
            // gradient
            const float *lse, *g, *scale;
            float*       rest; // what rounding took from the target's entry of P
            int64_t      rowsP; // of a segment of P
            CUtensorMap  mapP;
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

        // Loss: one pass over a tile's logits in registers, maximum then sum of exponentials; what leaves the SM are two
        // floats for 128 logits.
        struct LossEpi : HeadSums<256>
        {
            using Args                 = HeadArgs;
            using Sums                 = HeadSums<256>;
            static constexpr int kSide = 0;
            static constexpr bool kSplit = false;
            static constexpr bool kParted = false;
            static constexpr int ROOM  = 0; // shared memory behind the stages
            const Args&          a;

            __device__ LossEpi(const Args& args, int, int, unsigned char*, volatile int*)
                : a(args)
            {
            }
            __device__ __forceinline__ void begin(int64_t) {}
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
                const uint64_t alpha2 = pack2(a.alpha, a.alpha), log2e2 = pack2(kLog2e, kLog2e);
                float          m  = -INFINITY;
                const int      n  = int(min(int64_t(COLS), a.n - col));
#pragma unroll
                for(int i = 0; i < COLS / 2; i++)
                {
                    acc[i]         = mul2(acc[i], alpha2);
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
                    const float2 f = unpack2(mul2(add2(acc[i], less), log2e2));
                    sum[i & 3]     = add2(sum[i & 3], pack2(exp2f(f.x), exp2f(f.y)));
                }
                const float2 s = unpack2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])));
                a.part[(col / COLS) * a.T + row] = make_float2(m, s.x + s.y);
            }
            __device__ __forceinline__ void leave() {}
        };

        // Gradient: P = (exp(z - lse) - [class is the target]) * g * alpha, rounded to the operands' type for the two products
        // that follow (the products' sums are f32). The target's entry outweighs the others: what its rounding takes is kept and
        // added to dH and dW in f32, which leaves both with the error of their own rounding (512 x 20000 x 4096: 1.66e-3 in bf16, as
        // with P in 64 bits; dW without it 2.2e-3). The others' rounding, at most 2^-8 (f16: 2^-11) of each, is a twentieth of that
        // there. PARTS > 1: P as a sum of that many numbers, each what rounding took from the ones before, in
        // segments of rowsP rows (a multiple of 32; rows past the tokens hold zeros there).
        template <typename TP, int PARTS>
        struct ProbabilityEpi : HeadSums<256>
        {
            using Args                 = HeadArgs;
            using Sums                 = HeadSums<256>;
            static constexpr int kSide = 0;
            static constexpr bool kSplit = false;
            static constexpr bool kParted = false;
            static constexpr int ROUND = 64; // columns of a slot: rows of 128 bytes
            static constexpr int SLOTS = 1;
            static constexpr int ROOM  = 8 * SLOTS * 4096;
            const Args&          a;
            const int            lane;
            const uint32_t       slot;
            int                  stores;

            __device__ ProbabilityEpi(const Args& args, int w, int l, unsigned char* smem, volatile int*)
                : a(args)
                , lane(l)
                , slot(smemAddr(smem) + uint32_t(w * SLOTS * 4096))
                , stores(0)
            {
            }
            __device__ __forceinline__ void begin(int64_t) {}
            template <class Release>
            __device__ __forceinline__ void add(uint32_t taddr, bool first, Release release)
            {
                Sums::addSums(taddr, first, release);
            }
            __device__ __forceinline__ void end(int64_t row, int64_t col)
            {
                int64_t target = -1;
                float   lse = 0.f, f = 0.f;
                bool    live = false;
                if(row < a.T)
                {
                    target = a.targets[row];
                    live   = counts(target, a.ignore, a.V);
                    if(live)
                    {
                        lse = a.lse[row];
                        f = a.g[row] * a.alpha * (a.scale ? a.scale[0] : 1.f);
                    }
                }
                const uint64_t alpha2 = pack2(a.alpha, a.alpha), lse2 = pack2(-lse, -lse), log2e2 = pack2(kLog2e, kLog2e);
                const int      t  = live && target - a.v0 - col >= 0 && target - a.v0 - col < COLS ? int(target - a.v0 - col) : -1;
                // P takes the sums' place
#pragma unroll
                for(int i = 0; i < COLS / 2; i++)
                {
                    float p0, p1;
                    if constexpr(PARTS == 3)
                    {
                        // f32: an exponent of 15 as one of powers of two is rounded by 2^-20, which would be P's largest error
                        const float2 z = unpack2(acc[i]);
                        p0 = expf(fmaf(z.x, a.alpha, -lse));
                        p1 = expf(fmaf(z.y, a.alpha, -lse));
                    }
                    else
                    {
                        const float2 x = unpack2(mul2(fma2(acc[i], alpha2, lse2), log2e2));
                        p0 = exp2f(x.x);
                        p1 = exp2f(x.y);
                    }
                    if(t == 2 * i)
                        p0 -= 1.f;
                    if(t == 2 * i + 1)
                        p1 -= 1.f;
                    acc[i] = live ? pack2(p0 * f, p1 * f) : 0;
                }
                if(PARTS < 3 && t >= 0)
                {
                    const float p = Sums::at(t);
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
                                uint64_t&    pair = acc[(r + 8 * u + 2 * j) / 2];
                                const float2 x    = unpack2(pair);
                                const TP     lo = narrow<TP>(x.x), hi = narrow<TP>(x.y);
                                if constexpr(PARTS > 1)
                                    pair = pack2(x.x - widen(lo), x.y - widen(hi)); // for the next part
                                q[j] = uint32_t(reinterpret_cast<const unsigned short&>(lo))
                                       | (uint32_t(reinterpret_cast<const unsigned short&>(hi)) << 16);
                            }
                            // 16-byte units permuted as the map's swizzle has them
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + uint32_t(lane * 128 + ((u ^ (lane & 7)) << 4))),
                                         "r"(q[0]), "r"(q[1]), "r"(q[2]), "r"(q[3])
                                         : "memory");
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if(lane == 0)
                        {
                            // a block that begins outside has nothing to store; of one that ends outside the map clips the
                            // columns and, with one part, the rows (more parts: rowsP is a multiple of 32)
                            if(row < a.rowsP && col + r < a.n)
                                asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(&a.mapP), "r"(at),
                                             "r"(int(col + r)), "r"(int(low * a.rowsP + row))
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
            // what rounding took from the targets' entries of P (no lists: nothing is added), and H, rows of 16-bit elements ldh apart
            TokenLists            lists;
            const float*          rest;
            const unsigned short* H;
            int64_t               ldh, T, v0;
            int                   half; // H is f16, else bf16
            CUtensorMap           mapD;
        };
        // SLOTS: of 4 KiB for a warp's results. A short sum (few tokens) is bound by its stores and takes two; a long one leaves the
        // room to the stages.
        template <typename TD, int SLOTS>
        struct WeightEpi : HeadSums<256>
        {
            using Args                   = WeightArgs;
            static constexpr int  kSide  = 0;
            static constexpr bool kSplit = false;
            static constexpr bool kParted = false;
            static constexpr int  ROUND  = 128 / int(sizeof(TD)); // columns of a slot: rows of 128 bytes
            static constexpr int  ROOM   = 8 * SLOTS * 4096;
            const Args&           a;
            const int             lane;
            const uint32_t        slot;
            int                   stores, mine;

            __device__ WeightEpi(const Args& args, int w, int l, unsigned char* smem, volatile int*)
                : a(args)
                , lane(l)
                , slot(smemAddr(smem) + uint32_t(w * SLOTS * 4096))
                , stores(0)
                , mine(-1)
            {
            }
            // (asked for here, so that it is there when the sums are)
            __device__ __forceinline__ void begin(int64_t row)
            {
                mine = a.lists.first && row < a.rows ? a.lists.first[a.v0 + row] : -1;
            }
            template <class Release>
            __device__ __forceinline__ void add(uint32_t taddr, bool first, Release release)
            {
                addSums(taddr, first, release);
            }
            // sums += rest[token] * H[token, col ..] for this thread's class
            __device__ __forceinline__ void addToken(int token, int64_t col)
            {
                constexpr int         LOADS = 8;
                const float           e   = a.rest[token];
                const uint64_t        e2  = pack2(e, e);
                const unsigned short* src = a.H + token * a.ldh + col;
#pragma unroll
                for(int c = 0; c < COLS; c += 8 * LOADS)
                {
                    uint4 q[LOADS]; // on their way together
#pragma unroll
                    for(int l = 0; l < LOADS; l++)
                        q[l] = col + c + 8 * l < a.ldh ? *reinterpret_cast<const uint4*>(src + c + 8 * l) : make_uint4(0, 0, 0, 0);
#pragma unroll
                    for(int j = 0; j < 4 * LOADS; j++)
                    {
                        const uint4&   v = q[j / 4];
                        const uint32_t w = j % 4 == 0 ? v.x : (j % 4 == 1 ? v.y : (j % 4 == 2 ? v.z : v.w));
                        const float2   f = a.half ? __half22float2(reinterpret_cast<const __half2&>(w))
                                                  : make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
                        acc[c / 2 + j] = fma2(pack2(f.x, f.y), e2, acc[c / 2 + j]);
                    }
                }
            }
            // The targets' entries outweigh the others in a class's row: what rounding took from them is added here, token by token, behind
            // the next tile's MMAs. With the lists it takes, of a gradient: nothing of 4096 x 128000 x 4096 (10.0 ms), 7 of 210 us of
            // 1024 x 32000 x 1024, 17 of 190 of 128 x 32000 x 4096 (a tile's sum is short there), 20 of 95 of 4096 x 1000 x 1024 (the lists'
            // 16 tokens for most classes); P as two numbers instead would add a third to the gradient's operations.
            __device__ __forceinline__ void addRests(int64_t col)
            {
                while(__any_sync(0xffffffffu, mine >= 0))
                    if(mine >= 0)
                    {
                        const int token = mine;
                        mine            = a.lists.next[token];
                        addToken(token, col);
                    }
            }
            __device__ __forceinline__ void end(int64_t row, int64_t col)
            {
                addRests(col);
                const float    f  = a.scale ? a.scale[1] : 1.f;
                const uint64_t f2 = pack2(f, f);
#pragma unroll
                for(int r = 0; r < COLS; r += ROUND)
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
                            if constexpr(sizeof(TD) == 4)
                            {
                                const float2 x = unpack2(mul2(acc[(r + 4 * u + j) / 2], f2));
                                q[j]           = __float_as_uint((j & 1) ? x.y : x.x);
                            }
                            else
                            {
                                const float2 x = unpack2(mul2(acc[(r + 8 * u + 2 * j) / 2], f2));
                                const TD     lo = narrow<TD>(x.x), hi = narrow<TD>(x.y);
                                q[j] = uint32_t(reinterpret_cast<const unsigned short&>(lo))
                                       | (uint32_t(reinterpret_cast<const unsigned short&>(hi)) << 16);
                            }
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

        // dH = P W over parts of the classes: f32 sums of every part, [part][rows][ld], stored or (later pieces) added by bulk
        // copies; each element has one writer, so results are the same every time.
        struct HiddenArgs
        {
            int64_t     T, ld;
            int64_t     tileRows; // of a part, in whole tiles
            int64_t     rows; // of a part in the result: a multiple of 32
            int         add;
            CUtensorMap mapOut;
        };
        struct HiddenEpi : HeadSums<256>
        {
            using Args                    = HiddenArgs;
            static constexpr int  kSide   = 0;
            static constexpr bool kSplit  = false;
            static constexpr bool kParted = true;
            static constexpr int  SLOTS   = 1;
            static constexpr int  ROOM    = 8 * SLOTS * 4096;
            const Args&           a;
            const int             lane;
            const uint32_t        slot;

            __device__ HiddenEpi(const Args& args, int w, int l, unsigned char* smem, volatile int*)
                : a(args)
                , lane(l)
                , slot(smemAddr(smem) + uint32_t(w * SLOTS * 4096))
            {
            }
            __device__ __forceinline__ void begin(int64_t) {}
            template <class Release>
            __device__ __forceinline__ void add(uint32_t taddr, bool first, Release release)
            {
                addSums(taddr, first, release);
            }
            __device__ __forceinline__ void end(int64_t row, int64_t col)
            {
                const int64_t part = row / a.tileRows, t = row - part * a.tileRows;
#pragma unroll
                for(int r = 0; r < COLS; r += 32)
                {
                    if(lane == 0)
                        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); // the slot's last copy has read it
                    __syncwarp();
#pragma unroll
                    for(int u = 0; u < 8; u++)
                    {
                        const float2 x = unpack2(acc[(r + 4 * u) / 2]), y = unpack2(acc[(r + 4 * u) / 2 + 1]);
                        asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(slot + uint32_t(lane * 128 + ((u ^ (lane & 7)) << 4))),
                                     "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y)
                                     : "memory");
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if(lane == 0)
                    {
                        if(t < a.T && col + r < a.ld)
                        {
                            if(a.add)
                                asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(&a.mapOut),
                                             "r"(slot), "r"(int(col + r)), "r"(int(part * a.rows + t))
                                             : "memory");
                            else
                                asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(&a.mapOut), "r"(slot),
                                             "r"(int(col + r)), "r"(int(part * a.rows + t))
                                             : "memory");
                        }
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
                        joinSums(m, s, p[j].x, p[j].y);
                }
                for(; i < groups; i += kJoinWarps)
                {
                    const float2 p = part[i * T + t];
                    joinSums(m, s, p.x, p.y);
                }
            }
            mine[warp][lane] = make_float2(m, s);
            __syncthreads();
            if(warp != 0 || t >= T)
                return;
            for(int w = 1; w < kJoinWarps; w++)
                joinSums(m, s, mine[w][lane].x, mine[w][lane].y);
            if(!first)
                joinSums(m, s, state[t], state[T + t]);
            if(!last)
            {
                state[t]     = m;
                state[T + t] = s;
                return;
            }
            const float   ref = reference(m), l = logf(s);
            const int64_t target = targets[t];
            lse[t] = ref + l;
            if(target == ignore)
                loss[t] = 0.f;
            else if(target < 0 || target >= V)
            {
                loss[t] = __int_as_float(0x7fc00000);
                atomicExch_system(status, kStatusBadTarget);
            }
            else
                loss[t] = (ref - state[2 * T + t]) + l; // at least 0, and 0 where nothing but the target has a share
        }

        bool encodeMatrix(PFN_encodeTiled encode, CUtensorMap* map, const void* base, int64_t cols, int64_t rows, int64_t ld, int boxCols, int boxRows,
                          bool f32 = false)
        {
            const int64_t size    = f32 ? 4 : 2, unit = 16 / size;
            cuuint64_t    gdim[2] = {cuuint64_t(cols), cuuint64_t(rows)}, gstr[1] = {cuuint64_t((rows > 1 ? ld : (cols + unit - 1) / unit * unit) * size)};
            cuuint32_t    bx[2] = {cuuint32_t(boxCols), cuuint32_t(boxRows)}, estr[2] = {1, 1};
            return encode(map, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(base), gdim, gstr, bx, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE)
                   == CUDA_SUCCESS;
        }

        // The pairs of segments that are multiplied when X is a sum of nx numbers and Y of ny: the products that are left out
        // are at most 2^-24 of the whole, 2^-27 in the mean.
        void segmentPairs(int nx, int ny, AccArgs& a, int kBlocksOfOne)
        {
            int pairs = 0;
            a.segX = a.segY = 0;
            for(int sum = std::min(nx + ny - 2, 2); sum >= 0; sum--) // small products first
                for(int x = 0; x < nx; x++)
                {
                    const int y = sum - x;
                    if(y < 0 || y >= ny)
                        continue;
                    a.segX |= uint32_t(x) << (4 * pairs);
                    a.segY |= uint32_t(y) << (4 * pairs);
                    pairs++;
                }
            if(nx > 1 && ny > 1)
                a.chunk = 4; // f32's accuracy: shorter truncated sums
            a.segBlocks = kBlocksOfOne;
            a.kBlocks   = pairs * kBlocksOfOne;
        }

        template <class T>
        struct Named // a type as an argument
        {
            using Type = T;
        };

        // what every launch has in common; xRows: rows of X that a CTA loads
        template <class Epi, bool PAIR>
        void fillCommon(AccArgs& a, int64_t rows, int64_t cols, int xRows, int64_t bytesOfRow, int* status)
        {
            constexpr int  TILE   = PAIR ? 256 : 128;
            const uint32_t block  = (uint32_t(xRows) + (PAIR ? 128u : 256u)) * 128u, behind = uint32_t(128 - xRows) * 128u;
            const int      room   = 226 * 1024 - 1024 - Epi::ROOM - int(behind);
            a.tilesM     = int((rows + TILE - 1) / TILE);
            a.tilesN     = int((cols + 255) / 256);
            a.groupM     = int(std::max<int64_t>(1, std::min<int64_t>(a.tilesM, (int64_t(32) << 20) / (TILE * bytesOfRow))));
            a.chunk      = 16;
            a.kElems     = 64;
            a.xRows      = xRows;
            a.yRows      = 256;
            a.ksplit     = 1;
            a.kParts     = 1;
            // Waits and commits between MMAs cost the issuing thread several hundred cycles: two K blocks a stage (1024 cycles
            // of MMAs) where three stages of them fit
            a.sub        = room / int(2 * block) >= 3 ? 2 : 1;
            a.stages     = std::min<int>(kAccMaxStages, room / int(block * a.sub));
            a.stageBytes = (uint32_t(a.stages * a.sub) * block + behind + 1023) / 1024 * 1024;
            a.status     = status;
            a.statusCode = kStatusSoftmax;
        }
        // f32 sums, both operands f16 or bf16, transposed ones, N / 8, M / 16
        uint32_t instruction(bool f16, bool pair, bool xMn, bool yMn)
        {
            return (1u << 4) | (f16 ? 0u : (1u << 7) | (1u << 10)) | (xMn ? 1u << 15 : 0u) | (yMn ? 1u << 16 : 0u) | (uint32_t(256 >> 3) << 17)
                   | (uint32_t((pair ? 256 : 128) >> 4) << 24);
        }

        template <class Epi, bool PAIR, bool XMN, bool YMN>
        cudaError_t launchAccumulate(const CUtensorMap& mapX, const CUtensorMap& mapY, const AccArgs& a, const typename Epi::Args& ea, int smCount,
                                     cudaStream_t stream, const char* name)
        {
            auto                     kernel = accumulate_kernel<Epi, PAIR, 256, false, XMN, YMN>;
            static const cudaError_t regs   = accCheckRegs((const void*)kernel, 256);
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

        // 128 x 256 tiles of one CTA each, or 256 x 256 tiles of CTA pairs, which load less. Up to 128 tokens a tile of 128 is
        // enough and the classes' rows are the traffic (1 token, 32000 x 4096: 54 us; with tiles of 128 classes 60, of 64 94: a
        // K block costs the same however narrow). Beyond, the form with the shorter sequence of tiles, one of a single CTA
        // taking about 1.4 times a pair's (it is bound by what it loads).
        bool singleTiles(int64_t T, int64_t columns, int sms)
        {
            if(T <= 128)
                return true;
            const int64_t single = ((T + 127) / 128 * columns + sms - 1) / sms, pairs = ((T + 255) / 256 * columns + sms / 2 - 1) / (sms / 2);
            return 7 * single < 5 * pairs;
        }
        int rowsLoaded(int64_t T) // no more rows than there are tokens
        {
            return int(std::min<int64_t>(128, (T + 7) / 8 * 8));
        }

        template <class Epi, bool PAIR>
        cudaError_t launchHeadForm(const HeadProduct& h, HeadArgs& ea, int smCount, int* status, cudaStream_t stream, const char* name)
        {
            PFN_encodeTiled encode = tensorMapEncoder();
            const int       xRows  = PAIR ? 128 : rowsLoaded(h.T);
            CUtensorMap     mapX, mapY;
            if(!encode || !encodeMatrix(encode, &mapX, h.H, h.D, h.segments > 1 ? h.segments * h.segH : h.T, h.ldh, 64, xRows)
               || !encodeMatrix(encode, &mapY, h.W, h.D, h.segments > 1 ? h.segments * h.segW : h.n, h.ldw, 64, PAIR ? 128 : 256))
                return cudaErrorNotSupported;
            AccArgs a{};
            fillCommon<Epi, PAIR>(a, h.T, h.n, xRows, h.D * 2 * h.segments, status);
            segmentPairs(h.segments, h.segments, a, int((h.D + 63) / 64));
            a.xSegR = int(h.segH), a.ySegR = int(h.segW);
            a.idesc = instruction(h.type == CUDA_R_16F, PAIR, false, false);
            return launchAccumulate<Epi, PAIR, false, false>(mapX, mapY, a, ea, smCount, stream, name);
        }

        cudaError_t noted(const char* name)
        {
            const cudaError_t e = cudaGetLastError();
            if(e == cudaSuccess)
                noteLaunch(name);
            return e;
        }
    } // namespace

    namespace
    {
        int smsOf(int smCount)
        {
            return smCount > 0 ? smCount : 148;
        }
    } // namespace

    int probabilityParts(int type, int64_t T)
    {
        // A row of dW is a sum over the tokens of which the class's own ones outweigh the others: over few tokens the rounding
        // of P does not average out (up to 1.5 times the rounding of dW itself). P is then handed over as two numbers,
        // which doubles a short sum that is bound by the bytes of dW all the same. f32: three bf16 numbers, as H and W.
        return type == CUDA_R_32F ? 3 : (T <= 64 ? 2 : 1);
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
        return singleTiles(h.T, (h.n + 255) / 256, smsOf(smCount)) ? launchHeadForm<LossEpi, false>(h, ea, smCount, status, stream, "cross_entropy_head")
                               : launchHeadForm<LossEpi, true>(h, ea, smCount, status, stream, "cross_entropy_head_pair");
    }

    cudaError_t launchLossJoin(const void* part, int64_t n, int64_t T, float* state, bool first, bool last, int64_t V, int64_t ignore,
                               const int64_t* targets, float* loss, float* lse, int* status, cudaStream_t stream)
    {
        join_kernel<<<unsigned((T + 31) / 32), 32 * kJoinWarps, 0, stream>>>(static_cast<const float2*>(part), (n + kHeadGroup - 1) / kHeadGroup, T,
                                                                            state, first, last, V, ignore, targets, loss, lse, status);
        return noted("cross_entropy_join");
    }

    cudaError_t launchHeadGradient(const HeadProduct& h, int64_t v0, int64_t V, int64_t ignore, const int64_t* targets, const float* lse,
                                   const float* g, float alpha, const float* scale, const Probabilities& P, float* rest, int smCount, int* status,
                                   cudaStream_t stream)
    {
        HeadArgs ea{};
        ea.T = h.T, ea.n = h.n, ea.v0 = v0, ea.V = V, ea.ignore = ignore;
        ea.targets = targets, ea.alpha = alpha, ea.lse = lse, ea.g = g, ea.scale = scale, ea.rest = rest;
        ea.rowsP               = P.rows;
        PFN_encodeTiled encode = tensorMapEncoder();
        if(!encode || !encodeMatrix(encode, &ea.mapP, P.data, h.n, P.parts * P.rows, P.ld, 64, 32))
            return cudaErrorNotSupported;
        const char *name = "cross_entropy_head_gradient", *pairName = "cross_entropy_head_gradient_pair";
        const bool  half = h.type == CUDA_R_16F, narrow = singleTiles(h.T, (h.n + 255) / 256, smsOf(smCount));
        if(P.parts == 3)
            return narrow ? launchHeadForm<ProbabilityEpi<__nv_bfloat16, 3>, false>(h, ea, smCount, status, stream, name)
                          : launchHeadForm<ProbabilityEpi<__nv_bfloat16, 3>, true>(h, ea, smCount, status, stream, pairName);
        if(P.parts == 2) // few tokens, single tiles
            return half ? launchHeadForm<ProbabilityEpi<__half, 2>, false>(h, ea, smCount, status, stream, name)
                        : launchHeadForm<ProbabilityEpi<__nv_bfloat16, 2>, false>(h, ea, smCount, status, stream, name);
        if(narrow)
            return half ? launchHeadForm<ProbabilityEpi<__half, 1>, false>(h, ea, smCount, status, stream, name)
                        : launchHeadForm<ProbabilityEpi<__nv_bfloat16, 1>, false>(h, ea, smCount, status, stream, name);
        return half ? launchHeadForm<ProbabilityEpi<__half, 1>, true>(h, ea, smCount, status, stream, pairName)
                    : launchHeadForm<ProbabilityEpi<__nv_bfloat16, 1>, true>(h, ea, smCount, status, stream, pairName);
    }

    // How many parts of the classes dH's products run in, side by side: the tiles of [T, D] alone would leave SMs idle when
    // there are few, or in their last round when there are some. A round of tiles over n classes takes about n x 5.9 ns
    // (measured rate of a pair), a part more T x D x 8 bytes of traffic; a part's sums have at least 1024 terms. `piece`: classes
    // times the products that an element's product is made of.
    int hiddenParts(int64_t T, int64_t D, int64_t piece, int sms)
    {
        const bool    single = T <= 128;
        const int64_t tiles  = (D + 255) / 256 * (single ? 1 : (T + 255) / 256), units = single ? sms : sms / 2;
        int           best   = 1;
        double        least  = 0;
        for(int parts = 1; parts <= sms && (parts == 1 || parts * 1024 <= piece); parts++)
        {
            const double rounds = double((tiles * parts + units - 1) / units) / parts;
            const double time   = rounds * double(piece) * 5.9e-9 + parts * double(T) * double(D) * 8 / 6.5e12;
            if(parts == 1 || time < least)
            {
                least = time;
                best  = parts;
            }
        }
        return best;
    }

    int64_t hiddenRows(int64_t T)
    {
        return (T + 31) / 32 * 32;
    }

    cudaError_t launchHiddenGradient(const HeadProduct& h, const Probabilities& P, int parts, float* out, int64_t ldo, bool add, int smCount,
                                     int* status, cudaStream_t stream)
    {
        PFN_encodeTiled encode = tensorMapEncoder();
        const bool      narrow = h.T <= 128;
        const int       xRows = narrow ? rowsLoaded(h.T) : 128, segP = h.segments > 1 ? P.parts : 1; // the second part of few tokens is for dW
        CUtensorMap     mapX, mapY;
        if(!encode || !encodeMatrix(encode, &mapX, P.data, h.n, P.parts * P.rows, P.ld, 64, xRows)
           || !encodeMatrix(encode, &mapY, h.W, h.D, h.segments > 1 ? h.segments * h.segW : h.n, h.ldw, 64, 64))
            return cudaErrorNotSupported;
        AccArgs a{};
        if(narrow)
            fillCommon<HiddenEpi, false>(a, h.T, h.D, xRows, h.n * 2 * segP, status);
        else
            fillCommon<HiddenEpi, true>(a, h.T, h.D, xRows, h.n * 2 * segP, status);
        segmentPairs(segP, h.segments, a, int((h.n + 63) / 64));
        a.xSegR = int(P.rows), a.ySegK = int(h.segW);
        a.idesc  = instruction(h.type == CUDA_R_16F, !narrow, false, true);
        a.kParts = std::min(parts, a.kBlocks); // a short last piece: every part has something to add
        HiddenArgs ea{};
        ea.T = h.T, ea.ld = ldo, ea.add = add;
        ea.rows     = hiddenRows(h.T);
        ea.tileRows = int64_t(a.tilesM) * (narrow ? 128 : 256);
        if(!encodeMatrix(encode, &ea.mapOut, out, ldo, parts * ea.rows, ldo, 32, 32, true))
            return cudaErrorNotSupported;
        a.groupM = a.tilesM *= a.kParts;
        return narrow ? launchAccumulate<HiddenEpi, false, false, true>(mapX, mapY, a, ea, smCount, stream, "cross_entropy_hidden")
                      : launchAccumulate<HiddenEpi, true, false, true>(mapX, mapY, a, ea, smCount, stream, "cross_entropy_hidden_pair");
    }

    cudaError_t launchWeightGradient(const HeadProduct& h, const Probabilities& P, int64_t v0, const TokenLists& lists, const float* rest, const float* scale,
                                     int typeOut, void* dW, int64_t ldw, int smCount, int* status, cudaStream_t stream)
    {
        PFN_encodeTiled encode = tensorMapEncoder();
        const bool      wide   = typeOut == CUDA_R_32F;
        WeightArgs      ea{};
        ea.rows = h.n, ea.cols = h.D, ea.scale = scale;
        ea.lists = lists;
        ea.rest = rest, ea.H = static_cast<const unsigned short*>(h.H), ea.ldh = h.ldh, ea.T = h.T, ea.v0 = v0;
        ea.half = h.type == CUDA_R_16F;
        CUtensorMap mapX, mapY;
        // one segment: rows past the tokens are not there (zeros); more: they hold zeros
        if(!encode || !encodeMatrix(encode, &mapX, P.data, h.n, P.parts > 1 ? P.parts * P.rows : h.T, P.ld, 64, 64)
           || !encodeMatrix(encode, &mapY, h.H, h.D, h.segments > 1 ? h.segments * h.segH : h.T, h.ldh, 64, 64)
           || !encodeMatrix(encode, &ea.mapD, dW, h.D, h.n, ldw, wide ? 32 : 64, 32, wide))
            return cudaErrorNotSupported;
        const bool  few  = h.T * P.parts <= 256;
        const char* name = "cross_entropy_weight";
        auto        run  = [&](auto epi) {
            using Epi = decltype(epi);
            AccArgs a{};
            fillCommon<typename Epi::Type, true>(a, h.n, h.D, 128, h.T * 2 * P.parts, status);
            segmentPairs(P.parts, h.segments, a, int((h.T + 63) / 64));
            a.xSegK = int(P.rows), a.ySegK = int(h.segH);
            a.idesc = instruction(h.type == CUDA_R_16F, true, true, true);
            return launchAccumulate<typename Epi::Type, true, true, true>(mapX, mapY, a, ea, smCount, stream, name);
        };
        if(wide)
            return few ? run(Named<WeightEpi<float, 2>>{}) : run(Named<WeightEpi<float, 1>>{});
        if(typeOut == CUDA_R_16F)
            return few ? run(Named<WeightEpi<__half, 2>>{}) : run(Named<WeightEpi<__half, 1>>{});
        return few ? run(Named<WeightEpi<__nv_bfloat16, 2>>{}) : run(Named<WeightEpi<__nv_bfloat16, 1>>{});
    }

    cudaError_t launchPackRows(int type, const void* X, const TokenRows& rows, int64_t count, int64_t total, int64_t cols, int64_t ld, void* X2,
                               const int64_t* targets, int64_t ignore, int64_t V, const TokenLists& lists, int* status, cudaStream_t stream)
    {
        const RowShape  s   = rowShape(total, ld / 8);
        unsigned short* out = static_cast<unsigned short*>(X2);
        if(type == CUDA_R_32F)
            pack_rows_kernel<float, true><<<s.grid, s.block, 0, stream>>>((const float*)X, rows, count, total, cols, ld, out, targets, ignore, V, lists.classes, status,
                                                                          rowsAligned(rows, X, 4, 4));
        else if(type == CUDA_R_16F)
            pack_rows_kernel<__half, false><<<s.grid, s.block, 0, stream>>>((const __half*)X, rows, count, total, cols, ld, out, targets, ignore, V, lists.classes,
                                                                            status, rowsAligned(rows, X, 8, 2));
        else
            pack_rows_kernel<__nv_bfloat16, false><<<s.grid, s.block, 0, stream>>>((const __nv_bfloat16*)X, rows, count, total, cols, ld, out, targets,
                                                                                   ignore, V, lists.classes, status, rowsAligned(rows, X, 8, 2));
        return noted("cross_entropy_pack");
    }

    cudaError_t launchTokenLists(const TokenLists& lists, int64_t T, int64_t V, cudaStream_t stream)
    {
        token_lists_kernel<<<unsigned((V + 31) / 32), 32 * kListWarps, 0, stream>>>(lists, T, V);
        return noted("cross_entropy_lists");
    }

    cudaError_t launchGradientScale(const float* g, float alpha, int64_t T, const int64_t* targets, int64_t ignore, int64_t V, float* scale,
                                    cudaStream_t stream)
    {
        gradient_scale_kernel<<<1, 1024, 0, stream>>>(g, alpha, T, targets, ignore, V, scale);
        return noted("cross_entropy_scale");
    }

    cudaError_t launchStoreRows(int type, const float* X, int64_t ldx, int64_t count, int64_t cols, const float* scale, void* Y,
                                const TokenRows& rows, const TargetRest& rest, int parts, int64_t partRows, cudaStream_t stream)
    {
        const RowShape s   = rowShape(count, (cols + 3) / 4);
        const bool     vec = rowsAligned(rows, Y, 4, type == CUDA_R_32F ? 4 : 2);
        if(type == CUDA_R_32F)
            store_rows_kernel<float><<<s.grid, s.block, 0, stream>>>(X, ldx, count, cols, scale, (float*)Y, rows, rest, parts, partRows, vec);
        else if(type == CUDA_R_16F)
            store_rows_kernel<__half><<<s.grid, s.block, 0, stream>>>(X, ldx, count, cols, scale, (__half*)Y, rows, rest, parts, partRows, vec);
        else
            store_rows_kernel<__nv_bfloat16><<<s.grid, s.block, 0, stream>>>(X, ldx, count, cols, scale, (__nv_bfloat16*)Y, rows, rest, parts, partRows, vec);
        return noted("cross_entropy_store");
    }
} // namespace htb
