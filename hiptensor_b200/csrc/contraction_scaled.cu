// Block-scaled 8-bit contraction: D[m, n] = alpha * sum over blocks of 128 of k of
// scaleA * scaleB * sum_k A[m, k] B[n, k], + beta * C[m, n]; operands e4m3 / e5m2, sums in f32.
//
// The scales forbid to sum over blocks in tensor memory: each block's sums are taken from there, scaled and added in registers
// (accumulate.cuh). What bounds the large products is that hand-over: with two accumulators of 256 columns (all of tensor
// memory), a block costs the start and end of its MMAs (1000 cycles, 512 of them MMAs), the reads with the additions in
// between (540) and the way back to the issuer (350), over two blocks in flight: about 950 cycles. 8192^3 to bf16: 720 us
// one after the other (1.52 PFLOP/s, the card at its power limit), 610 after a pause; the same pipeline without the additions
// takes 400. A scale per column as well (weight gradients) doubles the additions, which then bound it: 8192^3 820 to 850 us,
// 4096 x 4096 x 8192 added to f32 280 (1.0 PFLOP/s). Narrow tiles are bound by what an
// SM loads (about 39 bytes a cycle): few tokens are cut along K over clusters to load with more SMs (4096 x 4096: 1 token
// 10.7 us, 128 tokens 12.6). Operands that no such load can read take the FMA kernel: 4096^3 8.1 ms, 777 x 2057 x 1001 262 us
// (18 in rows of whole 16-byte words).
#include <cuda_fp8.h>

#include <algorithm>

#include "accumulate.cuh"
#include "convert.cuh"
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
        // Any strides and extents: 64 x 64 tiles, 16 x 16 threads with 4 x 4 results each, byte loads into shared memory as
        // f32, FMA. A block's products are summed by themselves and scaled once.
        template <typename TD>
        __global__ void __launch_bounds__(256) scaled_simt_kernel(const unsigned char* __restrict__ A, const float* __restrict__ sA,
                                                                  const unsigned char* __restrict__ B, const float* __restrict__ sB,
                                                                  const TD* C, TD* D, float alpha, float beta, const __grid_constant__ ScaledPlan p)
        {
            constexpr int    kStep = 32;
            __shared__ float a[kStep][65], b[kStep][65];
            const int        tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
            const bool       aWide = p.typeA == CUDA_R_8F_E5M2, bWide = p.typeB == CUDA_R_8F_E5M2;
            const int64_t    m0 = int64_t(blockIdx.x) * 64;
            for(int64_t n0 = int64_t(blockIdx.y) * 64; n0 < p.N; n0 += int64_t(gridDim.y) * 64)
            {
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
                            sum[i][j] = fmaf(part[i][j], x[i] * y[j], sum[i][j]);
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
        }

        // ------------------------------------------------------------------ tensor-core path
        struct ScaledArgs
        {
            const float *sX, *sY; // scales of the operand on the rows' / columns' side of the tiles
            int64_t      sxRow, sxK, syRow, syK;
            int          blockX, blockY;
            int          quadX, quadY; // scales of four blocks in one aligned 16-byte word
            int64_t      rows, cols; // of the product
            const void*  C;
            void*        D;
            int64_t      dRow, dCol;
            float        alpha, beta;
            int          vec; // columns contiguous
            int          tma; // the result goes out as bulk tensor stores (no C; rows at multiples of 16 bytes)
            CUtensorMap  mapD, mapC;
        };

        // Epilogue of accumulate_kernel: a chunk is one block of 128 along k. A thread multiplies the block's sums of its row by
        // scaleX (one per row and block) and scaleY (VECY: one per column and block; else one for 128 columns) and adds
        // them to its running sums, two columns per instruction. Both come through the side ring: 128 rows, then TN
        // columns (VECY) or the two halves of the columns.
        // BULK: the result goes out as bulk tensor stores; WITHC: C comes in by bulk loads, too.
        template <typename TD, int TN, bool VECY, bool BULK, bool WITHC>
        struct ScaledEpi
        {
            using Args                 = ScaledArgs;
            static constexpr int COLS  = TN / 2;
            static constexpr int CH    = COLS < 32 ? COLS : 32; // columns per round of stores
            static constexpr int CL    = (VECY && COLS == 128) ? 16 : CH; // columns per load from tensor memory, as registers allow
            static constexpr int kSide = 128 + (VECY ? TN : 4);
            // K blocks whose scales are fetched together: a fetch takes a trip to memory, and narrow tiles need a block's every
            // few hundred cycles
            static constexpr int kGroup = TN <= 64 ? 16 : (VECY ? 8 : 4);
            static constexpr int SLOTS = 2; // of 4 KiB, per warp, for the result
            static constexpr bool kSplit = !BULK;
            static constexpr bool kParted = false;
            static constexpr int BYTES = kSideSlots * kGroup * kSide * 4; // of the ring, in front of them
            static constexpr int ROUND = 128 / int(sizeof(TD)); // columns of a slot: rows of 128 bytes

            // Scales along k are mostly contiguous (sxK == 1): four blocks come as one 16-byte load, one value at a time would
            // touch a line per row and block, more lines than fit beside the shared memory (4096^3 with a scale per
            // column: 218 us). Batches of four loads, then four stores each into the rows of the ring.
            struct Side
            {
                const Args& a;
                const int   lane;
                int64_t     row, col;

                __device__ Side(const Args& args, int l)
                    : a(args)
                    , lane(l)
                {
                }
                __device__ __forceinline__ void begin(int64_t r, int64_t c)
                {
                    row = r + lane;
                    col = VECY ? c + lane : c + (lane & 1) * COLS;
                }
                // values kb .. end - 1 of N rows (32 apart from `first`) into ring[kb % group][at + 32 i + lane]
                template <int N>
                __device__ __forceinline__ void batch(float* ring, int at, const float* src, int64_t first, int64_t limit, int block, int64_t sRow,
                                                      int64_t sK, bool quad, int kb, int end, bool mine)
                {
                    float v[N][kGroup];
#pragma unroll
                    for(int i = 0; i < N; i++)
                    {
                        const int64_t r = first + i * 32;
                        const float*  p = src + (block > 1 ? r / kScaleBlock : r) * sRow + kb * sK;
#pragma unroll
                        for(int j = 0; j < kGroup; j += 4)
                        {
                            float4 q = make_float4(0.f, 0.f, 0.f, 0.f); // rows and columns past the result
                            if(mine && r < limit && kb + j < end)
                            {
                                // (a group begins at a multiple of four blocks unless a K split cuts it)
                                if(quad && kb + j + 4 <= end && (kb & 3) == 0)
                                    q = __ldg(reinterpret_cast<const float4*>(p + j));
                                else
                                {
                                    q.x = __ldg(p + j * sK);
                                    if(kb + j + 1 < end)
                                        q.y = __ldg(p + (j + 1) * sK);
                                    if(kb + j + 2 < end)
                                        q.z = __ldg(p + (j + 2) * sK);
                                    if(kb + j + 3 < end)
                                        q.w = __ldg(p + (j + 3) * sK);
                                }
                            }
                            v[i][j] = q.x, v[i][j + 1] = q.y, v[i][j + 2] = q.z, v[i][j + 3] = q.w;
                        }
                    }
                    if(!mine)
                        return;
#pragma unroll
                    for(int i = 0; i < N; i++)
#pragma unroll
                        for(int j = 0; j < kGroup; j++)
                            if(kb + j < end)
                                ring[(kb % kGroup + j) * kSide + at + i * 32 + lane] = v[i][j];
                }
                __device__ __forceinline__ void fetch(float* ring, int kb, int end)
                {
                    batch<4>(ring, 0, a.sX, row, a.rows, a.blockX, a.sxRow, a.sxK, a.quadX != 0, kb, end, true);
                    if constexpr(VECY)
                    {
                        constexpr int N = TN / 32 < 4 ? TN / 32 : 4;
#pragma unroll 1
                        for(int i = 0; i < TN / 32; i += N)
                            batch<N>(ring, 128 + i * 32, a.sY, col + i * 32, a.cols, 1, a.syRow, a.syK, a.quadY != 0, kb, end, true);
                    }
                    else
                        batch<1>(ring, 128, a.sY, col, a.cols, kScaleBlock, a.syRow, a.syK, a.quadY != 0, kb, end, lane < 2);
                }
            };

            const Args&  a;
            const int    lane;
            float*       slot;
            int          stores; // bulk stores of this warp so far, they take the slots in turn
            volatile int* abort;
            uint32_t     bar;
            const float* ys;
            uint64_t     s;
            uint64_t     acc[COLS / 2];

            __device__ ScaledEpi(const Args& args, int w, int l, unsigned char* smem, volatile int* abortFlag)
                : a(args)
                , lane(l)
                , slot(reinterpret_cast<float*>(smem + (BYTES + 1023) / 1024 * 1024 + w * (SLOTS * 4096)))
                , stores(0)
                , abort(abortFlag)
            {
                if constexpr(WITHC)
                {
                    // one barrier for each slot: C's blocks on their way into it
                    __shared__ __align__(8) unsigned long long bars[8 * SLOTS];
                    bar = smemAddr(&bars[w * SLOTS]);
                    if(l == 0)
                    {
                        for(int i = 0; i < SLOTS; i++)
                            mbarInit(bar + 8 * i, 1);
                        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
                    }
                    __syncwarp();
                }
            }
            __device__ __forceinline__ void begin(int64_t)
            {
#pragma unroll
                for(int j = 0; j < COLS / 2; j++)
                    acc[j] = 0;
            }
            __device__ __forceinline__ void side(const float* v, int row, int half)
            {
                const float x = v[row];
                ys            = v + 128 + half * COLS;
                const float m = VECY ? x : x * v[128 + half];
                s             = pack2(m, m);
            }
            template <class Release>
            __device__ __forceinline__ void add(uint32_t taddr, bool, Release release)
            {
                auto scaleAdd = [&](const uint32_t(&v)[CL], int c) {
#pragma unroll
                    for(int j = 0; j < CL; j += 4)
                    {
                        uint64_t s0 = s, s1 = s;
                        if constexpr(VECY)
                        {
                            const float4 q = *reinterpret_cast<const float4*>(ys + c + j);
                            s0             = mul2(s, pack2(q.x, q.y));
                            s1             = mul2(s, pack2(q.z, q.w));
                        }
                        acc[(c + j) / 2]     = fma2(pack2(v[j], v[j + 1]), s0, acc[(c + j) / 2]);
                        acc[(c + j) / 2 + 1] = fma2(pack2(v[j + 2], v[j + 3]), s1, acc[(c + j) / 2 + 1]);
                    }
                };
                // Two loads at a time (a wait is for all that are on their way), the next two behind the first additions
                uint32_t v0[CL], v1[CL];
                tmemLoad<CL>(taddr, v0);
                if constexpr(CL < COLS)
                    tmemLoad<CL>(taddr + CL, v1);
#pragma unroll
                for(int c = 0; c < COLS; c += 2 * CL)
                {
                    tmemWait();
                    if(c + 2 * CL >= COLS)
                        release();
                    scaleAdd(v0, c);
                    if(c + 2 * CL < COLS)
                        tmemLoad<CL>(taddr + c + 2 * CL, v0);
                    if(c + CL < COLS)
                        scaleAdd(v1, c + CL);
                    if(c + 3 * CL < COLS)
                        tmemLoad<CL>(taddr + c + 3 * CL, v1);
                }
            }
            __device__ __forceinline__ float sum(int j) const
            {
                const float2 f = unpack2(acc[j / 2]);
                return (j & 1) ? f.y : f.x;
            }
            static __device__ __forceinline__ TD finish(const Args& a, float v, int64_t at)
            {
                v *= a.alpha;
                return narrow<TD>(a.C ? fmaf(a.beta, widen(static_cast<const TD*>(a.C)[at]), v) : v);
            }
            // Columns col0 .. col0 + W - 1 of row `row` as they are: neighbouring lanes write neighbouring rows
            template <int W>
            __device__ __forceinline__ void storeDirect(const float (&w)[W], int64_t row, int64_t col0)
            {
                if(row >= a.rows)
                    return;
                int64_t at = row * a.dRow + col0 * a.dCol;
#pragma unroll
                for(int j = 0; j < W; j++, at += a.dCol)
                    if(col0 + j < a.cols)
                        static_cast<TD*>(a.D)[at] = finish(a, w[j], at);
            }
            // The same through shared memory when the columns are contiguous: lanes that follow each other write (and read C)
            // along a row, one element each, so that any row stride and start will do (rows of odd length: 4096 x 4097 x 4096
            // in bf16 takes 120 us, 260 with every lane on a row of its own; 87 by bulk stores
            // when N is 4096). Eight rows' worth of C is read ahead of their stores.
            template <int W>
            __device__ __forceinline__ void store(const float (&w)[W], int64_t row, int64_t col0)
            {
                constexpr int U = W / 4, STEP = 32 / W; // 16-byte units of a row, XORed with the row against bank conflicts; rows at a time
                __syncwarp(); // the round before has been read
#pragma unroll
                for(int u = 0; u < U; u++)
                    *reinterpret_cast<float4*>(slot + lane * W + ((u ^ (lane & (U - 1))) << 2))
                        = make_float4(w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
                __syncwarp();
                const int     j = lane % W, first = lane / W;
                const int64_t row0 = row - lane, c = col0 + j;
                const int     rows = int(min(int64_t(32), a.rows - row0)); // may be negative
                if(c >= a.cols)
                    return;
                int64_t at = (row0 + first) * a.dRow + c;
                TD*     D  = static_cast<TD*>(a.D);
#pragma unroll 1
                for(int r = first; r < rows; r += 8 * STEP)
                {
                    TD in[8];
                    if(a.C)
                    {
#pragma unroll
                        for(int i = 0; i < 8; i++)
                            if(r + i * STEP < rows)
                                in[i] = static_cast<const TD*>(a.C)[at + i * STEP * a.dRow];
                    }
#pragma unroll
                    for(int i = 0; i < 8; i++)
                    {
                        const int rr = r + i * STEP;
                        if(rr < rows)
                        {
                            const float v = slot[rr * W + ((((j >> 2) ^ (rr & (U - 1))) << 2) | (j & 3))] * a.alpha;
                            D[at]         = narrow<TD>(a.C ? fmaf(a.beta, widen(in[i]), v) : v);
                        }
                        at += STEP * a.dRow;
                    }
                }
            }
            // lane 0: fetches C's block of columns col .. of the warp's rows into the slot of bulk store number n
            __device__ __forceinline__ void fetchC(int n, int64_t row, int64_t col)
            {
                const uint32_t b = bar + uint32_t(n % SLOTS) * 8u;
                if(row < a.rows && col < a.cols)
                {
                    mbarArriveExpectTx(b, 4096);
                    const int c[2] = {int(col), int(row)};
                    tmaLoad<2>(smemAddr(slot) + uint32_t((n % SLOTS) * 4096), &a.mapC, b, c);
                }
                else
                    mbarArrive(b);
            }
            // A slot of 32 rows x 128 bytes, 16-byte units permuted as the tensor map's 128-byte swizzle has them, and one
            // bulk store of it: the tile leaves while the next one is summed. With C (mapC), the slot holds C's block first.
            __device__ __forceinline__ void bulkStore(int c, int64_t row, int64_t col)
            {
                const uint32_t at = smemAddr(slot) + uint32_t((stores % SLOTS) * 4096), line = at + uint32_t(lane * 128);
                if constexpr(WITHC)
                    mbarWaitTight(bar + uint32_t(stores % SLOTS) * 8u, uint32_t(stores / SLOTS) & 1u, abort);
                else
                {
                    if(lane == 0)
                        asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(SLOTS - 1) : "memory"); // the slot's last store has read it
                }
                __syncwarp();
                stores++;
#pragma unroll
                for(int u = 0; u < 8; u++)
                {
                    constexpr int  PER  = 16 / int(sizeof(TD)); // columns of a unit
                    const uint32_t unit = line + uint32_t((u ^ (lane & 7)) << 4);
                    __align__(16) TD e[PER];
                    if constexpr(WITHC)
                    {
                        uint32_t q[4];
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]) : "r"(unit) : "memory");
                        const TD* in = reinterpret_cast<const TD*>(q);
#pragma unroll
                        for(int j = 0; j < PER; j++)
                            e[j] = narrow<TD>(fmaf(a.beta, widen(in[j]), sum(c + PER * u + j) * a.alpha));
                    }
                    else
                    {
#pragma unroll
                        for(int j = 0; j < PER; j++)
                            e[j] = narrow<TD>(sum(c + PER * u + j) * a.alpha);
                    }
                    const uint32_t* q = reinterpret_cast<const uint32_t*>(e);
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(unit), "r"(q[0]), "r"(q[1]), "r"(q[2]), "r"(q[3]) : "memory");
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if(lane == 0)
                {
                    // a block that begins outside the result has nothing to store (one that ends outside is clipped)
                    if(row < a.rows && col + c < a.cols)
                        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(&a.mapD), "r"(at),
                                     "r"(int(col + c)), "r"(int(row))
                                     : "memory");
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    if(WITHC && c + SLOTS * ROUND < COLS)
                    {
                        // the block after the next one, into this slot
                        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                        fetchC(stores + SLOTS - 1, row, col + c + SLOTS * ROUND);
                    }
                }
            }
            __device__ __forceinline__ void end(int64_t row, int64_t col)
            {
                if constexpr(BULK)
                {
                    if(WITHC && lane == 0)
                    {
                        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); // the slots are free
                        for(int i = 0; i < SLOTS && i * ROUND < COLS; i++)
                            fetchC(stores + i, row, col + i * ROUND);
                    }
#pragma unroll
                    for(int c = 0; c < COLS; c += ROUND)
                        bulkStore(c, row, col);
                }
                else
                {
#pragma unroll
                    for(int c = 0; c < COLS; c += CH)
                    {
                        float w[CH];
#pragma unroll
                        for(int j = 0; j < CH; j++)
                            w[j] = sum(c + j);
                        if(!a.vec)
                            storeDirect<CH>(w, row, col + c);
                        else
                            store<CH>(w, row, col + c);
                    }
                }
            }
            // before the block ends: the bulk stores have read their slots
            __device__ __forceinline__ void leave()
            {
                if(lane == 0) // (nothing to wait for where none was issued)
                    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            }
            // 32 rows of W columns by one bulk store, rows packed in a slot (a K split's results: the map's box is W wide)
            template <int W>
            __device__ __forceinline__ void bulkBlock(const float (&w)[W], int64_t row, int64_t col)
            {
                const uint32_t at = smemAddr(slot) + uint32_t((stores % SLOTS) * 4096);
                if(lane == 0)
                    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(SLOTS - 1) : "memory");
                __syncwarp();
                stores++;
                constexpr int PER = 16 / int(sizeof(TD)); // columns of a 16-byte word
#pragma unroll
                for(int u = 0; u < W / PER; u++)
                {
                    TD e[PER];
#pragma unroll
                    for(int j = 0; j < PER; j++)
                        e[j] = narrow<TD>(w[u * PER + j] * a.alpha);
                    const uint32_t* q = reinterpret_cast<const uint32_t*>(e);
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + uint32_t(lane * (W * int(sizeof(TD))) + u * 16)), "r"(q[0]),
                                 "r"(q[1]), "r"(q[2]), "r"(q[3])
                                 : "memory");
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if(lane == 0)
                {
                    if(row < a.rows && col < a.cols)
                        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(&a.mapD), "r"(at),
                                     "r"(int(col)), "r"(int(row))
                                     : "memory");
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                }
            }
            // K split over KS = 2 or 4 CTAs: CTA q finishes columns q TN / KS .. of the tile. A thread's columns are KS / 2 slices,
            // each of one CTA. Exchange zone in the stages of CTA q: [sending rank][four columns][128 rows] of 16 bytes.
            template <int KS>
            __device__ __forceinline__ void sendTo(uint32_t zone, uint32_t rank, int row, int half)
            {
                constexpr int WIDE = TN / KS, SLICES = KS / 2;
#pragma unroll
                for(int s = 0; s < SLICES; s++)
                {
                    const uint32_t q = uint32_t(half * SLICES + s);
                    if(q == rank)
                        continue;
                    const uint32_t dst = mapToRank(zone + rank * uint32_t(WIDE * 512) + uint32_t(row) * 16u, q);
#pragma unroll
                    for(int j = 0; j < WIDE; j += 4)
                    {
                        const float2 x = unpack2(acc[(s * WIDE + j) / 2]), y = unpack2(acc[(s * WIDE + j) / 2 + 1]);
                        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dst + uint32_t(j / 4) * 2048u), "f"(x.x), "f"(x.y),
                                     "f"(y.x), "f"(y.y)
                                     : "memory");
                    }
                }
            }
            template <int KS>
            __device__ __forceinline__ void finishSplit(uint32_t zone, uint32_t rank, int row, int half, int64_t r, int64_t col0)
            {
                constexpr int WIDE = TN / KS, SLICES = KS / 2, W = WIDE < 32 ? WIDE : 32;
#pragma unroll
                for(int s = 0; s < SLICES; s++)
                {
                    if(uint32_t(half * SLICES + s) != rank)
                        continue;
#pragma unroll
                    for(int c = 0; c < WIDE; c += W)
                    {
                        float w[W];
#pragma unroll
                        for(int j = 0; j < W; j += 4)
                        {
                            float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                            for(int q = 0; q < KS; q++) // in the order of the ranks
                            {
                                const float2 x = unpack2(acc[(s * WIDE + c + j) / 2]), y = unpack2(acc[(s * WIDE + c + j) / 2 + 1]);
                                float4       v = make_float4(x.x, x.y, y.x, y.y);
                                if(uint32_t(q) != rank)
                                    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                                                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                                                 : "r"(zone + uint32_t(q * WIDE * 512) + uint32_t((c + j) / 4) * 2048u + uint32_t(row) * 16u)
                                                 : "memory");
                                t = make_float4(t.x + v.x, t.y + v.y, t.z + v.z, t.w + v.w);
                            }
                            w[j] = t.x, w[j + 1] = t.y, w[j + 2] = t.z, w[j + 3] = t.w;
                        }
                        const int64_t col = col0 + half * COLS + s * WIDE + c;
                        if(!a.vec)
                            storeDirect<W>(w, r, col);
                        else if(a.tma)
                            bulkBlock<W>(w, r, col);
                        else
                            store<W>(w, r, col);
                    }
                }
            }
            __device__ __forceinline__ void send(uint32_t zone, uint32_t rank, int ksplit, int row, int half)
            {
                if(ksplit == 2)
                    sendTo<2>(zone, rank, row, half);
                else
                    sendTo<4>(zone, rank, row, half);
            }
            __device__ __forceinline__ void endSplit(uint32_t zone, uint32_t rank, int ksplit, int row, int half, int64_t r, int64_t col0)
            {
                if(ksplit == 2)
                    finishSplit<2>(zone, rank, row, half, r, col0);
                else
                    finishSplit<4>(zone, rank, row, half, r, col0);
            }
        };

        bool encodeRows(PFN_encodeTiled encode, CUtensorMap* map, const void* base, int64_t k, int64_t rows, int64_t stride, int box)
        {
            cuuint64_t gdim[2] = {cuuint64_t(k), cuuint64_t(rows)}, gstr[1] = {rows > 1 ? cuuint64_t(stride) : cuuint64_t((k + 15) / 16 * 16)};
            cuuint32_t bx[2] = {128, cuuint32_t(box)}, estr[2] = {1, 1};
            return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), gdim, gstr, bx, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE)
                   == CUDA_SUCCESS;
        }
        // box: 32 rows of `boxCols` columns, or (0) of 128 bytes in the swizzled layout
        bool encodeResult(PFN_encodeTiled encode, CUtensorMap* map, int type, void* base, int64_t cols, int64_t rows, int64_t strideBytes, int boxCols)
        {
            const bool wide    = type == CUDA_R_32F;
            cuuint64_t gdim[2] = {cuuint64_t(cols), cuuint64_t(rows)}, gstr[1] = {cuuint64_t(strideBytes)};
            cuuint32_t bx[2] = {boxCols ? cuuint32_t(boxCols) : (wide ? 32u : 64u), 32}, estr[2] = {1, 1};
            return encode(map, wide ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, base, gdim, gstr, bx, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, boxCols ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE)
                   == CUDA_SUCCESS;
        }
        // rows contiguous along k, starting at multiples of 16 bytes, no two of them in one place
        bool rowsForTma(const void* base, int64_t k, int64_t rows, int64_t sK, int64_t sRow)
        {
            return (uintptr_t(base) & 15) == 0 && (sK == 1 || k == 1)
                   && (rows == 1 || (sRow % 16 == 0 && sRow >= k && sRow < (int64_t(1) << 40)));
        }

        // which kernel a problem runs on
        struct ScaledForm
        {
            bool swap; // B on the rows' side of the tiles
            bool pair;
            int  tn, ksplit;
        };
        ScaledForm formOf(const ScaledPlan& p, int sms)
        {
            ScaledForm    f{};
            const int64_t kb = (p.K + 127) / 128, small = std::min(p.M, p.N);
            // few rows on one side (a token, a few of them): that side becomes the columns of narrow tiles, the other
            // one, the weights, fills the 128 rows
            if(small <= 64)
            {
                f.swap = p.M < p.N;
                f.tn   = small <= 32 ? 32 : 64;
            }
            else
            {
                f.swap = p.dN != 1 && p.dM == 1; // the result contiguous along the columns of the tiles
                f.pair = ((p.M + 255) / 256) * ((p.N + 255) / 256) >= sms / 2 * 3 / 4;
                f.tn   = f.pair ? 256 : 128;
            }
            f.ksplit            = 1;
            const int64_t tiles = f.pair ? 0 : ((f.swap ? p.N : p.M) + 127) / 128 * (((f.swap ? p.M : p.N) + f.tn - 1) / f.tn);
            while(!f.pair && f.ksplit < 4 && tiles * f.ksplit * 2 <= sms && kb >= f.ksplit * 4)
                f.ksplit *= 2;
            return f;
        }

        template <typename TD, bool PAIR, int TN, bool VECY, bool BULK, bool WITHC = false>
        cudaError_t launchTensor(const CUtensorMap& mapX, const CUtensorMap& mapY, AccArgs a, const ScaledArgs& ea, int smCount,
                                 cudaStream_t stream)
        {
            using Epi               = ScaledEpi<TD, TN, VECY, BULK, WITHC>;
            auto           kernel   = accumulate_kernel<Epi, PAIR, TN, true>;
            constexpr uint32_t stage = 16384u + (PAIR ? 128u : uint32_t(TN)) * 128u;
            // the ring of scales, two slots of 4 KiB per warp for the result, and room to align the stages
            constexpr uint32_t room = (Epi::BYTES + 1023) / 1024 * 1024 + 8 * Epi::SLOTS * 4096 + 1024;
            a.stages                = std::min<int>(kAccMaxStages, int((226 * 1024 - room) / stage)) & ~1; // even: see the issuers
            static_assert((226 * 1024 - room) / stage >= 4, "as many stages as accumulators");
            const size_t smem       = size_t(a.stages) * stage + room;
            static const cudaError_t regs = accCheckRegs((const void*)kernel, TN);
            if(regs != cudaSuccess)
                return regs;
            if(cudaError_t e = ensureDynamicSmem((const void*)kernel, int(smem)))
                return e;
            a.xRows                   = 128;
            a.yRows                   = PAIR ? 128 : std::min(TN, (int(std::min<int64_t>(ea.cols, TN)) + 7) / 8 * 8); // no more than there are
            a.stageBytes              = uint32_t(a.stages) * stage;
            const int           csize = PAIR ? 2 : a.ksplit;
            cudaLaunchConfig_t  cfg{};
            cudaLaunchAttribute attr[2];
            attr[0].id                                         = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x                           = unsigned(csize);
            attr[0].val.clusterDim.y                           = 1;
            attr[0].val.clusterDim.z                           = 1;
            attr[1].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr[1].val.programmaticStreamSerializationAllowed = 1;
            const int64_t units                                = int64_t(a.tilesM) * a.tilesN;
            // a split tile is a cluster's only one; else the grid is resident and walks the tiles
            cfg.gridDim          = dim3(unsigned(csize * (a.ksplit > 1 ? units : std::min<int64_t>(units, smCount / csize))));
            cfg.blockDim         = dim3(kAccThreads);
            cfg.dynamicSmemBytes = smem;
            cfg.stream           = stream;
            cfg.attrs            = attr;
            cfg.numAttrs         = 2;
            cudaError_t e        = cudaLaunchKernelEx(&cfg, kernel, mapX, mapY, a, ea);
            if(e == cudaSuccess)
                noteLaunch(PAIR ? "scaled_pair" : "scaled_tile");
            return e;
        }

        template <typename TD, bool VECY>
        cudaError_t launchForm(const ScaledForm& f, const CUtensorMap& mapX, const CUtensorMap& mapY, const AccArgs& a,
                               const ScaledArgs& ea, int smCount, cudaStream_t stream)
        {
            if(f.pair)
                return !ea.tma ? launchTensor<TD, true, 256, VECY, false>(mapX, mapY, a, ea, smCount, stream)
                       : ea.C  ? launchTensor<TD, true, 256, VECY, true, true>(mapX, mapY, a, ea, smCount, stream)
                               : launchTensor<TD, true, 256, VECY, true>(mapX, mapY, a, ea, smCount, stream);
            if(f.tn == 128)
                return !ea.tma || f.ksplit > 1 ? launchTensor<TD, false, 128, VECY, false>(mapX, mapY, a, ea, smCount, stream)
                       : ea.C                  ? launchTensor<TD, false, 128, VECY, true, true>(mapX, mapY, a, ea, smCount, stream)
                                               : launchTensor<TD, false, 128, VECY, true>(mapX, mapY, a, ea, smCount, stream);
            if(f.tn == 64)
                return launchTensor<TD, false, 64, VECY, false>(mapX, mapY, a, ea, smCount, stream);
            return launchTensor<TD, false, 32, VECY, false>(mapX, mapY, a, ea, smCount, stream);
        }

        template <typename TD>
        cudaError_t launchTyped(const ScaledPlan& p, float alpha, const void* A, const float* sA, const void* B, const float* sB,
                                float beta, const void* C, void* D, int smCount, int* status, cudaStream_t stream)
        {
            const int sms = smCount > 0 ? smCount : 148;
            PFN_encodeTiled encode = tensorMapEncoder();
            // (a fold of modes may have more rows than a tensor map's coordinates reach)
            const int64_t most = (int64_t(1) << 31) - 512;
            if(encode && p.K > 0 && p.M < most && p.N < most && rowsForTma(A, p.K, p.M, p.aK, p.aM) && rowsForTma(B, p.K, p.N, p.bK, p.bN))
            {
                const ScaledForm f = formOf(p, sms);
                CUtensorMap      mapX, mapY;
                const int64_t    rows = f.swap ? p.N : p.M, cols = f.swap ? p.M : p.N, tileRows = f.pair ? 256 : 128;
                const int        rowsX = 128, rowsY = f.pair ? 128 : std::min(f.tn, (int(std::min<int64_t>(cols, f.tn)) + 7) / 8 * 8);
                const bool       ok = f.swap ? (encodeRows(encode, &mapX, B, p.K, p.N, p.bN, rowsX) && encodeRows(encode, &mapY, A, p.K, p.M, p.aM, rowsY))
                                             : (encodeRows(encode, &mapX, A, p.K, p.M, p.aM, rowsX) && encodeRows(encode, &mapY, B, p.K, p.N, p.bN, rowsY));
                const int64_t    tilesM = (rows + tileRows - 1) / tileRows, tilesN = (cols + f.tn - 1) / f.tn;
                if(ok && tilesM * tilesN < (int64_t(1) << 30))
                {
                    AccArgs a{};
                    a.tilesM     = int(tilesM);
                    a.tilesN     = int(tilesN);
                    a.kBlocks    = int((p.K + 127) / 128);
                    a.chunk      = 1;
                    a.sub        = 1;
                    a.kParts     = 1;
                    a.kElems     = 128;
                    a.ksplit     = f.ksplit;
                    a.groupM     = int(std::max<int64_t>(1, std::min<int64_t>(tilesM, (int64_t(32) << 20) / (tileRows * p.K))));
                    a.status     = status;
                    a.statusCode = kStatusScaled;
                    // f32 sums; formats of X and Y (0 e4m3, 1 e5m2); N / 8; M / 16
                    const int tX = f.swap ? p.typeB : p.typeA, tY = f.swap ? p.typeA : p.typeB;
                    a.idesc = (1u << 4) | (tX == CUDA_R_8F_E5M2 ? 1u << 7 : 0u) | (tY == CUDA_R_8F_E5M2 ? 1u << 10 : 0u)
                              | (uint32_t(f.tn >> 3) << 17) | (uint32_t(tileRows >> 4) << 24);
                    ScaledArgs ea{};
                    ea.sX = f.swap ? sB : sA, ea.sY = f.swap ? sA : sB;
                    ea.sxRow = f.swap ? p.sbN : p.saM, ea.sxK = f.swap ? p.sbK : p.saK;
                    ea.syRow = f.swap ? p.saM : p.sbN, ea.syK = f.swap ? p.saK : p.sbK;
                    auto quad = [](const float* s, int64_t sRow, int64_t sK) { return sK == 1 && sRow % 4 == 0 && (uintptr_t(s) & 15) == 0; };
                    ea.quadX = quad(ea.sX, ea.sxRow, ea.sxK), ea.quadY = quad(ea.sY, ea.syRow, ea.syK);
                    ea.blockX = f.swap ? p.blockN : p.blockM, ea.blockY = f.swap ? p.blockM : p.blockN;
                    ea.rows = rows, ea.cols = cols;
                    ea.C = C, ea.D = D;
                    ea.dRow = f.swap ? p.dN : p.dM, ea.dCol = f.swap ? p.dM : p.dN;
                    ea.alpha = alpha, ea.beta = beta;
                    ea.vec = ea.dCol == 1 || cols == 1;
                    // bulk stores: the wide forms (a slot's row is 128 bytes of the result) and, without C, K splits
                    // (not where a row ends inside 16 bytes: a bulk store writes all of them, into what lies behind the row)
                    const int64_t size = int64_t(sizeof(TD)), ld = rows > 1 ? ea.dRow : (cols + 15) / 16 * 16;
                    const int boxCols = f.ksplit > 1 ? std::min(f.tn / f.ksplit, 32) : 0;
                    ea.tma = (f.tn >= 128 || f.ksplit > 1) && (!C || f.ksplit == 1) && (ea.dCol == 1 || cols == 1) && ld * size % 16 == 0 && cols * size % 16 == 0 && ld >= cols
                             && ld < (int64_t(1) << 36) && ((uintptr_t(D) | uintptr_t(C)) & 15) == 0 && encodeResult(encode, &ea.mapD, p.typeD, D, cols, rows, ld * size, boxCols)
                             && (!C || encodeResult(encode, &ea.mapC, p.typeD, const_cast<void*>(C), cols, rows, ld * size, 0));
                    return ea.blockY > 1 ? launchForm<TD, false>(f, mapX, mapY, a, ea, sms, stream)
                                         : launchForm<TD, true>(f, mapX, mapY, a, ea, sms, stream);
                }
            }
            const int64_t gx = (p.M + 63) / 64, gy = std::min<int64_t>((p.N + 63) / 64, 65535);
            if(gx > 0x7fffffffll)
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
        switch(p.typeD)
        {
        case CUDA_R_32F: return launchTyped<float>(p, alpha, A, scaleA, B, scaleB, beta, C, D, smCount, deviceStatus, stream);
        case CUDA_R_16F: return launchTyped<__half>(p, alpha, A, scaleA, B, scaleB, beta, C, D, smCount, deviceStatus, stream);
        case CUDA_R_16BF: return launchTyped<__nv_bfloat16>(p, alpha, A, scaleA, B, scaleB, beta, C, D, smCount, deviceStatus, stream);
        }
        return cudaErrorNotSupported;
    }
} // namespace htb
