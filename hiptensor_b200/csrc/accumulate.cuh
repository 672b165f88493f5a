// Pipeline shared by the block-scaled 8-bit contraction and the cross-entropy kernels: tiles of X Y^T (two K-major matrices)
// on the 5th-generation tensor cores whose sums are carried on in REGISTERS. The K range of a tile is cut into chunks; each
// chunk is summed in tensor memory from zero and then added to the running sums of the epilogue threads:
//   * 8-bit operands with scales per block of 128: a chunk is one block, its sums are multiplied by the block's scales on
//     the way;
//   * half-precision operands: the tensor cores truncate when they add a product sum to an accumulator (measured: sums over
//     4096 elements are short by 3.6e-6 of their value), so a long sum is made of chunks of 1024 whose sums are added with
//     rounding.
//
// Roles: warp 0 loads by TMA, one thread of warp 1 (8 bit: of warps 1 and 2) issues the MMAs, warp 3 fetches scales, warps 4 .. 11 are the epilogue. Tensor memory holds two
// chunks or four: while one is read, the next are summed. Epilogue warp w reads lanes 32 (w % 4) .. + 31 (rows of the tile) and half
// (w - 4) / 4 of the columns, so a thread owns one row and TN / 2 neighbouring columns of the tile.
//
// PAIR: two CTAs work on a 256 x 256 tile (cta_group::2), each with 128 rows of X and half of the 256 rows of Y in shared
// memory; halves what a CTA loads for Y. Otherwise a CTA has a 128 x TN tile, and a cluster of `ksplit` CTAs may cut a
// tile's K range.
#pragma once

#include "tcgen05_util.cuh"

namespace htb
{
    namespace
    {
        constexpr int kAccThreads = 384; // three warpgroups: loads and MMAs, two of the epilogue
        constexpr int kAccEpi     = 256; // epilogue threads
        // Registers a thread: 168 at launch (384 x 168 = 64512 of the SM's 65536). Wide tiles need more for the running sums:
        // the first warpgroup gives some back, the epilogue takes them: 128 x 72 + 256 x 216 = 64512.
        constexpr int kAccRegs = 168, kAccRegsLoad = 72, kAccRegsEpi = 216;
        static_assert(128 * kAccRegsLoad + 256 * kAccRegsEpi <= kAccThreads * kAccRegs, "the shares exceed what the launch has");
        constexpr int kAccMaxStages = 16;
        constexpr int kSideSlots    = 2; // groups of Epi::kGroup K blocks in the side ring

        struct AccArgs
        {
            int      tilesM, tilesN; // tiles of (PAIR ? 256 : 128) rows and TN columns
            int      groupM; // tiles of M that are walked together, for the sake of L2
            int      kBlocks; // 128-byte blocks along K
            int      chunk; // K blocks per chunk (1 for 8-bit operands)
            int      sub; // K blocks per stage (1 for 8-bit operands); chunks are multiples of it
            int      kParts; // parts of the K range whose sums stay apart; tm counts the tiles of rows part by part
            int      kElems; // elements of a 128-byte block: 128 (8 bit) or 64
            // Operands that are sums of several matrices (f32 numbers as three bf16 ones, [segment][rows][cols]): the K range is a
            // list of pairs of segments, segBlocks K blocks each; bits 4 i .. of segX / segY name the pair's segments, which
            // lie xSegR / ySegR rows of the tile's side or xSegK / ySegK elements of K apart. One pair: segBlocks = kBlocks.
            int      segBlocks;
            uint32_t segX, segY;
            int      xSegR, xSegK, ySegR, ySegK;
            int      xRows, yRows; // not PAIR: rows of X and Y that are loaded, multiples of 8
            int      ksplit; // CTAs of a cluster that share a tile (not PAIR)
            int      stages;
            uint32_t stageBytes; // of all stages, and what the MMAs may read behind them: a multiple of 1024
            uint32_t idesc;
            int*     status;
            int      statusCode;
        };

        __device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi)
        {
            uint64_t r;
            asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
            return r;
        }
        __device__ __forceinline__ uint64_t pack2(float lo, float hi)
        {
            return pack2(__float_as_uint(lo), __float_as_uint(hi));
        }
        __device__ __forceinline__ float2 unpack2(uint64_t v)
        {
            uint32_t lo, hi;
            asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(v));
            return make_float2(__uint_as_float(lo), __uint_as_float(hi));
        }
        __device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
        {
            uint64_t r;
            asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
            return r;
        }
        __device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b)
        {
            uint64_t r;
            asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
            return r;
        }
        __device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
        {
            uint64_t r;
            asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
            return r;
        }

        // N columns of this warp's 32 lanes, one row a thread; the values are there after tmemWait()
        template <int N>
        __device__ __forceinline__ void tmemLoad(uint32_t addr, uint32_t (&v)[N])
        {
            if constexpr(N == 32)
                asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                             "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                             "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                             : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                               "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
                               "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]),
                               "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]),
                               "=r"(v[30]), "=r"(v[31])
                             : "r"(addr)
                             : "memory");
            else
                asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                             "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                             : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                               "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                             : "r"(addr)
                             : "memory");
        }
        __device__ __forceinline__ void tmemWait()
        {
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        }

        __device__ __forceinline__ void tmaLoadPair2(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1)
        {
            asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
                         "[%2];" ::"r"(dst),
                         "l"(map), "r"(bar), "r"(c0), "r"(c1)
                         : "memory");
        }

        __device__ __forceinline__ bool mbarTest(uint32_t bar, uint32_t parity)
        {
            uint32_t done;
            asm volatile("{\n\t.reg .pred p;\n\t"
                         "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                         "selp.u32 %0, 1, 0, p;\n\t}"
                         : "=r"(done)
                         : "r"(bar), "r"(parity)
                         : "memory");
            return done != 0;
        }

        template <bool PAIR, bool F8>
        __device__ __forceinline__ void issueMma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
        {
            if constexpr(PAIR && F8)
                asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                             "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                             "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
                             : "memory");
            else if constexpr(PAIR)
                asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                             "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                             "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
                             : "memory");
            else if constexpr(F8)
                asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                             "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                             "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
                             : "memory");
            else
                asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                             "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                             "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
                             : "memory");
        }
        template <bool PAIR>
        __device__ __forceinline__ void commitTo(uint32_t bar)
        {
            if constexpr(PAIR)
                asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                             "h"((unsigned short)3)
                             : "memory");
            else
                asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
        }

        // tile u of the walk: groups of groupM tiles of M, inside a group M fastest
        __device__ __forceinline__ void tileOf(const AccArgs& a, int u, int& tm, int& tn)
        {
            const int per = a.groupM * a.tilesN, g = u / per, in = u - g * per;
            const int gm  = min(a.groupM, a.tilesM - g * a.groupM);
            tn            = in / gm;
            tm            = g * a.groupM + in - tn * gm;
        }

        // Registers that a kernel with wide tiles was built with must be what the shares above add up to: a smaller
        // launch would make the epilogue wait for registers that are not there.
        inline cudaError_t accCheckRegs(const void* kernel, int tn)
        {
            if(tn < 128)
                return cudaSuccess;
            cudaFuncAttributes  at;
            const cudaError_t e = cudaFuncGetAttributes(&at, kernel);
            if(e != cudaSuccess)
                return e;
            return at.numRegs >= kAccRegs ? cudaSuccess : cudaErrorInvalidKernelImage;
        }

        // Epi: the epilogue, one object per epilogue thread:
        //   Epi(args, warp 0 .. 7, lane, shared memory behind the stages, flag of waits that ran out)
        //   begin(row)                      a tile begins, row is this thread's
        //   side(values, row in the tile, half of the columns)  with kSide: this K block's side values
        //   add(taddr, first, release)      reads the chunk's sums from tensor memory, calls release, and adds them
        //   end(row, col)                   the tile's sums are complete
        //   leave()                         no tile follows
        //   kParted                         whether AccArgs::kParts may be above 1
        //   send(..), endSplit(..)          with kSplit: the exchange of a tile whose K range is cut
        // With Epi::kSide > 0, warp 3 fetches kSide floats for every K block (the scales), a group of kGroup blocks at a time,
        // into a ring of kSideSlots groups, ahead of the epilogue and across tiles:
        //   Side(args, lane), begin(first row of this CTA, first column), fetch(slot, first K block, past the last one)
        // XMN, YMN: the operand is contiguous along its rows (a matrix with one row per k; half precision): 64-row chunks of
        // [64 k][128 bytes] instead of rows of 128 bytes along k, transposed descriptors.
        template <class Epi, bool PAIR, int TN, bool F8, bool XMN = false, bool YMN = false>
        __global__ void __launch_bounds__(kAccThreads, 1)
            accumulate_kernel(const __grid_constant__ CUtensorMap mapX, const __grid_constant__ CUtensorMap mapY, const __grid_constant__ AccArgs a,
                              const __grid_constant__ typename Epi::Args ea)
        {
            constexpr int      ROWS   = PAIR ? 256 : 128;
            // A K block: PAIR 128 rows of X, then this CTA's 128 rows of Y; else TN rows of Y, then the rows of X that there are
            // (a.xRows, a.yRows: a few tokens need not fill a tile's rows, the MMAs read what lies there and nobody looks at
            // those rows of the sums)
            constexpr uint32_t yOff   = PAIR ? 16384u : uint32_t(TN) * 128u;
            const uint32_t     kBlock = PAIR ? 32768u : yOff + uint32_t(a.xRows) * 128u; // of one K block
            const uint32_t     kStage = kBlock * uint32_t(a.sub);
            // accumulators in tensor memory: what the two hand-overs of a chunk take (1000 cycles and more) passes behind the other
            // ones' sums; narrow tiles have room for more than two
            constexpr uint32_t NBUF   = (F8 && TN <= 128) ? 4 : 2;
            constexpr uint32_t kCols  = NBUF * TN;
            extern __shared__ unsigned char smemRaw[];
            unsigned char* tiles = (unsigned char*)((uintptr_t(smemRaw) + 1023) & ~uintptr_t(1023));
            __shared__ __align__(8) unsigned long long fullBar[kAccMaxStages], emptyBar[kAccMaxStages];
            __shared__ __align__(8) unsigned long long tmemFullBar[2], tmemEmptyBar[4];
            __shared__ uint32_t tmemBase;
            __shared__ int      abortFlag;
            __shared__ __align__(8) unsigned long long sideFullBar[kSideSlots], sideEmptyBar[kSideSlots];

            const int      warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
            const uint32_t rank = (PAIR || a.ksplit > 1) ? clusterRank() : 0u;
            const bool     leader = !PAIR || rank == 0;
            const int      csize = PAIR ? 2 : a.ksplit;
            const int      clusterId = int(blockIdx.x) / csize, numClusters = int(gridDim.x) / csize;
            const bool     clustered = csize > 1;

            asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
            if(threadIdx.x == 32)
            {
                prefetchTensorMap(&mapX);
                prefetchTensorMap(&mapY);
            }
            if(threadIdx.x == 0)
            {
                abortFlag = 0;
                for(int s = 0; s < a.stages; s++)
                {
                    mbarInit(smemAddr(&fullBar[s]), 1);
                    mbarInit(smemAddr(&emptyBar[s]), 1);
                }
                for(int i = 0; i < 2; i++)
                    mbarInit(smemAddr(&tmemFullBar[i]), 1);
                for(int i = 0; i < int(NBUF); i++)
                    mbarInit(smemAddr(&tmemEmptyBar[i]), (PAIR ? 2 : 1) * (kAccEpi / 32));
                for(int i = 0; i < kSideSlots; i++)
                {
                    mbarInit(smemAddr(&sideFullBar[i]), 32);
                    mbarInit(smemAddr(&sideEmptyBar[i]), kAccEpi / 32);
                }
                asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            }
            if(warp == 1)
            {
                if constexpr(PAIR)
                {
                    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smemAddr(&tmemBase)), "r"(kCols)
                                 : "memory");
                    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
                }
                else
                {
                    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smemAddr(&tmemBase)), "r"(kCols)
                                 : "memory");
                    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncthreads();
            if(clustered)
                clusterSync(); // the peers' barriers exist before anything signals them
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t tmem   = tmemBase;
            volatile int*  abortP = &abortFlag;
            const uint32_t tilesAddr = smemAddr(tiles), fullAddr = smemAddr(&fullBar[0]), emptyAddr = smemAddr(&emptyBar[0]);
            const int      units = a.tilesM * a.tilesN;
            // K blocks of this CTA: all, or its part of a split tile
            int  kbBegin = PAIR ? 0 : int((long long)a.kBlocks * int(rank) / a.ksplit);
            int  kbEnd   = PAIR ? a.kBlocks : int((long long)a.kBlocks * (int(rank) + 1) / a.ksplit);
            auto part    = [&](int& tm) { // kParts: the K range is the tile's
                if(Epi::kParted && a.kParts > 1)
                {
                    const int tiles = a.tilesM / a.kParts, p = tm / tiles;
                    kbBegin = int((long long)a.kBlocks * p / a.kParts);
                    kbEnd   = int((long long)a.kBlocks * (p + 1) / a.kParts);
                    tm -= p * tiles;
                }
            };
            // global memory is read and written from here on: the grid ahead of this one must be complete
            asm volatile("griddepcontrol.wait;" ::: "memory");

            constexpr bool kMoreRegs = TN >= 128;
            if(warp < 4)
            {
                if constexpr(kMoreRegs)
                    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kAccRegsLoad));
            if(warp == 0)
            {
                if(lane == 0)
                {
                    const uint32_t leaderFull = PAIR ? mapToRank(fullAddr, 0) : fullAddr;
                    uint32_t       stage = 0, phase = 0;
                    bool           ok = true;
                    for(int u = clusterId; ok && u < units; u += numClusters)
                    {
                        int tm, tn;
                        tileOf(a, u, tm, tn);
                        part(tm);
                        const int x0 = tm * ROWS + (PAIR ? int(rank) * 128 : 0), y0 = tn * TN + (PAIR ? int(rank) * 128 : 0);
                        for(int kb = kbBegin; kb < kbEnd; kb += a.sub)
                        {
                            ok = mbarWaitTight(emptyAddr + 8 * stage, phase ^ 1, abortP);
                            if(!ok)
                                break;
                            const uint32_t bar = leaderFull + 8 * stage;
                            const int      blocks = min(a.sub, kbEnd - kb);
                            if(leader)
                                mbarArriveExpectTx(fullAddr + 8 * stage, (PAIR ? 2 * 32768u : uint32_t(a.xRows + a.yRows) * 128u) * uint32_t(blocks));
                            for(int i = 0; i < blocks; i++)
                            {
                                const uint32_t dst = tilesAddr + stage * kStage + i * kBlock;
                                const uint32_t dstX = PAIR ? dst : dst + yOff, dstY = PAIR ? dst + 16384 : dst;
                                int k0 = (kb + i) * a.kElems, xr = x0, yr = y0, kx = k0, ky = k0;
                                if(!F8 && a.segBlocks != a.kBlocks)
                                {
                                    const int pair = (kb + i) / a.segBlocks, sx = int(a.segX >> (4 * pair)) & 15, sy = int(a.segY >> (4 * pair)) & 15;
                                    k0 -= pair * a.segBlocks * a.kElems;
                                    kx = k0 + sx * a.xSegK, xr += sx * a.xSegR;
                                    ky = k0 + sy * a.ySegK, yr += sy * a.ySegR;
                                }
                                static_assert(!(XMN || YMN) || !F8, "only half precision");
                                static_assert(!XMN || PAIR, "128 rows of X in two chunks");
                                if constexpr(XMN)
                                {
                                    tmaLoadPair2(dstX, &mapX, bar, xr, kx);
                                    tmaLoadPair2(dstX + 8192, &mapX, bar, xr + 64, kx);
                                }
                                else if constexpr(PAIR)
                                    tmaLoadPair2(dstX, &mapX, bar, kx, xr);
                                else
                                {
                                    const int c[2] = {kx, xr};
                                    tmaLoad<2>(dstX, &mapX, bar, c);
                                }
                                if constexpr(YMN)
                                {
#pragma unroll
                                    for(int c0 = 0; c0 < (PAIR ? 128 : TN); c0 += 64)
                                    {
                                        const int c[2] = {yr + c0, ky};
                                        if constexpr(PAIR)
                                            tmaLoadPair2(dstY + c0 * 128, &mapY, bar, c[0], c[1]);
                                        else
                                            tmaLoad<2>(dstY + c0 * 128, &mapY, bar, c);
                                    }
                                }
                                else if constexpr(PAIR)
                                    tmaLoadPair2(dstY, &mapY, bar, ky, yr);
                                else
                                {
                                    const int c[2] = {ky, yr};
                                    tmaLoad<2>(dstY, &mapY, bar, c);
                                }
                            }
                            if(++stage == uint32_t(a.stages))
                            {
                                stage = 0;
                                phase ^= 1;
                            }
                        }
                    }
                }
                if(!PAIR && clustered)
                {
                    __syncwarp();
                    clusterSync(); // the two meeting points of the exchange (see the epilogue)
                    clusterSync();
                }
            }
            else if(warp <= 2)
            {
                // 8 bit: two issuers, warp 1 takes the even chunks (first accumulator), warp 2 the odd ones. An MMA is accepted
                // only shortly before the one ahead of it is done, so what a thread does between its MMAs (the waits, the
                // commits: 700 cycles around 512 of MMAs for a chunk of one block) would leave the tensor cores idle. A
                // barrier tells apart two rounds of the stages only, so no issuer may look more than a round ahead: the number
                // of stages is even (checked by the launcher), so a stage is always the same issuer's, which waits for its
                // rounds in order.
                // Half precision: long chunks, one issuer.
                constexpr uint32_t ISSUERS = F8 ? 2 : 1;
                if(lane == 0 && leader && uint32_t(warp) <= ISSUERS)
                {
                    const uint32_t addrX = tilesAddr + (PAIR ? 0u : yOff), addrY = tilesAddr + (PAIR ? 16384u : 0u);
                    const uint64_t descX = XMN ? smemDescMn(addrX) : smemDesc(addrX), descY = YMN ? smemDescMn(addrY) : smemDesc(addrY);
                    constexpr int  stepX = XMN ? 128 : 2, stepY = YMN ? 128 : 2; // a K step of 32 bytes (MN: of 16 rows), in 16 bytes
                    const uint32_t self = uint32_t(warp) - 1;
                    uint32_t       stage = 0, phase = 0, seq = 0;
                    bool           ok = true;
                    for(int u = clusterId; ok && u < units; u += numClusters)
                    {
                        if constexpr(Epi::kParted)
                        {
                            int tm, tn;
                            tileOf(a, u, tm, tn);
                            part(tm);
                        }
                        for(int kb = kbBegin; ok && kb < kbEnd; kb += a.chunk, seq++)
                        {
                            const uint32_t buf = seq % NBUF;
                            if(ISSUERS == 2 && (seq & 1) != self)
                            {
                                if(++stage == uint32_t(a.stages)) // the other issuer's stage (a chunk is one block)
                                {
                                    stage = 0;
                                    phase ^= 1;
                                }
                                continue;
                            }
                            const int      end = min(kb + a.chunk, kbEnd);
                            const uint32_t d   = tmem + buf * TN;
                            // the first stage before the accumulator: the latter is what comes late, and nothing should
                            // stand between its release and the MMAs
                            ok = mbarWaitTight(fullAddr + 8 * stage, phase, abortP)
                                 && mbarWaitTight(smemAddr(&tmemEmptyBar[buf]), ((seq / NBUF) & 1) ^ 1, abortP);
                            if(!ok)
                                break;
                            for(int k = kb; k < end; k += a.sub)
                            {
                                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                                const uint32_t now = stage;
                                if(++stage == uint32_t(a.stages))
                                {
                                    stage = 0;
                                    phase ^= 1;
                                }
                                bool      ready  = false;
                                const int blocks = min(a.sub, end - k);
                                for(int i = 0; i < blocks; i++)
                                {
                                    const uint64_t off = uint64_t((now * kStage + i * kBlock) >> 4);
#pragma unroll
                                    for(int s = 0; s < 4; s++) // 32 bytes of K each
                                    {
                                        if(s == 2 && i + 1 == blocks && k + a.sub < end) // a look at the next stage while MMAs are queued
                                            ready = mbarTest(fullAddr + 8 * stage, phase);
                                        issueMma<PAIR, F8>(d, descX + off + stepX * s, descY + off + stepY * s, a.idesc,
                                                           (k != kb || i != 0 || s != 0) ? 1u : 0u);
                                    }
                                }
                                // frees the stage once these MMAs have read it, which with one block a chunk (F8) also says
                                // that the chunk is summed
                                commitTo<PAIR>(emptyAddr + 8 * now);
                                if(k + a.sub < end && !ready)
                                    ok = mbarWaitTight(fullAddr + 8 * stage, phase, abortP);
                                if(!ok)
                                    break;
                            }
                            if(!F8 && ok)
                                commitTo<PAIR>(smemAddr(&tmemFullBar[buf]));
                        }
                    }
                }
                if(!PAIR && clustered)
                {
                    __syncwarp();
                    clusterSync();
                    clusterSync();
                }
            }
            else
            {
                if constexpr(Epi::kSide > 0)
                {
                    float* const       ring = reinterpret_cast<float*>(tiles + a.stageBytes);
                    typename Epi::Side side(ea, lane);
                    uint32_t           slot = 0, phase = 0;
                    bool               ok = true;
                    for(int u = clusterId; ok && u < units; u += numClusters)
                    {
                        int tm, tn;
                        tileOf(a, u, tm, tn);
                        part(tm);
                        side.begin(int64_t(tm) * ROWS + (PAIR ? int(rank) * 128 : 0), int64_t(tn) * TN);
                        for(int kb = kbBegin; kb < kbEnd;)
                        {
                            ok = __all_sync(0xffffffffu, mbarWaitTight(smemAddr(&sideEmptyBar[slot]), phase ^ 1, abortP));
                            if(!ok)
                                break;
                            const int end = min((kb / Epi::kGroup + 1) * Epi::kGroup, kbEnd);
                            side.fetch(ring + slot * (Epi::kSide * Epi::kGroup), kb, end);
                            mbarArrive(smemAddr(&sideFullBar[slot]));
                            kb = end;
                            if(++slot == kSideSlots)
                            {
                                slot = 0;
                                phase ^= 1;
                            }
                        }
                    }
                    __syncwarp();
                }
                if(!PAIR && clustered)
                {
                    clusterSync();
                    clusterSync();
                }
            }
            }
            else
            {
                if constexpr(kMoreRegs)
                    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kAccRegsEpi));
                const int quad = warp & 3, half = (warp - 4) >> 2;
                Epi       epi(ea, warp - 4, lane, tiles + a.stageBytes, abortP);
                uint32_t  buf = 0, bufPhase = 0, stage = 0, phase = 0; // stage and phase: F8, a chunk is one stage
                uint32_t  slot = 0, slotPhase = 0;
                const float* ring = reinterpret_cast<const float*>(tiles + a.stageBytes);
                bool      ok = true;
                int       syncs = 0;
                const uint32_t emptyLeader = PAIR ? mapToRank(smemAddr(&tmemEmptyBar[0]), 0) : smemAddr(&tmemEmptyBar[0]);
                for(int u = clusterId; ok && u < units; u += numClusters)
                {
                    int tm, tn;
                    tileOf(a, u, tm, tn);
                    const int tile = tm; // with kParts the rows of the parts' results follow each other
                    part(tm);
                    const int     row = quad * 32 + lane;
                    const int64_t r = int64_t(tile) * ROWS + (PAIR ? int(rank) * 128 : 0) + row, c = int64_t(tn) * TN + half * (TN / 2);
                    epi.begin(r);
                    for(int kb = kbBegin; kb < kbEnd; kb += a.chunk)
                    {
                        if constexpr(Epi::kSide > 0)
                        {
                            if(kb == kbBegin || kb % Epi::kGroup == 0)
                                ok = __all_sync(0xffffffffu, mbarWaitTight(smemAddr(&sideFullBar[slot]), slotPhase, abortP));
                            if(!ok)
                                break;
                            epi.side(ring + (slot * Epi::kGroup + kb % Epi::kGroup) * Epi::kSide, row, half);
                        }
                        ok = __all_sync(0xffffffffu, F8 ? mbarWaitTight(emptyAddr + 8 * stage, phase, abortP)
                                                        : mbarWaitTight(smemAddr(&tmemFullBar[buf]), bufPhase, abortP));
                        if(!ok)
                            break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        // called once the chunk is out of tensor memory: hands the accumulator back
                        auto release = [&]() {
                            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                            __syncwarp();
                            if(lane == 0)
                            {
                                // At CTA scope even where the barrier is the other CTA's: nothing but the completed reads
                                // of tensor memory is handed over, and a release at cluster scope is a fence that waits
                                // for the scales on their way (8 bit, 4096^3: 1.4 times the time)
                                if constexpr(PAIR)
                                    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(emptyLeader + 8 * buf) : "memory");
                                else
                                    mbarArrive(emptyLeader + 8 * buf);
                            }
                        };
                        epi.add(tmem + (uint32_t(quad * 32) << 16) + buf * TN + uint32_t(half * (TN / 2)), kb == kbBegin, release);
                        if constexpr(Epi::kSide > 0)
                        {
                            if(kb + 1 == kbEnd || (kb + 1) % Epi::kGroup == 0) // the group's last block
                            {
                                __syncwarp();
                                if(lane == 0)
                                    mbarArrive(smemAddr(&sideEmptyBar[slot]));
                                if(++slot == kSideSlots)
                                {
                                    slot = 0;
                                    slotPhase ^= 1;
                                }
                            }
                        }
                        if(++buf == NBUF)
                        {
                            buf = 0;
                            bufPhase ^= 1;
                        }
                        if(++stage == uint32_t(a.stages))
                        {
                            stage = 0;
                            phase ^= 1;
                        }
                    }
                    if(!ok)
                        break;
                    if constexpr(!PAIR && Epi::kSplit)
                    {
                        if(clustered)
                        {
                            // K split: CTA r of the cluster finishes columns r TN / ksplit .. of the tile. Every CTA sends
                            // the others their columns of its sums, into the (by then idle) stages, and adds what it
                            // gets in the order of the ranks.
                            clusterSync(); // every CTA of the cluster has its sums: all stages are idle
                            epi.send(tilesAddr, rank, a.ksplit, row, half);
                            clusterSync(); // the others' sums have arrived
                            syncs = 2;
                            epi.endSplit(tilesAddr, rank, a.ksplit, row, half, r, int64_t(tn) * TN);
                            continue;
                        }
                    }
                    epi.end(r, c);
                }
                epi.leave();
                for(; !PAIR && clustered && syncs < 2; syncs++)
                    clusterSync(); // a CTA whose wait ran out still meets the others
            }

            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncthreads();
            if(abortFlag)
            {
                // a wait ran out: loads and MMAs may still be on their way into memory that is given up below (about a
                // millisecond is many times what they can take)
                const long long t0 = clock64();
                while(clock64() - t0 < 2000000)
                    ;
            }
            if(clustered)
                clusterSync(); // all CTAs are done with tensor memory and with each other's barriers and shared memory
            if(threadIdx.x == 0 && abortFlag && a.status)
                atomicExch_system(a.status, a.statusCode);
            if(warp == 1)
            {
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if constexpr(PAIR)
                    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
                else
                    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
            }
        }
    } // namespace
} // namespace htb
