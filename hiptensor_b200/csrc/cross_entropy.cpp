// Host side of the linear cross entropy and its gradient: mode folding, the layout of the workspace, the walk over the
// pieces of the vocabulary.
#include <algorithm>

#include <hiptensor/hiptensor.hpp>

#include "cross_entropy.hpp"
#include "kernels.hpp"

namespace htb
{
    namespace
    {
        constexpr int64_t  kPieceUnit   = 256; // classes: a tile's columns
        constexpr int64_t  kIndexRange  = (int64_t(1) << 31) - 512; // of a load's coordinate, and a tile behind it
        constexpr uint64_t kRecommended = uint64_t(1) << 30; // bytes of the pieces' buffers under WORKSPACE_RECOMMENDED

        int64_t roundUp(int64_t n, int64_t to)
        {
            return (n + to - 1) / to * to;
        }
        int find(const int32_t* modes, int n, int32_t m)
        {
            for(int i = 0; i < n; i++)
                if(modes[i] == m)
                    return i;
            return -1;
        }
        bool sane(const hiptensorTensorDescriptor_t& d)
        {
            if(d.mLengths.size() != d.mStrides.size() || d.mLengths.empty() || d.mLengths.size() > std::size_t(kMaxRank))
                return false;
            for(std::size_t i = 0; i < d.mLengths.size(); i++)
                if(int64_t(d.mLengths[i]) < 0 || int64_t(d.mLengths[i]) >= (int64_t(1) << 31) || int64_t(d.mStrides[i]) < 0
                   || (d.mLengths[i] > 1 && d.mStrides[i] == 0))
                    return false;
            return true;
        }

        // Whether and how a call runs in one pass over W (few tokens; this and the tensor cores in us): gradients of 8 tokens of f32
        // (x 32000 x 1024: 103 and 247) and of rows that no TMA load can read (f16, x 30011 x 1001: 154 and 207), of 4 tokens of
        // others (bf16, x 11722 x 2064: 56 and 73; 8 tokens x 32000 x 4096: 376 and 230); losses of 8 tokens of f32 (x 32000 x 1024:
        // 64 and 126) and of 4 of rows that no TMA load can read (bf16, x 30011 x 1001: 48 and 72, 8 tokens 73 and 71).
        FewShape fewShape(const CrossEntropyPlan& p, bool gradient)
        {
            FewShape      f{};
            const int64_t size = dtypeSize(p.type), unit = 16 / size;
            f.tokens = 1;
            while(f.tokens < p.T && f.tokens < 8)
                f.tokens *= 2;
            const int64_t smem = f.tokens * p.D * (size + (gradient ? 4 : 0)) + 16;
            const bool    words = (p.wD == 1 || p.D == 1) && p.D % unit == 0 && (p.V == 1 || p.wV % unit == 0);
            const int     most  = size == 4 ? 8 : (gradient ? (words ? 4 : 8) : (words ? 0 : 4));
            if(p.T < 1 || p.T > most || (p.wD != 1 && p.D > 1) || smem > 200 * 1024)
                return f;
            f.use     = true;
            f.unit    = words ? int(unit) : (p.D % 2 == 0 && (p.V == 1 || p.wV % 2 == 0) ? 2 : 1);
            f.units   = p.D / f.unit;
            f.ldh     = roundUp(p.D, 4);
            f.smem    = int(smem);
            // equal rounds over a row's units; 512 threads per SM (their registers) as far as shared memory allows. Fewer threads
            // per block, and more blocks, are slower: one token x 32000 x 1024 f32 47 us in one round, 69 in four.
            const int64_t rounds = (f.units + 255) / 256;
            f.threads            = int(roundUp((f.units + rounds - 1) / rounds, 32));
            const int64_t each   = std::max<int64_t>(1, std::min<int64_t>(512 / f.threads, (227 << 10) / (smem + 5120)));
            int64_t       n      = std::min(p.sms * each, (p.V + 3) / 4);
            if(gradient)
                n = std::min(n, std::max<int64_t>(1, p.V * size / (4 * p.T)));
            f.blocks = int(n);
            return f;
        }

        // The layout for pieces of `piece` classes. Every buffer starts at a multiple of 256 bytes.
        CrossEntropyLayout layoutFor(const CrossEntropyPlan& p, bool gradient, int64_t piece)
        {
            CrossEntropyLayout l{};
            const int64_t      unit = 16 / dtypeSize(p.type);
            const bool         f32  = p.type == CUDA_R_32F;
            const bool wordsH = p.nt <= 1 && p.hD == 1 && (p.T == 1 || (p.tStride[0] % unit == 0 && p.tStride[0] >= p.D));
            const bool wordsW = p.wD == 1 && (p.V == 1 || (p.wV % unit == 0 && p.wV >= p.D));
            // the gradient reads a copy of H whose rows of ignored tokens are zeros: what lies there (padding, NaN) must not
            // reach dW through 0 * NaN
            l.packH    = gradient || f32 || !wordsH;
            l.packW    = f32 || !wordsW;
            l.direct   = wordsW && p.D % unit == 0; // a bulk store writes whole words of 16 bytes, behind a row's end too
            l.segments = f32 ? 3 : 1;
            l.ld       = roundUp(p.D, 8);
            l.piece    = piece;
            const int partsP = gradient ? probabilityParts(p.type, p.T) : 1;
            // segments of tokens are contracted in blocks of 64: zeros up to there
            l.rowsT = l.segments > 1 || partsP > 1 ? roundUp(p.T, 64) : p.T;
            const int pairs = f32 ? 6 : 1;
            l.parts         = gradient ? int(std::max<int64_t>(1, std::min<int64_t>(p.parts, piece * pairs / 1024))) : 1;
            uint64_t at   = 0;
            auto     take = [&](bool wanted, uint64_t bytes) {
                const uint64_t here = at;
                if(wanted)
                    at += (bytes + 255) / 256 * 256;
                return here;
            };
            const uint64_t T = uint64_t(p.T), n = uint64_t(piece), ld = uint64_t(l.ld), seg = uint64_t(l.segments);
            l.hOff           = take(l.packH, seg * uint64_t(l.rowsT) * ld * 2);
            l.stateOff       = take(!gradient, T * 12);
            l.scaleOff       = take(gradient, 8);
            l.restOff        = take(gradient, T * 4);
            l.lists          = gradient && partsP == 1;
            l.listOff        = take(l.lists, uint64_t(2 * roundUp(p.T, 64) + p.V) * 4);
            l.dhOff          = take(gradient, uint64_t(l.parts) * uint64_t(hiddenRows(p.T)) * ld * 4);
            l.wOff           = take(l.packW, seg * n * ld * 2);
            l.partOff        = take(!gradient, n / kHeadGroup * T * 8);
            l.pOff           = take(gradient, uint64_t(partsP) * uint64_t(l.rowsT) * n * 2);
            l.dwOff          = take(gradient && !l.direct, n * ld * 4);
            l.bytes          = at + 256; // room to align the caller's pointer
            return l;
        }
        // of a call in one pass
        CrossEntropyLayout layoutFew(const CrossEntropyPlan& p, const FewShape& f, bool gradient)
        {
            CrossEntropyLayout l{};
            const uint64_t     T = uint64_t(p.T), n = uint64_t(f.blocks);
            l.stateOff = l.dhOff = 0;
            l.partOff            = (T * 12 + 255) / 256 * 256;
            l.bytes              = 256 + (gradient ? n * T * uint64_t(f.ldh) * 4 : l.partOff + n * T * 8);
            return l;
        }
        // Units of the largest piece there may be. Coordinates of loads are 32-bit numbers: the three parts of an f32 piece lie behind
        // each other (3 n rows), and the classes that dH's product contracts are counted through all six products (6 n).
        int64_t mostUnits(const CrossEntropyPlan& p, bool gradient)
        {
            const int64_t all = roundUp(p.V, kPieceUnit) / kPieceUnit;
            return p.type == CUDA_R_32F ? std::min(all, kIndexRange / ((gradient ? 6 : 3) * kPieceUnit)) : all;
        }
        // the largest pieces that fit into `bytes`; piece = 0 when not even the smallest do
        CrossEntropyLayout layoutIn(const CrossEntropyPlan& p, bool gradient, uint64_t bytes)
        {
            int64_t lo = 0, hi = mostUnits(p, gradient); // pieces of lo units fit
            while(lo < hi)
            {
                const int64_t mid = (lo + hi + 1) / 2;
                if(layoutFor(p, gradient, mid * kPieceUnit).bytes <= bytes)
                    lo = mid;
                else
                    hi = mid - 1;
            }
            if(lo > 0)
            {
                // pieces of equal size, no more of them than that
                const int64_t units = roundUp(p.V, kPieceUnit) / kPieceUnit, count = (units + lo - 1) / lo;
                lo = (units + count - 1) / count;
            }
            return layoutFor(p, gradient, lo * kPieceUnit);
        }

        TokenRows rowsOfH(const CrossEntropyPlan& p)
        {
            TokenRows r{};
            r.nt = p.nt;
            for(int i = 0; i < p.nt; i++)
            {
                r.ext[i]    = p.tExt[i];
                r.stride[i] = p.tStride[i];
            }
            r.elem = p.hD;
            return r;
        }
        TokenRows plainRows(int64_t stride, int64_t elem, int64_t count)
        {
            TokenRows r{};
            r.nt        = 1;
            r.ext[0]    = count;
            r.stride[0] = stride;
            r.elem      = elem;
            return r;
        }

        int64_t rowStride(const CrossEntropyPlan& p, const CrossEntropyLayout& l)
        {
            return p.T > 1 ? p.tStride[0] : l.ld;
        }

#define HTB_TRY(call)                    \
    do                                   \
    {                                    \
        const cudaError_t e_ = (call);   \
        if(e_ != cudaSuccess)            \
            return launchResult(fn, e_); \
    } while(0)
    } // namespace

    int planCrossEntropy(const hiptensorTensorDescriptor_t& H, const int32_t* modeH, const hiptensorTensorDescriptor_t& W,
                         const int32_t* modeW, int64_t ignoreIndex, int typeCompute, int smCount, CrossEntropyPlan* out)
    {
        const int type = H.mType;
        if((type != CUDA_R_16F && type != CUDA_R_16BF && type != CUDA_R_32F) || W.mType != type || typeCompute != HIPTENSOR_COMPUTE_32F
           || H.mUnaryOp != HIPTENSOR_OP_IDENTITY || W.mUnaryOp != HIPTENSOR_OP_IDENTITY)
            return HIPTENSOR_STATUS_NOT_SUPPORTED;
        if(!sane(H) || !sane(W))
            return HIPTENSOR_STATUS_INVALID_VALUE;
        const int rH = int(H.mLengths.size()), rW = int(W.mLengths.size());
        for(int i = 0; i < rH; i++)
            if(find(modeH, i, modeH[i]) >= 0)
                return HIPTENSOR_STATUS_INVALID_VALUE;
        CrossEntropyPlan p{};
        p.type   = type;
        p.ignore = ignoreIndex;
        p.sms    = smCount > 0 ? smCount : 148;
        p.T = p.V = p.D = 1;
        p.hD = p.wD = 1;
        p.wV        = 1;
        int  nv = 0, nd = 0;
        bool empty = false;
        for(int i = 0; i < rW; i++)
        {
            const int64_t ext = int64_t(W.mLengths[i]), s = int64_t(W.mStrides[i]);
            if(find(modeW, i, modeW[i]) >= 0)
                return HIPTENSOR_STATUS_INVALID_VALUE;
            if(ext == 0)
                return HIPTENSOR_STATUS_INVALID_VALUE; // a softmax over nothing, or logits of nothing
            const int j = find(modeH, rH, modeW[i]);
            if(j >= 0 && int64_t(H.mLengths[j]) != ext)
                return HIPTENSOR_STATUS_INVALID_VALUE;
            if(ext == 1)
                continue;
            if(j >= 0)
            {
                // contracted modes: one, or several that follow each other without a gap in both tensors
                const int64_t sh = int64_t(H.mStrides[j]);
                if(nd && p.wD == s * ext && p.hD == sh * ext)
                    p.D *= ext;
                else if(nd)
                    return HIPTENSOR_STATUS_NOT_SUPPORTED;
                else
                    p.D = ext;
                p.wD = s;
                p.hD = sh;
                nd++;
            }
            else
            {
                if(nv && p.wV == s * ext)
                    p.V *= ext;
                else if(nv)
                    return HIPTENSOR_STATUS_NOT_SUPPORTED;
                else
                    p.V = ext;
                p.wV = s;
                nv++;
            }
        }
        int contracted = 0;
        for(int i = 0; i < rH; i++)
        {
            if(find(modeW, rW, modeH[i]) >= 0)
            {
                contracted++;
                continue;
            }
            const int64_t ext = int64_t(H.mLengths[i]), s = int64_t(H.mStrides[i]);
            empty |= ext == 0;
            if(ext == 1)
                continue;
            p.T *= ext;
            if(p.nt > 0 && p.tStride[p.nt - 1] == s * ext)
            {
                p.tExt[p.nt - 1] *= ext;
                p.tStride[p.nt - 1] = s;
                continue;
            }
            if(p.nt == kMaxGroup)
                return HIPTENSOR_STATUS_NOT_SUPPORTED;
            p.tExt[p.nt]      = ext;
            p.tStride[p.nt++] = s;
        }
        if(contracted == 0)
            return HIPTENSOR_STATUS_INVALID_VALUE;
        if(empty)
            p.T = 0;
        // (f32: the tokens' three parts lie behind each other, in rows of a multiple of 64)
        if(p.V >= kIndexRange || p.T >= kIndexRange || (type == CUDA_R_32F && 3 * roundUp(p.T, 64) >= kIndexRange) || p.D > (int64_t(1) << 26))
            return HIPTENSOR_STATUS_NOT_SUPPORTED;
        p.parts = p.T > 0 ? hiddenParts(p.T, p.D, p.V * (type == CUDA_R_32F ? 6 : 1), p.sms) : 1;
        *out    = p;
        return HIPTENSOR_STATUS_SUCCESS;
    }

    uint64_t crossEntropyWorkspace(const CrossEntropyPlan& p, bool gradient, int pref)
    {
        if(p.T == 0)
            return 0;
        if(const FewShape f = fewShape(p, gradient); f.use)
            return layoutFew(p, f, gradient).bytes;
        const uint64_t least = layoutFor(p, gradient, kPieceUnit).bytes, most = layoutFor(p, gradient, mostUnits(p, gradient) * kPieceUnit).bytes;
        if(pref == HIPTENSOR_WORKSPACE_MIN)
            return least;
        if(pref == HIPTENSOR_WORKSPACE_MAX)
            return most;
        return layoutIn(p, gradient, std::max(least, std::min(most, least + kRecommended))).bytes;
    }

    int crossEntropy(const hiptensorHandle_t* handle, const CrossEntropyPlan* plan, const void* alpha, const void* H, const void* W,
                     const int64_t* targets, float* loss, float* lse, void* workspace, uint64_t workspaceSize, void* stream_)
    {
        const char* fn = "htCrossEntropy";
        HTB_LOG_API(fn, "handle=%p, plan=%p, alpha=%p, H=%p, W=%p, targets=%p, loss=%p, lse=%p, workspace=%p, workspaceSize=%llu, stream=%p",
                    (const void*)handle, (const void*)plan, alpha, H, W, (const void*)targets, (void*)loss, (void*)lse, workspace,
                    (unsigned long long)workspaceSize, stream_);
        if(!handle || !plan)
            return HIPTENSOR_STATUS_NOT_INITIALIZED;
        const HandleState* st = stateOf(handle);
        if(!st)
            return HIPTENSOR_STATUS_NOT_INITIALIZED;
        if(auto s = checkDevice(fn, st); s != HIPTENSOR_STATUS_SUCCESS)
            return s;
        const CrossEntropyPlan& p = *plan;
        if(p.T == 0)
            return HIPTENSOR_STATUS_SUCCESS;
        if(!alpha || !H || !W || !targets || !loss || !lse || ((uintptr_t(H) | uintptr_t(W)) & 15) || (uintptr_t(targets) & 7)
           || ((uintptr_t(loss) | uintptr_t(lse)) & 3))
        {
            HTB_LOG_ERROR(fn, "Input Parameter Error : a required pointer is nullptr or not aligned (%s)",
                          hiptensorGetErrorString(HIPTENSOR_STATUS_INVALID_VALUE));
            return HIPTENSOR_STATUS_INVALID_VALUE;
        }
        const FewShape           f    = fewShape(p, false);
        const uint64_t           room = workspace ? workspaceSize : 0;
        const CrossEntropyLayout l    = f.use ? layoutFew(p, f, false) : layoutIn(p, false, room);
        if(f.use ? l.bytes > room : l.piece == 0)
        {
            HTB_LOG_ERROR(fn, "Insufficient workspace: req: %llu alloc: %llu (%s)",
                          (unsigned long long)crossEntropyWorkspace(p, false, HIPTENSOR_WORKSPACE_MIN), (unsigned long long)workspaceSize,
                          hiptensorGetErrorString(HIPTENSOR_STATUS_INSUFFICIENT_WORKSPACE));
            return HIPTENSOR_STATUS_INSUFFICIENT_WORKSPACE;
        }
        const cudaStream_t stream = cudaStream_t(stream_);
        unsigned char*     ws     = reinterpret_cast<unsigned char*>((uintptr_t(workspace) + 255) & ~uintptr_t(255));
        const float        a      = *(const float*)alpha;
        const int64_t      size   = dtypeSize(p.type);
        const int          type16 = p.type == CUDA_R_16F ? CUDA_R_16F : CUDA_R_16BF;
        float*             state  = reinterpret_cast<float*>(ws + l.stateOff);
        if(f.use)
        {
            HTB_TRY(launchFewLoss(p, f, H, rowsOfH(p), W, targets, a, ws + l.partOff, state, st->deviceStatus, stream));
            HTB_TRY(launchLossJoin(ws + l.partOff, int64_t(f.blocks) * kHeadGroup, p.T, state, true, true, p.V, p.ignore, targets, loss, lse,
                                   st->deviceStatus, stream));
            return HIPTENSOR_STATUS_SUCCESS;
        }
        const void*        h      = H;
        int64_t            ldh    = rowStride(p, l);
        if(l.packH)
        {
            HTB_TRY(launchPackRows(p.type, H, rowsOfH(p), p.T, l.rowsT, p.D, l.ld, ws + l.hOff, nullptr, 0, 0, TokenLists{}, nullptr, stream));
            h   = ws + l.hOff;
            ldh = l.ld;
        }
        for(int64_t v0 = 0; v0 < p.V; v0 += l.piece)
        {
            const int64_t n   = std::min(l.piece, p.V - v0);
            const void*   w   = static_cast<const unsigned char*>(W) + v0 * p.wV * size;
            int64_t       ldw = p.wV;
            if(l.packW)
            {
                HTB_TRY(launchPackRows(p.type, w, plainRows(p.wV, p.wD, n), n, n, p.D, l.ld, ws + l.wOff, nullptr, 0, 0, TokenLists{}, nullptr, stream));
                w   = ws + l.wOff;
                ldw = l.ld;
            }
            HTB_TRY(launchHeadLoss(HeadProduct{h, w, p.T, n, p.D, ldh, ldw, type16, l.segments, l.rowsT, n}, v0, targets, a, ws + l.partOff, state,
                                   st->smCount, st->deviceStatus, stream));
            HTB_TRY(launchLossJoin(ws + l.partOff, n, p.T, state, v0 == 0, v0 + n == p.V, p.V, p.ignore, targets, loss, lse, st->deviceStatus,
                                   stream));
        }
        return HIPTENSOR_STATUS_SUCCESS;
    }

    int crossEntropyGradient(const hiptensorHandle_t* handle, const CrossEntropyPlan* plan, const void* alpha, const void* H,
                             const void* W, const int64_t* targets, const float* lse, const float* gradLoss, void* dH, void* dW,
                             void* workspace, uint64_t workspaceSize, void* stream_)
    {
        const char* fn = "htCrossEntropyGradient";
        HTB_LOG_API(fn, "handle=%p, plan=%p, alpha=%p, H=%p, W=%p, targets=%p, lse=%p, gradLoss=%p, dH=%p, dW=%p, workspace=%p, workspaceSize=%llu, stream=%p",
                    (const void*)handle, (const void*)plan, alpha, H, W, (const void*)targets, (const void*)lse, (const void*)gradLoss, dH, dW,
                    workspace, (unsigned long long)workspaceSize, stream_);
        if(!handle || !plan)
            return HIPTENSOR_STATUS_NOT_INITIALIZED;
        const HandleState* st = stateOf(handle);
        if(!st)
            return HIPTENSOR_STATUS_NOT_INITIALIZED;
        if(auto s = checkDevice(fn, st); s != HIPTENSOR_STATUS_SUCCESS)
            return s;
        const CrossEntropyPlan& p      = *plan;
        const int64_t           size   = dtypeSize(p.type);
        const cudaStream_t      stream = cudaStream_t(stream_);
        if(!dH && !dW)
            return HIPTENSOR_STATUS_SUCCESS;
        if((p.T > 0 && (!alpha || !H || !W || !targets || !lse || !gradLoss)) || ((uintptr_t(H) | uintptr_t(W)) & 15)
           || ((uintptr_t(dH) | uintptr_t(dW)) & 15) || (uintptr_t(targets) & 7) || ((uintptr_t(lse) | uintptr_t(gradLoss)) & 3))
        {
            HTB_LOG_ERROR(fn, "Input Parameter Error : a required pointer is nullptr or not aligned (%s)",
                          hiptensorGetErrorString(HIPTENSOR_STATUS_INVALID_VALUE));
            return HIPTENSOR_STATUS_INVALID_VALUE;
        }
        if(p.T == 0)
        {
            if(dW) // no token, no gradient
                HTB_TRY(launchStoreRows(p.type, nullptr, 0, p.V, p.D, nullptr, dW, plainRows(p.wV, p.wD, p.V), TargetRest{}, 0, 0, stream));
            return HIPTENSOR_STATUS_SUCCESS;
        }
        const FewShape           f    = fewShape(p, true);
        const uint64_t           room = workspace ? workspaceSize : 0;
        const CrossEntropyLayout l    = f.use ? layoutFew(p, f, true) : layoutIn(p, true, room);
        if(f.use ? l.bytes > room : l.piece == 0)
        {
            HTB_LOG_ERROR(fn, "Insufficient workspace: req: %llu alloc: %llu (%s)",
                          (unsigned long long)crossEntropyWorkspace(p, true, HIPTENSOR_WORKSPACE_MIN), (unsigned long long)workspaceSize,
                          hiptensorGetErrorString(HIPTENSOR_STATUS_INSUFFICIENT_WORKSPACE));
            return HIPTENSOR_STATUS_INSUFFICIENT_WORKSPACE;
        }
        unsigned char* ws     = reinterpret_cast<unsigned char*>((uintptr_t(workspace) + 255) & ~uintptr_t(255));
        const float    a      = *(const float*)alpha;
        if(f.use)
        {
            HTB_TRY(launchFewGradient(p, f, H, rowsOfH(p), W, targets, lse, gradLoss, a, reinterpret_cast<float*>(ws + l.dhOff), dH, dW,
                                      st->deviceStatus, stream));
            return HIPTENSOR_STATUS_SUCCESS;
        }
        const int      type16 = p.type == CUDA_R_16F ? CUDA_R_16F : CUDA_R_16BF;
        float*         scale  = nullptr;
        if(p.type == CUDA_R_16F)
        {
            scale = reinterpret_cast<float*>(ws + l.scaleOff);
            HTB_TRY(launchGradientScale(gradLoss, a, p.T, targets, p.ignore, p.V, scale, stream));
        }
        void* h       = ws + l.hOff;
        TokenLists lists{};
        if(l.lists)
        {
            lists.classes = reinterpret_cast<int*>(ws + l.listOff); // (read in whole words of 16 bytes)
            lists.next    = lists.classes + roundUp(p.T, 64);
            lists.first   = lists.next + roundUp(p.T, 64);
        }
        HTB_TRY(launchPackRows(p.type, H, rowsOfH(p), p.T, l.rowsT, p.D, l.ld, h, targets, p.ignore, p.V, lists, st->deviceStatus, stream));
        if(l.lists && dW)
            HTB_TRY(launchTokenLists(lists, p.T, p.V, stream));
        float*              dh   = reinterpret_cast<float*>(ws + l.dhOff);
        float*              dw   = reinterpret_cast<float*>(ws + l.dwOff);
        float*              rest = reinterpret_cast<float*>(ws + l.restOff);
        const Probabilities P{ws + l.pOff, probabilityParts(p.type, p.T), l.rowsT, l.piece};
        for(int64_t v0 = 0; v0 < p.V; v0 += l.piece)
        {
            const int64_t n = std::min(l.piece, p.V - v0);
            // segments of classes are contracted in blocks of 64: zeros up to there
            const int64_t rowsW = l.segments > 1 ? roundUp(n, 64) : n;
            const void*   w     = static_cast<const unsigned char*>(W) + v0 * p.wV * size;
            int64_t       ldw   = p.wV;
            if(l.packW)
            {
                HTB_TRY(launchPackRows(p.type, w, plainRows(p.wV, p.wD, n), n, rowsW, p.D, l.ld, ws + l.wOff, nullptr, 0, 0, TokenLists{}, nullptr, stream));
                w   = ws + l.wOff;
                ldw = l.ld;
            }
            const HeadProduct head{h, w, p.T, n, p.D, l.ld, ldw, type16, l.segments, l.rowsT, rowsW};
            HTB_TRY(launchHeadGradient(head, v0, p.V, p.ignore, targets, lse, gradLoss, a, scale, P, rest, st->smCount, st->deviceStatus, stream));
            if(dH)
                HTB_TRY(launchHiddenGradient(head, P, l.parts, dh, l.ld, v0 > 0, st->smCount, st->deviceStatus, stream));
            if(dW)
            {
                unsigned char* out = static_cast<unsigned char*>(dW) + v0 * p.wV * size;
                if(l.direct)
                    HTB_TRY(launchWeightGradient(head, P, v0, lists, rest, scale, p.type, out, p.wV, st->smCount, st->deviceStatus, stream));
                else
                {
                    // rows of W that no bulk store can write: through f32 in the workspace
                    HTB_TRY(launchWeightGradient(head, P, v0, lists, rest, nullptr, CUDA_R_32F, dw, l.ld, st->smCount, st->deviceStatus, stream));
                    HTB_TRY(launchStoreRows(p.type, dw, l.ld, n, p.D, scale, out, plainRows(p.wV, p.wD, n), TargetRest{}, 1, 0, stream));
                }
            }
        }
        if(dH)
            HTB_TRY(launchStoreRows(p.type, dh, l.ld, p.T, p.D, scale, dH, rowsOfH(p),
                                    TargetRest{P.parts == 3 ? nullptr : rest, targets, p.ignore, p.V, p.wV, p.wD, W}, l.parts, hiddenRows(p.T),
                                    stream));
        return HIPTENSOR_STATUS_SUCCESS;
    }
} // namespace htb
