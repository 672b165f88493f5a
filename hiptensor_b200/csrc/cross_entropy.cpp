// Host side of the linear cross entropy and its gradient: mode folding, the layout of the workspace, the walk over the
// pieces of the vocabulary. The products are this library's own contractions.
#include <algorithm>

#include <hiptensor/hiptensor.hpp>

#include "cross_entropy.hpp"
#include "kernels.hpp"

namespace htb
{
    namespace
    {
        constexpr int64_t  kPieceUnit   = 256; // classes; a piece's rows then start at multiples of 16 bytes in every type
        constexpr uint64_t kRecommended = uint64_t(512) << 20; // bytes of the pieces' buffers under WORKSPACE_RECOMMENDED

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

        // The layout for pieces of `piece` classes. Every buffer starts at a multiple of 256 bytes.
        CrossEntropyLayout layoutFor(const CrossEntropyPlan& p, bool gradient, int64_t piece)
        {
            CrossEntropyLayout l{};
            const uint64_t     size = uint64_t(dtypeSize(p.type));
            const int64_t      unit = 16 / int64_t(size);
            const bool wordsH = p.nt <= 1 && p.hD == 1 && (p.T == 1 || (p.tStride[0] % unit == 0 && p.tStride[0] >= p.D));
            // (the gradient's products read W along its rows, too: their length has to be one of whole 16-byte words)
            const bool wordsW = p.wD == 1 && (p.V == 1 || (p.wV % unit == 0 && p.wV >= p.D)) && (!gradient || p.D % unit == 0);
            // the gradient reads a copy of H whose rows of ignored tokens are zeros: what lies there (padding, NaN) must not
            // reach dW through 0 * NaN
            l.packH  = gradient || !wordsH;
            l.packW  = !wordsW;
            l.ld     = roundUp(p.D, unit);
            l.piece  = piece;
            uint64_t at   = 0;
            auto     take = [&](bool wanted, uint64_t bytes) {
                const uint64_t here = at;
                if(wanted)
                    at += (bytes + 255) / 256 * 256;
                return here;
            };
            const uint64_t T = uint64_t(p.T), n = uint64_t(piece);
            const bool f32   = p.type == CUDA_R_32F, two = gradient && !f32 && splitProbabilities(p.T);
            l.hOff           = take(l.packH, (two ? 2 : 1) * T * uint64_t(l.ld) * size);
            l.stateOff       = take(!gradient, T * 12);
            l.scaleOff       = take(gradient, 8);
            l.restOff        = take(gradient, T * 4);
            l.parts          = f32 ? 0 : hiddenParts(p.T, l.ld, piece);
            l.dhOff          = take(gradient, uint64_t(std::max(l.parts, 1)) * T * uint64_t(l.ld) * 4);
            l.wOff           = take(l.packW, n * uint64_t(l.ld) * size);
            l.zOff           = take(f32, T * n * 4);
            l.partOff        = take(!f32 && !gradient, (n + kHeadGroup - 1) / kHeadGroup * T * 8);
            l.pOff           = take(!f32 && gradient, (two ? 2 : 1) * T * n * size);
            l.dwOff          = take(gradient && !f32 && l.packW, n * uint64_t(l.ld) * 4);
            l.bytes          = at + 256; // room to align the caller's pointer
            return l;
        }
        // the largest pieces that fit into `bytes`; piece = 0 when not even the smallest do
        CrossEntropyLayout layoutIn(const CrossEntropyPlan& p, bool gradient, uint64_t bytes)
        {
            int64_t lo = 0, hi = roundUp(p.V, kPieceUnit) / kPieceUnit; // pieces of lo units fit
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

        // D[m, n] = alpha * sum_k A B + beta * D through the library's contraction planner: matrices given by extents and
        // the strides of their two modes
        struct Matrix
        {
            const void* data;
            int64_t     rows, cols, sRow, sCol;
            int         type;
        };
        cudaError_t product(const Matrix& A, int aRow, int aCol, const Matrix& B, int bRow, int bCol, const Matrix& D, int dRow, int dCol,
                            float alpha, float beta, const HandleState* st, cudaStream_t stream)
        {
            const int64_t   lA[2] = {A.rows, A.cols}, sA[2] = {A.sRow, A.sCol}, lB[2] = {B.rows, B.cols}, sB[2] = {B.sRow, B.sCol},
                          lD[2] = {D.rows, D.cols}, sD[2] = {D.sRow, D.sCol};
            const int32_t   mA[2] = {aRow, aCol}, mB[2] = {bRow, bCol}, mD[2] = {dRow, dCol};
            ContractionPlan plan;
            const int rc = planContraction(TensorView{2, lA, sA, mA, A.type}, TensorView{2, lB, sB, mB, B.type},
                                           TensorView{2, lD, sD, mD, D.type}, D.type, beta != 0.f, HIPTENSOR_COMPUTE_32F, st->smCount, &plan, 0);
            if(rc != PLAN_OK)
                return cudaErrorNotSupported;
            return launchContraction(plan, alpha, A.data, B.data, beta, beta != 0.f ? D.data : nullptr, const_cast<void*>(D.data), nullptr, 0,
                                     st->smCount, st->deviceStatus, stream);
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
                         const int32_t* modeW, int64_t ignoreIndex, int typeCompute, CrossEntropyPlan* out)
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
        if(p.V >= (int64_t(1) << 31) - 512 || p.T >= (int64_t(1) << 31) - 512 || p.D >= (int64_t(1) << 31) - 512)
            return HIPTENSOR_STATUS_NOT_SUPPORTED;
        *out = p;
        return HIPTENSOR_STATUS_SUCCESS;
    }

    uint64_t crossEntropyWorkspace(const CrossEntropyPlan& p, bool gradient, int pref)
    {
        if(p.T == 0)
            return 0;
        const uint64_t least = layoutFor(p, gradient, kPieceUnit).bytes, most = layoutFor(p, gradient, roundUp(p.V, kPieceUnit)).bytes;
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
        const CrossEntropyLayout l = layoutIn(p, false, workspace ? workspaceSize : 0);
        if(l.piece == 0)
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
        float*             state  = reinterpret_cast<float*>(ws + l.stateOff);
        const void*        h      = H;
        int64_t            ldh    = p.nt ? p.tStride[0] : l.ld;
        if(l.packH)
        {
            HTB_TRY(launchPackRows(p.type, H, rowsOfH(p), p.T, p.D, l.ld, ws + l.hOff, nullptr, 0, 0, nullptr, false, stream));
            h   = ws + l.hOff;
            ldh = l.ld;
        }
        const bool f32 = p.type == CUDA_R_32F;
        float*     z   = reinterpret_cast<float*>(ws + l.zOff);
        for(int64_t v0 = 0; v0 < p.V; v0 += l.piece)
        {
            const int64_t n   = std::min(l.piece, p.V - v0);
            const void*   w   = static_cast<const unsigned char*>(W) + v0 * p.wV * size;
            int64_t       ldw = p.wV;
            if(l.packW)
            {
                HTB_TRY(launchPackRows(p.type, w, plainRows(p.wV, p.wD, n), n, p.D, l.ld, ws + l.wOff, nullptr, 0, 0, nullptr, false, stream));
                w   = ws + l.wOff;
                ldw = l.ld;
            }
            if(f32)
            {
                HTB_TRY(product(Matrix{h, p.T, p.D, ldh, 1, p.type}, 0, 2, Matrix{w, n, p.D, ldw, 1, p.type}, 1, 2,
                                Matrix{z, p.T, n, l.piece, 1, CUDA_R_32F}, 0, 1, a, 0.f, st, stream));
                HTB_TRY(launchSoftmaxPiece(z, l.piece, p.T, v0, n, targets, state, stream));
            }
            else
            {
                HTB_TRY(launchHeadLoss(HeadProduct{h, w, p.T, n, p.D, ldh, ldw, p.type}, v0, targets, a, ws + l.partOff, state, st->smCount,
                                       st->deviceStatus, stream));
                HTB_TRY(launchLossJoin(ws + l.partOff, n, p.T, state, v0 == 0, v0 + n == p.V, p.V, p.ignore, targets, loss, lse,
                                       st->deviceStatus, stream));
            }
        }
        if(f32)
            HTB_TRY(launchLossFinish(state, p.T, p.V, p.ignore, targets, loss, lse, st->deviceStatus, stream));
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
                HTB_TRY(launchStoreRows(p.type, nullptr, 0, p.V, p.D, nullptr, dW, plainRows(p.wV, p.wD, p.V), TargetRest{}, 0, stream));
            return HIPTENSOR_STATUS_SUCCESS;
        }
        const CrossEntropyLayout l = layoutIn(p, true, workspace ? workspaceSize : 0);
        if(l.piece == 0)
        {
            HTB_LOG_ERROR(fn, "Insufficient workspace: req: %llu alloc: %llu (%s)",
                          (unsigned long long)crossEntropyWorkspace(p, true, HIPTENSOR_WORKSPACE_MIN), (unsigned long long)workspaceSize,
                          hiptensorGetErrorString(HIPTENSOR_STATUS_INSUFFICIENT_WORKSPACE));
            return HIPTENSOR_STATUS_INSUFFICIENT_WORKSPACE;
        }
        unsigned char* ws    = reinterpret_cast<unsigned char*>((uintptr_t(workspace) + 255) & ~uintptr_t(255));
        const float    a     = *(const float*)alpha;
        const bool     f32   = p.type == CUDA_R_32F;
        float*         scale = nullptr;
        if(p.type == CUDA_R_16F)
        {
            scale = reinterpret_cast<float*>(ws + l.scaleOff);
            HTB_TRY(launchGradientScale(gradLoss, a, p.T, scale, stream));
        }
        const bool    two   = !f32 && splitProbabilities(p.T);
        const int64_t rowsK = two ? 2 * p.T : p.T; // of P and H in the weights' product
        void*         h     = ws + l.hOff;
        HTB_TRY(launchPackRows(p.type, H, rowsOfH(p), p.T, p.D, l.ld, h, targets, p.ignore, p.V, st->deviceStatus, two, stream));
        float*       z   = reinterpret_cast<float*>(ws + l.zOff);
        void*        P   = f32 ? (void*)z : (void*)(ws + l.pOff);
        float*       dh  = reinterpret_cast<float*>(ws + l.dhOff);
        float*       dw  = reinterpret_cast<float*>(ws + l.dwOff);
        float*       rest = reinterpret_cast<float*>(ws + l.restOff);
        // the copies are as wide as their rows (zeros behind D), and so are the results' buffers
        const Matrix Hm{h, p.T, l.ld, l.ld, 1, p.type};
        for(int64_t v0 = 0; v0 < p.V; v0 += l.piece)
        {
            const int64_t n   = std::min(l.piece, p.V - v0);
            const void*   w   = static_cast<const unsigned char*>(W) + v0 * p.wV * size;
            int64_t       ldw = p.wV;
            if(l.packW)
            {
                HTB_TRY(launchPackRows(p.type, w, plainRows(p.wV, p.wD, n), n, p.D, l.ld, ws + l.wOff, nullptr, 0, 0, nullptr, false, stream));
                w   = ws + l.wOff;
                ldw = l.ld;
            }
            const Matrix Wm{w, n, l.ld, ldw, 1, p.type}, Pm{P, p.T, n, l.piece, 1, p.type};
            if(f32)
            {
                HTB_TRY(product(Hm, 0, 2, Wm, 1, 2, Matrix{z, p.T, n, l.piece, 1, CUDA_R_32F}, 0, 1, a, 0.f, st, stream));
                HTB_TRY(launchProbabilities(z, l.piece, p.T, v0, n, p.V, p.ignore, targets, lse, gradLoss, a, stream));
            }
            else
                HTB_TRY(launchHeadGradient(HeadProduct{h, w, p.T, n, p.D, l.ld, ldw, p.type}, v0, p.V, p.ignore, targets, lse, gradLoss, a,
                                           scale, P, l.piece, rest, st->smCount, st->deviceStatus, stream));
            if(dH && l.parts > 0)
                HTB_TRY(launchHiddenGradient(p.type, P, l.piece, w, ldw, p.T, n, l.ld, l.parts, dh, l.ld, v0 > 0, st->smCount, st->deviceStatus,
                                             stream));
            else if(dH)
                HTB_TRY(product(Pm, 0, 1, Wm, 1, 2, Matrix{dh, p.T, l.ld, l.ld, 1, CUDA_R_32F}, 0, 2, 1.f, v0 ? 1.f : 0.f, st, stream));
            if(dW)
            {
                unsigned char* out = static_cast<unsigned char*>(dW) + v0 * p.wV * size;
                if(!f32 && !l.packW)
                    HTB_TRY(launchWeightGradient(p.type, P, l.piece, h, l.ld, rowsK, n, p.D, scale, out, p.wV, st->smCount, st->deviceStatus,
                                                 stream));
                else if(!f32)
                {
                    // rows of W that no bulk store can write: through f32 in the workspace
                    const Matrix P2{P, rowsK, n, l.piece, 1, p.type}, H2{h, rowsK, l.ld, l.ld, 1, p.type};
                    HTB_TRY(product(P2, 0, 1, H2, 0, 2, Matrix{dw, n, l.ld, l.ld, 1, CUDA_R_32F}, 1, 2, 1.f, 0.f, st, stream));
                    HTB_TRY(launchStoreRows(p.type, dw, l.ld, n, p.D, scale, out, plainRows(p.wV, p.wD, n), TargetRest{}, 1, stream));
                }
                else
                    HTB_TRY(product(Pm, 0, 1, Matrix{h, p.T, p.D, l.ld, 1, p.type}, 0, 2, Matrix{out, n, p.D, p.wV, p.wD, p.type}, 1, 2, 1.f, 0.f, st, stream));
            }
        }
        if(dH)
            HTB_TRY(launchStoreRows(p.type, dh, l.ld, p.T, p.D, scale, dH, rowsOfH(p),
                                    f32 ? TargetRest{} : TargetRest{rest, targets, p.ignore, p.V, p.wV, p.wD, W}, std::max(l.parts, 1), stream));
        return HIPTENSOR_STATUS_SUCCESS;
    }
} // namespace htb
