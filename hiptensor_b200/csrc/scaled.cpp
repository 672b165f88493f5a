// Host side of block quantisation and of the block-scaled 8-bit contraction: argument checks and mode folding.
// Everything works on fixed arrays: nothing here allocates or throws.
#include <algorithm>
#include <iterator>

#include <hiptensor/hiptensor.hpp>

#include "kernels.hpp"
#include "scaled.hpp"

namespace htb
{
    namespace
    {
        bool is8Bit(int t)
        {
            return t == CUDA_R_8F_E4M3 || t == CUDA_R_8F_E5M2;
        }
        bool isReal(int t)
        {
            return t == CUDA_R_16F || t == CUDA_R_16BF || t == CUDA_R_32F;
        }

        // one mode seen in up to three tensors
        struct Mode
        {
            int64_t  ext;
            int64_t  s[3];
            uint32_t block;
        };

        int indexOf(const int32_t* modes, int n, int32_t mode)
        {
            for(int i = 0; i < n; i++)
                if(modes[i] == mode)
                    return i;
            return -1;
        }
        bool distinct(const int32_t* modes, int n)
        {
            for(int i = 0; i < n; i++)
                if(indexOf(modes, i, modes[i]) >= 0)
                    return false;
            return true;
        }
        bool sane(const hiptensorTensorDescriptor_t& d)
        {
            if(d.mLengths.size() != d.mStrides.size() || d.mLengths.size() > std::size_t(kMaxRank))
                return false;
            for(std::size_t i = 0; i < d.mLengths.size(); i++)
                if(int64_t(d.mLengths[i]) < 0 || int64_t(d.mLengths[i]) >= (int64_t(1) << 31) || int64_t(d.mStrides[i]) < 0)
                    return false;
            return true;
        }
        // the extents of a scale tensor: one for each block along every mode, in the order of the tensor's modes
        bool scalesMatch(const hiptensorTensorDescriptor_t& X, const uint32_t* block, const hiptensorTensorDescriptor_t& S)
        {
            if(S.mType != CUDA_R_32F || S.mLengths.size() != X.mLengths.size())
                return false;
            for(std::size_t i = 0; i < X.mLengths.size(); i++)
            {
                if(block[i] != 1 && block[i] != uint32_t(kScaleBlock))
                    return false;
                if(S.mLengths[i] != (X.mLengths[i] + block[i] - 1) / block[i])
                    return false;
            }
            return true;
        }
        // Folds the modes (all of block 1) of a group whose neighbours follow each other without a gap in every tensor:
        // sorted by descending stride in the first tensor; returns the new count.
        int fold(Mode* m, int n)
        {
            std::sort(m, m + n, [](const Mode& a, const Mode& b) { return a.s[0] > b.s[0]; });
            int k = 0;
            for(int i = 0; i < n; i++)
            {
                bool merge = k > 0;
                for(int t = 0; t < 3 && merge; t++)
                    merge = m[k - 1].s[t] == m[i].s[t] * m[i].ext;
                if(merge)
                {
                    const int64_t ext = m[k - 1].ext * m[i].ext;
                    m[k - 1]          = m[i];
                    m[k - 1].ext      = ext;
                }
                else
                    m[k++] = m[i];
            }
            return k;
        }
    } // namespace

    int planQuantize(const hiptensorTensorDescriptor_t& A, const int32_t* modeA, const uint32_t* blockA,
                     const hiptensorTensorDescriptor_t& Q, const int32_t* modeQ, const hiptensorTensorDescriptor_t& S,
                     QuantPlan* out)
    {
        if(!isReal(A.mType) || !is8Bit(Q.mType) || A.mUnaryOp != HIPTENSOR_OP_IDENTITY || Q.mUnaryOp != HIPTENSOR_OP_IDENTITY
           || S.mUnaryOp != HIPTENSOR_OP_IDENTITY)
            return HIPTENSOR_STATUS_NOT_SUPPORTED;
        const int rank = int(A.mLengths.size());
        if(!sane(A) || !sane(Q) || !sane(S) || rank < 1 || int(Q.mLengths.size()) != rank || !distinct(modeA, rank)
           || !distinct(modeQ, rank) || !scalesMatch(A, blockA, S))
            return HIPTENSOR_STATUS_INVALID_VALUE;
        Mode free[kMaxRank], block[kMaxRank];
        int  nf = 0, nb = 0, blocked = 0;
        bool empty = false;
        for(int i = 0; i < rank; i++)
        {
            const int j = indexOf(modeQ, rank, modeA[i]);
            if(j < 0 || Q.mLengths[j] != A.mLengths[i])
                return HIPTENSOR_STATUS_INVALID_VALUE;
            const Mode m{int64_t(A.mLengths[i]), {int64_t(A.mStrides[i]), int64_t(Q.mStrides[j]), int64_t(S.mStrides[i])}, blockA[i]};
            blocked += m.block > 1;
            empty |= m.ext == 0;
            if(m.ext == 1)
                continue;
            if(m.ext > 1 && (m.s[1] == 0 || m.s[2] == 0) && !(m.block > 1 && S.mLengths[i] == 1 && m.s[1] != 0))
                return HIPTENSOR_STATUS_INVALID_VALUE; // two elements of an output in one place
            if(m.block > 1)
                block[nb++] = m;
            else
                free[nf++] = m;
        }
        if(blocked == 0)
            return HIPTENSOR_STATUS_INVALID_VALUE;
        if(nb > 2)
            return HIPTENSOR_STATUS_NOT_SUPPORTED;
        QuantPlan p{};
        p.typeA = A.mType;
        p.typeQ = Q.mType;
        if(empty)
        {
            *out = p; // rows = cols = 0: nothing to do
            return HIPTENSOR_STATUS_SUCCESS;
        }
        nf = fold(free, nf);
        const Mode one{1, {0, 0, 0}, 1}, oneBlock{1, {0, 0, 0}, uint32_t(kScaleBlock)};
        Mode       r, c, b = one;
        if(nb == 2)
        {
            if(nf > 1)
                return HIPTENSOR_STATUS_NOT_SUPPORTED;
            r = block[0];
            c = block[1];
            if(nf == 1)
                b = free[0];
        }
        else
        {
            if(nf > 2)
                return HIPTENSOR_STATUS_NOT_SUPPORTED;
            c = nb == 1 ? block[0] : oneBlock;
            r = one;
            if(nf == 1)
                r = free[0];
            if(nf == 2)
            {
                // the mode that A, else Q, is contiguous along shares the tiles with the blocked one; the other is a batch
                auto score = [](const Mode& m) { return (m.s[0] == 1 ? 2 : 0) + (m.s[1] == 1 ? 1 : 0); };
                const int  first
                    = score(free[0]) != score(free[1]) ? (score(free[0]) > score(free[1]) ? 0 : 1) : (free[0].ext >= free[1].ext ? 0 : 1);
                r = free[first];
                b = free[1 - first];
            }
        }
        if(r.s[0] == 1 && r.ext > 1 && c.s[0] != 1)
            std::swap(r, c);
        p.batch = b.ext;
        p.rows  = r.ext;
        p.cols  = c.ext;
        p.aB = b.s[0], p.qB = b.s[1], p.sB = b.s[2];
        p.aR = r.s[0], p.qR = r.s[1], p.sR = r.s[2];
        p.aC = c.s[0], p.qC = c.s[1], p.sC = c.s[2];
        p.blockR = int(r.block), p.blockC = int(c.block);
        *out     = p;
        return HIPTENSOR_STATUS_SUCCESS;
    }

    namespace
    {
        // The free modes of one operand as one mode (ext, stride in X, in its scales, in D, block), or a status.
        int freeMode(const hiptensorTensorDescriptor_t& X, const int32_t* modeX, const hiptensorTensorDescriptor_t& SX,
                     const uint32_t* blockX, const hiptensorTensorDescriptor_t& D, const int32_t* modeD, Mode* out)
        {
            Mode free[kMaxRank];
            int  n = 0, blocked = 0;
            bool empty = false;
            for(std::size_t i = 0; i < X.mLengths.size(); i++)
            {
                const int j = indexOf(modeD, int(D.mLengths.size()), modeX[i]);
                if(j < 0)
                    continue;
                if(D.mLengths[j] != X.mLengths[i])
                    return HIPTENSOR_STATUS_INVALID_VALUE;
                empty |= X.mLengths[i] == 0;
                if(X.mLengths[i] == 1)
                    continue;
                if(D.mStrides[j] == 0 && X.mLengths[i] > 1)
                    return HIPTENSOR_STATUS_INVALID_VALUE;
                free[n++] = Mode{int64_t(X.mLengths[i]), {int64_t(X.mStrides[i]), int64_t(SX.mStrides[i]), int64_t(D.mStrides[j])}, blockX[i]};
                blocked += blockX[i] > 1;
            }
            if(empty)
            {
                *out = Mode{0, {0, 0, 0}, 1};
                return HIPTENSOR_STATUS_SUCCESS;
            }
            if(blocked > 1 || (blocked == 1 && n > 1))
                return HIPTENSOR_STATUS_NOT_SUPPORTED;
            if(blocked == 0)
                n = fold(free, n);
            if(n > 1)
                return HIPTENSOR_STATUS_NOT_SUPPORTED;
            *out = n == 1 ? free[0] : Mode{1, {0, 0, 0}, 1};
            return HIPTENSOR_STATUS_SUCCESS;
        }
    } // namespace

    int planScaled(const hiptensorTensorDescriptor_t& A, const int32_t* modeA, const hiptensorTensorDescriptor_t& scaleA,
                   const uint32_t* blockA, const hiptensorTensorDescriptor_t& B, const int32_t* modeB,
                   const hiptensorTensorDescriptor_t& scaleB, const uint32_t* blockB, const hiptensorTensorDescriptor_t* C,
                   const hiptensorTensorDescriptor_t& D, const int32_t* modeD, int typeCompute, ScaledPlan* out)
    {
        for(const hiptensorTensorDescriptor_t* d : {&A, &scaleA, &B, &scaleB, &D})
            if(d->mUnaryOp != HIPTENSOR_OP_IDENTITY)
                return HIPTENSOR_STATUS_NOT_SUPPORTED;
        if(!is8Bit(A.mType) || !is8Bit(B.mType) || !isReal(D.mType) || typeCompute != HIPTENSOR_COMPUTE_32F)
            return HIPTENSOR_STATUS_NOT_SUPPORTED;
        for(const hiptensorTensorDescriptor_t* d : {&A, &scaleA, &B, &scaleB, &D})
            if(!sane(*d))
                return HIPTENSOR_STATUS_INVALID_VALUE;
        const int rA = int(A.mLengths.size()), rB = int(B.mLengths.size()), rD = int(D.mLengths.size());
        if(rA < 1 || rB < 1 || !distinct(modeA, rA) || !distinct(modeB, rB) || !distinct(modeD, rD)
           || !scalesMatch(A, blockA, scaleA) || !scalesMatch(B, blockB, scaleB))
            return HIPTENSOR_STATUS_INVALID_VALUE;
        if(C && (C->mType != D.mType || C->mLengths != D.mLengths || C->mStrides != D.mStrides || C->mUnaryOp != D.mUnaryOp))
            return HIPTENSOR_STATUS_NOT_SUPPORTED;
        ScaledPlan p{};
        p.K = 1;
        int contracted = 0;
        for(int i = 0; i < rA; i++)
        {
            const int j = indexOf(modeB, rB, modeA[i]), d = indexOf(modeD, rD, modeA[i]);
            if(j >= 0 && d >= 0)
                return HIPTENSOR_STATUS_NOT_SUPPORTED; // a batch mode, as in hiptensorContraction
            if(j < 0 && d < 0)
                return HIPTENSOR_STATUS_INVALID_VALUE; // neither contracted nor kept
            if(j < 0)
                continue;
            if(A.mLengths[i] != B.mLengths[j])
                return HIPTENSOR_STATUS_INVALID_VALUE;
            if(blockA[i] != uint32_t(kScaleBlock) || blockB[j] != uint32_t(kScaleBlock))
                return HIPTENSOR_STATUS_NOT_SUPPORTED; // the contracted mode is the one in blocks
            if(A.mLengths[i] == 1)
                continue;
            if(contracted++)
                return HIPTENSOR_STATUS_NOT_SUPPORTED;
            p.K = int64_t(A.mLengths[i]);
            p.aK = int64_t(A.mStrides[i]), p.bK = int64_t(B.mStrides[j]);
            p.saK = int64_t(scaleA.mStrides[i]), p.sbK = int64_t(scaleB.mStrides[j]);
        }
        for(int i = 0; i < rB; i++)
            if(indexOf(modeA, rA, modeB[i]) < 0 && indexOf(modeD, rD, modeB[i]) < 0)
                return HIPTENSOR_STATUS_INVALID_VALUE;
        for(int i = 0; i < rD; i++)
            if(indexOf(modeA, rA, modeD[i]) < 0 && indexOf(modeB, rB, modeD[i]) < 0)
                return HIPTENSOR_STATUS_INVALID_VALUE;
        Mode m, n;
        if(int rc = freeMode(A, modeA, scaleA, blockA, D, modeD, &m))
            return rc;
        if(int rc = freeMode(B, modeB, scaleB, blockB, D, modeD, &n))
            return rc;
        p.M = m.ext, p.aM = m.s[0], p.saM = m.s[1], p.dM = m.s[2], p.blockM = int(m.block);
        p.N = n.ext, p.bN = n.s[0], p.sbN = n.s[1], p.dN = n.s[2], p.blockN = int(n.block);
        p.typeA = A.mType, p.typeB = B.mType, p.typeD = D.mType;
        p.hasC = C != nullptr;
        *out   = p;
        return HIPTENSOR_STATUS_SUCCESS;
    }

    int blockQuantize(const hiptensorHandle_t* handle, const void* A, const hiptensorTensorDescriptor_t* descA,
                      const int32_t* modeA, const uint32_t* blockA, void* Q, const hiptensorTensorDescriptor_t* descQ,
                      const int32_t* modeQ, float* S, const hiptensorTensorDescriptor_t* descS, void* stream)
    {
        const char* fn = "htBlockQuantize";
        HTB_LOG_API(fn, "handle=%p, A=%p, descA=%p, Q=%p, descQ=%p, S=%p, descS=%p, stream=%p", (const void*)handle, A,
                    (const void*)descA, Q, (const void*)descQ, (void*)S, (const void*)descS, stream);
        if(!handle || !descA || !modeA || !blockA || !descQ || !modeQ || !descS)
            return HIPTENSOR_STATUS_NOT_INITIALIZED;
        QuantPlan p;
        if(int rc = planQuantize(*descA, modeA, blockA, *descQ, modeQ, *descS, &p))
        {
            HTB_LOG_ERROR(fn, "these tensors cannot be quantised in blocks (%s)", hiptensorGetErrorString(hiptensorStatus_t(rc)));
            return rc;
        }
        const HandleState* st = stateOf(handle);
        if(!st)
            return HIPTENSOR_STATUS_NOT_INITIALIZED;
        if(auto s = checkDevice(fn, st); s != HIPTENSOR_STATUS_SUCCESS)
            return s;
        if(p.rows == 0 || p.cols == 0)
            return HIPTENSOR_STATUS_SUCCESS;
        if(!A || !Q || !S || (uintptr_t(A) % uintptr_t(dtypeSize(p.typeA))) || (uintptr_t(S) & 3))
            return HIPTENSOR_STATUS_INVALID_VALUE;
        return launchResult(fn, launchQuantize(p, A, Q, S, cudaStream_t(stream)));
    }

    int scaledContraction(const hiptensorHandle_t* handle, const ScaledPlan* plan, const void* alpha, const void* A,
                          const float* scaleA, const void* B, const float* scaleB, const void* beta, const void* C, void* D,
                          void* stream)
    {
        const char* fn = "htScaledContraction";
        HTB_LOG_API(fn, "handle=%p, plan=%p, alpha=%p, A=%p, scaleA=%p, B=%p, scaleB=%p, beta=%p, C=%p, D=%p, stream=%p",
                    (const void*)handle, (const void*)plan, alpha, A, (const void*)scaleA, B, (const void*)scaleB, beta, C, D, stream);
        if(!handle || !plan)
            return HIPTENSOR_STATUS_NOT_INITIALIZED;
        const HandleState* st = stateOf(handle);
        if(!st)
            return HIPTENSOR_STATUS_NOT_INITIALIZED;
        if(auto s = checkDevice(fn, st); s != HIPTENSOR_STATUS_SUCCESS)
            return s;
        if(plan->M == 0 || plan->N == 0)
            return HIPTENSOR_STATUS_SUCCESS;
        const uintptr_t sizeD = uintptr_t(dtypeSize(plan->typeD));
        if(!alpha || !D || (plan->K > 0 && (!A || !scaleA || !B || !scaleB)) || (plan->hasC && (!beta || !C)) || (uintptr_t(D) % sizeD)
           || (plan->hasC && uintptr_t(C) % sizeD) || ((uintptr_t(scaleA) | uintptr_t(scaleB)) & 3))
        {
            HTB_LOG_ERROR(fn, "Input Parameter Error : a required pointer is nullptr or not aligned to its type (%s)",
                          hiptensorGetErrorString(HIPTENSOR_STATUS_INVALID_VALUE));
            return HIPTENSOR_STATUS_INVALID_VALUE;
        }
        return launchResult(fn, launchScaled(*plan, *(const float*)alpha, A, scaleA, B, scaleB, plan->hasC ? *(const float*)beta : 0.f,
                                             plan->hasC ? C : nullptr, D, st->smCount, st->deviceStatus, cudaStream_t(stream)));
    }
} // namespace htb
