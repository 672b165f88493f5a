// Softmax cross entropy of a linear head, z[t, v] = alpha * sum_d H[t, d] W[v, d], in pieces of the vocabulary and without
// keeping the logits, and its gradient. Plan, kernels' launch entry points and the bodies of the flat entry points.
#pragma once

#include <cstdint>

#include <cuda_runtime_api.h>

#include <hiptensor/hiptensor_types.hpp>

#include "planner.hpp"

namespace htb
{
    struct CrossEntropyPlan
    {
        int64_t T, V, D; // tokens, classes, contracted extent
        int     type; // of H, W, dH, dW
        // H's token modes (order of the descriptor, folded): a token's number counts them with the last one fastest
        int     nt;
        int64_t tExt[kMaxGroup], tStride[kMaxGroup];
        int64_t hD, wV, wD; // strides in elements
        int64_t ignore;
    };

    // What one call does, piece by piece, and where its scratch lies (byte offsets into the workspace).
    struct CrossEntropyLayout
    {
        bool     packH, packW; // operands copied into the workspace as packed rows of ld elements
        int64_t  ld;
        int      parts; // sums of dH that are kept apart
        int64_t  piece; // classes of a piece (a multiple of kPieceUnit, or all of them)
        uint64_t hOff, wOff, stateOff, zOff, partOff, pOff, dhOff, dwOff, scaleOff, restOff;
        uint64_t bytes;
    };

    int planCrossEntropy(const hiptensorTensorDescriptor_t& H, const int32_t* modeH, const hiptensorTensorDescriptor_t& W,
                         const int32_t* modeW, int64_t ignoreIndex, int typeCompute, CrossEntropyPlan* out);
    uint64_t crossEntropyWorkspace(const CrossEntropyPlan& p, bool gradient, int pref);

    // token rows of a strided tensor
    struct TokenRows
    {
        int     nt;
        int64_t ext[kMaxGroup], stride[kMaxGroup];
        int64_t elem; // stride along the contracted mode
    };
    // X2[r, 0 .. ld) = X[row r, 0 .. cols), zeros behind. With targets: rows whose target is `ignore` or no class become zeros,
    // and the latter raise the status word. twice: the rows again behind the first `count`.
    cudaError_t launchPackRows(int type, const void* X, const TokenRows& rows, int64_t count, int64_t cols, int64_t ld, void* X2,
                               const int64_t* targets, int64_t ignore, int64_t V, int* status, bool twice, cudaStream_t stream);

    // f16 / bf16: logits of n classes from v0 on, used where they are made
    struct HeadProduct
    {
        const void *H, *W; // rows of D elements, ldh / ldw apart, at multiples of 16 bytes
        int64_t     T, n, D, ldh, ldw;
        int         type;
    };
    constexpr int kHeadGroup = 128; // classes that share one partial maximum and sum
    // part: ceil(n / kHeadGroup) x T pairs of floats; the target logits go to state[2T .. 3T)
    cudaError_t launchHeadLoss(const HeadProduct& h, int64_t v0, const int64_t* targets, float alpha, void* part, float* state, int smCount,
                               int* status, cudaStream_t stream);
    // joins a piece's partial results with state[0 .. 2T) (maximum, sum in powers of two); after the last piece loss and lse
    cudaError_t launchLossJoin(const void* part, int64_t n, int64_t T, float* state, bool first, bool last, int64_t V, int64_t ignore,
                               const int64_t* targets, float* loss, float* lse, int* status, cudaStream_t stream);
    // P[t, v] = (exp(z - lse) - [v0 + v == target]) * g * alpha (* scale[0]); rest[t]: what rounding took from the target's entry;
    // with splitProbabilities(T) what it took from every entry in T more rows
    bool splitProbabilities(int64_t T);
    cudaError_t launchHeadGradient(const HeadProduct& h, int64_t v0, int64_t V, int64_t ignore, const int64_t* targets, const float* lse,
                                   const float* g, float alpha, const float* scale, void* P, int64_t ldp, float* rest, int smCount, int* status,
                                   cudaStream_t stream);

    // out[part][t, d] = (add: +=) sum over a part of the classes of P[t, v] W[v, d], `parts` of them side by side
    int         hiddenParts(int64_t T, int64_t D, int64_t piece);
    cudaError_t launchHiddenGradient(int type, const void* P, int64_t ldp, const void* W, int64_t ldw, int64_t T, int64_t n, int64_t D, int parts,
                                     float* out, int64_t ldo, bool add, int smCount, int* status, cudaStream_t stream);
    // dW[v, d] = sum over K rows of P[k, v] H[k, d] (* scale[1]); rows of dW ldw apart, at multiples of 16 bytes
    cudaError_t launchWeightGradient(int type, const void* P, int64_t ldp, const void* H, int64_t ldh, int64_t K, int64_t n, int64_t D,
                                     const float* scale, void* dW, int64_t ldw, int smCount, int* status, cudaStream_t stream);

    // f32: logits of a piece in memory, z[t, v] with rows ldz apart
    // running maximum / sum / target logit per token: state[0 .. T), [T .. 2T), [2T .. 3T)
    cudaError_t launchSoftmaxPiece(const float* z, int64_t ldz, int64_t T, int64_t v0, int64_t count, const int64_t* targets, float* state,
                                   cudaStream_t stream);
    cudaError_t launchLossFinish(const float* state, int64_t T, int64_t V, int64_t ignore, const int64_t* targets, float* loss, float* lse,
                                 int* deviceStatus, cudaStream_t stream);
    // z becomes P in place
    cudaError_t launchProbabilities(float* z, int64_t ldz, int64_t T, int64_t v0, int64_t count, int64_t V, int64_t ignore,
                                    const int64_t* targets, const float* lse, const float* g, float alpha, cudaStream_t stream);

    // f16: scale[0] = a power of two that brings max |g * alpha| close to the top of the range, scale[1] = its reciprocal
    cudaError_t launchGradientScale(const float* g, float alpha, int64_t T, float* scale, cudaStream_t stream);
    // Y[row r, c] = (sum of `parts` X[r, c] + rest[r] * W[target of r, c]) (* scale[1]) rounded to `type`; parts 0: zeros; rest null: none
    struct TargetRest
    {
        const float*   rest;
        const int64_t* targets;
        int64_t        ignore, V, wV, wD;
        const void*    W;
    };
    cudaError_t launchStoreRows(int type, const float* X, int64_t ldx, int64_t count, int64_t cols, const float* scale, void* Y,
                                const TokenRows& rows, const TargetRest& rest, int parts, cudaStream_t stream);

    int crossEntropy(const hiptensorHandle_t* handle, const CrossEntropyPlan* plan, const void* alpha, const void* H, const void* W,
                     const int64_t* targets, float* loss, float* lse, void* workspace, uint64_t workspaceSize, void* stream);
    int crossEntropyGradient(const hiptensorHandle_t* handle, const CrossEntropyPlan* plan, const void* alpha, const void* H,
                             const void* W, const int64_t* targets, const float* lse, const float* gradLoss, void* dH, void* dW,
                             void* workspace, uint64_t workspaceSize, void* stream);
} // namespace htb
