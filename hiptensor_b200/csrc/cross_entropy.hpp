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
        int64_t  piece; // classes of a piece (a multiple of kPieceUnit, or all of them)
        uint64_t hOff, wOff, stateOff, zOff, pOff, dhOff, dwOff, scaleOff;
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
    // X2[r, 0 .. ld) = X[row r, 0 .. cols), zeros behind; rows whose target is `ignore` or outside [0, V) become zeros when
    // targets are given
    cudaError_t launchPackRows(int type, const void* X, const TokenRows& rows, int64_t count, int64_t cols, int64_t ld, void* X2,
                               const int64_t* targets, int64_t ignore, int64_t V, cudaStream_t stream);
    // running maximum / sum / target logit per token: state[0 .. T), [T .. 2T), [2T .. 3T)
    cudaError_t launchSoftmaxPiece(const float* z, int64_t ldz, int64_t T, int64_t v0, int64_t count, const int64_t* targets, float* state,
                                   cudaStream_t stream);
    cudaError_t launchLossFinish(const float* state, int64_t T, int64_t V, int64_t ignore, const int64_t* targets, float* loss, float* lse,
                                 int* deviceStatus, cudaStream_t stream);
    // scale[0] = a power of two that brings max |g * alpha| close to the top of f16's range, scale[1] = its reciprocal
    cudaError_t launchGradientScale(const float* g, float alpha, int64_t T, float* scale, cudaStream_t stream);
    // P[t, v] = (exp(z - lse) - [v0 + v == target]) * g * alpha (* scale[0])
    cudaError_t launchProbabilities(int type, const float* z, int64_t ldz, int64_t T, int64_t v0, int64_t count, int64_t V, int64_t ignore,
                                    const int64_t* targets, const float* lse, const float* g, float alpha, const float* scale, void* P,
                                    int64_t ldp, int* deviceStatus, cudaStream_t stream);
    // Y[row r, c] = X[r, c] (* scale[1]) rounded to `type`
    cudaError_t launchStoreRows(int type, const float* X, int64_t ldx, int64_t count, int64_t cols, const float* scale, void* Y,
                                const TokenRows& rows, cudaStream_t stream);

    int crossEntropy(const hiptensorHandle_t* handle, const CrossEntropyPlan* plan, const void* alpha, const void* H, const void* W,
                     const int64_t* targets, float* loss, float* lse, void* workspace, uint64_t workspaceSize, void* stream);
    int crossEntropyGradient(const hiptensorHandle_t* handle, const CrossEntropyPlan* plan, const void* alpha, const void* H,
                             const void* W, const int64_t* targets, const float* lse, const float* gradLoss, void* dH, void* dW,
                             void* workspace, uint64_t workspaceSize, void* stream);
} // namespace htb
