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
        int     sms; // of the handle's device
        int     parts; // of dH's products (hiddenParts for the whole vocabulary)
        int64_t ignore;
    };

    // What one call does, piece by piece, and where its scratch lies (byte offsets into the workspace).
    struct CrossEntropyLayout
    {
        bool     packH, packW; // operands copied into the workspace as packed rows of ld 16-bit elements
        bool     direct; // rows of dW can be written by bulk stores
        int      segments; // numbers of 16 bits that an element of the copies is a sum of: 3 for f32
        int64_t  rowsT; // of a segment of H's copy and of P
        int64_t  ld;
        int      parts; // sums of dH that are kept apart
        int64_t  piece; // classes of a piece, a multiple of 256
        bool     lists; // of the tokens of each class
        uint64_t hOff, wOff, stateOff, partOff, pOff, dhOff, dwOff, scaleOff, restOff, listOff;
        uint64_t bytes;
    };

    int planCrossEntropy(const hiptensorTensorDescriptor_t& H, const int32_t* modeH, const hiptensorTensorDescriptor_t& W,
                         const int32_t* modeW, int64_t ignoreIndex, int typeCompute, int smCount, CrossEntropyPlan* out);
    uint64_t crossEntropyWorkspace(const CrossEntropyPlan& p, bool gradient, int pref);

    // The tokens of every class (null: not wanted): `first` has a class's first token, `next` a token's follower, -1 where there is none.
    // A list ends after kListed tokens (it may go on for as many). `classes`: every token's class (-1: does not count).
    constexpr int kListed = 16;
    struct TokenLists
    {
        int *classes, *next, *first;
    };
    cudaError_t launchTokenLists(const TokenLists& lists, int64_t T, int64_t V, cudaStream_t stream);

    // token rows of a strided tensor
    struct TokenRows
    {
        int     nt;
        int64_t ext[kMaxGroup], stride[kMaxGroup];
        int64_t elem; // stride along the contracted mode
    };
    // X2[r, 0 .. ld) = X[row r, 0 .. cols), zeros behind and in rows count .. total - 1; f32 as three segments of `total` rows. With
    // targets: rows whose target is `ignore` or no class become zeros, and the latter raise the status word. lists: `classes` is
    // written.
    cudaError_t launchPackRows(int type, const void* X, const TokenRows& rows, int64_t count, int64_t total, int64_t cols, int64_t ld, void* X2,
                               const int64_t* targets, int64_t ignore, int64_t V, const TokenLists& lists, int* status, cudaStream_t stream);

    // the logits of n classes, used where they are made: operands in 16 bits, `segments` of segH / segW rows each
    struct HeadProduct
    {
        const void *H, *W; // rows of D elements, ldh / ldw apart, at multiples of 16 bytes
        int64_t     T, n, D, ldh, ldw;
        int         type; // CUDA_R_16F or CUDA_R_16BF
        int         segments;
        int64_t     segH, segW;
    };
    // P, [parts][rows][ld] in 16 bits
    struct Probabilities
    {
        void*   data;
        int     parts;
        int64_t rows, ld;
    };
    int           probabilityParts(int type, int64_t T);
    constexpr int kHeadGroup = 128; // classes that share one partial maximum and sum
    // part: ceil(n / kHeadGroup) x T pairs of floats; the target logits go to state[2T .. 3T)
    cudaError_t launchHeadLoss(const HeadProduct& h, int64_t v0, const int64_t* targets, float alpha, void* part, float* state, int smCount,
                               int* status, cudaStream_t stream);
    // joins a piece's partial results with state[0 .. 2T) (maximum, sum of exponentials); after the last piece loss and lse
    cudaError_t launchLossJoin(const void* part, int64_t n, int64_t T, float* state, bool first, bool last, int64_t V, int64_t ignore,
                               const int64_t* targets, float* loss, float* lse, int* status, cudaStream_t stream);
    // P[t, v] = (exp(z - lse) - [v0 + v == target]) * g * alpha (* scale[0]); rest[t]: what rounding took from the target's entry
    cudaError_t launchHeadGradient(const HeadProduct& h, int64_t v0, int64_t V, int64_t ignore, const int64_t* targets, const float* lse,
                                   const float* g, float alpha, const float* scale, const Probabilities& P, float* rest, int smCount, int* status,
                                   cudaStream_t stream);
    // out[part][t, d] = (add: +=) sum over a part of the classes of P[t, v] W[v, d], `parts` of them side by side
    int64_t     hiddenRows(int64_t T); // of a part in `out`
    int         hiddenParts(int64_t T, int64_t D, int64_t piece, int sms);
    cudaError_t launchHiddenGradient(const HeadProduct& h, const Probabilities& P, int parts, float* out, int64_t ldo, bool add, int smCount,
                                     int* status, cudaStream_t stream);
    // dW[v, d] = sum over the tokens of P[t, v] H[t, d] (* scale[1]); rows of dW ldw apart, at multiples of 16 bytes. With
    // lists, rest[t] H[t, d] is added for the listed tokens t of class v.
    cudaError_t launchWeightGradient(const HeadProduct& h, const Probabilities& P, int64_t v0, const TokenLists& lists, const float* rest, const float* scale,
                                     int typeOut, void* dW, int64_t ldw, int smCount, int* status, cudaStream_t stream);

    // f16: scale[0] = a power of two that brings max |g * alpha| over the tokens that count (finite ones) close to the top of the range,
    // scale[1] = its reciprocal
    cudaError_t launchGradientScale(const float* g, float alpha, int64_t T, const int64_t* targets, int64_t ignore, int64_t V, float* scale,
                                    cudaStream_t stream);
    // Y[row r, c] = (sum of `parts` X[r, c], partRows rows apart, + rest[r] * W[target of r, c]) (* scale[1]) rounded to `type`; parts 0: zeros; rest null:
    // none. With targets: 0 in the rows of tokens that do not count.
    struct TargetRest
    {
        const float*   rest;
        const int64_t* targets;
        int64_t        ignore, V, wV, wD;
        const void*    W;
    };
    cudaError_t launchStoreRows(int type, const float* X, int64_t ldx, int64_t count, int64_t cols, const float* scale, void* Y,
                                const TokenRows& rows, const TargetRest& rest, int parts, int64_t partRows, cudaStream_t stream);

    // A few tokens, in one pass over W (cross_entropy_few.cu)
    struct FewShape
    {
        bool    use;
        int     unit; // elements of a row that are read at a time: 16 bytes, two elements or one
        int     tokens; // rounded up to a power of two
        int     threads, smem, blocks;
        int64_t units, ldh;
    };
    // part: `blocks` x T pairs of floats, as launchLossJoin reads them; the target logits go to state[2T .. 3T)
    cudaError_t launchFewLoss(const CrossEntropyPlan& p, const FewShape& f, const void* H, const TokenRows& rows, const void* W, const int64_t* targets,
                              float alpha, void* part, float* state, int* status, cudaStream_t stream);
    // part: [blocks][T][ldh] floats; dH or dW may be null
    cudaError_t launchFewGradient(const CrossEntropyPlan& p, const FewShape& f, const void* H, const TokenRows& rows, const void* W,
                                  const int64_t* targets, const float* lse, const float* g, float alpha, float* part, void* dH, void* dW, int* status,
                                  cudaStream_t stream);

    int crossEntropy(const hiptensorHandle_t* handle, const CrossEntropyPlan* plan, const void* alpha, const void* H, const void* W,
                     const int64_t* targets, float* loss, float* lse, void* workspace, uint64_t workspaceSize, void* stream);
    int crossEntropyGradient(const hiptensorHandle_t* handle, const CrossEntropyPlan* plan, const void* alpha, const void* H,
                             const void* W, const int64_t* targets, const float* lse, const float* gradLoss, void* dH, void* dW,
                             void* workspace, uint64_t workspaceSize, void* stream);
} // namespace htb
