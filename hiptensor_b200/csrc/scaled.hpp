// 8-bit tensors with a scale for each block of 128: block quantisation and the contraction of two such tensors.
// Host-side plans (plain data, passed by value to the kernels) and the launch entry points.
#pragma once

#include <cstdint>

#include <cuda_runtime_api.h>

#include <hiptensor/hiptensor_types.hpp>

namespace htb
{
    constexpr int kScaleBlock = 128;

    // Q[b, r, c] = rn_8bit(A[b, r, c] * R), S[b, r / blockR, c / blockC]: strides in elements. c is the mode along which A
    // is contiguous when there is one.
    struct QuantPlan
    {
        int64_t batch, rows, cols;
        int64_t aB, aR, aC, qB, qR, qC, sB, sR, sC;
        int     blockR, blockC; // 1 or kScaleBlock, at least one of them kScaleBlock
        int     typeA, typeQ;
    };

    // D[m, n] = alpha * sum_k scaleA[m / blockM, k / 128] A[m, k] * scaleB[n / blockN, k / 128] B[n, k] + beta * C[m, n];
    // C has D's layout. Strides in elements.
    struct ScaledPlan
    {
        int64_t M, N, K;
        int64_t aM, aK, bN, bK, dM, dN;
        int64_t saM, saK, sbN, sbK;
        int     blockM, blockN; // 1 or kScaleBlock
        int     typeA, typeB, typeD;
        int     hasC;
    };

    // Both return a hiptensorStatus_t. Descriptors and mode lists as in include/hiptensor_b200.h.
    int planQuantize(const hiptensorTensorDescriptor_t& A, const int32_t* modeA, const uint32_t* blockA,
                     const hiptensorTensorDescriptor_t& Q, const int32_t* modeQ, const hiptensorTensorDescriptor_t& S,
                     QuantPlan* out);
    int planScaled(const hiptensorTensorDescriptor_t& A, const int32_t* modeA, const hiptensorTensorDescriptor_t& scaleA,
                   const uint32_t* blockA, const hiptensorTensorDescriptor_t& B, const int32_t* modeB,
                   const hiptensorTensorDescriptor_t& scaleB, const uint32_t* blockB, const hiptensorTensorDescriptor_t* C,
                   const hiptensorTensorDescriptor_t& D, const int32_t* modeD, int typeCompute, ScaledPlan* out);

    cudaError_t launchQuantize(const QuantPlan& p, const void* A, void* Q, float* S, cudaStream_t stream);
    cudaError_t launchScaled(const ScaledPlan& p, float alpha, const void* A, const float* scaleA, const void* B,
                             const float* scaleB, float beta, const void* C, void* D, int smCount, int* deviceStatus,
                             cudaStream_t stream);

    // bodies of the flat entry points
    int blockQuantize(const hiptensorHandle_t* handle, const void* A, const hiptensorTensorDescriptor_t* descA,
                      const int32_t* modeA, const uint32_t* blockA, void* Q, const hiptensorTensorDescriptor_t* descQ,
                      const int32_t* modeQ, float* S, const hiptensorTensorDescriptor_t* descS, void* stream);
    int scaledContraction(const hiptensorHandle_t* handle, const ScaledPlan* plan, const void* alpha, const void* A,
                          const float* scaleA, const void* B, const float* scaleB, const void* beta, const void* C, void* D,
                          void* stream);
} // namespace htb
