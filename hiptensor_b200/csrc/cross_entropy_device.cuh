// What the kernels of the linear cross entropy share: rows of a strided tensor, joining of partial softmax sums.
#pragma once

#include "convert.cuh"
#include "cross_entropy.hpp"

namespace htb
{
    namespace
    {
        __device__ __forceinline__ int64_t rowOffset(const TokenRows& r, int64_t row)
        {
            int64_t off = 0;
            for(int i = r.nt - 1; i >= 0; i--)
            {
                const int64_t q = i ? row / r.ext[i] : 0;
                off += (row - q * r.ext[i]) * r.stride[i];
                row = q;
            }
            return off;
        }
        __device__ __forceinline__ bool counts(int64_t target, int64_t ignore, int64_t V)
        {
            return target != ignore && target >= 0 && target < V;
        }

        constexpr float kLog2e = 1.4426950408889634f;

        __device__ __forceinline__ float maxNan(float a, float b)
        {
            float r;
            asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
            return r;
        }
        // the value that exponents are taken relative to: 0 where a maximum is infinite
        __device__ __forceinline__ float reference(float m)
        {
            return fabsf(m) == INFINITY ? 0.f : m;
        }
        // (m, s): a maximum and a sum of exponentials relative to it; takes (m2, s2) in. Logits stay in natural units until the maximum
        // is taken away from them: a product with log2(e) before that would overflow for a mask of the type's lowest value, and round
        // the target's logit otherwise than the maximum (losses below 0).
        __device__ __forceinline__ void joinSums(float& m, float& s, float m2, float s2)
        {
            const float top = maxNan(m, m2), ref = reference(top);
            // nothing yet, or nothing above -infinity: not 0 * exp2(0 - ref), which is NaN far below 0
            s = (m == -INFINITY ? 0.f : s * exp2f((reference(m) - ref) * kLog2e)) + (m2 == -INFINITY ? 0.f : s2 * exp2f((reference(m2) - ref) * kLog2e));
            m = top;
        }
    } // namespace
} // namespace htb
