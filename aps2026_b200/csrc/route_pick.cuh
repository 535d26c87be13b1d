// Top-2 expert selection of one token, shared by the routing kernels
// (moe.cu) and the decode step's expert layer (moe_decode.cu).
#pragma once

#include "common.cuh"

namespace b2 {
namespace {

constexpr int kMaxExperts = 32;

// sign(s) * floorf(|s| / quantum + 0.5f) * quantum, the reference's
// canonicalisation (src/tensor.cu:1301-1305), with every operation rounded
// separately (no contraction is possible in the reference expression).
__device__ __forceinline__ float quantize(float s, float quantum) {
    const float r = __fmul_rn(floorf(__fadd_rn(__fdiv_rn(fabsf(s), quantum), 0.5f)), quantum);
    return s < 0.0f ? -r : r;
}

// The E router logits of one token, into registers.
__device__ __forceinline__ void load_scores(const float* row, unsigned E, float (&sc)[kMaxExperts]) {
    if ((E & 3u) == 0 && aligned16(row)) {
#pragma unroll
        for (unsigned e = 0; e < kMaxExperts; e += 4)
            if (e < E) {
                const float4 v = ld_stream(reinterpret_cast<const float4*>(row + e));
                sc[e] = v.x; sc[e + 1] = v.y; sc[e + 2] = v.z; sc[e + 3] = v.w;
            }
    } else {
#pragma unroll
        for (unsigned e = 0; e < kMaxExperts; ++e)
            if (e < E) sc[e] = __ldg(row + e);
    }
}

// The token's two experts, first | second << 8, as k_moe_top2 picks them
// (src/tensor.cu:1299-1328): the first scan takes an expert when its
// quantized score beats the best so far by more than tie_eps, the second
// scan does the same skipping the first pick. Quantizes sc in place.
__device__ __forceinline__ unsigned top2_of_scores(float (&sc)[kMaxExperts], unsigned E, float quantum,
                                                   float tie_eps) {
    int first = -1;
    float first_value = -3.402823466e+38F;
#pragma unroll
    for (unsigned e = 0; e < kMaxExperts; ++e)
        if (e < E) {
            sc[e] = quantize(sc[e], quantum);
            if (first < 0 || sc[e] > __fadd_rn(first_value, tie_eps)) {
                first = static_cast<int>(e);
                first_value = sc[e];
            }
        }
    int second = -1;
    float second_value = -3.402823466e+38F;
#pragma unroll
    for (unsigned e = 0; e < kMaxExperts; ++e)
        if (e < E && static_cast<int>(e) != first) {
            if (second < 0 || sc[e] > __fadd_rn(second_value, tie_eps)) {
                second = static_cast<int>(e);
                second_value = sc[e];
            }
        }
    return static_cast<unsigned>(first) | (static_cast<unsigned>(second) << 8);
}

}  // namespace
}  // namespace b2
