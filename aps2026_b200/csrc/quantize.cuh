// What the two implementations of the top-2 routing rule have in common: the
// router scores' grid and the number of experts. moe.cu scans a token's experts
// in one thread, for many tokens; moe_decode.cu with a lane per expert, for few.
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

}  // namespace
}  // namespace b2
