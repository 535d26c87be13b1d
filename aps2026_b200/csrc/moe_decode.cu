// The expert layer for a few tokens (b2_moe_decode): top-2 routing, the gated
// expert products and the weighted sum, in two launches.
//
// Mathematics: for token t and each of its two experts e,
//   a(t, e) = silu(Wg[e] x[t]) * (Wu[e] x[t]),   out[t] = sum_e g(t, e) Wd[e] a(t, e).
//
// One warp per dot product: (assignment, row of gate and up), then (token,
// row of out). A plain form that is right for every case.
#include <cuda_bf16.h>

#include "route_pick.cuh"

namespace b2 {
namespace {

constexpr std::size_t kMaxDecodeTokens = 128;

struct MoeDecodeArgs {
    const void* x;
    std::size_t ld_x;
    const float* logits;
    unsigned T, H, E, I;
    float quantum, tie_eps;
    unsigned gates;
    const void* w_gate_up;
    const void* w_down;
    void* out;
    std::size_t ld_out;
    float* act;  // [2T, I]
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

// The token's experts in ascending order and their gates.
__device__ __forceinline__ void route(const MoeDecodeArgs& a, unsigned t, unsigned (&e)[2], float (&g)[2]) {
    float sc[kMaxExperts];
    const float* row = a.logits + static_cast<std::size_t>(t) * a.E;
    load_scores(row, a.E, sc);
    const unsigned pair = top2_of_scores(sc, a.E, a.quantum, a.tie_eps);
    e[0] = min(pair & 0xFFu, pair >> 8);
    e[1] = max(pair & 0xFFu, pair >> 8);
    g[0] = g[1] = 0.5f;
    if (a.gates == B2_GATES_SOFTMAX) {
        const float x0 = __ldg(row + e[0]), x1 = __ldg(row + e[1]), m = fmaxf(x0, x1);
        const float p0 = expf(x0 - m), p1 = expf(x1 - m);
        g[0] = p0 / (p0 + p1);
        g[1] = p1 / (p0 + p1);
    }
}

template <typename T, typename W>
__global__ void __launch_bounds__(256)
moe_gate_up_rows(MoeDecodeArgs a) {
    pdl_begin();
    const unsigned lane = threadIdx.x & 31;
    const std::size_t units = static_cast<std::size_t>(2) * a.T * a.I;
    for (std::size_t u = static_cast<std::size_t>(blockIdx.x) * 8 + threadIdx.x / 32; u < units;
         u += static_cast<std::size_t>(gridDim.x) * 8) {
        const unsigned p = static_cast<unsigned>(u / a.I), i = static_cast<unsigned>(u % a.I);
        unsigned e[2];
        float g[2];
        route(a, p / 2, e, g);
        const T* x = static_cast<const T*>(a.x) + (p / 2) * a.ld_x;
        const W* wg = static_cast<const W*>(a.w_gate_up) + (static_cast<std::size_t>(e[p & 1]) * 2 * a.I + i) * a.H;
        const W* wu = wg + static_cast<std::size_t>(a.I) * a.H;
        float sg = 0.0f, su = 0.0f;
        for (unsigned h = lane; h < a.H; h += 32) {
            sg += to_f(wg[h]) * to_f(x[h]);
            su += to_f(wu[h]) * to_f(x[h]);
        }
        sg = warp_sum(sg);
        su = warp_sum(su);
        if (lane == 0) a.act[u] = sg / (1.0f + expf(-sg)) * su;
    }
}

template <typename T, typename W>
__global__ void __launch_bounds__(256)
moe_down_rows(MoeDecodeArgs a) {
    pdl_begin();
    const unsigned lane = threadIdx.x & 31;
    const std::size_t units = static_cast<std::size_t>(a.T) * a.H;
    for (std::size_t u = static_cast<std::size_t>(blockIdx.x) * 8 + threadIdx.x / 32; u < units;
         u += static_cast<std::size_t>(gridDim.x) * 8) {
        const unsigned t = static_cast<unsigned>(u / a.H), h = static_cast<unsigned>(u % a.H);
        unsigned e[2];
        float g[2];
        route(a, t, e, g);
        float y = 0.0f;
        for (unsigned s = 0; s < 2; ++s) {
            const W* w = static_cast<const W*>(a.w_down) + (static_cast<std::size_t>(e[s]) * a.H + h) * a.I;
            const float* act = a.act + (static_cast<std::size_t>(2) * t + s) * a.I;
            float d = 0.0f;
            for (unsigned i = lane; i < a.I; i += 32) d += to_f(w[i]) * act[i];
            y += g[s] * warp_sum(d);
        }
        if (lane == 0) {
            T* out = static_cast<T*>(a.out) + t * a.ld_out + h;
            if constexpr (sizeof(T) == 2) *out = __float2bfloat16_rn(y);
            else *out = y;
        }
    }
}

template <typename T, typename W>
void launch_moe(const MoeDecodeArgs& a, cudaStream_t s) {
    const std::size_t up = static_cast<std::size_t>(2) * a.T * a.I, down = static_cast<std::size_t>(a.T) * a.H;
    auto k1 = moe_gate_up_rows<T, W>;
    auto k2 = moe_down_rows<T, W>;
    launch_pdl(k1, wave_grid(reinterpret_cast<const void*>(k1), 256, 0, (up + 7) / 8), 256, 0, s, a);
    launch_pdl(k2, wave_grid(reinterpret_cast<const void*>(k2), 256, 0, (down + 7) / 8), 256, 0, s, a);
}

}  // namespace
}  // namespace b2

extern "C" {

int b2_moe_decode_workspace_size(size_t T, size_t I, size_t* bytes) {
    using namespace b2;
    if (!bytes) return invalid("b2_moe_decode_workspace_size: null pointer");
    if (T > kMaxDecodeTokens || I > 0x7FFFFFFu)
        return invalid("b2_moe_decode_workspace_size: T must be 128 at most, I below 2^27");
    *bytes = 2 * T * I * sizeof(float) + 16;
    return B2_OK;
}

int b2_moe_decode(const void* x, size_t ld_x, uint32_t x_dtype, const float* logits, size_t T, size_t H, size_t E,
                  size_t I, float quantum, float tie_eps, uint32_t gates, const void* w_gate_up,
                  const void* w_down, uint32_t w_dtype, void* out, size_t ld_out, void* workspace,
                  size_t workspace_bytes, b2_stream_t stream) {
    using namespace b2;
    if (E < 2 || E > static_cast<size_t>(kMaxExperts)) return invalid("b2_moe_decode: E must be in [2, 32]");
    if (x_dtype > B2_DTYPE_BF16 || w_dtype > B2_DTYPE_BF16) return invalid("b2_moe_decode: unknown dtype");
    if (gates > B2_GATES_SOFTMAX) return invalid("b2_moe_decode: unknown gates");
    if (T > kMaxDecodeTokens)
        return set_error(B2_ERR_UNSUPPORTED, "b2_moe_decode: more than 128 tokens (route with b2_moe_route)");
    if (T == 0) return B2_OK;
    if (H == 0 || I == 0 || H > 0x7FFFFFFu || I > 0x7FFFFFFu) return invalid("b2_moe_decode: H and I must be in [1, 2^27)");
    if (ld_x < H || ld_out < H) return invalid("b2_moe_decode: row stride below H");
    if (!x || !logits || !w_gate_up || !w_down || !out || !workspace) return invalid("b2_moe_decode: null pointer");
    std::size_t need = 0;
    b2_moe_decode_workspace_size(T, I, &need);
    if (workspace_bytes < need) return invalid("b2_moe_decode: workspace too small");
    if (!aligned16(workspace)) return invalid("b2_moe_decode: misaligned workspace");
    MoeDecodeArgs a{};
    a.x = x; a.ld_x = ld_x; a.logits = logits;
    a.T = static_cast<unsigned>(T); a.H = static_cast<unsigned>(H);
    a.E = static_cast<unsigned>(E); a.I = static_cast<unsigned>(I);
    a.quantum = quantum; a.tie_eps = tie_eps; a.gates = gates;
    a.w_gate_up = w_gate_up; a.w_down = w_down; a.out = out; a.ld_out = ld_out;
    a.act = static_cast<float*>(workspace);
    cudaStream_t s = as_stream(stream);
    if (x_dtype == B2_DTYPE_F32) {
        if (w_dtype == B2_DTYPE_F32) launch_moe<float, float>(a, s);
        else launch_moe<float, __nv_bfloat16>(a, s);
    } else {
        if (w_dtype == B2_DTYPE_F32) launch_moe<__nv_bfloat16, float>(a, s);
        else launch_moe<__nv_bfloat16, __nv_bfloat16>(a, s);
    }
    return launch_result("b2_moe_decode");
}

}  // extern "C"
