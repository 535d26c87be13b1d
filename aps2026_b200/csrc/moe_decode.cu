// The expert layer for a few tokens (b2_moe_decode): top-2 routing, the gated
// expert products and the weighted sum, in two launches.
//
// Mathematics: for token t and each of its two experts e,
//   a(t, e) = silu(Wg[e] x[t]) * (Wu[e] x[t]),   out[t] = sum_e g(t, e) Wd[e] a(t, e).
//
// HBM bound: with T <= 128 tokens every weight of an expert that is reached
// is read once and meets few tokens, so the weights stream from HBM through a
// ring of cp.async stages in shared memory. Which k a lane holds of the
// matrix instruction's M = 16 operand is free as long as both operands agree,
// so a lane takes 16 neighbouring bytes of its rows: it copies exactly what
// it will use, every ring is private to a lane, and no barrier is needed. Up
// to 16 tokens are the instruction's N, staged the same way.
// The instruction multiplies bf16 or TF32; fp32's accuracy is kept in
// parts: bf16 weights meet fp32 activations as three bf16 parts (24 bits),
// fp32 weights as TF32 hi and lo (hi hi + hi lo + lo hi). Its accumulator
// truncates, so chains are short (2 blocks) and added in registers.
//
// Launch 1, moe_gate_up: an item is (expert with up to 8 NT of its tokens,
// 8 MT rows of gate and the same of up); a CTA takes equally many items, one
// after the other through the same rings. Its warps interleave the k blocks,
// so together they read whole lines, and add up in shared memory. Launch 2,
// moe_down: CTA = 16 rows of the output for all tokens; warps take (expert,
// token chunk, part of k) and meet in shared memory, where a token's two
// experts are summed in ascending order: no atomics, results repeat. Each
// CTA routes for itself (T x E logits). Launch 2 starts under launch 1 and
// has routed and requested its first weights before it waits.
#include <algorithm>

#include <cuda_bf16.h>

#include "route_pick.cuh"

namespace b2 {
namespace {

constexpr unsigned kMaxDecodeTokens = 128;
constexpr unsigned kMaxGroups = kMaxExperts + 2 * kMaxDecodeTokens / 16;
constexpr unsigned kChain = 2;           // blocks between two additions in registers
constexpr unsigned kDownPartials = 256;  // (part of k, assignment) sums of moe_down
constexpr unsigned kUpRing = 8192, kDownRing = 10240;  // bytes of a warp's stages

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
    float* act;       // [2T, act_ld]: assignment 2t + s, s = 0 the lower expert
    unsigned act_ld;  // I rounded up to 8; zeros past I
};

// ---- routing, per CTA ----------------------------------------------------------

struct Plan {
    unsigned mask[kMaxDecodeTokens / 32][kMaxExperts];     // tokens of each expert, by bit
    unsigned char lists[kMaxExperts][kMaxDecodeTokens];    // assignments of each expert, tokens ascending
    float gate[2 * kMaxDecodeTokens];
    unsigned group[kMaxGroups];                            // expert | first in list << 8 | count << 16
    unsigned groups;
};
__device__ __forceinline__ unsigned group_expert(unsigned g) { return g & 0xFFu; }
__device__ __forceinline__ unsigned group_first(unsigned g) { return (g >> 8) & 0xFFu; }
__device__ __forceinline__ unsigned group_count(unsigned g) { return g >> 16; }

// Routes the tokens and cuts every expert's into groups of CHUNK. THREADS >=
// 256. Ends with a barrier.
template <unsigned CHUNK>
__device__ __forceinline__ void make_plan(const MoeDecodeArgs& a, Plan& p) {
    const unsigned t = threadIdx.x, lane = t & 31, warp = t / 32;
    const unsigned words = (a.T + 31) / 32;
    unsigned lo = 0xFFu, hi = 0xFFu;
    if (warp < words) {
        if (t < a.T) {
            float sc[kMaxExperts];
            const float* row = a.logits + static_cast<std::size_t>(t) * a.E;
            load_scores(row, a.E, sc);
            const unsigned pair = top2_of_scores(sc, a.E, a.quantum, a.tie_eps);
            lo = min(pair & 0xFFu, pair >> 8);
            hi = max(pair & 0xFFu, pair >> 8);
            float g0 = 0.5f, g1 = 0.5f;
            if (a.gates == B2_GATES_SOFTMAX) {
                const float x0 = __ldg(row + lo), x1 = __ldg(row + hi), m = fmaxf(x0, x1);
                const float p0 = expf(x0 - m), p1 = expf(x1 - m);
                g0 = p0 / (p0 + p1);
                g1 = p1 / (p0 + p1);
            }
            p.gate[2 * t] = g0;
            p.gate[2 * t + 1] = g1;
        }
        unsigned mine = 0;
        for (unsigned e = 0; e < a.E; ++e) {
            const unsigned m = __ballot_sync(0xffffffffu, lo == e || hi == e);
            if (lane == e) mine = m;
        }
        p.mask[warp][lane] = mine;
    }
    __syncthreads();
    if (t < a.T) {
        const unsigned below = (1u << lane) - 1u;
        unsigned r0 = __popc(p.mask[warp][lo] & below), r1 = __popc(p.mask[warp][hi] & below);
        for (unsigned w = 0; w < warp; ++w) {
            r0 += __popc(p.mask[w][lo]);
            r1 += __popc(p.mask[w][hi]);
        }
        p.lists[lo][r0] = static_cast<unsigned char>(2 * t);
        p.lists[hi][r1] = static_cast<unsigned char>(2 * t + 1);
    }
    if (warp == 7) {
        unsigned n = 0;
        for (unsigned w = 0; w < words; ++w) n += __popc(p.mask[w][lane]);
        const unsigned chunks = (n + CHUNK - 1) / CHUNK;
        unsigned end = chunks;
#pragma unroll
        for (unsigned o = 1; o < 32; o <<= 1) {
            const unsigned v = __shfl_up_sync(0xffffffffu, end, o);
            if (lane >= o) end += v;
        }
        for (unsigned i = 0; i < chunks; ++i)
            p.group[end - chunks + i] = lane | (i * CHUNK) << 8 | min(CHUNK, n - i * CHUNK) << 16;
        if (lane == 31) p.groups = end;
    }
    __syncthreads();
}

// ---- the products -------------------------------------------------------------------

__device__ __forceinline__ void mma_bf16(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                         unsigned b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                         unsigned b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&p);
}
__device__ __forceinline__ uint4 lds16(unsigned addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint2 lds8(unsigned addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
    return v;
}
// SIZE bytes of src, or zeros.
template <int SIZE>
__device__ __forceinline__ void copy_async(unsigned dst, const void* src, bool have) {
    const int bytes = have ? SIZE : 0;
    if constexpr (SIZE == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(bytes), "n"(SIZE)
                     : "memory");
}
// The same through L1: a token's two 16-byte pieces share sectors.
__device__ __forceinline__ void copy_async_l1(unsigned dst, const void* src, bool have) {
    const int bytes = have ? 16 : 0;
    asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// A block is 64 bytes of a weight row: 32 bf16 or 16 fp32; lane c of four
// holds 16 of them, k = c * PER .. + PER.
template <typename W>
constexpr unsigned kPer = 16 / sizeof(W);
template <typename W>
constexpr unsigned kBlock = 4 * kPer<W>;
// Parts of an activation that meet a weight.
template <typename X, typename W>
constexpr unsigned kParts = sizeof(X) == 2 ? 1 : sizeof(W) == 2 ? 3 : 2;

// The stages of one warp: MT 16-row tiles of a weight block (lane's rows r and
// r + 8 of each) and NT 8-token tiles of activations (lane's token r), each
// lane's bytes at its own place. VEC: every 16 bytes of a row of weights (XVEC:
// the activations that meet them) are aligned, and inside the row or past it.
template <typename X, typename W, unsigned MT, unsigned NT, unsigned RING, bool VEC, bool XVEC>
struct Ring {
    static constexpr unsigned PER = kPer<W>, BLOCK = kBlock<W>;
    static constexpr unsigned XB = PER * sizeof(X);  // bytes of a token per lane: 32, 16 or 8
    static constexpr unsigned WEIGHTS = MT * 2 * 512, STAGE = WEIGHTS + NT * 32 * XB;
    static constexpr unsigned STAGES = RING / STAGE < 6 ? RING / STAGE : 6;
    static_assert(STAGES >= 2, "a ring of one stage");
    unsigned char* raw;     // the lane's place in the warp's first stage
    unsigned base, get, put;  // shared addresses of the lane's place: first stage, next to use, next to fill

    __device__ __forceinline__ void init(unsigned char* warp_base, unsigned lane) {
        raw = warp_base + lane * 16;
        base = get = put = smem_addr(raw);
    }
    static __device__ __forceinline__ void step(unsigned& at, unsigned base) {
        at += STAGE;
        if (at == base + STAGES * STAGE) at = base;
    }

    // w[m][i]: the lane's weights (row's start + k); ok: bit 2m + i set where
    // the row is there; left: weights from k to the row's end, if positive.
    __device__ __forceinline__ void put_weights(const W* const (&w)[MT][2], unsigned ok, int left, const void* any) {
#pragma unroll
        for (unsigned m = 0; m < MT; ++m)
#pragma unroll
            for (unsigned i = 0; i < 2; ++i) {
                const bool row = (ok >> (2 * m + i)) & 1u;
                if (VEC) {
                    const bool have = row && left > 0;
                    copy_async<16>(put + (m * 2 + i) * 512, have ? w[m][i] : any, have);
                } else {
                    W v[PER];
#pragma unroll
                    for (unsigned e = 0; e < PER; ++e) v[e] = row && static_cast<int>(e) < left ? w[m][i][e] : W(0.0f);
                    W* dst = reinterpret_cast<W*>(raw + (put - base) + (m * 2 + i) * 512);
#pragma unroll
                    for (unsigned e = 0; e < PER; ++e) dst[e] = v[e];
                }
            }
    }
    // x[n]: the lane's activations of token tile n, null where there is no
    // token (its place is left as it is: a column nobody reads).
    __device__ __forceinline__ void put_acts(const X* const (&x)[NT], int left, unsigned lane) {
#pragma unroll
        for (unsigned n = 0; n < NT; ++n) {
            if (!x[n]) continue;
            const unsigned at = put + WEIGHTS + n * 32 * XB;
            if (XVEC) {
                const bool have = left > 0;
                const X* src = x[n];  // not read where there is none
                if constexpr (XB == 32) {
                    copy_async_l1(at, src, have);
                    copy_async_l1(at + 512, src + 4, have);
                } else if constexpr (XB == 16) {
                    copy_async<16>(at, src, have);
                } else {
                    copy_async<8>(at - lane * 8, src, have);
                }
            } else {
                constexpr unsigned PIECE = XB >= 16 ? 16 / sizeof(X) : PER;  // elements per place
                X v[PER];
#pragma unroll
                for (unsigned e = 0; e < PER; ++e) v[e] = static_cast<int>(e) < left ? x[n][e] : X(0.0f);
                unsigned char* dst = raw + (at - base) - (XB == 8 ? lane * 8 : 0);
#pragma unroll
                for (unsigned e = 0; e < PER; ++e) reinterpret_cast<X*>(dst + e / PIECE * 512)[e % PIECE] = v[e];
            }
        }
    }

    // part[n] += the stage's products for nt token tiles.
    __device__ __forceinline__ void multiply(unsigned nt, float (&part)[NT][MT][4], unsigned lane) {
        constexpr unsigned PARTS = kParts<X, W>;
        uint4 w[MT][2];
#pragma unroll
        for (unsigned m = 0; m < MT; ++m) {
            w[m][0] = lds16(get + m * 1024);
            w[m][1] = lds16(get + m * 1024 + 512);
        }
#pragma unroll
        for (unsigned n = 0; n < NT; ++n) {
            if (n >= nt) break;
            const unsigned at = get + WEIGHTS + n * 32 * XB;
            unsigned b[PARTS][4];
            if constexpr (sizeof(X) == 4 && sizeof(W) == 2) {  // x = three bf16 parts
                const uint4 lo = lds16(at), hi = lds16(at + 512);
                const unsigned v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                for (unsigned i = 0; i < 4; ++i) {
                    unsigned long long rest = f2_pack(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
#pragma unroll
                    for (unsigned q = 0; q < 3; ++q) {
                        const float2 f = f2_unpack(rest);
                        b[q][i] = pack_bf16(f.x, f.y);
                        if (q < 2)
                            rest = f2_fma(f2_pack(__uint_as_float(b[q][i] << 16), __uint_as_float(b[q][i] & 0xFFFF0000u)),
                                          f2_pack(-1.0f, -1.0f), rest);
                    }
                }
            } else if constexpr (sizeof(W) == 2) {
                const uint4 v = lds16(at);
                b[0][0] = v.x; b[0][1] = v.y; b[0][2] = v.z; b[0][3] = v.w;
            } else if constexpr (sizeof(X) == 4) {  // x = TF32 hi + lo
                const uint4 v = lds16(at);
                split_tf32(v.x, b[0][0], b[1][0]);
                split_tf32(v.y, b[0][1], b[1][1]);
                split_tf32(v.z, b[0][2], b[1][2]);
                split_tf32(v.w, b[0][3], b[1][3]);
            } else {
                const uint2 v = lds8(at - lane * 8);
                b[0][0] = v.x << 16; b[0][1] = v.x & 0xFFFF0000u;
                b[0][2] = v.y << 16; b[0][3] = v.y & 0xFFFF0000u;
            }
            if constexpr (sizeof(W) == 2) {
#pragma unroll
                for (unsigned q = PARTS; q-- > 0;)
#pragma unroll
                    for (unsigned m = 0; m < MT; ++m) {
                        mma_bf16(part[n][m], w[m][0].x, w[m][1].x, w[m][0].y, w[m][1].y, b[q][0], b[q][1]);
                        mma_bf16(part[n][m], w[m][0].z, w[m][1].z, w[m][0].w, w[m][1].w, b[q][2], b[q][3]);
                    }
            } else {
#pragma unroll
                for (unsigned m = 0; m < MT; ++m) {
                    const unsigned r0[4] = {w[m][0].x, w[m][0].y, w[m][0].z, w[m][0].w};
                    const unsigned r1[4] = {w[m][1].x, w[m][1].y, w[m][1].z, w[m][1].w};
                    unsigned h0[4], l0[4], h1[4], l1[4];
#pragma unroll
                    for (unsigned i = 0; i < 4; ++i) {
                        split_tf32(r0[i], h0[i], l0[i]);
                        split_tf32(r1[i], h1[i], l1[i]);
                    }
#pragma unroll
                    for (unsigned i = 0; i < 4; i += 2) {
                        mma_tf32(part[n][m], l0[i], l1[i], l0[i + 1], l1[i + 1], b[0][i], b[0][i + 1]);
                        if (PARTS == 2)
                            mma_tf32(part[n][m], h0[i], h1[i], h0[i + 1], h1[i + 1], b[PARTS - 1][i], b[PARTS - 1][i + 1]);
                        mma_tf32(part[n][m], h0[i], h1[i], h0[i + 1], h1[i + 1], b[0][i], b[0][i + 1]);
                    }
                }
            }
        }
    }
    // w = hi + lo in TF32, hi rounded to nearest.
    static __device__ __forceinline__ void split_tf32(unsigned w, unsigned& hi, unsigned& lo) {
        hi = (w + 0x1000u) & 0xFFFFE000u;
        lo = __float_as_uint(__uint_as_float(w) - __uint_as_float(hi));
    }
};

template <unsigned NT, unsigned MT>
__device__ __forceinline__ void clear(float (&v)[NT][MT][4]) {
#pragma unroll
    for (unsigned n = 0; n < NT; ++n)
#pragma unroll
        for (unsigned m = 0; m < MT; ++m) v[n][m][0] = v[n][m][1] = v[n][m][2] = v[n][m][3] = 0.0f;
}
// acc += part, part = 0.
template <unsigned NT, unsigned MT>
__device__ __forceinline__ void flush(float (&acc)[NT][MT][4], float (&part)[NT][MT][4]) {
#pragma unroll
    for (unsigned n = 0; n < NT; ++n)
#pragma unroll
        for (unsigned m = 0; m < MT; ++m)
#pragma unroll
            for (unsigned i = 0; i < 4; ++i) acc[n][m][i] += part[n][m][i];
    clear(part);
}

// ---- launch 1 ---------------------------------------------------------------------------

// Item j: group j / tiles, rows j % tiles * 8 MT ... of its gate and up.
template <typename X, typename W, unsigned MT, unsigned NT, unsigned WARPS, bool VEC>
struct Up {
    using R = Ring<X, W, MT, NT, kUpRing, VEC, VEC>;
    static constexpr unsigned CHUNK = 8 * NT;
    struct Smem {
        alignas(16) unsigned char ring[WARPS][kUpRing];
        float sums[2][WARPS][MT * 16][CHUNK + 1];  // of items j and j + 1
        Plan plan;
    };
};

template <typename X, typename W, unsigned MT, unsigned NT, unsigned WARPS, bool VEC>
__global__ void __launch_bounds__(WARPS * 32, 16 / WARPS)
moe_gate_up(MoeDecodeArgs a, unsigned tiles) {
    using U = Up<X, W, MT, NT, WARPS, VEC>;
    using R = typename U::R;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    typename U::Smem& sm = *reinterpret_cast<typename U::Smem*>(smem_raw);
    pdl_begin();
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x / 32, r = lane / 4, c = lane % 4;
    make_plan<U::CHUNK>(a, sm.plan);
    // equally many items per CTA, on as many CTAs as that takes
    const unsigned items = sm.plan.groups * tiles;
    const unsigned rounds = (items + gridDim.x - 1) / gridDim.x;
    const unsigned ctas = (items + rounds - 1) / rounds;
    if (blockIdx.x >= ctas) return;

    const unsigned blocks = (a.H + R::BLOCK - 1) / R::BLOCK;
    const unsigned count = blocks > warp ? (blocks - warp + WARPS - 1) / WARPS : 0u;  // per item
    R ring;
    ring.init(sm.ring[warp], lane);
    // the end that fills
    unsigned put_item = blockIdx.x, put_left = 0, ok = 0;
    int left = 0;
    const W* w[MT][2] = {};
    const X* x[NT] = {};
    const auto put_step = [&]() {
        if (put_left == 0) {
            if (put_item >= items || count == 0) return;
            const unsigned g = sm.plan.group[put_item / tiles], i0 = put_item % tiles * 8 * MT;
            const unsigned e = group_expert(g), k = warp * R::BLOCK + c * R::PER;
            ok = 0;
#pragma unroll
            for (unsigned m = 0; m < MT; ++m) {
                const unsigned i = i0 + m * 8 + r;
                if (i < a.I) ok |= 3u << (2 * m);
                w[m][0] = static_cast<const W*>(a.w_gate_up) + (static_cast<std::size_t>(e) * 2 * a.I + i) * a.H + k;
                w[m][1] = w[m][0] + static_cast<std::size_t>(a.I) * a.H;
            }
#pragma unroll
            for (unsigned t = 0; t < NT; ++t)
                x[t] = t * 8 + r < group_count(g)
                           ? static_cast<const X*>(a.x) + (sm.plan.lists[e][group_first(g) + t * 8 + r] / 2) * a.ld_x + k
                           : nullptr;
            left = static_cast<int>(a.H) - static_cast<int>(k);
            put_left = count;
            put_item += ctas;
        }
        ring.put_weights(w, ok, left, a.w_gate_up);
        ring.put_acts(x, left, lane);
        R::step(ring.put, ring.base);
#pragma unroll
        for (unsigned m = 0; m < MT; ++m) {
            w[m][0] += WARPS * R::BLOCK;
            w[m][1] += WARPS * R::BLOCK;
        }
#pragma unroll
        for (unsigned t = 0; t < NT; ++t)
            if (x[t]) x[t] += WARPS * R::BLOCK;
        left -= static_cast<int>(WARPS * R::BLOCK);
        --put_left;
    };
#pragma unroll
    for (unsigned i = 0; i < R::STAGES - 1; ++i) {
        put_step();
        cp_async_commit();
    }
    unsigned buffer = 0;
    for (unsigned item = blockIdx.x; item < items; item += ctas, buffer ^= 1) {
        const unsigned g = sm.plan.group[item / tiles], i0 = item % tiles * 8 * MT;
        const unsigned e = group_expert(g), n = group_count(g), nt = (n + 7) / 8;
        float acc[NT][MT][4], part[NT][MT][4];
        clear(acc);
        clear(part);
        for (unsigned i = 0; i < count; ++i) {
            put_step();
            cp_async_commit();
            cp_async_wait<R::STAGES - 1>();
            ring.multiply(nt, part, lane);
            R::step(ring.get, ring.base);
            if (i % kChain == kChain - 1) flush(acc, part);
        }
        flush(acc, part);
        auto& sums = sm.sums[buffer];
#pragma unroll
        for (unsigned t = 0; t < NT; ++t)
            if (t < nt)
#pragma unroll
                for (unsigned m = 0; m < MT; ++m)
#pragma unroll
                    for (unsigned i = 0; i < 4; ++i)
                        sums[warp][m * 16 + r + i / 2 * 8][t * 8 + 2 * c + i % 2] = acc[t][m][i];
        __syncthreads();  // also: everyone has read the other buffer
        for (unsigned i = threadIdx.x; i < n * 8 * MT; i += WARPS * 32) {
            const unsigned row = i % (8 * MT), t = i / (8 * MT), at = row / 8 * 16 + row % 8;
            if (i0 + row >= a.act_ld) continue;
            float gate = 0.0f, up = 0.0f;
#pragma unroll
            for (unsigned v = 0; v < WARPS; ++v) {
                gate += sums[v][at][t];
                up += sums[v][at + 8][t];
            }
            const unsigned to = sm.plan.lists[e][group_first(g) + t];
            a.act[static_cast<std::size_t>(to) * a.act_ld + i0 + row] =
                i0 + row < a.I ? gate / (1.0f + expf(-gate)) * up : 0.0f;
        }
    }
}

// ---- launch 2 ---------------------------------------------------------------------------

template <typename W, unsigned NT, bool VEC>
struct Down {
    static constexpr unsigned WARPS = 8, CHUNK = 8 * NT;
    using R = Ring<float, W, 1, NT, kDownRing, VEC, true>;
    struct Smem {
        alignas(16) unsigned char ring[WARPS][kDownRing];
        float sums[kDownPartials][17];
        Plan plan;
    };
};

template <typename X, typename W, unsigned NT, bool VEC>
__global__ void __launch_bounds__(256, 2)
moe_down(MoeDecodeArgs a) {
    using D = Down<W, NT, VEC>;
    using R = typename D::R;
    constexpr unsigned WARPS = D::WARPS;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    typename D::Smem& sm = *reinterpret_cast<typename D::Smem*>(smem_raw);
    // No wait yet: what is read up to it -- logits and weights -- was written
    // before launch 1, whose CTAs all waited for that before they let this
    // launch start.
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x / 32, r = lane / 4, c = lane % 4;
    make_plan<D::CHUNK>(a, sm.plan);
    // k is cut in 2^shift parts so that the warps' loads even out: the fewest
    // rounds of (a part's blocks + 4, what a unit costs besides)
    const unsigned groups = sm.plan.groups, blocks = (a.I + R::BLOCK - 1) / R::BLOCK;
    unsigned shift = 0, best = ~0u;
#pragma unroll
    for (unsigned s = 0; s < 4; ++s) {
        const unsigned cost = (((groups << s) + WARPS - 1) / WARPS) * (((blocks + (1u << s) - 1) >> s) + 4);
        if (((2 * a.T) << s) <= kDownPartials && (1u << s) <= blocks && cost < best) {
            best = cost;
            shift = s;
        }
    }
    const unsigned parts = 1u << shift, units = groups << shift, h0 = blockIdx.x * 16;
    const auto blocks_of = [&](unsigned u) { return (blocks - (u & (parts - 1)) + parts - 1) >> shift; };
    R ring;
    ring.init(sm.ring[warp], lane);

    // The warp's blocks are those of its units u = warp, warp + WARPS, ...,
    // one after the other through the ring.
    unsigned put_u = warp, put_left = 0, ok = 0;
    int left = 0;
    const W* w[1][2] = {};
    const float* x[NT] = {};
    const auto put_step = [&](bool with_weights, bool with_acts) {
        if (put_left == 0) {
            if (put_u >= units) return;
            const unsigned g = sm.plan.group[put_u >> shift], e = group_expert(g);
            const unsigned k = (put_u & (parts - 1)) * R::BLOCK + c * R::PER;
            const unsigned h = h0 + r;
            w[0][0] = static_cast<const W*>(a.w_down) + (static_cast<std::size_t>(e) * a.H + h) * a.I + k;
            w[0][1] = w[0][0] + static_cast<std::size_t>(8) * a.I;
            ok = (h < a.H ? 1u : 0u) | (h + 8 < a.H ? 2u : 0u);
#pragma unroll
            for (unsigned t = 0; t < NT; ++t)
                x[t] = t * 8 + r < group_count(g)
                           ? a.act + static_cast<std::size_t>(sm.plan.lists[e][group_first(g) + t * 8 + r]) * a.act_ld + k
                           : nullptr;
            left = static_cast<int>(a.I) - static_cast<int>(k);
            put_left = blocks_of(put_u);
            put_u += WARPS;
        }
        if (with_weights) ring.put_weights(w, ok, left, a.w_down);
        // past I the row is padded with zeros to act_ld
        if (with_acts) ring.put_acts(x, static_cast<int>(a.act_ld) - static_cast<int>(a.I) + left, lane);
        R::step(ring.put, ring.base);
        w[0][0] += parts * R::BLOCK;
        w[0][1] += parts * R::BLOCK;
#pragma unroll
        for (unsigned t = 0; t < NT; ++t)
            if (x[t]) x[t] += parts * R::BLOCK;
        left -= static_cast<int>(parts * R::BLOCK);
        --put_left;
    };
    // weights of the first stages, then launch 1's activations
    for (unsigned i = 0; i < R::STAGES - 1; ++i) put_step(true, false);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    put_u = warp;
    put_left = 0;
    ring.put = ring.base;
    for (unsigned i = 0; i < R::STAGES - 1; ++i) {
        put_step(false, true);
        cp_async_commit();
    }
    for (unsigned u = warp; u < units; u += WARPS) {
        const unsigned g = sm.plan.group[u >> shift], n = group_count(g), nt = (n + 7) / 8;
        const unsigned count = blocks_of(u);
        float acc[NT][1][4], part[NT][1][4];
        clear(acc);
        clear(part);
        for (unsigned b = 0; b < count; ++b) {
            put_step(true, true);
            cp_async_commit();
            cp_async_wait<R::STAGES - 1>();
            ring.multiply(nt, part, lane);
            R::step(ring.get, ring.base);
            if (b % kChain == kChain - 1) flush(acc, part);
        }
        flush(acc, part);
#pragma unroll
        for (unsigned t = 0; t < NT; ++t)
#pragma unroll
            for (unsigned i = 0; i < 4; ++i) {
                const unsigned j = t * 8 + 2 * c + i % 2;
                if (j < n)
                    sm.sums[(u & (parts - 1)) * 2 * a.T + sm.plan.lists[group_expert(g)][group_first(g) + j]]
                           [r + i / 2 * 8] = acc[t][0][i];
            }
    }
    __syncthreads();
    for (unsigned i = threadIdx.x; i < a.T * 16; i += WARPS * 32) {
        const unsigned t = i / 16, h = i % 16;
        if (h0 + h >= a.H) continue;
        float y[2] = {0.0f, 0.0f};
        for (unsigned p = 0; p < parts; ++p) {
            y[0] += sm.sums[p * 2 * a.T + 2 * t][h];
            y[1] += sm.sums[p * 2 * a.T + 2 * t + 1][h];
        }
        const float v = sm.plan.gate[2 * t] * y[0] + sm.plan.gate[2 * t + 1] * y[1];
        X* out = static_cast<X*>(a.out) + t * a.ld_out + h0 + h;
        if constexpr (sizeof(X) == 2) *out = __float2bfloat16_rn(v);
        else *out = v;
    }
}

template <typename X, typename W, unsigned MT, unsigned NT, unsigned WARPS, bool VEC>
cudaError_t launch_tiled(const MoeDecodeArgs& a, cudaStream_t s) {
    const unsigned tiles = (a.I + 8 * MT - 1) / (8 * MT), chunk = 8 * NT;
    // an expert's last group may be partial, the others hold `chunk` assignments
    const unsigned groups = std::min(2 * a.T, std::min(a.E, 2 * a.T) + 2 * a.T / chunk);
    const unsigned slots = static_cast<unsigned>(sm_count()) * (16 / WARPS);
    const auto up = moe_gate_up<X, W, MT, NT, WARPS, VEC>;
    const auto down = moe_down<X, W, NT, VEC>;
    const std::size_t up_smem = sizeof(typename Up<X, W, MT, NT, WARPS, VEC>::Smem);
    const std::size_t down_smem = sizeof(typename Down<W, NT, VEC>::Smem);
    cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void*>(up), up_smem);
    if (e == cudaSuccess) e = allow_dynamic_smem(reinterpret_cast<const void*>(down), down_smem);
    if (e == cudaSuccess) e = launch_pdl(up, std::min(groups * tiles, slots), WARPS * 32, up_smem, s, a, tiles);
    if (e == cudaSuccess) e = launch_pdl(down, (a.H + 15) / 16, 256, down_smem, s, a);
    return e;
}

template <typename X, typename W>
cudaError_t launch_moe(const MoeDecodeArgs& a, cudaStream_t s) {
    const bool vec = a.H % 8 == 0 && a.I % kPer<W> == 0 && a.ld_x % 8 == 0 && aligned16(a.x) &&
                     aligned16(a.w_gate_up) && aligned16(a.w_down);
    // up to 8 tokens: one 8-token tile holds any expert's, and the finest row
    // tiles and k slices give the few experts' rows to the most warps
    if (!vec) return launch_tiled<X, W, 2, 2, 8, false>(a, s);
    if (a.T <= 8) return launch_tiled<X, W, 1, 1, 16, true>(a, s);
    return launch_tiled<X, W, 2, 2, 8, true>(a, s);
}

}  // namespace
}  // namespace b2

extern "C" {

int b2_moe_decode_workspace_size(size_t T, size_t I, size_t* bytes) {
    using namespace b2;
    if (!bytes) return invalid("b2_moe_decode_workspace_size: null pointer");
    if (T > kMaxDecodeTokens || I > 0x7FFFFFFu)
        return invalid("b2_moe_decode_workspace_size: T must be 128 at most, I below 2^27");
    *bytes = 2 * T * ((I + 7) / 8 * 8) * sizeof(float) + 16;
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
    a.act_ld = static_cast<unsigned>((I + 7) / 8 * 8);
    cudaStream_t s = as_stream(stream);
    cudaError_t e;
    if (x_dtype == B2_DTYPE_F32)
        e = w_dtype == B2_DTYPE_F32 ? launch_moe<float, float>(a, s) : launch_moe<float, __nv_bfloat16>(a, s);
    else
        e = w_dtype == B2_DTYPE_F32 ? launch_moe<__nv_bfloat16, float>(a, s)
                                    : launch_moe<__nv_bfloat16, __nv_bfloat16>(a, s);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return set_error(B2_ERR_CUDA, std::string("b2_moe_decode: ") + cudaGetErrorString(e));
    }
    return launch_result("b2_moe_decode");
}

}  // extern "C"
