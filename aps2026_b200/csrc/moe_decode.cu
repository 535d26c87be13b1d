// The expert layer for a few tokens (b2_moe_decode): top-2 routing, the gated
// expert products and the weighted sum, in two launches.
//
// Mathematics: for token t and each of its two experts e,
//   a(t, e) = silu(Wg[e] x[t]) * (Wu[e] x[t]),   out[t] = sum_e g(t, e) Wd[e] a(t, e).
//
// The weights stream from HBM once (groups of one expert read them again, from
// L2) and meet few tokens. Which k a lane holds of the matrix instruction's
// M = 16 operand is free as long as both operands agree, so a lane takes 16
// neighbouring bytes of its rows: it copies exactly what it will use, through
// its own ring of cp.async stages in shared memory, without barriers. The
// tokens are the instruction's N, staged the same way. Rows that start at any
// element cannot be copied so: their 16-byte chunks are brought by the row's
// four lanes, as asynchronously, and read across them, shifted (5 tokens of
// 3001 x 201 28 us; of 2944 x 201, where only launch 2 has such rows, 21).
// The instruction multiplies bf16 or TF32; fp32's accuracy is kept in parts:
// bf16 weights meet fp32 activations as three bf16 parts (24 bits), fp32
// weights as TF32 hi and lo (hi hi + hi lo + lo hi). Its accumulator
// truncates, a bias that grows with the chain, so a chain is one block long
// and blocks are added in registers (61 tokens in fp32: error 6.6e-7 of the
// output; two blocks per chain 9.6e-7, and 4 us more).
//
// Launch 1, moe_gate_up: an item is (expert with up to 8 NT of its tokens,
// 8 MT rows of gate and the same of up); a CTA takes equally many items, one
// after the other through the same rings. The warps of an item interleave its
// k blocks, so together they read whole lines, and add up in shared memory.
// It leaves the activations in their parts. Launch 2, moe_down: CTA = 16 MT
// rows of the output for its tokens; warps take (expert, 8 NT of its tokens,
// part of k) and meet in shared memory, where a token's two experts are
// summed in ascending order: no float atomics, results repeat. Each CTA
// routes for itself (T x E logits). Launch 2 starts under launch 1 and has
// routed and requested its first weights before it waits.
//
// What bounds it: one token, the two launches' latencies (routing, first
// weights, the meeting, the hand-over: 12.7 us at 4096 x 448 x 16 in bf16,
// 3.4 us of HBM time). 9 tokens, HBM with those latencies (27 to 31 us, 19 of
// HBM time). 61 tokens in fp32, fixed latencies: weights split into TF32 parts
// and chains of three products each, in 16 warps per SM (launch 1: 60 us, issue
// 54% active, matrix unit 35%; both 88, HBM time 55). 128 tokens, splitting
// the activations anew for every 16 rows (41 us at 1001 x 333 x 7; at 4096 x 448
// x 16 85, HBM time 28, and 67 with bf16 activations, which are not split).
#include <algorithm>

#include <cuda_bf16.h>

#include "quantize.cuh"

namespace b2 {
namespace {

constexpr unsigned kMaxDecodeTokens = 128;
constexpr unsigned kMaxGroups = kMaxExperts + 2 * kMaxDecodeTokens / 8;
constexpr unsigned kDownPartials = 256;  // (part of k, assignment) sums of moe_down
constexpr unsigned kWarps = 16;          // one CTA per SM: all its shared memory is rings
constexpr unsigned kRing = 11264;        // bytes of a warp's stages: 16 rings, the sums and the plan fill 227 KB

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
    void* act;        // [parts][2T][act_ld]: assignment 2t + s, s = 0 the lower expert
    unsigned act_ld;  // I rounded up to 8; zeros past I
};

// ---- routing, per CTA ----------------------------------------------------------

struct Plan {
    unsigned mask[kMaxDecodeTokens / 32][kMaxExperts];   // tokens of each expert, by bit
    unsigned char lists[kMaxExperts][kMaxDecodeTokens];  // assignments of each expert, tokens ascending
    unsigned short pair[kMaxDecodeTokens];               // lower expert | higher << 8
    float gate[2 * kMaxDecodeTokens];
    unsigned group[kMaxGroups];                          // expert | first in list << 8 | count << 16
    unsigned groups;
};
__device__ __forceinline__ unsigned group_expert(unsigned g) { return g & 0xFFu; }
__device__ __forceinline__ unsigned group_first(unsigned g) { return (g >> 8) & 0xFFu; }
__device__ __forceinline__ unsigned group_count(unsigned g) { return g >> 16; }

// The expert that b2_moe_route's ascending scan ends with, among those of
// `alive` (one lane per expert, SUB lanes per token, score: this lane's): it
// starts with the lowest and moves to the next one that beats it by more than
// tie_eps. Each step of the loop is one such move.
template <unsigned SUB>
__device__ __forceinline__ unsigned scan_best(float score, unsigned lane, unsigned alive, float tie_eps) {
    const unsigned base = lane / SUB * SUB;
    const unsigned mine = SUB == 32 ? alive : (alive >> base) & 0xFFFFu;
    unsigned best = __ffs(mine) - 1;  // two are alive at least
    for (;;) {
        const float bar = __fadd_rn(__shfl_sync(0xffffffffu, score, base + best), tie_eps);
        const unsigned beats = __ballot_sync(0xffffffffu, score > bar) & alive;
        const unsigned after = (SUB == 32 ? beats : (beats >> base) & 0xFFFFu) & (0xFFFFFFFEu << best);
        if (after) best = __ffs(after) - 1;
        if (!__any_sync(0xffffffffu, after != 0)) return best;
    }
}

// A lane per expert, 32 / SUB tokens per warp at a time: the code stays short
// (it runs once per CTA, from a cold instruction cache).
template <unsigned SUB>
__device__ __forceinline__ void pick_experts(const MoeDecodeArgs& a, unsigned from, unsigned tokens, Plan& p) {
    constexpr unsigned AT_ONCE = 32 / SUB, BATCH = 4;
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x / 32, e = lane % SUB;
    for (unsigned t0 = warp * AT_ONCE; t0 < tokens; t0 += kWarps * AT_ONCE * BATCH) {
        float raw[BATCH];
#pragma unroll
        for (unsigned i = 0; i < BATCH; ++i) {
            const unsigned t = t0 + i * kWarps * AT_ONCE + lane / SUB;
            raw[i] = t < tokens && e < a.E ? __ldg(a.logits + static_cast<std::size_t>(from + t) * a.E + e) : 0.0f;
        }
#pragma unroll 1
        for (unsigned i = 0; i < BATCH && t0 + i * kWarps * AT_ONCE < tokens; ++i) {
            const unsigned t = t0 + i * kWarps * AT_ONCE + lane / SUB;
            const float x = i == 0 ? raw[0] : i == 1 ? raw[1] : i == 2 ? raw[2] : raw[3];
            const float score = quantize(x, a.quantum);
            const unsigned alive = __ballot_sync(0xffffffffu, e < a.E);
            const unsigned first = scan_best<SUB>(score, lane, alive, a.tie_eps);
            const unsigned rest = alive & ~__ballot_sync(0xffffffffu, e == first);
            const unsigned second = scan_best<SUB>(score, lane, rest, a.tie_eps);
            const unsigned lo = min(first, second), hi = max(first, second);
            const float x0 = __shfl_sync(0xffffffffu, x, lane / SUB * SUB + lo);
            const float x1 = __shfl_sync(0xffffffffu, x, lane / SUB * SUB + hi);
            if (e == 0 && t < tokens) {
                float g0 = 0.5f, g1 = 0.5f;
                if (a.gates == B2_GATES_SOFTMAX) {
                    const float m = fmaxf(x0, x1), p0 = expf(x0 - m), p1 = expf(x1 - m);
                    g0 = p0 / (p0 + p1);
                    g1 = p1 / (p0 + p1);
                }
                p.pair[t] = static_cast<unsigned short>(lo | hi << 8);
                p.gate[2 * t] = g0;
                p.gate[2 * t + 1] = g1;
                atomicOr(&p.mask[t / 32][lo], 1u << (t & 31));
                atomicOr(&p.mask[t / 32][hi], 1u << (t & 31));
            }
        }
    }
}

// Routes tokens from .. from + tokens - 1 (counted from 0 in the plan) and cuts
// every expert's into groups of CHUNK. Ends with a barrier.
template <unsigned CHUNK>
__device__ __forceinline__ void make_plan(const MoeDecodeArgs& a, unsigned from, unsigned tokens, Plan& p) {
    const unsigned t = threadIdx.x, lane = t & 31, warp = t / 32;
    if (warp < kMaxDecodeTokens / 32) p.mask[warp][lane] = 0;
    __syncthreads();
    if (a.E <= 16) pick_experts<16>(a, from, tokens, p);
    else pick_experts<32>(a, from, tokens, p);
    __syncthreads();
    if (t < 2 * tokens) {  // assignment t
        const unsigned token = t / 2, e = t % 2 ? p.pair[token] >> 8 : p.pair[token] & 0xFFu;
        unsigned rank = __popc(p.mask[token / 32][e] & ((1u << (token & 31)) - 1u));
        for (unsigned w = 0; w < token / 32; ++w) rank += __popc(p.mask[w][e]);
        p.lists[e][rank] = static_cast<unsigned char>(t);
    }
    if (warp == kWarps - 1) {
        unsigned n = 0;
#pragma unroll
        for (unsigned w = 0; w < kMaxDecodeTokens / 32; ++w) n += __popc(p.mask[w][lane]);
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
__device__ __forceinline__ void copy_async16(unsigned dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
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
// Activations as launch 1 leaves them for launch 2: kParts<float, W> planes.
template <typename W>
struct Planes {};
template <typename X, typename W>
struct ActOf {  // raw: one place of PER elements
    using type = X;
    static constexpr unsigned planes = 0;
};
template <typename W>
struct ActOf<Planes<W>, W> {
    using type = W;  // bf16 parts or TF32 parts
    static constexpr unsigned planes = kParts<float, W>;
};

// w = hi + lo in TF32, hi rounded to nearest.
__device__ __forceinline__ void split_tf32(unsigned w, unsigned& hi, unsigned& lo) {
    hi = (w + 0x1000u) & 0xFFFFE000u;
    lo = __float_as_uint(__uint_as_float(w) - __uint_as_float(hi));
}

// Where a row that starts at any element lies in a stage: the 16-byte chunks
// of memory that its block touches, side by side, zeros past the row's end.
// They are brought by the four lanes of the row and read across them from byte
// `skip` on.
template <typename T>
__device__ __forceinline__ unsigned skip_of(const T* row) {
    return static_cast<unsigned>(reinterpret_cast<std::uintptr_t>(row)) & 15u;
}
__device__ __forceinline__ const unsigned char* chunk_of(const void* p) {
    return reinterpret_cast<const unsigned char*>(reinterpret_cast<std::uintptr_t>(p) & ~std::uintptr_t(15));
}
// Lane c's share of a block of BYTES bytes and of the chunks around them:
// chunks c, c + 4, ... of the row's, the first of which is at `chunk` and goes
// to `dst`. there: bytes from `chunk` to the row's end. whole: all the chunks
// are inside the tensor, which begins at `tensor`, and before the row's end.
template <typename T, unsigned BYTES>
__device__ __forceinline__ void copy_chunks(unsigned char* dst, const void* chunk, unsigned c, const void* tensor, int there,
                                            bool whole) {
    const unsigned char* from = static_cast<const unsigned char*>(chunk);
    if (whole) {
        const unsigned to = smem_addr(dst);
#pragma unroll
        for (unsigned i = 0; i < BYTES / 16 + 1; i += 4)
            if (i + 4 <= BYTES / 16 + 1 || i + c <= BYTES / 16)
                asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(to + i * 16), "l"(from + i * 16) : "memory");
        return;
    }
#pragma unroll 1
    for (unsigned i = 0; i + c <= BYTES / 16; i += 4, from += 64, dst += 64, there -= 64) {
        const int bytes = max(0, min(there, 16));
        if (from >= tensor || bytes == 0) {
            asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)),
                         "l"(bytes ? from : chunk_of(tensor) + 16), "r"(bytes)
                         : "memory");
        } else {  // a tensor that starts inside a chunk
            for (int e = 0; e < 16; e += sizeof(T))
                *reinterpret_cast<T*>(dst + e) =
                    from + e >= tensor && e < bytes ? *reinterpret_cast<const T*>(from + e) : T(0.0f);
        }
    }
}
// Where lane c's chunks of a row begin, at its block `at`.
template <typename T>
__device__ __forceinline__ const T* lane_chunk(const T* row, unsigned block_bytes, unsigned at, unsigned c) {
    return reinterpret_cast<const T*>(chunk_of(row) + (static_cast<std::size_t>(at) * block_bytes + c * 16));
}
// Lane c's WORDS words of a row in a stage.
template <typename T, unsigned WORDS>
__device__ __forceinline__ void read_skewed(unsigned row, unsigned skip, unsigned c, unsigned (&v)[WORDS]) {
    const unsigned at = row + (skip & 12u) + c * WORDS * 4;
    unsigned w[WORDS + 1];
#pragma unroll
    for (unsigned i = 0; i < WORDS + (sizeof(T) == 2); ++i)
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[i]) : "r"(at + i * 4));
#pragma unroll
    for (unsigned i = 0; i < WORDS; ++i) v[i] = sizeof(T) == 2 ? __funnelshift_r(w[i], w[i + 1], (skip & 2u) * 8) : w[i];
}
// skip_of the lane's rows.
template <unsigned MT, unsigned NT>
struct Skew {
    unsigned w[MT][2], x[NT];
};

template <unsigned NT, unsigned MT>
__device__ __forceinline__ void clear(float (&v)[NT][MT][4]) {
#pragma unroll
    for (unsigned n = 0; n < NT; ++n)
#pragma unroll
        for (unsigned m = 0; m < MT; ++m) v[n][m][0] = v[n][m][1] = v[n][m][2] = v[n][m][3] = 0.0f;
}
// The stages of one warp: MT 16-row tiles of a weight block (lane's rows r and
// r + 8 of each) and NT 8-token tiles of activations (lane's token r). VEC:
// every 16 bytes of a row of weights (XVEC: the activations that meet them)
// are aligned, and inside the row or past it; then each lane's bytes have
// their own place, and only the lane itself touches them. Else rows lie as
// copy_chunks puts them.
template <typename A, typename W, unsigned MT, unsigned NT, bool VEC, bool XVEC>
struct Ring {
    using X = typename ActOf<A, W>::type;
    static constexpr unsigned PLANES = ActOf<A, W>::planes;
    static constexpr unsigned PER = kPer<W>, BLOCK = kBlock<W>;
    static constexpr unsigned XB = PLANES ? PLANES * 16 : PER * sizeof(X);  // bytes of a token per lane
    static constexpr unsigned WROW = 80, XROW = BLOCK * sizeof(X) + 16;     // bytes of an unaligned row
    static constexpr unsigned WEIGHTS = MT * 2 * (VEC ? 512 : 8 * WROW), XTILE = XVEC ? 32 * XB : 8 * XROW;
    static constexpr unsigned STAGE = WEIGHTS + NT * XTILE;
    static constexpr unsigned STAGES = kRing / STAGE < 6 ? kRing / STAGE : 6;
    static_assert(STAGES >= 2, "a ring of one stage");
    unsigned char* raw;       // the lane's place in the warp's first stage
    unsigned base, get, put;  // shared addresses of the lane's place: first stage, next to use, next to fill

    __device__ __forceinline__ void init(unsigned char* warp_base, unsigned lane) {
        raw = warp_base + lane * 16;
        base = get = put = smem_addr(raw);
    }
    static __device__ __forceinline__ void step(unsigned& at, unsigned base) {
        at += STAGE;
        if (at == base + STAGES * STAGE) at = base;
    }
    // Rows that lanes share: every lane has read the stage that is filled next
    // (before put), every lane's copies are there (before multiply).
    static __device__ __forceinline__ void meet() {
        if (!VEC || !XVEC) __syncwarp();
    }

    // A stage that is inside its rows for all lanes. Rows and tokens that are
    // not there are left as they are: sums that nobody reads.
    __device__ __forceinline__ void put_whole(const W* const (&w)[MT][2], unsigned ok, bool with_weights,
                                              const X* const (&x)[NT], unsigned x_ok, bool with_acts, unsigned lane,
                                              std::size_t plane) {
        static_assert(VEC && XVEC, "aligned rows");
        if (with_weights)
#pragma unroll
            for (unsigned i = 0; i < 2 * MT; ++i)
                if ((ok >> i) & 1u) copy_async16(put + i * 512, w[i / 2][i % 2]);
        if (with_acts)
#pragma unroll
            for (unsigned n = 0; n < NT; ++n)
                if ((x_ok >> n) & 1u) {
                    const unsigned at = put + WEIGHTS + n * XTILE;
                    if constexpr (PLANES > 0) {
#pragma unroll
                        for (unsigned q = 0; q < PLANES; ++q) copy_async16(at + q * 512, x[n] + q * plane);
                    } else if constexpr (XB == 32) {
                        copy_async_l1(at, x[n], true);
                        copy_async_l1(at + 512, x[n] + 4, true);
                    } else if constexpr (XB == 16) {
                        copy_async16(at, x[n]);
                    } else {
                        copy_async<8>(at - lane * 8, x[n], true);
                    }
                }
    }
    // w[m][i]: the lane's weights (row's start + k); ok: bit 2m + i set where
    // the row is there; left: weights from k to the row's end, if positive.
    __device__ __forceinline__ void put_weights(const W* const (&w)[MT][2], unsigned ok, int left, const W* tensor,
                                                const Skew<MT, NT>& skew, bool inside, unsigned lane) {
#pragma unroll
        for (unsigned m = 0; m < MT; ++m)
#pragma unroll
            for (unsigned i = 0; i < 2; ++i) {
                const bool row = (ok >> (2 * m + i)) & 1u;
                if (VEC) {
                    const bool have = row && left > 0;
                    copy_async<16>(put + (m * 2 + i) * 512, have ? w[m][i] : tensor, have);
                } else if (row) {
                    const unsigned c = lane % 4;  // w[m][i]: the lane's chunk
                    const int rest = (left + static_cast<int>(c * PER)) * static_cast<int>(sizeof(W));  // of the row, from the block on
                    copy_chunks<W, 64>(raw + (put - base) - (lane - c) * 16 + ((m * 2 + i) * 8 + lane / 4) * WROW, w[m][i], c,
                                       tensor, rest + static_cast<int>(skew.w[m][i] - c * 16), inside && rest >= 80);
                }
            }
    }
    // x[n]: the lane's activations of token tile n (of the first plane); x_ok:
    // bit n set where there is a token.
    __device__ __forceinline__ void put_acts(const X* const (&x)[NT], unsigned x_ok, int left, unsigned lane,
                                             std::size_t plane, const X* tensor, const Skew<MT, NT>& skew, bool inside) {
#pragma unroll
        for (unsigned n = 0; n < NT; ++n) {
            if (!((x_ok >> n) & 1u)) continue;
            const unsigned at = put + WEIGHTS + n * XTILE;
            if (XVEC) {
                const bool have = left > 0;  // x[n] is not read where there is none
                if constexpr (PLANES > 0) {
#pragma unroll
                    for (unsigned q = 0; q < PLANES; ++q) copy_async<16>(at + q * 512, x[n] + q * plane, have);
                } else if constexpr (XB == 32) {
                    copy_async_l1(at, x[n], have);
                    copy_async_l1(at + 512, x[n] + 4, have);
                } else if constexpr (XB == 16) {
                    copy_async<16>(at, x[n], have);
                } else {
                    copy_async<8>(at - lane * 8, x[n], have);
                }
            } else {
                const unsigned c = lane % 4;
                const int rest = (left + static_cast<int>(c * PER)) * static_cast<int>(sizeof(X));
                copy_chunks<X, BLOCK * sizeof(X)>(raw + (at - base) - (lane - c) * 16 + lane / 4 * XROW, x[n], c, tensor,
                                                  rest + static_cast<int>(skew.x[n] - c * 16),
                                                  inside && rest >= static_cast<int>(BLOCK * sizeof(X) + 16));
            }
        }
    }

    // acc[n] += the stage's products for nt token tiles.
    __device__ __forceinline__ void multiply(unsigned nt, float (&acc)[NT][MT][4], unsigned lane,
                                             const Skew<MT, NT>& skew) {
        constexpr unsigned PARTS = PLANES ? PLANES : kParts<X, W>;
        uint4 w[MT][2];
#pragma unroll
        for (unsigned m = 0; m < MT; ++m) {
            if constexpr (VEC) {
                w[m][0] = lds16(get + m * 1024);
                w[m][1] = lds16(get + m * 1024 + 512);
            } else {
#pragma unroll
                for (unsigned i = 0; i < 2; ++i) {
                    unsigned v[4];
                    read_skewed<W>(get - lane * 16 + ((m * 2 + i) * 8 + lane / 4) * WROW, skew.w[m][i], lane % 4, v);
                    w[m][i] = make_uint4(v[0], v[1], v[2], v[3]);
                }
            }
        }
#pragma unroll
        for (unsigned n = 0; n < NT; ++n) {
            if (n >= nt) break;
            const unsigned at = get + WEIGHTS + n * XTILE;
            unsigned v[PLANES ? 1 : XB / 4];  // raw activations
            if constexpr (PLANES == 0) {
                if constexpr (!XVEC) {
                    read_skewed<X>(at - lane * 16 + lane / 4 * XROW, skew.x[n], lane % 4, v);
                } else if constexpr (XB == 8) {
                    const uint2 y = lds8(at - lane * 8);
                    v[0] = y.x; v[1] = y.y;
                } else {
#pragma unroll
                    for (unsigned i = 0; i < XB / 16; ++i) {
                        const uint4 y = lds16(at + i * 512);
                        v[4 * i] = y.x; v[4 * i + 1] = y.y; v[4 * i + 2] = y.z; v[4 * i + 3] = y.w;
                    }
                }
            }
            unsigned b[PARTS][4];
            if constexpr (PLANES > 0) {  // in parts as it lies
#pragma unroll
                for (unsigned q = 0; q < PARTS; ++q) {
                    const uint4 y = lds16(at + q * 512);
                    b[q][0] = y.x; b[q][1] = y.y; b[q][2] = y.z; b[q][3] = y.w;
                }
            } else if constexpr (sizeof(X) == 2 && sizeof(W) == 2) {
#pragma unroll
                for (unsigned i = 0; i < 4; ++i) b[0][i] = v[i];
            } else if constexpr (sizeof(W) == 2) {  // x = three bf16 parts
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
            } else if constexpr (sizeof(X) == 4) {  // x = TF32 hi + lo
#pragma unroll
                for (unsigned i = 0; i < 4; ++i) split_tf32(v[i], b[0][i], b[PARTS - 1][i]);
            } else {
                b[0][0] = v[0] << 16; b[0][1] = v[0] & 0xFFFF0000u;
                b[0][2] = v[1] << 16; b[0][3] = v[1] & 0xFFFF0000u;
            }
            float part[1][MT][4];  // of this block alone
            clear(part);
            if constexpr (sizeof(W) == 2) {
#pragma unroll
                for (unsigned q = PARTS; q-- > 0;)
#pragma unroll
                    for (unsigned m = 0; m < MT; ++m) {
                        mma_bf16(part[0][m], w[m][0].x, w[m][1].x, w[m][0].y, w[m][1].y, b[q][0], b[q][1]);
                        mma_bf16(part[0][m], w[m][0].z, w[m][1].z, w[m][0].w, w[m][1].w, b[q][2], b[q][3]);
                    }
            } else {
#pragma unroll
                for (unsigned m = 0; m < MT; ++m) {
                    const unsigned r0[4] = {w[m][0].x, w[m][0].y, w[m][0].z, w[m][0].w};
                    const unsigned r1[4] = {w[m][1].x, w[m][1].y, w[m][1].z, w[m][1].w};
                    unsigned h0[4], l0[4], h1[4], l1[4];
#pragma unroll
                    for (unsigned i = 0; i < 4; ++i) {
                        // hi truncated: its rounding would cost another operation
                        // per weight; lo then has 13 bits, of which TF32 keeps 11
                        h0[i] = r0[i] & 0xFFFFE000u;
                        l0[i] = __float_as_uint(__uint_as_float(r0[i]) - __uint_as_float(h0[i]));
                        h1[i] = r1[i] & 0xFFFFE000u;
                        l1[i] = __float_as_uint(__uint_as_float(r1[i]) - __uint_as_float(h1[i]));
                    }
#pragma unroll
                    for (unsigned i = 0; i < 4; i += 2) {
                        mma_tf32(part[0][m], l0[i], l1[i], l0[i + 1], l1[i + 1], b[0][i], b[0][i + 1]);
                        if (PARTS == 2)
                            mma_tf32(part[0][m], h0[i], h1[i], h0[i + 1], h1[i + 1], b[PARTS - 1][i], b[PARTS - 1][i + 1]);
                        mma_tf32(part[0][m], h0[i], h1[i], h0[i + 1], h1[i + 1], b[0][i], b[0][i + 1]);
                    }
                }
            }
#pragma unroll
            for (unsigned m = 0; m < MT; ++m)
#pragma unroll
                for (unsigned i = 0; i < 4; ++i) acc[n][m][i] += part[0][m][i];
        }
    }
};

// ---- infinities ---------------------------------------------------------------------------
//
// In parts an infinite operand is inf - inf, and so is a finite one whose high
// part rounds up to infinity; a part that is 0 makes an infinite weight a NaN.
// All of that ends in a NaN sum, so a sum that is NaN is taken once more
// without parts: it comes out infinite, or finite, where a plain fp32 sum does.
// Only that case costs time (a token of NaN: its rows' sums up to the first NaN).
__device__ __forceinline__ float wide(float v) { return v; }
__device__ __forceinline__ float wide(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename X, typename W>
__device__ float plain_dot(const X* x, const W* w, unsigned n) {
    float sum = 0.0f;
    for (unsigned k = 0; k < n && sum == sum; ++k) sum = fmaf(wide(w[k]), wide(x[k]), sum);
    return sum;
}
// An activation from here on, or NaN, is unusual: the largest bf16, up to which
// rounding makes no part infinite.
constexpr float kUnusual = 3.3895313892515355e38f;
// Stores activation v, which is unusual, in its parts: taken again where it is
// NaN; its high parts truncated, and an infinite one alone.
template <typename X, typename W>
__device__ __noinline__ void put_unusual(float v, const X* x, const W* gate_row, std::size_t to_up, unsigned H, void* act,
                                         std::size_t at, std::size_t plane) {
    if (v != v && sizeof(X) + sizeof(W) > 4) {  // else nothing was in parts
        const float gate = plain_dot(x, gate_row, H), up = plain_dot(x, gate_row + to_up, H);
        v = gate / (1.0f + expf(-gate)) * up;
    }
    constexpr unsigned PARTS = kParts<float, W>;
    for (unsigned q = 0; q < PARTS; ++q) {
        const float b = sizeof(W) == 2 ? wide(__float2bfloat16_rz(v))
                                       : v != v ? v : __uint_as_float(__float_as_uint(v) & 0xFFFFE000u);
        if constexpr (sizeof(W) == 2) static_cast<__nv_bfloat16*>(act)[q * plane + at] = __float2bfloat16_rz(v);
        else static_cast<float*>(act)[q * plane + at] = b;
        v = isinf(v) ? 0.0f : v - b;
    }
}
// sum_k w[k] act[k], activations in their planes.
template <typename W>
__device__ float plain_dot_planes(const void* act, std::size_t at, std::size_t plane, const W* w, unsigned n) {
    float sum = 0.0f;
    for (unsigned k = 0; k < n && sum == sum; ++k) {
        float v;
        if constexpr (sizeof(W) == 2) {
            const __nv_bfloat16* a = static_cast<const __nv_bfloat16*>(act) + at + k;
            v = wide(a[0]) + wide(a[plane]) + wide(a[2 * plane]);
        } else {
            const float* a = static_cast<const float*>(act) + at + k;
            v = a[0] + a[plane];
        }
        sum = fmaf(wide(w[k]), v, sum);
    }
    return sum;
}
// A token's output that is NaN, taken again: y0, y1 its experts' sums, `at`
// its first expert's activations, w0 and w1 its rows of w_down.
template <typename W>
__device__ __noinline__ float output_again(float y0, float y1, float g0, float g1, const void* act, std::size_t at,
                                           std::size_t act_ld, std::size_t plane, const W* w0, const W* w1, unsigned n) {
    if (y0 != y0) y0 = plain_dot_planes(act, at, plane, w0, n);
    if (y1 != y1) y1 = plain_dot_planes(act, at + act_ld, plane, w1, n);
    return g0 * y0 + g1 * y1;
}

// ---- launch 1 ---------------------------------------------------------------------------

// Item j: group j / tiles, rows j % tiles * 8 MT ... of its gate and up.
template <typename X, typename W, unsigned MT, unsigned NT, bool VEC>
struct Up {
    using R = Ring<X, W, MT, NT, VEC, VEC>;
    static constexpr unsigned ROWS = 8 * MT, CHUNK = 8 * NT;
    static constexpr unsigned BUFFERS = MT == 1 ? 2 : 1;
    struct Smem {
        alignas(16) unsigned char ring[kWarps][kRing];
        float sums[BUFFERS][kWarps][16 * MT][CHUNK + 1];
        Plan plan;
    };
};

template <typename X, typename W, unsigned MT, unsigned NT, bool VEC>
__global__ void __launch_bounds__(kWarps * 32, 1)
moe_gate_up(MoeDecodeArgs a, unsigned tiles) {
    using U = Up<X, W, MT, NT, VEC>;
    using R = typename U::R;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    typename U::Smem& sm = *reinterpret_cast<typename U::Smem*>(smem_raw);
    pdl_begin();
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x / 32, r = lane / 4, c = lane % 4;
    make_plan<U::CHUNK>(a, 0, a.T, sm.plan);
    // A round of a CTA is 2^shift items, kWarps >> shift warps each. With few k
    // blocks a warp has little to do between two rounds' ends, which cost it
    // what 2 blocks do; then fewer warps per item are better, if that fits the
    // number of items (H = 256: 23 instead of 39 us; from 4 blocks per warp on,
    // nothing is gained). Equally many rounds per CTA, on as many CTAs as that takes.
    const unsigned items = sm.plan.groups * tiles, blocks = (a.H + R::BLOCK - 1) / R::BLOCK;
    unsigned shift = 0, ctas = 0;
    for (unsigned s = 0, best = ~0u; s < (MT == 1 ? 3 : 2); ++s) {
        if (s && blocks << s > 4 * kWarps) break;
        const unsigned sets = (items + (1u << s) - 1) >> s, rounds = (sets + gridDim.x - 1) / gridDim.x;
        const unsigned cost = rounds * ((((blocks << s) + kWarps - 1) / kWarps) + 2);
        if (cost < best) {
            best = cost;
            shift = s;
            ctas = (sets + rounds - 1) / rounds;
        }
    }
    if (blockIdx.x >= ctas) return;
    const unsigned team = kWarps >> shift, mine = warp / team, at = warp % team, step = team * R::BLOCK;
    const unsigned count = blocks > at ? (blocks - at + team - 1) / team : 0u;  // of a warp, per item
    R ring;
    ring.init(sm.ring[warp], lane);
    // the end that fills
    unsigned put_set = blockIdx.x, put_left = 0, ok = 0, x_ok = 0;
    int left = 0;
    bool w_inside = false, x_inside = false;
    Skew<MT, NT> put_skew{};
    const W* w[MT][2] = {};
    const X* x[NT] = {};
    const auto put_step = [&]() {
        if (put_left == 0) {
            const unsigned item = (put_set << shift) + mine;
            if (item >= items || count == 0) return;
            const unsigned g = sm.plan.group[item / tiles], i = item % tiles * U::ROWS + r;
            const unsigned e = group_expert(g), k = at * R::BLOCK + c * R::PER;
            ok = 0;
            w_inside = x_inside = !VEC;
#pragma unroll
            for (unsigned m = 0; m < MT; ++m) {
                if (i + m * 8 >= a.I) continue;
                ok |= 3u << 2 * m;
#pragma unroll
                for (unsigned up = 0; up < 2; ++up) {
                    const W* row = static_cast<const W*>(a.w_gate_up) +
                                   ((static_cast<std::size_t>(e) * 2 + up) * a.I + i + m * 8) * a.H;
                    w[m][up] = VEC ? row + k : lane_chunk(row, 64, at, c);
                    put_skew.w[m][up] = skip_of(row);
                    if (!VEC) w_inside &= chunk_of(row) >= a.w_gate_up;
                }
            }
            x_ok = 0;
#pragma unroll
            for (unsigned t = 0; t < NT; ++t)
                if (t * 8 + r < group_count(g)) {
                    x_ok |= 1u << t;
                    const X* row = static_cast<const X*>(a.x) + (sm.plan.lists[e][group_first(g) + t * 8 + r] / 2) * a.ld_x;
                    x[t] = VEC ? row + k : lane_chunk(row, R::BLOCK * sizeof(X), at, c);
                    put_skew.x[t] = skip_of(row);
                    if (!VEC) x_inside &= chunk_of(row) >= a.x;
                }
            left = static_cast<int>(a.H) - static_cast<int>(k);
            put_left = count;
            put_set += ctas;
        }
        if (VEC && left >= static_cast<int>(R::BLOCK - c * R::PER)) {
            if constexpr (VEC) ring.put_whole(w, ok, true, x, x_ok, true, lane, 0);
        } else {
            ring.put_weights(w, ok, left, static_cast<const W*>(a.w_gate_up), put_skew, w_inside, lane);
            ring.put_acts(x, x_ok, left, lane, 0, static_cast<const X*>(a.x), put_skew, x_inside);
        }
        R::step(ring.put, ring.base);
#pragma unroll
        for (unsigned i = 0; i < 2 * MT; ++i) w[i / 2][i % 2] += step;
#pragma unroll
        for (unsigned t = 0; t < NT; ++t) x[t] += step;
        left -= static_cast<int>(step);
        --put_left;
    };
#pragma unroll 1
    for (unsigned i = 0; i < R::STAGES - 1; ++i) {
        put_step();
        cp_async_commit();
    }
    unsigned buffer = 0;
    for (unsigned set = blockIdx.x; set << shift < items; set += ctas, buffer = U::BUFFERS - 1 - buffer) {
        auto& sums = sm.sums[buffer];
        const unsigned item = (set << shift) + mine;
        if (item < items) {
            const unsigned g = sm.plan.group[item / tiles], n = group_count(g), nt = (n + 7) / 8;
            float acc[NT][MT][4];
            clear(acc);
            Skew<MT, NT> skew{};
            if constexpr (!VEC) {
                const unsigned e = group_expert(g), i = item % tiles * U::ROWS + r;
                const W* row = static_cast<const W*>(a.w_gate_up) + (static_cast<std::size_t>(e) * 2 * a.I + i) * a.H;
#pragma unroll
                for (unsigned m = 0; m < MT; ++m) {
                    skew.w[m][0] = skip_of(row + std::size_t(8 * m) * a.H);
                    skew.w[m][1] = skip_of(row + (std::size_t(a.I) + 8 * m) * a.H);
                }
#pragma unroll
                for (unsigned t = 0; t < NT; ++t)
                    if (t * 8 + r < n)
                        skew.x[t] = skip_of(static_cast<const X*>(a.x) + sm.plan.lists[e][group_first(g) + t * 8 + r] / 2 * a.ld_x);
            }
            for (unsigned i = 0; i < count; ++i) {
                R::meet();
                put_step();
                cp_async_commit();
                cp_async_wait<R::STAGES - 1>();
                R::meet();
                ring.multiply(nt, acc, lane, skew);
                R::step(ring.get, ring.base);
            }
#pragma unroll
            for (unsigned t = 0; t < NT; ++t)
                if (t < nt)
#pragma unroll
                    for (unsigned i = 0; i < 4 * MT; ++i)
                        sums[warp][i / 4 * 16 + r + i / 2 % 2 * 8][t * 8 + 2 * c + i % 2] = acc[t][i / 4][i % 4];
        }
        __syncthreads();  // also: everyone has read the other buffer
        const unsigned row = threadIdx.x % U::ROWS, t = threadIdx.x / U::ROWS % U::CHUNK;
        const unsigned which = threadIdx.x / (U::ROWS * U::CHUNK), done = (set << shift) + which;
        const unsigned i0 = done % tiles * U::ROWS, g = done < items ? sm.plan.group[done / tiles] : 0u, e = group_expert(g);
        if (which >> shift == 0 && t < group_count(g) && i0 + row < a.act_ld) {
            float gate = 0.0f, up = 0.0f;
#pragma unroll
            for (unsigned v = 0; v < kWarps; ++v) {
                if (v >= team) break;
                gate += sums[which * team + v][row / 8 * 16 + row % 8][t];
                up += sums[which * team + v][row / 8 * 16 + row % 8 + 8][t];
            }
            const unsigned to = sm.plan.lists[e][group_first(g) + t];
            const std::size_t at = static_cast<std::size_t>(to) * a.act_ld + i0 + row;
            const std::size_t plane = static_cast<std::size_t>(2) * a.T * a.act_ld;
            float v = i0 + row < a.I ? gate / (1.0f + expf(-gate)) * up : 0.0f;
            if (!(fabsf(v) < kUnusual)) {
                put_unusual(v, static_cast<const X*>(a.x) + to / 2 * a.ld_x,
                            static_cast<const W*>(a.w_gate_up) + (static_cast<std::size_t>(e) * 2 * a.I + i0 + row) * a.H,
                            static_cast<std::size_t>(a.I) * a.H, a.H, a.act, at, plane);
            } else if constexpr (sizeof(W) == 2) {
                __nv_bfloat16* act = static_cast<__nv_bfloat16*>(a.act);
#pragma unroll
                for (unsigned q = 0; q < 3; ++q) {
                    const __nv_bfloat16 b = __float2bfloat16_rn(v);
                    act[q * plane + at] = b;
                    v -= __bfloat162float(b);
                }
            } else {
                unsigned hi, lo;
                split_tf32(__float_as_uint(v), hi, lo);
                static_cast<unsigned*>(a.act)[at] = hi;
                static_cast<unsigned*>(a.act)[plane + at] = lo;
            }
        }
        if (U::BUFFERS == 1) __syncthreads();
    }
}

// ---- launch 2 ---------------------------------------------------------------------------

template <typename W, unsigned MT, unsigned NT, bool VEC>
struct Down {
    using R = Ring<Planes<W>, W, MT, NT, VEC, true>;
    struct Smem {
        alignas(16) unsigned char ring[kWarps][kRing];
        float sums[kDownPartials][16 * MT + 1];
        Plan plan;
    };
};

template <typename X, typename W, unsigned MT, unsigned NT, bool VEC>
__global__ void __launch_bounds__(kWarps * 32, 1)
moe_down(MoeDecodeArgs a, unsigned per) {
    using D = Down<W, MT, NT, VEC>;
    using R = typename D::R;
    using Act = typename R::X;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    typename D::Smem& sm = *reinterpret_cast<typename D::Smem*>(smem_raw);
    // No wait yet: what is read up to it -- logits and weights -- was written
    // before launch 1, whose CTAs all waited for that before they let this
    // launch start.
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x / 32, r = lane / 4, c = lane % 4;
    const unsigned t0 = blockIdx.y * per, T = min(per, a.T - t0);  // the CTA's tokens
    make_plan<8 * NT>(a, t0, T, sm.plan);
    // k is cut in 2^shift parts so that the warps' loads even out: the fewest
    // rounds of (a part's blocks + 4, what a unit costs besides)
    const unsigned groups = sm.plan.groups, blocks = (a.I + R::BLOCK - 1) / R::BLOCK;
    unsigned shift = 0, best = ~0u;
#pragma unroll
    for (unsigned s = 0; s < 4; ++s) {
        const unsigned cost = (((groups << s) + kWarps - 1) / kWarps) * (((blocks + (1u << s) - 1) >> s) + 4);
        if (((2 * T) << s) <= kDownPartials && (1u << s) <= blocks && cost < best) {
            best = cost;
            shift = s;
        }
    }
    const unsigned parts = 1u << shift, units = groups << shift, h0 = blockIdx.x * 16 * MT;
    const auto blocks_of = [&](unsigned u) { return (blocks - (u & (parts - 1)) + parts - 1) >> shift; };
    const std::size_t plane = static_cast<std::size_t>(2) * a.T * a.act_ld;
    R ring;
    ring.init(sm.ring[warp], lane);
    // The warp's blocks are those of its units u = warp, warp + kWarps, ...,
    // one after the other through the ring.
    unsigned put_u = warp, put_left = 0, ok = 0, x_ok = 0;
    int left = 0;
    bool inside = false;
    Skew<MT, NT> put_skew{};
    const W* w[MT][2] = {};
    const Act* x[NT] = {};
    const auto put_step = [&](bool with_weights, bool with_acts) {
        if (put_left == 0) {
            if (put_u >= units) return;
            const unsigned g = sm.plan.group[put_u >> shift], e = group_expert(g);
            const unsigned k = (put_u & (parts - 1)) * R::BLOCK + c * R::PER;
            ok = 0;
            inside = !VEC;
#pragma unroll
            for (unsigned i = 0; i < 2 * MT; ++i) {
                const unsigned h = h0 + r + 8 * i;
                const W* row = static_cast<const W*>(a.w_down) + (static_cast<std::size_t>(e) * a.H + h) * a.I;
                w[i / 2][i % 2] = VEC ? row + k : lane_chunk(row, 64, put_u & (parts - 1), c);
                if (h < a.H) ok |= 1u << i;
                put_skew.w[i / 2][i % 2] = skip_of(row);
                if (!VEC && h < a.H) inside &= chunk_of(row) >= a.w_down;
            }
            x_ok = 0;
#pragma unroll
            for (unsigned t = 0; t < NT; ++t)
                if (t * 8 + r < group_count(g)) {
                    x_ok |= 1u << t;
                    x[t] = static_cast<const Act*>(a.act) +
                           static_cast<std::size_t>(2 * t0 + sm.plan.lists[e][group_first(g) + t * 8 + r]) * a.act_ld + k;
                }
            left = static_cast<int>(a.I) - static_cast<int>(k);
            put_left = blocks_of(put_u);
            put_u += kWarps;
        }
        if (VEC && left >= static_cast<int>(R::BLOCK - c * R::PER)) {
            if constexpr (VEC) ring.put_whole(w, ok, with_weights, x, x_ok, with_acts, lane, plane);
        } else {
            if (with_weights) ring.put_weights(w, ok, left, static_cast<const W*>(a.w_down), put_skew, inside, lane);
            // past I the row is padded with zeros to act_ld
            if (with_acts) ring.put_acts(x, x_ok, static_cast<int>(a.act_ld - a.I) + left, lane, plane, nullptr, put_skew, false);
        }
        R::step(ring.put, ring.base);
#pragma unroll
        for (unsigned i = 0; i < 2 * MT; ++i) w[i / 2][i % 2] += parts * R::BLOCK;
#pragma unroll
        for (unsigned t = 0; t < NT; ++t) x[t] += parts * R::BLOCK;
        left -= static_cast<int>(parts * R::BLOCK);
        --put_left;
    };
    // weights of the first stages, then launch 1's activations
    bool first = true;
#pragma unroll 1
    for (unsigned i = 0; i < 2 * (R::STAGES - 1); ++i) {
        if (i == R::STAGES - 1) {
            asm volatile("griddepcontrol.wait;" ::: "memory");
            put_u = warp;
            put_left = 0;
            ring.put = ring.base;
            first = false;
        }
        put_step(first, !first);
        if (!first) cp_async_commit();
    }
    for (unsigned u = warp; u < units; u += kWarps) {
        const unsigned g = sm.plan.group[u >> shift], n = group_count(g);
        const unsigned count = blocks_of(u);
        float acc[NT][MT][4];
        clear(acc);
        Skew<MT, NT> skew{};
        if constexpr (!VEC) {
#pragma unroll
            for (unsigned i = 0; i < 2 * MT; ++i)
                skew.w[i / 2][i % 2] = skip_of(static_cast<const W*>(a.w_down) +
                                               (static_cast<std::size_t>(group_expert(g)) * a.H + h0 + r + 8 * i) * a.I);
        }
        for (unsigned b = 0; b < count; ++b) {
            R::meet();
            put_step(true, true);
            cp_async_commit();
            cp_async_wait<R::STAGES - 1>();
            R::meet();
            ring.multiply((n + 7) / 8, acc, lane, skew);
            R::step(ring.get, ring.base);
        }
#pragma unroll
        for (unsigned t = 0; t < 2 * NT; ++t) {
            const unsigned at = t / 2 * 8 + 2 * c + t % 2;
            if (at < n) {
                float* sums = sm.sums[(u & (parts - 1)) * 2 * T + sm.plan.lists[group_expert(g)][group_first(g) + at]];
#pragma unroll
                for (unsigned m = 0; m < MT; ++m) {
                    sums[m * 16 + r] = acc[t / 2][m][t % 2];
                    sums[m * 16 + r + 8] = acc[t / 2][m][2 + t % 2];
                }
            }
        }
    }
    __syncthreads();
    for (unsigned i = threadIdx.x; i < T * 16 * MT; i += kWarps * 32) {
        const unsigned t = i / (16 * MT), h = i % (16 * MT);
        if (h0 + h >= a.H) continue;
        float y[2] = {0.0f, 0.0f};
        for (unsigned p = 0; p < parts; ++p) {
            y[0] += sm.sums[p * 2 * T + 2 * t][h];
            y[1] += sm.sums[p * 2 * T + 2 * t + 1][h];
        }
        const float g0 = sm.plan.gate[2 * t], g1 = sm.plan.gate[2 * t + 1];
        float v = g0 * y[0] + g1 * y[1];
        if (v != v) {
            const W* rows = static_cast<const W*>(a.w_down) + static_cast<std::size_t>(h0 + h) * a.I;
            const std::size_t of_expert = static_cast<std::size_t>(a.H) * a.I;
            v = output_again(y[0], y[1], g0, g1, a.act, static_cast<std::size_t>(2 * (t0 + t)) * a.act_ld, a.act_ld, plane,
                             rows + (sm.plan.pair[t] & 0xFFu) * of_expert, rows + (sm.plan.pair[t] >> 8) * of_expert, a.I);
        }
        X* out = static_cast<X*>(a.out) + (t0 + t) * a.ld_out + h0 + h;
        if constexpr (sizeof(X) == 2) *out = __float2bfloat16_rn(v);
        else *out = v;
    }
}

template <typename X, typename W, unsigned MT, unsigned NT, bool VEC>
cudaError_t launch_up(const MoeDecodeArgs& a, cudaStream_t s) {
    using U = Up<X, W, MT, NT, VEC>;
    const unsigned tiles = (a.I + U::ROWS - 1) / U::ROWS;
    // an expert's last group may be partial, the others hold CHUNK assignments
    const unsigned groups = std::min(2 * a.T, std::min(a.E, 2 * a.T) + 2 * a.T / U::CHUNK);
    const auto kernel = moe_gate_up<X, W, MT, NT, VEC>;
    const std::size_t smem = sizeof(typename U::Smem);
    const cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
    if (e != cudaSuccess) return e;
    return launch_pdl(kernel, std::min(groups * tiles, static_cast<unsigned>(sm_count())), kWarps * 32, smem, s, a, tiles);
}

template <typename X, typename W, unsigned MT, unsigned NT, bool VEC>
cudaError_t launch_down(const MoeDecodeArgs& a, cudaStream_t s) {
    const auto kernel = moe_down<X, W, MT, NT, VEC>;
    const std::size_t smem = sizeof(typename Down<W, MT, NT, VEC>::Smem);
    const cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
    if (e != cudaSuccess) return e;
    // as long as rows alone leave SMs without a CTA, the tokens are cut in two,
    // down to 8 (60 tokens of 320 x 800: 18.5 us, down to 16 20.9; to 4 no better)
    const unsigned rows = (a.H + 16 * MT - 1) / (16 * MT);
    unsigned cuts = 1;
    while (2 * cuts * rows <= static_cast<unsigned>(sm_count()) && a.T >= 16 * cuts) cuts *= 2;
    const unsigned per = (a.T + cuts - 1) / cuts;
    return launch_pdl(kernel, dim3(rows, (a.T + per - 1) / per), kWarps * 32, smem, s, a, per);
}

template <typename X, typename W>
cudaError_t launch_moe(const MoeDecodeArgs& a, cudaStream_t s) {
    // rows of 16-byte pieces, for each launch by itself
    const bool vec_up = a.H % 8 == 0 && a.ld_x % 8 == 0 && aligned16(a.x) && aligned16(a.w_gate_up);
    const bool vec_down = a.I % kPer<W> == 0 && aligned16(a.w_down);
    // 16 tokens per group, and 16 rows of gate and up per item, where the
    // experts have more than 4 tokens on average: fewer experts are read twice,
    // fewer activations split twice (128 tokens of 4096 x 448 x 16: 85 us, with
    // 8 rows 107); else 8 of each, whose smaller stages leave more weights in flight
    const bool wide = 2 * a.T > 4 * a.E;
    cudaError_t e = vec_up ? wide ? launch_up<X, W, 2, 2, true>(a, s) : launch_up<X, W, 1, 1, true>(a, s)
                           : wide ? launch_up<X, W, 2, 2, false>(a, s) : launch_up<X, W, 1, 1, false>(a, s);
    if (e != cudaSuccess) return e;
    // 32 output rows per CTA as long as that reaches most SMs: the activations
    // are read once for both tiles, and 16 rows would leave a second round of CTAs
    const bool tall = a.H > 16u * static_cast<unsigned>(sm_count());
    if (vec_down) return tall ? launch_down<X, W, 2, 1, true>(a, s) : launch_down<X, W, 1, 1, true>(a, s);
    if (tall) return wide ? launch_down<X, W, 2, 2, false>(a, s) : launch_down<X, W, 2, 1, false>(a, s);
    return wide ? launch_down<X, W, 1, 2, false>(a, s) : launch_down<X, W, 1, 1, false>(a, s);
}

}  // namespace
}  // namespace b2

extern "C" {

int b2_moe_decode_workspace_size(size_t T, size_t I, size_t* bytes) {
    using namespace b2;
    if (!bytes) return invalid("b2_moe_decode_workspace_size: null pointer");
    if (T > kMaxDecodeTokens || I > 0x7FFFFFFu)
        return invalid("b2_moe_decode_workspace_size: T must be 128 at most, I below 2^27");
    *bytes = 2 * T * ((I + 7) / 8 * 8) * 8 + 16;  // up to two fp32 parts
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
    a.act = workspace;
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
