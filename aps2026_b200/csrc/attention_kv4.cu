// Attention of each sequence's newest rows over its 4-bit paged cache
// (b2_attention_kv4).
//
// Mathematics: one pass over a row's visible keys with a running reference R
// and sum L of its softmax, p_j = 2^(x_j - R), x in base 2. A key is never
// expanded: with k_j = s c + m per 64 dimensions, q . k_j = sum over groups
// of s (q . (c - 8)) + (m + 8 s)(sum q), so the tensor cores multiply the
// codes -- c - 8 is exact in fp16: a nibble masked into the mantissa of 1024
// (of 1024 / 16 steps for the odd nibbles) and one packed FMA -- and s and m
// are applied in fp32. Likewise sum_j p_j v_j = (p_j s_j) . (c_j - 8) +
// sum p_j (m_j + 8 s_j). (A nibble left as an fp16 subnormal needs no FMA, but
// the matrix unit aligns by the exponent field: it cost 7 bits.)
// The other operands keep fp32's accuracy as two fp16 parts each: queries,
// scaled by a power of two per row, as the upper and lower 8 rows of one M =
// 16 operand; p s as two operands of one accumulator. R is raised only when
// some p s would pass 2^15 (fp16's end), so most tiles rescale nothing.
//
// HBM bound: 144 bytes per visible position and KV head (head_dim 128). A
// warp takes 32 positions a step from its own cp.async ring, S = Q K^T with
// 8 query rows (heads x new tokens of one KV head), then O^T += V^T P^T; in
// these two orders a thread's P is already the operand the second product
// wants. The matrix unit adds to its accumulator with truncation, a bias
// that grows with the chain; so a chain is one step long (4 instructions)
// and the steps are added in registers.
//
// All (row tile, KV head) pairs' steps form one list that is cut into equal
// shares, one per CTA, two CTAs per SM: ragged lengths and one long sequence
// load every SM alike. A share holds the end of one pair, whole pairs, and
// the start of another; parts meet in the workspace, where the last CTA to
// arrive adds them in the list's order, so results repeat bit for bit.
#include <algorithm>

#include <cuda_fp16.h>

#include "kv4.cuh"

namespace b2 {
namespace {

constexpr unsigned kWarps = 8;           // warps per CTA
constexpr unsigned kStep = 32;           // positions per warp step
constexpr unsigned kRows = 8;            // query rows per tile
constexpr unsigned kPairCache = 256;     // pairs whose sizes a CTA keeps
constexpr unsigned kMaxGrid = 2 * 160;   // CTAs the workspace is sized for
constexpr float kNegInf = -INFINITY;

struct AttnKv4Args {
    const void* q;
    void* out;
    std::size_t q_row, q_head;
    unsigned rows, q_heads, group;      // group = q_heads / kv_heads
    const std::uint32_t* q_offsets;
    const std::uint32_t* lens;
    unsigned max_queries, max_len;
    unsigned tiles;                     // row tiles per sequence: ceil(max_queries * group / 8)
    float scale_log2;                   // scale * log2(e)
    unsigned window, sinks;
    unsigned* counters;                 // [kMaxGrid], zero between calls
    float* part_ml;                     // [2 kMaxGrid][8][2]: reference, sum
    float* part_o;                      // [2 kMaxGrid][8][D]
    Kv4View cache;
};

// One row tile of one sequence: 8 of its (query, head in group) rows.
struct Tile {
    unsigned first_row;   // row of q of the sequence's first query
    unsigned queries, len;
    unsigned flat;        // first flat index query * group + head
    unsigned rows;        // rows in the tile, 8 at most
    int p_min, p_max;     // positions of its first and last row
    unsigned sinks, low;  // visible: [0, sinks) and [low, p_max]
    unsigned total;       // number of visible keys
};

template <unsigned D>
struct Shape {
    static constexpr unsigned groups = D / kKv4Group;
    static constexpr unsigned stages = D == 128 ? 2 : 4;
    static constexpr unsigned codes = kStep * D / 2;          // bytes of a step's K (V) codes
    static constexpr unsigned params = kStep * 4 * groups;
    static constexpr unsigned stage = 2 * (codes + params);
    static constexpr unsigned ring = kWarps * stages * stage;
};

template <unsigned D>
struct Smem {
    alignas(128) unsigned char ring[Shape<D>::ring];  // also the warps' O at a segment's end
    uint4 q[D / 16][32];                              // A operands: k-step, lane
    float q_sum[kRows][2];                            // sum of q per group, times scale * log2 e
    float q_scale[kRows];                             // score per unit of accumulated product
    unsigned valid[kWarps][Shape<D>::stages];         // positions of the step that exist
    float ref[kWarps][kRows], sum[kWarps][kRows], mean[kWarps][kRows][2];
    float row_ref[kRows], row_sum[kRows];
    unsigned pair_units[kPairCache];
    unsigned scan[kWarps], scan_total, found_pair, found_before, last;
};

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint4& a, unsigned b0, unsigned b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// `bytes` of the copy are read, the rest of SIZE is zero.
template <int SIZE>
__device__ __forceinline__ void copy_async(unsigned dst, const void* src, bool have) {
    const int bytes = have ? SIZE : 0;
    if constexpr (SIZE == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(bytes), "n"(SIZE)
                     : "memory");
}

__device__ __forceinline__ unsigned half_pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ float2 half_unpack(unsigned w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// The tile `index` of sequence `seq`; total = 0 if it sees nothing, rows = 0
// if it does not exist. `report`: flag what is out of range.
__device__ __forceinline__ Tile make_tile(const AttnKv4Args& a, unsigned seq, unsigned index, bool report) {
    Tile t{};
    t.first_row = a.q_offsets ? __ldg(a.q_offsets + seq) : seq;
    const unsigned end = a.q_offsets ? __ldg(a.q_offsets + seq + 1) : seq + 1;
    t.len = __ldg(a.lens + seq);
    if (end < t.first_row || end > a.rows || end - t.first_row > a.max_queries) {
        if (report) flag_check(B2_CHECK_KV4);
        return t;
    }
    t.queries = end - t.first_row;
    if (t.len > a.max_len || t.len > static_cast<std::size_t>(a.cache.max_pages) << a.cache.page_shift) {
        if (report) flag_check(B2_CHECK_KV4);
        t.len = 0;
    }
    t.flat = index * kRows;
    const unsigned all = t.queries * a.group;
    t.rows = t.flat < all ? min(kRows, all - t.flat) : 0u;
    if (t.rows == 0) return t;
    const int base = static_cast<int>(t.len) - static_cast<int>(t.queries);
    t.p_min = base + static_cast<int>(t.flat / a.group);
    t.p_max = base + static_cast<int>((t.flat + t.rows - 1) / a.group);
    if (t.len == 0 || t.p_max < 0) return t;
    const int low = a.window ? t.p_min - static_cast<int>(a.window) + 1 : 0;
    t.low = low > 0 ? static_cast<unsigned>(low) : 0u;
    t.sinks = min(a.sinks, t.low);
    t.total = t.sinks + static_cast<unsigned>(t.p_max) + 1 - t.low;
    return t;
}

// Position of the u-th visible key.
__device__ __forceinline__ unsigned key_position(const Tile& t, unsigned u) {
    return u < t.sinks ? u : u - t.sinks + t.low;
}

// Query row (flat index f of its sequence) in q / out.
__device__ __forceinline__ std::size_t row_of(const AttnKv4Args& a, const Tile& t, unsigned f) {
    return t.first_row + f / a.group;
}

// The page of this lane's position in the step from key u0; kKv4Padding when
// there is none.
__device__ __forceinline__ unsigned lane_page(const AttnKv4Args& a, const Tile& t, unsigned seq, unsigned u) {
    unsigned page = kKv4Padding;
    if (u < t.total && !kv4_page(a.cache, seq, key_position(t, u), &page)) {
        flag_check(B2_CHECK_KV4);
        page = kKv4Padding;
    }
    return page;
}

// Issues the copies of one step into `stage`; `page` is this lane's.
template <unsigned D>
__device__ __forceinline__ void stage_step(const AttnKv4Args& a, const Tile& t, unsigned head, unsigned u0,
                                           unsigned page, unsigned stage, unsigned* valid, unsigned lane) {
    using S = Shape<D>;
    constexpr unsigned PARTS = D / 32;       // 16-byte chunks of a row of codes
    constexpr unsigned COPIES = PARTS;       // chunks per lane
    const unsigned shift = a.cache.page_shift, slots = (1u << shift) - 1u;
    const unsigned have = __ballot_sync(0xffffffffu, page != kKv4Padding);
    if (lane == 0) *valid = have;
    const std::uint8_t* heads = a.cache.data + head * a.cache.head_stride;
    const unsigned part = lane % PARTS;
    constexpr unsigned P = 4 * S::groups;
    // V rows: 16-byte chunks swizzled inside 128-byte lines, so that the 8
    // bytes (4 at D = 64) that each of 4 x 8 lanes reads hit all banks
    const auto v_at = [&](unsigned tok) {
        const unsigned line = tok * (D / 2) / 128, at = tok * (D / 2) / 16 % 8 + part;
        return stage + S::codes + line * 128 + ((at ^ ((D == 128 ? line & 3u : line & 1u) << 1)) << 4);
    };
    const unsigned page0 = __shfl_sync(0xffffffffu, page, 0);
    const unsigned j0 = key_position(t, u0);
    if (__all_sync(0xffffffffu, page == page0) && page0 != kKv4Padding &&
        (u0 >= t.sinks || u0 + kStep <= t.sinks) && ((j0 ^ (j0 + kStep - 1)) >> shift) == 0) {
        // 32 neighbours of one page: four runs of memory
        const std::uint8_t* block = heads + page0 * a.cache.page_stride;
        const unsigned slot = j0 & slots;
        const std::uint8_t* codes = block + (slot * (D / 2) + lane * 16);
        const std::uint8_t* v_codes = codes + kv4_v_codes<D>(shift);
#pragma unroll
        for (unsigned i = 0; i < COPIES; ++i) {
            copy_async<16>(stage + lane * 16 + i * 512, codes + i * 512, true);
            copy_async<16>(v_at(i * (32 / PARTS) + lane / PARTS), v_codes + i * 512, true);
        }
        const std::uint8_t* params = block + kv4_k_params<D>(shift) + (slot + lane) * P;
        copy_async<P>(stage + 2 * S::codes + lane * P, params, true);
        copy_async<P>(stage + 2 * S::codes + S::params + lane * P, params + (P << shift), true);
        return;
    }
#pragma unroll
    for (unsigned i = 0; i < COPIES; ++i) {
        const unsigned tok = i * (32 / PARTS) + lane / PARTS;
        const unsigned pg = __shfl_sync(0xffffffffu, page, tok);
        const bool ok = pg != kKv4Padding;
        const unsigned slot = key_position(t, u0 + tok) & slots;
        const std::uint8_t* src =
            ok ? heads + pg * a.cache.page_stride + (slot * (D / 2) + part * 16) : a.cache.data;
        copy_async<16>(stage + tok * (D / 2) + part * 16, src, ok);
        copy_async<16>(v_at(tok), ok ? src + kv4_v_codes<D>(shift) : src, ok);
    }
    const bool ok = page != kKv4Padding;
    const unsigned slot = key_position(t, u0 + lane) & slots;
    const std::uint8_t* block = ok ? heads + page * a.cache.page_stride : a.cache.data;
    copy_async<P>(stage + 2 * S::codes + lane * P, block + (ok ? kv4_k_params<D>(shift) + slot * P : 0u), ok);
    copy_async<P>(stage + 2 * S::codes + S::params + lane * P, block + (ok ? kv4_v_params<D>(shift) + slot * P : 0u),
                  ok);
}

// Pairs of fp32 in one register pair: two results per instruction.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ f32x2 both(float v) { return f2_pack(v, v); }

// What a warp carries through its steps. Thread (r = lane / 4, c = lane % 4)
// holds row r's reference and its part of the row's sums (even and odd keys),
// and O^T for rows 2c and 2c + 1, dimensions g * 64 + r * 8 + ...: o[g][n][0]
// is dimension n of the octet, o[g][n][1] dimension 4 + n.
template <unsigned D>
struct WarpState {
    float ref;
    f32x2 sum, mean[Shape<D>::groups];
    f32x2 o[Shape<D>::groups][4][2];
};

// c - 8 of the low (SHIFTED: second) nibbles of both halves of w, in fp16.
template <bool SHIFTED>
__device__ __forceinline__ unsigned codes_f16(unsigned w) {
    unsigned d;
    if (SHIFTED) {  // (1024 + 16 c) / 16 - 72
        const unsigned x = (w & 0x00F000F0u) | 0x64006400u;
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(x), "r"(0x2C002C00u), "r"(0xD480D480u));
    } else {  // (1024 + c) - 1032
        const unsigned x = (w & 0x000F000Fu) | 0x64006400u;
        asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(0xE408E408u));
    }
    return d;
}

template <unsigned N>
__device__ __forceinline__ void lds_n(unsigned addr, unsigned* w) {
    if constexpr (N == 4)
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
    else if constexpr (N == 2)
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
    else
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
}

__device__ __forceinline__ bool nonfinite_params(unsigned w) {
    return (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u;
}

// One step of 32 keys. MASKED: some row does not see some of them.
template <unsigned D, bool MASKED>
__device__ __forceinline__ void attend_step(const AttnKv4Args& a, const Tile& t, const Smem<D>& sm, unsigned stage,
                                            unsigned u0, unsigned valid, int pos, float q_scale,
                                            const float (&q_sum)[Shape<D>::groups], unsigned lane,
                                            WarpState<D>& st) {
    using S = Shape<D>;
    constexpr unsigned G = S::groups;
    const unsigned r = lane / 4, c = lane % 4;

    // ---- scores: x[b] holds keys 8b + 2c and 8b + 2c + 1 of row r ----
    f32x2 x[4] = {0, 0, 0, 0};
    {
        unsigned kw[4][2 * G], kp[4][2 * G];
#pragma unroll
        for (unsigned b = 0; b < 4; ++b) {
            lds_n<2 * G>(stage + (8 * b + r) * (D / 2) + c * (D / 8), kw[b]);
            lds_n<2 * G>(stage + 2 * S::codes + (8 * b + 2 * c) * 4 * G, kp[b]);
        }
#pragma unroll
        for (unsigned g = 0; g < G; ++g) {
            float acc[4][4];
#pragma unroll
            for (unsigned b = 0; b < 4; ++b) acc[b][0] = acc[b][1] = acc[b][2] = acc[b][3] = 0.0f;
#pragma unroll
            for (unsigned k = 0; k < 4; ++k) {
                const uint4 q = sm.q[g * 4 + k][lane];
#pragma unroll
                for (unsigned b = 0; b < 4; ++b) {
                    const unsigned w = kw[b][g * 2 + k / 2] >> (k % 2 * 8);
                    mma_f16(acc[b], q, codes_f16<false>(w), codes_f16<true>(w));
                }
            }
#pragma unroll
            for (unsigned b = 0; b < 4; ++b) {
                const f32x2 dot = add2(f2_pack(acc[b][0], acc[b][1]), f2_pack(acc[b][2], acc[b][3]));
                const f32x2 step = f2_pack(bf16_low(kp[b][g]), bf16_low(kp[b][G + g]));
                const f32x2 mid = f2_fma(step, both(8.0f), f2_pack(bf16_high(kp[b][g]), bf16_high(kp[b][G + g])));
                x[b] = f2_fma(mul2(step, dot), both(q_scale), x[b]);
                x[b] = f2_fma(mid, both(q_sum[g]), x[b]);
            }
        }
    }
    unsigned vp[4][2 * G];
#pragma unroll
    for (unsigned b = 0; b < 4; ++b) lds_n<2 * G>(stage + 2 * S::codes + S::params + (8 * b + 2 * c) * 4 * G, vp[b]);
    if (MASKED) {
#pragma unroll
        for (unsigned b = 0; b < 4; ++b) {
            float2 y = f2_unpack(x[b]);
#pragma unroll
            for (unsigned e = 0; e < 2; ++e) {
                const unsigned tok = 8 * b + 2 * c + e;
                const int j = static_cast<int>(key_position(t, u0 + tok));
                const bool seen = ((valid >> tok) & 1u) && j <= pos &&
                                  (a.window == 0 || pos - j < static_cast<int>(a.window) || j < static_cast<int>(a.sinks));
                if (!seen) (e ? y.y : y.x) = kNegInf;
                // a value that is not finite reaches the rows that see it
                // (through the mean's sum), and not the others (0 * NaN)
#pragma unroll
                for (unsigned g = 0; g < G; ++g) {
                    unsigned& w = vp[b][e * G + g];
                    if (nonfinite_params(w)) {
                        w = 0;
                        if (seen) st.mean[g] = both(NAN);
                    }
                }
            }
            x[b] = f2_pack(y.x, y.y);
        }
    }

    // ---- the reference: p s is to stay below 2^15 ----
    unsigned top_s = 0;
#pragma unroll
    for (unsigned b = 0; b < 4; ++b)
#pragma unroll
        for (unsigned i = 0; i < 2 * G; ++i) top_s = max(top_s, vp[b][i] << 16);
    top_s = __reduce_max_sync(0xffffffffu, top_s);
    if (top_s >= 0x7F800000u) {  // a step that is not finite has no part in the reference
        top_s = 0;
#pragma unroll
        for (unsigned b = 0; b < 4; ++b)
#pragma unroll
            for (unsigned i = 0; i < 2 * G; ++i)
                if ((vp[b][i] << 16) < 0x7F800000u) top_s = max(top_s, vp[b][i] << 16);
        top_s = __reduce_max_sync(0xffffffffu, top_s);
    }
    const float s_log2 = static_cast<float>(max(static_cast<int>(top_s >> 23) - 126, -60));
    float top = kNegInf;
#pragma unroll
    for (unsigned b = 0; b < 4; ++b) {
        const float2 y = f2_unpack(x[b]);
        top = fmaxf(top, fmaxf(y.x, y.y));
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float need = top + s_log2 - 11.0f;
    const bool raise = need > st.ref + 4.0f;
    if (__any_sync(0xffffffffu, raise)) {
        const float ref = raise ? need : st.ref;
        const float alpha = raise ? exp2_approx(st.ref - ref) : 1.0f;
        st.ref = ref;
        st.sum = mul2(st.sum, both(alpha));
        const f32x2 cols = f2_pack(__shfl_sync(0xffffffffu, alpha, 8 * c), __shfl_sync(0xffffffffu, alpha, 8 * c + 4));
#pragma unroll
        for (unsigned g = 0; g < G; ++g) {
            st.mean[g] = mul2(st.mean[g], both(alpha));
#pragma unroll
            for (unsigned n = 0; n < 4; ++n) {
                st.o[g][n][0] = mul2(st.o[g][n][0], cols);
                st.o[g][n][1] = mul2(st.o[g][n][1], cols);
            }
        }
    }
    const float ref = st.ref == kNegInf ? 0.0f : st.ref;
    f32x2 steps[G][4];
#pragma unroll
    for (unsigned b = 0; b < 4; ++b) {
        const float2 y = f2_unpack(add2(x[b], both(-ref)));
        x[b] = f2_pack(exp2_approx(y.x), exp2_approx(y.y));
        st.sum = add2(st.sum, x[b]);
#pragma unroll
        for (unsigned g = 0; g < G; ++g) {
            steps[g][b] = f2_pack(bf16_low(vp[b][g]), bf16_low(vp[b][G + g]));
            const f32x2 mid =
                f2_fma(steps[g][b], both(8.0f), f2_pack(bf16_high(vp[b][g]), bf16_high(vp[b][G + g])));
            st.mean[g] = f2_fma(x[b], mid, st.mean[g]);
        }
    }

    // ---- O^T += V^T (p s)^T ----
    unsigned vw[8][G];
#pragma unroll
    for (unsigned b = 0; b < 4; ++b)
#pragma unroll
        for (unsigned e = 0; e < 2; ++e) {
            const unsigned tok = 8 * b + 2 * c + e;
            const unsigned line = tok * (D / 2) / 128, at = tok * (D / 2) / 16 % 8 + r * G * 4 / 16;
            const unsigned sw = at ^ ((D == 128 ? line & 3u : line & 1u) << 1);
            lds_n<G>(stage + S::codes + line * 128 + sw * 16 + (r * G * 4) % 16, vw[2 * b + e]);
        }
#pragma unroll
    for (unsigned g = 0; g < G; ++g) {
        unsigned hi[4], lo[4], xa[4], ya[4];
#pragma unroll
        for (unsigned b = 0; b < 4; ++b) {
            const f32x2 ps = mul2(x[b], steps[g][b]);
            const float2 y = f2_unpack(ps);
            hi[b] = half_pack(y.x, y.y);
            const float2 h = half_unpack(hi[b]);
            const float2 rest = f2_unpack(f2_fma(f2_pack(h.x, h.y), both(-1.0f), ps));
            lo[b] = half_pack(rest.x, rest.y);
            xa[b] = __byte_perm(vw[2 * b][g], vw[2 * b + 1][g], 0x5410);
            ya[b] = __byte_perm(vw[2 * b][g], vw[2 * b + 1][g], 0x7632);
        }
#pragma unroll
        for (unsigned n = 0; n < 4; ++n) {
            const unsigned sh = n / 2 * 8;
            float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (unsigned h = 0; h < 2; ++h) {
                const unsigned w[4] = {xa[2 * h] >> sh, ya[2 * h] >> sh, xa[2 * h + 1] >> sh, ya[2 * h + 1] >> sh};
                const uint4 v = n % 2 ? make_uint4(codes_f16<true>(w[0]), codes_f16<true>(w[1]), codes_f16<true>(w[2]),
                                                   codes_f16<true>(w[3]))
                                      : make_uint4(codes_f16<false>(w[0]), codes_f16<false>(w[1]),
                                                   codes_f16<false>(w[2]), codes_f16<false>(w[3]));
                mma_f16(acc, v, hi[2 * h], hi[2 * h + 1]);
                mma_f16(acc, v, lo[2 * h], lo[2 * h + 1]);
            }
            st.o[g][n][0] = add2(st.o[g][n][0], f2_pack(acc[0], acc[1]));
            st.o[g][n][1] = add2(st.o[g][n][1], f2_pack(acc[2], acc[3]));
        }
    }
}

// The tile's queries as A operands: hi parts in rows 0..7, lo parts in 8..15,
// each row scaled by a power of two to about 2^9 at most.
template <typename T, unsigned D>
__device__ __forceinline__ void load_queries(const AttnKv4Args& a, const Tile& t, unsigned head, Smem<D>& sm) {
    constexpr unsigned G = Shape<D>::groups;
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const unsigned f = t.flat + warp;
    const bool have = warp < t.rows;
    const T* q = static_cast<const T*>(a.q) + row_of(a, t, have ? f : t.flat) * a.q_row +
                 (head * a.group + (have ? f : t.flat) % a.group) * a.q_head;
    float v[D / 32], top = 0.0f, sum[G];
#pragma unroll
    for (unsigned g = 0; g < G; ++g) sum[g] = 0.0f;
#pragma unroll
    for (unsigned e = 0; e < D / 32; ++e) {
        v[e] = have ? as_float(q[lane + 32 * e]) : 0.0f;
        top = fmaxf(top, fabsf(v[e]));
        sum[e / 2] += v[e];
    }
    top = warp_max(top);
#pragma unroll
    for (unsigned g = 0; g < G; ++g) sum[g] = warp_sum(sum[g]);
    // 2^e with top * 2^e in [2^9, 2^10)
    int e = 136 - static_cast<int>(__float_as_uint(top) >> 23);
    e = top == 0.0f || e < -100 ? (top == 0.0f ? 0 : -100) : min(e, 100);
    const float up = __uint_as_float(static_cast<unsigned>(127 + e) << 23);
    if (lane == 0) {
        sm.q_scale[warp] = a.scale_log2 * __uint_as_float(static_cast<unsigned>(127 - e) << 23);
#pragma unroll
        for (unsigned g = 0; g < G; ++g) sm.q_sum[warp][g] = sum[g] * a.scale_log2;
    }
    // dimension d = w * 32 + c * 8 + i of lane (row, c): nibble i of word w.
    // Pair (i, i + 4) of one register.
    __half* words = reinterpret_cast<__half*>(sm.q);
#pragma unroll
    for (unsigned k = 0; k < D / 32; ++k) {
        const unsigned d = lane + 32 * k, w = d / 32, c = d % 32 / 8, i = d % 8;
        const float x = v[k] * up;
        const __half hi = __float2half_rn(x);
        const __half lo = __float2half_rn(x - __half2float(hi));
        const unsigned step = w * 2 + (i % 4) / 2, reg = (i & 1u) * 2, half = i / 4;
        const unsigned at = ((step * 32 + warp * 4 + c) * 4 + reg) * 2 + half;
        words[at] = hi;
        words[at + 2] = lo;
    }
}

template <typename T>
__device__ __forceinline__ void store_out(T* p, float y) {
    if constexpr (sizeof(T) == 2) *p = __float2bfloat16_rn(y);
    else *p = y;
}

// Adds up the parts of a pair that CTAs first .. last hold (in this order)
// and writes its rows. `begin`: first unit of the pair in the list.
template <typename T, unsigned D>
__device__ __forceinline__ void join_parts(const AttnKv4Args& a, const Tile& t, unsigned head, unsigned long long begin,
                                           unsigned long long share, unsigned first, unsigned last, Smem<D>& sm) {
    const unsigned n = last - first + 1;
    float* factor = reinterpret_cast<float*>(sm.ring);  // [8][n]
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const auto slot = [&](unsigned i) {
        return static_cast<std::size_t>(2) * (first + i) + (begin < (first + i) * share ? 0 : 1);
    };
    if (warp < t.rows) {
        float m = kNegInf, l = 0.0f;
        for (unsigned i = lane; i < n; i += 32) {
            const float2 v = __ldcg(reinterpret_cast<const float2*>(a.part_ml) + slot(i) * kRows + warp);
            factor[warp * n + i] = v.x;
            m = fmaxf(m, v.x);
        }
        m = warp_max(m);
        for (unsigned i = lane; i < n; i += 32) {
            const float ref = factor[warp * n + i];
            const float w = ref == kNegInf ? 0.0f : exp2_approx(ref - m);
            factor[warp * n + i] = w;
            l += w * __ldcg(a.part_ml + (slot(i) * kRows + warp) * 2 + 1);
        }
        l = warp_sum(l);
        if (lane == 0) sm.row_sum[warp] = l;
    }
    __syncthreads();
    for (unsigned i = threadIdx.x; i < t.rows * (D / 4); i += kWarps * 32) {
        const unsigned row = i / (D / 4), d4 = i % (D / 4);
        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
        for (unsigned k = 0; k < n; ++k) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(a.part_o) + (slot(k) * kRows + row) * (D / 4) + d4);
            const float w = factor[row * n + k];
            s.x = fmaf(w, v.x, s.x); s.y = fmaf(w, v.y, s.y); s.z = fmaf(w, v.z, s.z); s.w = fmaf(w, v.w, s.w);
        }
        const float l = sm.row_sum[row], inv = 1.0f / l;
        const unsigned f = t.flat + row;
        T* out = static_cast<T*>(a.out) + (row_of(a, t, f) * a.q_heads + head * a.group + f % a.group) * D + d4 * 4;
        store_out(out, l == 0.0f ? 0.0f : s.x * inv);
        store_out(out + 1, l == 0.0f ? 0.0f : s.y * inv);
        store_out(out + 2, l == 0.0f ? 0.0f : s.z * inv);
        store_out(out + 3, l == 0.0f ? 0.0f : s.w * inv);
    }
    __syncthreads();
}

// Units [from, to) of the pair (tile t of sequence seq, head): this CTA's
// part. whole: they are all of it.
template <typename T, unsigned D>
__device__ __forceinline__ void run_segment(const AttnKv4Args& a, const Tile& t, unsigned seq, unsigned head,
                                            unsigned from, unsigned to, bool whole, std::size_t slot, Smem<D>& sm) {
    using S = Shape<D>;
    constexpr unsigned G = S::groups;
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    load_queries<T, D>(a, t, head, sm);

    const unsigned steps = to - from > warp ? (to - from - warp + kWarps - 1) / kWarps : 0u;
    const auto key_of = [&](unsigned i) { return (from + warp + i * kWarps) * kStep; };
    const unsigned ring = smem_addr(sm.ring) + warp * S::stages * S::stage;
    unsigned pages[S::stages];
#pragma unroll
    for (unsigned i = 0; i < S::stages; ++i)
        pages[i] = i < steps ? lane_page(a, t, seq, key_of(i) + lane) : kKv4Padding;
#pragma unroll
    for (unsigned i = 0; i < S::stages; ++i) {
        if (i < steps) stage_step<D>(a, t, head, key_of(i), pages[i], ring + i * S::stage, &sm.valid[warp][i], lane);
        cp_async_commit();
    }
    unsigned next_page = S::stages < steps ? lane_page(a, t, seq, key_of(S::stages) + lane) : kKv4Padding;
    __syncthreads();  // queries

    const unsigned r = lane / 4;
    const float q_scale = sm.q_scale[r];
    float q_sum[G];
#pragma unroll
    for (unsigned g = 0; g < G; ++g) q_sum[g] = sm.q_sum[r][g];
    const int pos = r < t.rows ? static_cast<int>(t.len) - static_cast<int>(t.queries) +
                                     static_cast<int>((t.flat + r) / a.group)
                               : -1;
    WarpState<D> st;
    st.ref = kNegInf;
    st.sum = 0;
#pragma unroll
    for (unsigned g = 0; g < G; ++g) {
        st.mean[g] = 0;
#pragma unroll
        for (unsigned n = 0; n < 4; ++n) st.o[g][n][0] = st.o[g][n][1] = 0;
    }
    for (unsigned i = 0; i < steps; ++i) {
        cp_async_wait<S::stages - 1>();
        __syncwarp();
        const unsigned u0 = key_of(i), at = i % S::stages, stage = ring + at * S::stage;
        const unsigned valid = sm.valid[warp][at];
        // all rows see all 32 keys: they exist, none is ahead of the first
        // row, and none is behind the last row's window
        const bool clear = valid == 0xFFFFFFFFu && static_cast<int>(key_position(t, u0 + kStep - 1)) <= t.p_min &&
                           (a.window == 0 || u0 + kStep <= t.sinks ||
                            static_cast<int>(u0 < t.sinks ? t.low : key_position(t, u0)) >
                                t.p_max - static_cast<int>(a.window));
        if (clear) attend_step<D, false>(a, t, sm, stage, u0, valid, pos, q_scale, q_sum, lane, st);
        else attend_step<D, true>(a, t, sm, stage, u0, valid, pos, q_scale, q_sum, lane, st);
        __syncwarp();
        if (i + S::stages < steps) {
            stage_step<D>(a, t, head, key_of(i + S::stages), next_page, stage, &sm.valid[warp][at], lane);
            next_page = i + S::stages + 1 < steps ? lane_page(a, t, seq, key_of(i + S::stages + 1) + lane)
                                                  : kKv4Padding;
        }
        cp_async_commit();
    }
    cp_async_wait<0>();

    // ---- the warps' sums meet ----
    const auto row_total = [](f32x2 v) {
        const float2 y = f2_unpack(v);
        float total = y.x + y.y;
        total += __shfl_xor_sync(0xffffffffu, total, 1);
        return total + __shfl_xor_sync(0xffffffffu, total, 2);
    };
    const float sum = row_total(st.sum);
    float mean[G];
#pragma unroll
    for (unsigned g = 0; g < G; ++g) mean[g] = row_total(st.mean[g]);
    if (lane % 4 == 0) {
        sm.ref[warp][r] = st.ref;
        sm.sum[warp][r] = sum;
#pragma unroll
        for (unsigned g = 0; g < G; ++g) sm.mean[warp][r][g] = mean[g];
    }
    __syncthreads();  // every ring is drained: it becomes the warps' O
    float* o = reinterpret_cast<float*>(sm.ring);
    constexpr unsigned PITCH = D + 4;
    const unsigned used = min(to - from, kWarps);  // warps that had a step
    if (warp < used) {
        const unsigned c2 = lane % 4 * 2;
#pragma unroll
        for (unsigned e = 0; e < 2; ++e)
            if (c2 + e < t.rows) {
                float* row = o + (warp * kRows + c2 + e) * PITCH + r * 8;
#pragma unroll
                for (unsigned g = 0; g < G; ++g) {
                    float v[8];
#pragma unroll
                    for (unsigned n = 0; n < 4; ++n) {
                        const float2 y0 = f2_unpack(st.o[g][n][0]), y1 = f2_unpack(st.o[g][n][1]);
                        v[n] = e ? y0.y : y0.x;
                        v[4 + n] = e ? y1.y : y1.x;
                    }
                    *reinterpret_cast<float4*>(row + g * 64) = make_float4(v[0], v[1], v[2], v[3]);
                    *reinterpret_cast<float4*>(row + g * 64 + 4) = make_float4(v[4], v[5], v[6], v[7]);
                }
            }
    }
    if (threadIdx.x < kRows) {
        float m = kNegInf, l = 0.0f;
        for (unsigned w = 0; w < used; ++w) m = fmaxf(m, sm.ref[w][threadIdx.x]);
        for (unsigned w = 0; w < used; ++w) {
            const float ref = sm.ref[w][threadIdx.x];
            const float f = ref == kNegInf ? 0.0f : exp2_approx(ref - m);
            sm.ref[w][threadIdx.x] = f;
            l += f * sm.sum[w][threadIdx.x];
        }
        sm.row_ref[threadIdx.x] = m;
        sm.row_sum[threadIdx.x] = l;
    }
    __syncthreads();
    for (unsigned i = threadIdx.x; i < t.rows * D; i += kWarps * 32) {
        const unsigned row = i / D, d = i % D;
        float y = 0.0f;
        for (unsigned w = 0; w < used; ++w)
            y = fmaf(sm.ref[w][row], o[(w * kRows + row) * PITCH + d] + sm.mean[w][row][d / kKv4Group], y);
        if (whole) {
            const unsigned f = t.flat + row;
            const float l = sm.row_sum[row];
            store_out(static_cast<T*>(a.out) + (row_of(a, t, f) * a.q_heads + head * a.group + f % a.group) * D + d,
                      l == 0.0f ? 0.0f : y / l);
        } else {
            __stcg(a.part_o + (slot * kRows + row) * D + d, y);
        }
    }
    if (!whole && threadIdx.x < t.rows)
        __stcg(reinterpret_cast<float2*>(a.part_ml) + slot * kRows + threadIdx.x,
               make_float2(sm.row_ref[threadIdx.x], sm.row_sum[threadIdx.x]));
}

// Exclusive sum of v over the CTA's threads and the total, through sm.scan;
// returns whether any thread's flag is set.
template <unsigned D>
__device__ __forceinline__ bool scan_units(unsigned v, bool flag, Smem<D>& sm, unsigned* exclusive, unsigned* total) {
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    unsigned incl = v;
#pragma unroll
    for (unsigned o = 1; o < 32; o <<= 1) {
        const unsigned n = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += n;
    }
    if (lane == 31) sm.scan[warp] = incl;
    const bool any = __syncthreads_or(flag);
    unsigned before = 0, all = 0;
#pragma unroll
    for (unsigned w = 0; w < kWarps; ++w) {
        if (w < warp) before += sm.scan[w];
        all += sm.scan[w];
    }
    __syncthreads();
    *total = all;
    *exclusive = before + incl - v;
    return any;
}

// Zeros for this CTA's pairs of p0 .. p0 + kPairCache that see nothing.
template <typename T, unsigned D>
__device__ __forceinline__ void write_blank_rows(const AttnKv4Args& a, unsigned p0) {
    const unsigned heads = a.cache.kv_heads, pairs = a.cache.seqs * a.tiles;
    const unsigned end = min(pairs, p0 + kPairCache);
    for (unsigned p = p0 + (blockIdx.x + gridDim.x - p0 % gridDim.x) % gridDim.x; p < end; p += gridDim.x) {
        const Tile t = make_tile(a, p / a.tiles, p % a.tiles, false);
        if (t.total != 0) continue;
        for (unsigned i = threadIdx.x; i < t.rows * heads * D; i += kWarps * 32) {
            const unsigned f = t.flat + i / D / heads, h = i / D % heads;
            store_out(static_cast<T*>(a.out) + (row_of(a, t, f) * a.q_heads + h * a.group + f % a.group) * D + i % D,
                      0.0f);
        }
    }
}

template <typename T, unsigned D>
__global__ void __launch_bounds__(kWarps * 32, 2)
attention_kv4_shares(AttnKv4Args a) {
    extern __shared__ unsigned char smem_raw[];
    Smem<D>& sm = *reinterpret_cast<Smem<D>*>(smem_raw);
    pdl_begin();
    const unsigned heads = a.cache.kv_heads;
    const unsigned pairs = a.cache.seqs * a.tiles;

    // ---- sizes of all pairs; rows that see nothing are written here ----
    unsigned long long all_units = 0;
    unsigned kept = 0;  // units of pair threadIdx.x, for pairs <= kPairCache
    for (unsigned p0 = 0; p0 < pairs; p0 += kPairCache) {
        const unsigned p = p0 + threadIdx.x;
        unsigned units = 0;
        bool blank = false;  // rows that see nothing, this CTA's to write
        if (p < pairs) {
            const bool mine = p % gridDim.x == blockIdx.x;
            const Tile t = make_tile(a, p / a.tiles, p % a.tiles, mine);
            units = (t.total + kStep - 1) / kStep;
            blank = mine && units == 0 && t.rows;
        }
        unsigned before, total;
        if (scan_units(units, blank, sm, &before, &total)) write_blank_rows<T, D>(a, p0);
        all_units += total;
        kept = units;
    }

    // ---- this CTA's share of the list (pair-major, then head, then unit) ----
    const unsigned long long work = all_units * heads;
    unsigned long long share = (work + gridDim.x - 1) / gridDim.x;
    // short contexts: not less than a pair, up to a unit per warp, so that a
    // pair is not cut for nothing
    const unsigned long long per_pair = (work + static_cast<unsigned long long>(pairs) * heads - 1) /
                                        (static_cast<unsigned long long>(pairs) * heads);
    share = max(share, min(per_pair, static_cast<unsigned long long>(kWarps)));
    unsigned long long at = blockIdx.x * share;
    const unsigned long long stop = min(at + share, work);
    if (at >= stop) return;
    // the pair that holds unit `at`
    unsigned long long pair_begin = 0;  // units of earlier pairs, one head
    unsigned block0 = 0;                // first pair of the cached block
    for (unsigned p0 = 0; p0 < pairs; p0 += kPairCache) {
        const unsigned p = p0 + threadIdx.x;
        unsigned units = kept;
        if (pairs > kPairCache) {
            units = 0;
            if (p < pairs) units = (make_tile(a, p / a.tiles, p % a.tiles, false).total + kStep - 1) / kStep;
        }
        unsigned before, total;
        scan_units(units, false, sm, &before, &total);
        sm.pair_units[threadIdx.x] = units;
        const unsigned long long b = (pair_begin + before) * heads;
        if (units && at >= b && at < b + static_cast<unsigned long long>(units) * heads) {
            sm.found_pair = p;
            sm.found_before = before;
        }
        __syncthreads();
        block0 = p0;
        if (at < (pair_begin + total) * heads) {
            pair_begin += sm.found_before;
            break;
        }
        pair_begin += total;
    }
    unsigned pair = sm.found_pair;
    while (at < stop) {
        unsigned units = 0;
        for (;; ++pair) {  // skips pairs that see nothing
            units = pair - block0 < kPairCache
                        ? sm.pair_units[pair - block0]
                        : (make_tile(a, pair / a.tiles, pair % a.tiles, false).total + kStep - 1) / kStep;
            if (units) break;
        }
        const unsigned seq = pair / a.tiles;
        const Tile t = make_tile(a, seq, pair % a.tiles, false);
        while (at < stop && at < (pair_begin + units) * heads) {
            const unsigned head = static_cast<unsigned>((at - pair_begin * heads) / units);
            const unsigned long long begin = pair_begin * heads + static_cast<unsigned long long>(head) * units;
            const unsigned long long end = begin + units;
            const unsigned from = static_cast<unsigned>(at - begin);
            const unsigned to = static_cast<unsigned>(min(end, stop) - begin);
            const bool whole = from == 0 && to == units;
            // a part at the start of the share goes to slot 0, one at its end to slot 1
            const std::size_t slot = static_cast<std::size_t>(2) * blockIdx.x + (from == 0 ? 1 : 0);
            run_segment<T, D>(a, t, seq, head, from, to, whole, slot, sm);
            if (!whole) {
                const unsigned first = static_cast<unsigned>(begin / share);
                const unsigned last = static_cast<unsigned>((end - 1) / share);
                __threadfence();
                __syncthreads();
                if (threadIdx.x == 0) {
                    const unsigned arrived = atomicAdd(a.counters + first, 1u);
                    sm.last = arrived == last - first;
                    if (sm.last) a.counters[first] = 0;
                }
                __syncthreads();
                if (sm.last) {
                    __threadfence();
                    join_parts<T, D>(a, t, head, begin, share, first, last, sm);
                }
            }
            __syncthreads();  // the next segment's queries overwrite these
            at = begin + to;
        }
        pair_begin += units;
        ++pair;
    }
}

template <typename T, unsigned D>
cudaError_t launch_attention(const AttnKv4Args& a, cudaStream_t s) {
    auto kernel = attention_kv4_shares<T, D>;
    const std::size_t smem = sizeof(Smem<D>);
    const cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
    if (e != cudaSuccess) return e;
    // a CTA per pair at least, and no more than there can be shares of kWarps units
    const std::size_t keys = a.window ? std::min<std::size_t>(a.max_len, std::size_t(a.window) + a.sinks + a.max_queries)
                                      : a.max_len;
    const std::size_t pairs = static_cast<std::size_t>(a.cache.seqs) * a.tiles * a.cache.kv_heads;
    const std::size_t units = (keys + kStep - 1) / kStep * pairs;
    const std::size_t grid = std::min<std::size_t>(std::min<std::size_t>(2 * sm_count(), kMaxGrid),
                                                   std::max(pairs, (units + kWarps - 1) / kWarps));
    return launch_pdl(kernel, static_cast<unsigned>(grid), kWarps * 32, smem, s, a);
}

}  // namespace
}  // namespace b2

B2_DEFINE_CHECK_TAKER(attention_kv4)

extern "C" {

int b2_attention_kv4_workspace_size(size_t head_dim, size_t* bytes) {
    using namespace b2;
    if (!bytes) return invalid("b2_attention_kv4_workspace_size: null pointer");
    if (head_dim != 64 && head_dim != 128) return invalid("b2_attention_kv4_workspace_size: head_dim must be 64 or 128");
    *bytes = kMaxGrid * 4 + 2 * kMaxGrid * kRows * (2 + head_dim) * sizeof(float);
    return B2_OK;
}

int b2_attention_kv4(const void* q, size_t q_row_stride, size_t q_head_stride, void* out, uint32_t dtype,
                     size_t rows, size_t q_heads, const uint32_t* q_offsets, const uint32_t* lens,
                     size_t max_queries, size_t max_len, float scale, size_t window, size_t sinks,
                     const b2_kv4_cache* cache, void* workspace, size_t workspace_bytes, b2_stream_t stream) {
    using namespace b2;
    AttnKv4Args a{};
    int rc = kv4_view(cache, "b2_attention_kv4", &a.cache);
    if (rc != B2_OK) return rc;
    if (!kv4_dtype(dtype)) return invalid("b2_attention_kv4: unknown dtype");
    if (q_heads == 0 || q_heads % cache->kv_heads) return invalid("b2_attention_kv4: q_heads must be a multiple of kv_heads");
    if (rows == 0 || cache->seqs == 0) return B2_OK;
    if (!q || !out || !lens || !workspace) return invalid("b2_attention_kv4: null pointer");
    if (!q_offsets && rows != cache->seqs) return invalid("b2_attention_kv4: without q_offsets every sequence has one row");
    if (max_queries == 0) return invalid("b2_attention_kv4: max_queries must be 1 at least");
    if (rows > 0x7FFFFFFFu || q_heads > 0xFFFF || max_queries > 0x7FFFFFFFu / q_heads)
        return invalid("b2_attention_kv4: more than 2^31 query rows");
    if (max_len > std::size_t(1) << 28) return invalid("b2_attention_kv4: max_len past 2^28");
    std::size_t need = 0;
    b2_attention_kv4_workspace_size(cache->head_dim, &need);
    if (workspace_bytes < need) return invalid("b2_attention_kv4: workspace too small");
    if (!aligned16(out) || !aligned16(workspace)) return invalid("b2_attention_kv4: out and workspace must be 16-byte aligned");
    a.q = q; a.out = out; a.q_row = q_row_stride; a.q_head = q_head_stride;
    a.rows = static_cast<unsigned>(rows); a.q_heads = static_cast<unsigned>(q_heads);
    a.group = static_cast<unsigned>(q_heads / cache->kv_heads);
    a.q_offsets = q_offsets; a.lens = lens;
    a.max_queries = static_cast<unsigned>(max_queries); a.max_len = static_cast<unsigned>(max_len);
    a.scale_log2 = scale * 1.4426950408889634f;
    if (cache->seqs > 0x7FFFFFFFu / ((max_queries * a.group + kRows - 1) / kRows))
        return invalid("b2_attention_kv4: too many row tiles");
    a.tiles = static_cast<unsigned>((max_queries * a.group + kRows - 1) / kRows);
    a.counters = static_cast<unsigned*>(workspace);
    a.part_ml = reinterpret_cast<float*>(a.counters + kMaxGrid);
    a.part_o = a.part_ml + 2 * kMaxGrid * kRows * 2;
    a.window = static_cast<unsigned>(window < 0x7FFFFFFFu ? window : 0);  // a window past every length: none
    a.sinks = static_cast<unsigned>(sinks < 0x7FFFFFFFu ? sinks : 0x7FFFFFFFu);
    cudaStream_t s = as_stream(stream);
    cudaError_t e;
    if (dtype == B2_DTYPE_F32) {
        e = cache->head_dim == 128 ? launch_attention<float, 128>(a, s) : launch_attention<float, 64>(a, s);
    } else {
        e = cache->head_dim == 128 ? launch_attention<__nv_bfloat16, 128>(a, s)
                                   : launch_attention<__nv_bfloat16, 64>(a, s);
    }
    if (e != cudaSuccess) {
        cudaGetLastError();
        return set_error(B2_ERR_CUDA, std::string("b2_attention_kv4: ") + cudaGetErrorString(e));
    }
    return launch_result("b2_attention_kv4");
}

}  // extern "C"
