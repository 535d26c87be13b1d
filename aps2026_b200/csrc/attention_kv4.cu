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
// scaled by a power of two per row, and p s. R is raised only when some p s
// would pass 2^15 (fp16's end), so most steps rescale nothing. The matrix
// unit adds to its accumulator with truncation, a bias that grows with the
// chain; so a chain is one step long (4 instructions at most) and the steps
// are added in registers.
//
// A warp takes 32 positions a step from its own cp.async ring: S = Q K^T, then
// O^T += V^T P^T. Two forms of a tile of rows (heads x new tokens of one KV
// head): Wide, 8 rows, and Narrow, 4 rows, which a single token of a group of
// up to 4 heads takes, and where hi and lo parts share an instruction's
// columns (64 sequences of 4095 .. 32768 positions, 4 KV heads of 4 heads each:
// 178 us; with the same inputs in a row, partly from L2, 166, and 219 in Wide,
// half of its rows empty).
//
// The steps of all (row tile, KV head) pairs are cut into equal shares, one
// per CTA, two CTAs per SM, so that ragged lengths and one long sequence load
// every SM alike. When there are no more pairs than CTAs, each pair gets CTAs
// of its own, unless that leaves some CTA with 28 steps more than its share:
// a CTA with parts of two pairs pays a part's latencies twice (32 sequences of
// 129 .. 4096 positions, window 2047: 18.5 us, as one list 27.4; 16 of 4095 ..
// 32768, two tokens on 8 KV heads of 4 heads: 3 us more than as one list, of
// 115). A pair's parts
// meet in the workspace, where the last CTA to arrive adds them in the
// order of their keys, so results repeat bit for bit.
//
// What bounds it: with long contexts, the step's some 700 instructions (half
// of them turn nibbles into fp16) in 16 warps per SM at 128 registers, each of
// which runs QK, softmax and PV one after the other. 144 bytes per position and
// KV head (head_dim 128) would be 105 us of HBM time for the 679 MB of 64
// sequences; it takes 178, with issue 64% active, ALU 56%, matrix unit 24%, DRAM 3.8
// TB/s: no unit is at its limit, there is too little independent work. With
// little work per CTA, the chain of latencies: lengths, page numbers, keys, the
// warps' meeting, the parts' meeting (33 us for one sequence of 131,069, 11.7 us
// of HBM time; 7 us for one of 37). With the rows of a whole prompt, many short
// parts: shares count steps, so the CTA with a prompt's first rows gets some 200
// parts of 1 to 4 steps (2048 rows over 2048 positions 1038 us, over 8192 1287).
#include <algorithm>
#include <cmath>

#include <cuda_fp16.h>

#include "kv4.cuh"

namespace b2 {
namespace {

constexpr unsigned kWarps = 8;           // warps per CTA
constexpr unsigned kStep = 32;           // positions per warp step
constexpr unsigned kRows = 8;            // query rows per tile, at most
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
    unsigned tiles;                     // row tiles per sequence: ceil(max_queries * group / ROWS)
    float scale, q_sign;                // |scale| (1 for scale 0); the scale's sign, 0 for scale 0
    unsigned window, sinks;
    unsigned* counters;                 // [kMaxGrid], zero between calls
    float* part_ml;                     // [2 kMaxGrid][8][2]: reference, sum
    float* part_o;                      // [2 kMaxGrid][8][D]
    Kv4View cache;
};

// One row tile of one sequence: 4 or 8 of its (query, head in group) rows.
struct Tile {
    unsigned first_row;   // row of q of the sequence's first query
    unsigned queries, len;
    unsigned flat;        // first flat index query * group + head
    unsigned rows;        // rows in the tile
    int p_min, p_max;     // positions of its first and last row
    unsigned sinks, low;  // visible: [0, sinks) and [low, p_max]
    unsigned total;       // number of visible keys
    unsigned clear_from, clear_to;  // of these, the ones that every row sees
};

template <unsigned D>
struct Shape {
    static constexpr unsigned groups = D / kKv4Group;
    static constexpr unsigned stages = D == 128 ? 2 : 4;
    static constexpr unsigned codes = kStep * D / 2;          // bytes of a step's K (V) codes
    static constexpr unsigned params = kStep * 4 * groups;
    static constexpr unsigned stage = 2 * (codes + params);
};

template <unsigned D>
struct Smem {
    alignas(128) unsigned char ring[kWarps][Shape<D>::stages * Shape<D>::stage];  // also a warp's O at a segment's end
    alignas(16) __half q[D / 16][32][8];              // operands of QK: k-step, lane (4 halves used by Narrow)
    float q_sum[kRows][2];                            // sum of the scaled q per group
    float q_scale[kRows];                             // base-2 score per unit of product with the scaled q
    unsigned valid[kWarps][Shape<D>::stages];         // positions of the step that exist
    float ref[kWarps][kRows], sum[kWarps][kRows], mean[kWarps][kRows][2];
    float row_sum[kRows];
    unsigned pair_units[kPairCache];
    unsigned scan[kWarps], fits[kWarps], found_pair, found_before, last;
};

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint4& a, unsigned b0, unsigned b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

// The first of a chain: c = a b.
__device__ __forceinline__ void mma_f16_first(float (&c)[4], const uint4& a, unsigned b0, unsigned b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ void mma_bf16_first(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3,
                                               unsigned b0, unsigned b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// The 8 x 8 matrix of 16-bit values that lanes hold as row lane / 4, columns 2 (lane % 4), + 1, transposed.
__device__ __forceinline__ unsigned transpose_f16(unsigned v) {
    unsigned d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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

__device__ __forceinline__ unsigned half_pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ float2 half_unpack(unsigned w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// The tile `index` of sequence `seq`; total = 0 if it sees nothing, rows = 0
// if it does not exist. `report`: flag what is out of range.
template <unsigned ROWS>
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
    t.flat = index * ROWS;
    const unsigned all = t.queries * a.group;
    t.rows = t.flat < all ? min(ROWS, all - t.flat) : 0u;
    if (t.rows == 0) return t;
    const int base = static_cast<int>(t.len) - static_cast<int>(t.queries);
    t.p_min = base + static_cast<int>(t.flat / a.group);
    t.p_max = base + static_cast<int>((t.flat + t.rows - 1) / a.group);
    if (t.len == 0 || t.p_max < 0) return t;
    const int low = a.window ? t.p_min - static_cast<int>(a.window) + 1 : 0;
    t.low = low > 0 ? static_cast<unsigned>(low) : 0u;
    t.sinks = min(a.sinks, t.low);
    t.total = t.sinks + static_cast<unsigned>(t.p_max) + 1 - t.low;
    const int behind = t.p_max - static_cast<int>(a.window) + 1 - static_cast<int>(t.low);
    t.clear_from = a.window ? t.sinks + (behind > 0 ? static_cast<unsigned>(behind) : 0u) : 0u;
    t.clear_to = t.p_min < 0 ? 0u : t.sinks + static_cast<unsigned>(t.p_min) + 1 - t.low;
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

// Place of 16-byte chunk `part` of key tok's V row in a stage: swizzled inside
// 128-byte lines, so that the 4 bytes that each of 8 x 4 lanes reads of 4
// keys' rows hit all banks.
template <unsigned D>
__device__ __forceinline__ unsigned v_offset(unsigned tok, unsigned part) {
    const unsigned line = tok * (D / 2) / 128, at = tok * (D / 2) / 16 % 8 + part;
    return line * 128 + ((at ^ ((D == 128 ? line & 3u : line & 1u) << 1)) << 4);
}

// What a warp needs to bring a pair's steps into its ring.
template <unsigned D>
struct Feed {
    using S = Shape<D>;
    static constexpr unsigned PARTS = D / 32;  // 16-byte chunks of a row of codes = copies per lane
    static constexpr unsigned P = 4 * S::groups;
    const std::uint8_t* head;     // the KV head's block of page 0
    const std::uint32_t* table;   // the sequence's pages
    unsigned lane, v_at;          // v_at: place of the lane's first V chunk in a stage
    unsigned sinks, skip, total;  // key u is position u, past the sinks u + skip

    __device__ __forceinline__ void init(const AttnKv4Args& a, const Tile& t, unsigned seq, unsigned h, unsigned lane_) {
        head = a.cache.data + h * a.cache.head_stride;
        table = a.cache.table + static_cast<std::size_t>(seq) * a.cache.max_pages;
        lane = lane_;
        // keys lane / PARTS + i * (32 / PARTS): whole swizzle periods apart
        v_at = S::codes + v_offset<D>(lane / PARTS, lane % PARTS);
        sinks = t.sinks;
        skip = t.low - t.sinks;
        total = t.total;
    }
    __device__ __forceinline__ unsigned position(unsigned u) const { return u < sinks ? u : u + skip; }
    // Whether the step from key u0 is 32 neighbours of one page.
    __device__ __forceinline__ bool one_page(const AttnKv4Args& a, unsigned u0) const {
        const unsigned slots = (1u << a.cache.page_shift) - 1u;
        return u0 + kStep <= total && (u0 >= sinks || u0 + kStep <= sinks) && (position(u0) & slots) + kStep - 1 <= slots;
    }
    // The page of this lane's key of the step from u0 (the same for all lanes
    // of a one-page step); kKv4Padding where there is none. The length check
    // keeps positions inside the table.
    __device__ __forceinline__ unsigned page(const AttnKv4Args& a, unsigned u0) const {
        const unsigned u = u0 + lane;
        unsigned pg = kKv4Padding;
        if (u < total) {
            pg = __ldg(table + (position(u) >> a.cache.page_shift));
            if (pg >= a.cache.pages) {
                flag_check(B2_CHECK_KV4);
                pg = kKv4Padding;
            }
        }
        return pg;
    }
    // Issues the copies of the step from u0 into `stage`; pg: page(u0).
    __device__ __forceinline__ void copy(const AttnKv4Args& a, unsigned u0, unsigned pg, unsigned stage,
                                         unsigned* valid) const {
        const unsigned shift = a.cache.page_shift, slots = (1u << shift) - 1u;
        if (one_page(a, u0) && __any_sync(0xffffffffu, pg != kKv4Padding)) {  // four runs of memory
            if (lane == 0) *valid = 0xFFFFFFFFu;
            const unsigned slot = position(u0) & slots;
            const std::uint8_t* block = head + static_cast<unsigned long long>(pg) * a.cache.page_stride;
            const std::uint8_t* codes = block + (slot * (D / 2) + lane * 16);
            const std::uint8_t* v_codes = codes + kv4_v_codes<D>(shift);
            const unsigned k_dst = stage + lane * 16, v_dst = stage + v_at;
#pragma unroll
            for (unsigned i = 0; i < PARTS; ++i) {
                copy_async16(k_dst + i * 512, codes + i * 512);
                copy_async16(v_dst + i * 512, v_codes + i * 512);
            }
            const std::uint8_t* params = block + (kv4_k_params<D>(shift) + (slot + lane) * P);
            copy_async<P>(stage + 2 * S::codes + lane * P, params, true);
            copy_async<P>(stage + 2 * S::codes + S::params + lane * P, params + (P << shift), true);
            return;
        }
        const unsigned have = __ballot_sync(0xffffffffu, pg != kKv4Padding);
        if (lane == 0) *valid = have;
        const unsigned part = lane % PARTS;
#pragma unroll
        for (unsigned i = 0; i < PARTS; ++i) {
            const unsigned tok = i * (32 / PARTS) + lane / PARTS;
            const unsigned from = __shfl_sync(0xffffffffu, pg, tok);
            const bool ok = from != kKv4Padding;
            const unsigned slot = position(u0 + tok) & slots;
            const std::uint8_t* src = ok ? head + static_cast<unsigned long long>(from) * a.cache.page_stride +
                                               (slot * (D / 2) + part * 16)
                                         : a.cache.data;
            copy_async<16>(stage + tok * (D / 2) + part * 16, src, ok);
            copy_async<16>(stage + v_at + i * 512, ok ? src + kv4_v_codes<D>(shift) : src, ok);
        }
        const bool ok = pg != kKv4Padding;
        const unsigned slot = position(u0 + lane) & slots;
        const std::uint8_t* block = ok ? head + static_cast<unsigned long long>(pg) * a.cache.page_stride : a.cache.data;
        copy_async<P>(stage + 2 * S::codes + lane * P, block + (ok ? kv4_k_params<D>(shift) + slot * P : 0u), ok);
        copy_async<P>(stage + 2 * S::codes + S::params + lane * P, block + (ok ? kv4_v_params<D>(shift) + slot * P : 0u),
                      ok);
    }
};

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
__device__ __forceinline__ f32x2 sub2(f32x2 a, f32x2 b) {
    f32x2 d;
    asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ f32x2 both(float v) { return f2_pack(v, v); }

// (w & mask) | bits in one instruction.
__device__ __forceinline__ unsigned mask_or(unsigned w, unsigned mask, unsigned bits) {
    unsigned d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(w), "r"(mask), "r"(bits));
    return d;
}
// c - 8 of the low (SHIFTED: second) nibbles of both halves of w, in fp16: the
// conversion by fp16's exponent that Kim et al. published ("Who Says Elephants
// Can't Run", 2022), whose constants follow from the format.
template <bool SHIFTED>
__device__ __forceinline__ unsigned codes_f16(unsigned w) {
    unsigned d;
    if (SHIFTED)  // (1024 + 16 c) / 16 - 72
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(mask_or(w, 0x00F000F0u, 0x64006400u)), "r"(0x2C002C00u), "r"(0xD480D480u));
    else  // (1024 + c) - 1032
        asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(mask_or(w, 0x000F000Fu, 0x64006400u)), "r"(0xE408E408u));
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

// Columns first, first + 1 of a thread's O^T as rows of 128-bit stores.
template <unsigned PITCH, unsigned D>
__device__ __forceinline__ void put_columns(const f32x2 (&o)[Shape<D>::groups][4][2], float* warp_o, unsigned first,
                                            unsigned rows, unsigned r) {
#pragma unroll
    for (unsigned e = 0; e < 2; ++e)
        if (first + e < rows) {
            float* row = warp_o + (first + e) * PITCH + r * 8;
#pragma unroll
            for (unsigned g = 0; g < Shape<D>::groups; ++g) {
                float v[8];
#pragma unroll
                for (unsigned n = 0; n < 4; ++n) {
                    const float2 y0 = f2_unpack(o[g][n][0]), y1 = f2_unpack(o[g][n][1]);
                    v[n] = e ? y0.y : y0.x;
                    v[4 + n] = e ? y1.y : y1.x;
                }
                *reinterpret_cast<float4*>(row + g * 64) = make_float4(v[0], v[1], v[2], v[3]);
                *reinterpret_cast<float4*>(row + g * 64 + 4) = make_float4(v[4], v[5], v[6], v[7]);
            }
        }
}

// Position of the tile's row r; -1 past its rows.
__device__ __forceinline__ int row_position(const AttnKv4Args& a, const Tile& t, unsigned r) {
    return r < t.rows ? static_cast<int>(t.len) - static_cast<int>(t.queries) + static_cast<int>((t.flat + r) / a.group)
                      : -1;
}

// ---- a warp's steps ----------------------------------------------------------------
//
// Both kinds hold, for a step of 32 keys, the scores in fp32, p and p s, and
// O^T as accumulators of M = 16 dimensions x N = 8 columns: thread (r = lane /
// 4, c = lane % 4) has columns 2c and 2c + 1 of dimensions g * 64 + r * 8 +
// n (o[g][n][0]) and + 4 + n (o[g][n][1]), n < 4. Sums are parts that the
// end adds up: mean = sum p (m + 8 s) per group. m + 8 s, the middle of a
// key's range, is taken key by key: sums of p m and of p s alone are many times
// larger and cancel (over 32768 keys: error 3e-6 of the output, not 6e-7).

// The affine part of the scores, s (8 sum q) + m (sum q), is one product: the
// parameter words are (s, m) pairs in bf16 as they lie. (8 sum q, sum q) of
// group c % G in three bf16 parts: parts c / G (k = 2c) and 2 (k = 2c + 8).
template <unsigned G>
__device__ __forceinline__ void affine_operand(float q_sum, unsigned c, unsigned (&operand)[2]) {
    float a8 = 8.0f * q_sum, a1 = q_sum;
    unsigned p[3];
#pragma unroll
    for (unsigned i = 0; i < 3; ++i) {
        p[i] = bf16_pack(a8, a1);
        a8 -= bf16_low(p[i]);
        a1 -= bf16_high(p[i]);
    }
    operand[0] = c < G ? p[0] : c < 2 * G ? p[1] : 0u;
    operand[1] = c < G ? p[2] : 0u;
}

// What a step s < 2^(exponent - 126) asks of the reference above the score (in
// base 2): p s in [2^10, 2^11) there.
__device__ __forceinline__ float above_score(unsigned exponent) {
    return static_cast<float>(max(static_cast<int>(exponent) - 137, -71));
}
// What one key's parameters ask. A minimum counts as a step 2^80 below it, which
// keeps sums of p m over 2^28 keys in fp32 where steps are tiny or zero; what is
// not finite has no part in it.
template <unsigned G>
__device__ __forceinline__ float above_score_of(const unsigned* params) {
    int exponent = 0;
#pragma unroll
    for (unsigned g = 0; g < G; ++g) {
        const int s = params[g] >> 7 & 0xFFu, m = params[g] >> 23 & 0xFFu;
        if (s != 0xFF) exponent = max(exponent, s);
        if (m != 0xFF) exponent = max(exponent, m - 80);
    }
    return above_score(static_cast<unsigned>(exponent));
}
// Minima from here on may need that; below it p m is in range whatever the
// steps are (p < 2^75 at the least step that above_score counts).
constexpr float kLargeMinimum = 1048576.0f;
constexpr unsigned kLargeFlag = 0x8000u;  // beside a step's exponent
// The larger |m| of two parameter words: m is the word's high half, so the word
// is m but for its last bits.
__device__ __forceinline__ float larger_minimum(unsigned params0, unsigned params1) {
    return fmaxf(fabsf(__uint_as_float(params0)), fabsf(__uint_as_float(params1)));
}

__device__ __forceinline__ bool visible(const AttnKv4Args& a, unsigned valid, unsigned tok, int j, int pos) {
    return ((valid >> tok) & 1u) && j <= pos &&
           (a.window == 0 || pos - j < static_cast<int>(a.window) || j < static_cast<int>(a.sinks));
}

// Eight rows (5 new tokens of 4 heads on each of 4 KV heads, 12 sequences of
// 500 .. 4000: 27.1 us). Queries are the M = 16 operand of QK (hi parts in rows 0..7, lo
// in 8..15), so thread (r, c) gets the scores of row r and keys 8b + 2c, + 1,
// which is where the second product wants P^T (k = keys, n = rows).
template <unsigned D>
struct Wide {
    static constexpr unsigned ROWS = 8, G = Shape<D>::groups;
    using S = Shape<D>;
    unsigned lane, r, c, affine[2];
    float q_scale;
    int pos;
    float ref;
    f32x2 sum, mean[G];
    f32x2 o[G][4][2];

    __device__ __forceinline__ void init(const AttnKv4Args& a, const Tile& t, const Smem<D>& sm, unsigned lane_) {
        lane = lane_;
        r = lane / 4;
        c = lane % 4;
        q_scale = sm.q_scale[r];
        affine_operand<G>(sm.q_sum[r][c % G], c, affine);
        pos = row_position(a, t, r);
        ref = kNegInf;
        sum = 0;
#pragma unroll
        for (unsigned g = 0; g < G; ++g) {
            mean[g] = 0;
#pragma unroll
            for (unsigned n = 0; n < 4; ++n) o[g][n][0] = o[g][n][1] = 0;
        }
    }
    // Half `half` of pair (i, i + 4), i = 2 * (k-step % 2) + reg, of row `row`.
    static __device__ __forceinline__ void put_query(Smem<D>& sm, unsigned row, unsigned step, unsigned c, unsigned reg,
                                                     unsigned half, __half hi, __half lo) {
        __half* at = sm.q[step][row * 4 + c] + reg * 4 + half;
        at[0] = hi;
        at[2] = lo;
    }

    // clear: every row sees all of the keys.
    __device__ __forceinline__ void step(const AttnKv4Args& a, const Tile& t, const Smem<D>& sm, unsigned stage,
                                         unsigned u0, unsigned valid, bool clear) {
        // the step's largest s, and whether a minimum is large: a key per lane
        unsigned own[G];
        lds_n<G>(stage + 2 * S::codes + S::params + lane * 4 * G, own);
        const unsigned steps_top = __reduce_max_sync(
            0xffffffffu, ((G == 2 ? __vmaxu2(own[0], own[G - 1]) : own[0]) & 0x7F80u) |
                             (larger_minimum(own[0], own[G - 1]) >= kLargeMinimum ? kLargeFlag : 0u));
        // ---- scores: x[b] holds keys 8b + 2c and 8b + 2c + 1 of row r ----
        f32x2 x[4];
        {
#pragma unroll
            for (unsigned b = 0; b < 4; ++b) {
                unsigned w;
                lds_n<1>(stage + 2 * S::codes + (8 * b + r) * 4 * G + c % G * 4, &w);
                float y[4];
                mma_bf16_first(y, affine[0], 0u, affine[1], 0u, w, w);
                x[b] = f2_pack(y[0], y[1]);
            }
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
                for (unsigned k = 0; k < 4; ++k) {
                    const uint4 q = *reinterpret_cast<const uint4*>(sm.q[g * 4 + k][lane]);
#pragma unroll
                    for (unsigned b = 0; b < 4; ++b) {
                        const unsigned w = kw[b][g * 2 + k / 2] >> (k % 2 * 8);
                        if (k == 0) mma_f16_first(acc[b], q, codes_f16<false>(w), codes_f16<true>(w));
                        else mma_f16(acc[b], q, codes_f16<false>(w), codes_f16<true>(w));
                    }
                }
#pragma unroll
                for (unsigned b = 0; b < 4; ++b) {
                    const f32x2 dot = add2(f2_pack(acc[b][0], acc[b][1]), f2_pack(acc[b][2], acc[b][3]));
                    x[b] = f2_fma(f2_pack(bf16_low(kp[b][g]), bf16_low(kp[b][G + g])), dot, x[b]);
                }
            }
        }
        unsigned vp[4][2 * G];
#pragma unroll
        for (unsigned b = 0; b < 4; ++b) lds_n<2 * G>(stage + 2 * S::codes + S::params + (8 * b + 2 * c) * 4 * G, vp[b]);
        if (!clear) {
#pragma unroll
            for (unsigned b = 0; b < 4; ++b) {
                float2 y = f2_unpack(x[b]);
#pragma unroll
                for (unsigned e = 0; e < 2; ++e) {
                    const unsigned tok = 8 * b + 2 * c + e;
                    const int j = static_cast<int>(key_position(t, u0 + tok));
                    const bool seen = visible(a, valid, tok, j, pos);
                    if (!seen) (e ? y.y : y.x) = kNegInf;
                    // a value that is not finite reaches the rows that see it
                    // (through the mean's sum), and not the others (0 * NaN)
#pragma unroll
                    for (unsigned g = 0; g < G; ++g) {
                        unsigned& w = vp[b][e * G + g];
                        if (nonfinite_params(w)) {
                            w = 0;
                            if (seen) mean[g] = both(NAN);
                        }
                    }
                }
                x[b] = f2_pack(y.x, y.y);
            }
        }

        // ---- the reference: p s is to stay below 2^15 ----
        // A thread packs p s of its own keys only, so each tests its own, its top
        // score against the step's largest s first. Only where that may be too
        // much are keys taken one by one, each score with its own s -- a large s
        // of a key that the row does not see, or gives no weight, must not raise
        // the reference: the others' p s would sink below fp16 -- and exchanged.
        // (A key's parameters are taken apart by one lane and passed on: 12
        // sequences x 5 tokens 27.1 us; each thread with its own eight, 28.2.)
        float top = kNegInf;
#pragma unroll
        for (unsigned b = 0; b < 4; ++b) {
            const float2 y = f2_unpack(x[b]);
            top = fmaxf(top, fmaxf(y.x, y.y));
        }
        float need = fmaf(top, q_scale, above_score(steps_top >> 7 & 0xFFu));
        if (__any_sync(0xffffffffu, need > ref + 4.0f) || steps_top & kLargeFlag) {
            need = kNegInf;
            const float above = above_score_of<G>(own);
#pragma unroll
            for (unsigned b = 0; b < 4; ++b) {
                const float2 y = f2_unpack(x[b]);
                need = fmaxf(need, fmaf(y.x, q_scale, __shfl_sync(0xffffffffu, above, 8 * b + 2 * c)));
                need = fmaxf(need, fmaf(y.y, q_scale, __shfl_sync(0xffffffffu, above, 8 * b + 2 * c + 1)));
            }
            need = fmaxf(need, __shfl_xor_sync(0xffffffffu, need, 1));
            need = fmaxf(need, __shfl_xor_sync(0xffffffffu, need, 2));
            const float next = need > ref + 4.0f ? need : ref;
            const float alpha = next == ref ? 1.0f : exp2_approx(ref - next);
            ref = next;
            sum = mul2(sum, both(alpha));
            const f32x2 cols = f2_pack(__shfl_sync(0xffffffffu, alpha, 8 * c), __shfl_sync(0xffffffffu, alpha, 8 * c + 4));
#pragma unroll
            for (unsigned g = 0; g < G; ++g) {
                mean[g] = mul2(mean[g], both(alpha));
#pragma unroll
                for (unsigned n = 0; n < 4; ++n) {
                    o[g][n][0] = mul2(o[g][n][0], cols);
                    o[g][n][1] = mul2(o[g][n][1], cols);
                }
            }
        }
        const float at = ref == kNegInf ? 0.0f : ref;
        f32x2 steps[G][4];
#pragma unroll
        for (unsigned b = 0; b < 4; ++b) {
            const float2 y = f2_unpack(f2_fma(x[b], both(q_scale), both(-at)));
            x[b] = f2_pack(exp2_approx(y.x), exp2_approx(y.y));
            sum = add2(sum, x[b]);
#pragma unroll
            for (unsigned g = 0; g < G; ++g) {
                steps[g][b] = f2_pack(bf16_low(vp[b][g]), bf16_low(vp[b][G + g]));
                const f32x2 middle = f2_fma(steps[g][b], both(8.0f), f2_pack(bf16_high(vp[b][g]), bf16_high(vp[b][G + g])));
                mean[g] = f2_fma(x[b], middle, mean[g]);
            }
        }

        // ---- O^T += V^T (p s)^T ----
        const unsigned v_base = stage + S::codes + v_offset<D>(2 * c, r * G * 4 / 16) + r * G * 4 % 16;
        const unsigned v_next = stage + S::codes + v_offset<D>(2 * c + 1, r * G * 4 / 16) + r * G * 4 % 16;
        unsigned vw[8][G];  // the lane's octets of keys 8b + 2c and 8b + 2c + 1
#pragma unroll
        for (unsigned b = 0; b < 4; ++b) {
            lds_n<G>(v_base + 8 * b * (D / 2), vw[2 * b]);
            lds_n<G>(v_next + 8 * b * (D / 2), vw[2 * b + 1]);
        }
#pragma unroll
        for (unsigned g = 0; g < G; ++g) {
            unsigned hi[4], lo[4], xa[4], ya[4];
#pragma unroll
            for (unsigned b = 0; b < 4; ++b) {
                const unsigned w0 = vw[2 * b][g], w1 = vw[2 * b + 1][g];
                const f32x2 v = mul2(x[b], steps[g][b]);
                const float2 y = f2_unpack(v);
                hi[b] = half_pack(y.x, y.y);
                const float2 h = half_unpack(hi[b]);
                const float2 rest = f2_unpack(sub2(v, f2_pack(h.x, h.y)));
                lo[b] = half_pack(rest.x, rest.y);
                xa[b] = __byte_perm(w0, w1, 0x5410);
                ya[b] = __byte_perm(w0, w1, 0x7632);
            }
#pragma unroll
            for (unsigned n = 0; n < 4; ++n) {
                const unsigned sh = n / 2 * 8;
                float acc[4];
#pragma unroll
                for (unsigned h = 0; h < 2; ++h) {
                    const unsigned w[4] = {xa[2 * h] >> sh, ya[2 * h] >> sh, xa[2 * h + 1] >> sh, ya[2 * h + 1] >> sh};
                    const uint4 v = n % 2 ? make_uint4(codes_f16<true>(w[0]), codes_f16<true>(w[1]), codes_f16<true>(w[2]),
                                                       codes_f16<true>(w[3]))
                                          : make_uint4(codes_f16<false>(w[0]), codes_f16<false>(w[1]),
                                                       codes_f16<false>(w[2]), codes_f16<false>(w[3]));
                    if (h == 0) mma_f16_first(acc, v, hi[0], hi[1]);
                    else mma_f16(acc, v, hi[2], hi[3]);
                    mma_f16(acc, v, lo[2 * h], lo[2 * h + 1]);
                }
                o[g][n][0] = add2(o[g][n][0], f2_pack(acc[0], acc[1]));
                o[g][n][1] = add2(o[g][n][1], f2_pack(acc[2], acc[3]));
            }
        }
    }

    // The warp's sums into shared memory: references, sums and means now, O
    // (row pitch PITCH) once the rings are drained.
    __device__ __forceinline__ void put_sums(Smem<D>& sm, unsigned warp) {
        const auto total = [](f32x2 v) {
            const float2 y = f2_unpack(v);
            float x = y.x + y.y;
            x += __shfl_xor_sync(0xffffffffu, x, 1);
            return x + __shfl_xor_sync(0xffffffffu, x, 2);
        };
        const float l = total(sum);
        float m[G];
#pragma unroll
        for (unsigned g = 0; g < G; ++g) m[g] = total(mean[g]);
        if (c == 0) {
            sm.ref[warp][r] = ref;
            sm.sum[warp][r] = l;
#pragma unroll
            for (unsigned g = 0; g < G; ++g) sm.mean[warp][r][g] = m[g];
        }
    }
    template <unsigned PITCH>
    __device__ __forceinline__ void put_o(float* warp_o, unsigned rows) {
        put_columns<PITCH, D>(o, warp_o, 2 * c, rows, r);
    }
};

// Four rows (one token of a group of four heads): with eight columns each
// matrix instruction would be half empty, and these instructions are what a
// step costs most, so hi and lo parts share the columns: 34 of them instead
// of 68. Keys are the M = 16 operand of QK; columns n < 4 are the rows' hi
// parts, n >= 4 their lo parts, and the lanes of the two halves exchange, so
// that a thread ends with rows 2 (c & 1), + 1 of two keys: 16 (c >= 2) + 8 h +
// r. P s is split into hi and lo again, exchanged, and transposed by
// movmatrix into the operand of the second product.
template <unsigned D>
struct Narrow {
    static constexpr unsigned ROWS = 4, G = Shape<D>::groups;
    using S = Shape<D>;
    unsigned lane, r, c, affine[2];
    unsigned q[D / 16][2];
    f32x2 q_scale;
    int pos[2];
    f32x2 ref, sum, mean[G];
    f32x2 o[G][4][2];

    __device__ __forceinline__ void init(const AttnKv4Args& a, const Tile& t, const Smem<D>& sm, unsigned lane_) {
        lane = lane_;
        r = lane / 4;
        c = lane % 4;
        const unsigned row = 2 * (c & 1u);
        q_scale = f2_pack(sm.q_scale[row], sm.q_scale[row + 1]);
        affine_operand<G>(r < ROWS ? sm.q_sum[r][c % G] : 0.0f, c, affine);
        pos[0] = row_position(a, t, row);
        pos[1] = row_position(a, t, row + 1);
#pragma unroll
        for (unsigned k = 0; k < D / 16; ++k) {
            const uint2 v = *reinterpret_cast<const uint2*>(sm.q[k][lane]);
            q[k][0] = v.x;
            q[k][1] = v.y;
        }
        ref = both(kNegInf);
        sum = 0;
#pragma unroll
        for (unsigned g = 0; g < G; ++g) {
            mean[g] = 0;
#pragma unroll
            for (unsigned n = 0; n < 4; ++n) o[g][n][0] = o[g][n][1] = 0;
        }
    }
    static __device__ __forceinline__ void put_query(Smem<D>& sm, unsigned row, unsigned step, unsigned c, unsigned reg,
                                                     unsigned half, __half hi, __half lo) {
        sm.q[step][row * 4 + c][reg * 2 + half] = hi;
        sm.q[step][(row + ROWS) * 4 + c][reg * 2 + half] = lo;
    }

    __device__ __forceinline__ void step(const AttnKv4Args& a, const Tile& t, const Smem<D>&, unsigned stage, unsigned u0,
                                         unsigned valid, bool clear) {
        const bool upper = c & 2u;
        // ---- scores: y[k][h] is key 16k + 8h + r, columns 2c and 2c + 1 ----
        f32x2 y[2][2];
#pragma unroll
        for (unsigned k = 0; k < 2; ++k) {
            const unsigned tok = 16 * k + r, codes = stage + tok * (D / 2) + c * (D / 8);
            unsigned w0[2 * G], w1[2 * G], p0[G], p1[G];
            lds_n<2 * G>(codes, w0);
            lds_n<2 * G>(codes + 8 * (D / 2), w1);
            lds_n<G>(stage + 2 * S::codes + tok * 4 * G, p0);
            lds_n<G>(stage + 2 * S::codes + (tok + 8) * 4 * G, p1);
            {
                const unsigned a0 = G == 1 || !(c & 1u) ? p0[0] : p0[G - 1], a1 = G == 1 || !(c & 1u) ? p1[0] : p1[G - 1];
                float acc[4];
                mma_bf16_first(acc, a0, a1, a0, a1, affine[0], affine[1]);
                y[k][0] = f2_pack(acc[0], acc[1]);
                y[k][1] = f2_pack(acc[2], acc[3]);
            }
#pragma unroll
            for (unsigned g = 0; g < G; ++g) {
                float acc[4];
#pragma unroll
                for (unsigned i = 0; i < 4; ++i) {
                    const unsigned x0 = w0[g * 2 + i / 2] >> (i % 2 * 8), x1 = w1[g * 2 + i / 2] >> (i % 2 * 8);
                    const uint4 v = make_uint4(codes_f16<false>(x0), codes_f16<false>(x1), codes_f16<true>(x0),
                                               codes_f16<true>(x1));
                    if (i == 0) mma_f16_first(acc, v, q[g * 4][0], q[g * 4][1]);
                    else mma_f16(acc, v, q[g * 4 + i][0], q[g * 4 + i][1]);
                }
                y[k][0] = f2_fma(both(bf16_low(p0[g])), f2_pack(acc[0], acc[1]), y[k][0]);
                y[k][1] = f2_fma(both(bf16_low(p1[g])), f2_pack(acc[2], acc[3]), y[k][1]);
            }
        }
        // hi + lo: the lower lanes keep keys 0..15, the upper ones 16..31
        f32x2 x[2];
        unsigned vp[2][G];
        const unsigned first = (upper ? 16u : 0u) + r;
#pragma unroll
        for (unsigned h = 0; h < 2; ++h) {
            const float2 give = f2_unpack(upper ? y[0][h] : y[1][h]);
            x[h] = add2(upper ? y[1][h] : y[0][h], f2_pack(__shfl_xor_sync(0xffffffffu, give.x, 2),
                                                           __shfl_xor_sync(0xffffffffu, give.y, 2)));
            lds_n<G>(stage + 2 * S::codes + S::params + (first + 8 * h) * 4 * G, vp[h]);
        }
        if (!clear) {
#pragma unroll
            for (unsigned h = 0; h < 2; ++h) {
                const unsigned tok = first + 8 * h;
                const int j = static_cast<int>(key_position(t, u0 + tok));
                const bool seen0 = visible(a, valid, tok, j, pos[0]), seen1 = visible(a, valid, tok, j, pos[1]);
                const float2 v = f2_unpack(x[h]);
                x[h] = f2_pack(seen0 ? v.x : kNegInf, seen1 ? v.y : kNegInf);
                // a value that is not finite reaches the rows that see it
                // (through the mean's sum), and not the others (0 * NaN)
#pragma unroll
                for (unsigned g = 0; g < G; ++g)
                    if (nonfinite_params(vp[h][g])) {
                        vp[h][g] = 0;
                        mean[g] = add2(mean[g], f2_pack(seen0 ? NAN : 0.0f, seen1 ? NAN : 0.0f));
                    }
            }
        }

        // ---- the references: p s is to stay below 2^15 (as in Wide) ----
        {
            const float2 x0 = f2_unpack(x[0]), x1 = f2_unpack(x[1]), scale = f2_unpack(q_scale), old = f2_unpack(ref);
            const float top0 = fmaxf(x0.x, x1.x), top1 = fmaxf(x0.y, x1.y);
            unsigned top_w = __vmaxu2(vp[0][0], vp[1][0]);  // maxima of both halves: s is the lower
            if (G == 2) top_w = __vmaxu2(top_w, __vmaxu2(vp[0][G - 1], vp[1][G - 1]));
            const float above = above_score(top_w >> 7 & 0xFFu);
            const float top_m = fmaxf(larger_minimum(vp[0][0], vp[1][0]), larger_minimum(vp[0][G - 1], vp[1][G - 1]));
            float need0 = fmaf(top0, scale.x, above), need1 = fmaf(top1, scale.y, above);
            if (__any_sync(0xffffffffu, need0 > old.x + 4.0f || need1 > old.y + 4.0f || top_m >= kLargeMinimum)) {
                const float above0 = above_score_of<G>(vp[0]), above1 = above_score_of<G>(vp[1]);
                need0 = fmaxf(fmaf(x0.x, scale.x, above0), fmaf(x1.x, scale.x, above1));
                need1 = fmaxf(fmaf(x0.y, scale.y, above0), fmaf(x1.y, scale.y, above1));
#pragma unroll
                for (unsigned i = 2; i < 32; i *= 2) {
                    need0 = fmaxf(need0, __shfl_xor_sync(0xffffffffu, need0, i));
                    need1 = fmaxf(need1, __shfl_xor_sync(0xffffffffu, need1, i));
                }
                const float ref0 = need0 > old.x + 4.0f ? need0 : old.x, ref1 = need1 > old.y + 4.0f ? need1 : old.y;
                const f32x2 alpha = f2_pack(ref0 == old.x ? 1.0f : exp2_approx(old.x - ref0),
                                            ref1 == old.y ? 1.0f : exp2_approx(old.y - ref1));
                ref = f2_pack(ref0, ref1);
                sum = mul2(sum, alpha);
#pragma unroll
                for (unsigned g = 0; g < G; ++g) {
                    mean[g] = mul2(mean[g], alpha);
#pragma unroll
                    for (unsigned n = 0; n < 4; ++n) {
                        o[g][n][0] = mul2(o[g][n][0], alpha);
                        o[g][n][1] = mul2(o[g][n][1], alpha);
                    }
                }
            }
        }
        {
            const float2 at = f2_unpack(ref);
            const f32x2 minus = f2_pack(at.x == kNegInf ? 0.0f : -at.x, at.y == kNegInf ? 0.0f : -at.y);
#pragma unroll
            for (unsigned h = 0; h < 2; ++h) {
                const float2 v = f2_unpack(f2_fma(x[h], q_scale, minus));
                x[h] = f2_pack(exp2_approx(v.x), exp2_approx(v.y));
                sum = add2(sum, x[h]);
            }
        }

        // ---- O^T += V^T (p s)^T ----
        const unsigned v_base = stage + S::codes + v_offset<D>(2 * c, r * G * 4 / 16) + r * G * 4 % 16;
        const unsigned v_next = stage + S::codes + v_offset<D>(2 * c + 1, r * G * 4 / 16) + r * G * 4 % 16;
        unsigned vw[8][G];  // the lane's octets of keys 8b + 2c and 8b + 2c + 1
#pragma unroll
        for (unsigned b = 0; b < 4; ++b) {
            lds_n<G>(v_base + 8 * b * (D / 2), vw[2 * b]);
            lds_n<G>(v_next + 8 * b * (D / 2), vw[2 * b + 1]);
        }
#pragma unroll
        for (unsigned g = 0; g < G; ++g) {
            unsigned b[2][2];  // keys 16k + 8h + 2c, + 1 of column r
#pragma unroll
            for (unsigned h = 0; h < 2; ++h) {
                const float s = bf16_low(vp[h][g]);
                const f32x2 v = mul2(x[h], both(s));
                mean[g] = f2_fma(x[h], both(fmaf(8.0f, s, bf16_high(vp[h][g]))), mean[g]);
                const float2 f = f2_unpack(v);
                const unsigned hi = half_pack(f.x, f.y);
                const float2 up = half_unpack(hi);
                const float2 rest = f2_unpack(sub2(v, f2_pack(up.x, up.y)));
                const unsigned lo = half_pack(rest.x, rest.y);
                const unsigned got = __shfl_xor_sync(0xffffffffu, upper ? hi : lo, 2);
                b[0][h] = transpose_f16(upper ? got : hi);
                b[1][h] = transpose_f16(upper ? lo : got);
            }
            unsigned xa[4], ya[4];
#pragma unroll
            for (unsigned i = 0; i < 4; ++i) {
                xa[i] = __byte_perm(vw[2 * i][g], vw[2 * i + 1][g], 0x5410);
                ya[i] = __byte_perm(vw[2 * i][g], vw[2 * i + 1][g], 0x7632);
            }
#pragma unroll
            for (unsigned n = 0; n < 4; ++n) {
                const unsigned sh = n / 2 * 8;
                float acc[4];
#pragma unroll
                for (unsigned k = 0; k < 2; ++k) {
                    const unsigned w[4] = {xa[2 * k] >> sh, ya[2 * k] >> sh, xa[2 * k + 1] >> sh, ya[2 * k + 1] >> sh};
                    const uint4 v = n % 2 ? make_uint4(codes_f16<true>(w[0]), codes_f16<true>(w[1]), codes_f16<true>(w[2]),
                                                       codes_f16<true>(w[3]))
                                          : make_uint4(codes_f16<false>(w[0]), codes_f16<false>(w[1]),
                                                       codes_f16<false>(w[2]), codes_f16<false>(w[3]));
                    if (k == 0) mma_f16_first(acc, v, b[0][0], b[0][1]);
                    else mma_f16(acc, v, b[1][0], b[1][1]);
                }
                o[g][n][0] = add2(o[g][n][0], f2_pack(acc[0], acc[1]));
                o[g][n][1] = add2(o[g][n][1], f2_pack(acc[2], acc[3]));
            }
        }
    }

    __device__ __forceinline__ void put_sums(Smem<D>& sm, unsigned warp) {
        const auto total = [](f32x2 v) {
            float2 y = f2_unpack(v);
#pragma unroll
            for (unsigned i = 2; i < 32; i *= 2) {
                y.x += __shfl_xor_sync(0xffffffffu, y.x, i);
                y.y += __shfl_xor_sync(0xffffffffu, y.y, i);
            }
            return y;
        };
        const float2 l = total(sum), at = f2_unpack(ref);
        const unsigned row = 2 * (c & 1u);
        const bool writes = r == 0 && c < 2;
        if (writes) {
            sm.ref[warp][row] = at.x;
            sm.ref[warp][row + 1] = at.y;
            sm.sum[warp][row] = l.x;
            sm.sum[warp][row + 1] = l.y;
        }
#pragma unroll
        for (unsigned g = 0; g < G; ++g) {
            const float2 m = total(mean[g]);
            if (writes) {
                sm.mean[warp][row][g] = m.x;
                sm.mean[warp][row + 1][g] = m.y;
            }
        }
#pragma unroll
        for (unsigned g = 0; g < G; ++g)
#pragma unroll
            for (unsigned n = 0; n < 4; ++n)
#pragma unroll
                for (unsigned i = 0; i < 2; ++i) {  // hi + lo
                    const float2 v = f2_unpack(o[g][n][i]);
                    o[g][n][i] = add2(o[g][n][i], f2_pack(__shfl_xor_sync(0xffffffffu, v.x, 2),
                                                          __shfl_xor_sync(0xffffffffu, v.y, 2)));
                }
    }
    template <unsigned PITCH>
    __device__ __forceinline__ void put_o(float* warp_o, unsigned rows) {
        if (c < 2) put_columns<PITCH, D>(o, warp_o, 2 * c, rows, r);
    }
};

// The tile's queries as operands of QK, each row scaled by a power of two to
// about 2^9 at most and split into two fp16 parts. Warp w takes row w: lane's
// dimensions are lane, lane + 32, ...
template <typename T, unsigned D, unsigned ROWS>
__device__ __forceinline__ void fetch_query(const AttnKv4Args& a, const Tile& t, unsigned head, float (&v)[D / 32]) {
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x / 32;
#pragma unroll
    for (unsigned e = 0; e < D / 32; ++e) v[e] = 0.0f;
    if (warp >= t.rows) return;
    const unsigned f = t.flat + warp;
    const T* q = static_cast<const T*>(a.q) + row_of(a, t, f) * a.q_row + (head * a.group + f % a.group) * a.q_head;
#pragma unroll
    for (unsigned e = 0; e < D / 32; ++e) v[e] = as_float(q[lane + 32 * e]) * a.q_sign;
}
template <unsigned D, typename Rows>
__device__ __forceinline__ void place_query(const AttnKv4Args& a, const float (&v)[D / 32], Smem<D>& sm) {
    constexpr unsigned G = Shape<D>::groups;
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    if (warp >= Rows::ROWS) return;
    float top = 0.0f, sum[G];
#pragma unroll
    for (unsigned e = 0; e < D / 32; ++e) top = fmaxf(top, fabsf(v[e]));
    top = warp_max(top);
    // 2^e with top * 2^e in [2^9, 2^10)
    int e = 136 - static_cast<int>(__float_as_uint(top) >> 23);
    e = top == 0.0f ? 0 : max(-118, min(e, 100));
    const float up = __uint_as_float(static_cast<unsigned>(127 + e) << 23);
    // sums of scaled queries, and the scale back before log2(e): neither passes an end of fp32 on the way
#pragma unroll
    for (unsigned g = 0; g < G; ++g) sum[g] = warp_sum(v[2 * g] * up + v[2 * g + 1] * up);
    if (lane == 0) {
        const float down = a.scale * __uint_as_float(static_cast<unsigned>(127 - e) << 23);
        // positive, so that a masked score stays -inf
        sm.q_scale[warp] = fmaxf(down * 1.4426950408889634f, 1.17549435e-38f);
#pragma unroll
        for (unsigned g = 0; g < G; ++g) sm.q_sum[warp][g] = sum[g];
    }
    // dimension d = w * 32 + c * 8 + i: nibble i of word w of lane (row, c)
#pragma unroll
    for (unsigned k = 0; k < D / 32; ++k) {
        const unsigned c = lane / 8, i = lane % 8;
        const float x = v[k] * up;
        const __half hi = __float2half_rn(x);
        const __half lo = __float2half_rn(x - __half2float(hi));
        Rows::put_query(sm, warp, k * 2 + (i % 4) / 2, c, i % 2, i / 4, hi, lo);
    }
}

template <typename T>
__device__ __forceinline__ void store_out(T* p, float y) {
    if constexpr (sizeof(T) == 2) *p = __float2bfloat16_rn(y);
    else *p = y;
}

// Adds up the parts of a pair that CTAs first .. first + n - 1 hold, in this
// order, and writes its rows.
template <typename T, unsigned D>
__device__ __forceinline__ void join_parts(const AttnKv4Args& a, const Tile& t, unsigned head, unsigned first, unsigned n,
                                           Smem<D>& sm) {
    constexpr unsigned FEW = 4;
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const auto slot = [&](unsigned i) { return static_cast<std::size_t>(2) * (first + i) + (i == 0 ? 1u : 0u); };
    const float4* parts = reinterpret_cast<const float4*>(a.part_o);
    const float2* refs = reinterpret_cast<const float2*>(a.part_ml);
    const auto write = [&](unsigned row, unsigned d4, const float4& s, float l) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const unsigned f = t.flat + row;
        T* out = static_cast<T*>(a.out) + (row_of(a, t, f) * a.q_heads + head * a.group + f % a.group) * D + d4 * 4;
        // a row without keys has s = 0 and l = 0
        store_out(out, s.x * inv);
        store_out(out + 1, s.y * inv);
        store_out(out + 2, s.z * inv);
        store_out(out + 3, s.w * inv);
    };
    const auto add = [](float4& s, float w, const float4& v) {
        s.x = fmaf(w, v.x, s.x); s.y = fmaf(w, v.y, s.y); s.z = fmaf(w, v.z, s.z); s.w = fmaf(w, v.w, s.w);
    };
    if (n <= FEW) {  // everything in flight at once
        for (unsigned i = threadIdx.x; i < t.rows * (D / 4); i += kWarps * 32) {
            const unsigned row = i / (D / 4), d4 = i % (D / 4);
            float2 ml[FEW];
            float4 v[FEW];
#pragma unroll
            for (unsigned k = 0; k < FEW; ++k)
                if (k < n) {
                    ml[k] = __ldcg(refs + slot(k) * kRows + row);
                    v[k] = __ldcg(parts + (slot(k) * kRows + row) * (D / 4) + d4);
                } else {
                    ml[k] = make_float2(kNegInf, 0.0f);
                    v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
            float m = kNegInf, l = 0.0f;
#pragma unroll
            for (unsigned k = 0; k < FEW; ++k) m = fmaxf(m, ml[k].x);
            float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (unsigned k = 0; k < FEW; ++k) {
                const float w = ml[k].x == kNegInf ? 0.0f : exp2_approx(ml[k].x - m);
                l = fmaf(w, ml[k].y, l);
                if (w != 0.0f) add(s, w, v[k]);
            }
            write(row, d4, s, l);
        }
        return;
    }
    // References and sums first, then all parts' sums, cut among the threads
    // that a row's outputs leave idle, each cut added in order.
    float2* factor = reinterpret_cast<float2*>(sm.ring);  // [rows][n]
    if (warp < t.rows) {
        float2* mine = factor + warp * n;
        float m = kNegInf, l = 0.0f;
        for (unsigned i = lane; i < n; i += 32) {
            const float2 v = __ldcg(refs + slot(i) * kRows + warp);
            mine[i] = v;
            m = fmaxf(m, v.x);
        }
        m = warp_max(m);
        for (unsigned i = lane; i < n; i += 32) {
            const float w = mine[i].x == kNegInf ? 0.0f : exp2_approx(mine[i].x - m);
            l = fmaf(w, mine[i].y, l);
            mine[i].x = w;
        }
        l = warp_sum(l);
        if (lane == 0) sm.row_sum[warp] = l;
    }
    __syncthreads();
    const unsigned outputs = t.rows * (D / 4);
    const unsigned cuts = max(1u, min(kWarps * 32 / outputs, 8u)), per = (n + cuts - 1) / cuts;
    float4* sums = reinterpret_cast<float4*>(sm.ring) + kRows * kMaxGrid / 2;  // [cuts][outputs]
    for (unsigned i = threadIdx.x; i < outputs * cuts; i += kWarps * 32) {
        const unsigned cut = i / outputs, o = i % outputs, row = o / (D / 4), d4 = o % (D / 4);
        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const unsigned end = min(n, (cut + 1) * per);
#pragma unroll 10
        for (unsigned k = cut * per; k < end; ++k) {
            const float4 v = __ldcg(parts + (slot(k) * kRows + row) * (D / 4) + d4);
            const float w = factor[row * n + k].x;
            if (w != 0.0f) add(s, w, v);
        }
        sums[cut * outputs + o] = s;
    }
    __syncthreads();
    for (unsigned o = threadIdx.x; o < outputs; o += kWarps * 32) {
        float4 s = sums[o];
        for (unsigned cut = 1; cut < cuts; ++cut) add(s, 1.0f, sums[cut * outputs + o]);
        write(o / (D / 4), o % (D / 4), s, sm.row_sum[o / (D / 4)]);
    }
}

// Units [from, to) of the pair (tile t of sequence seq, head): this CTA's
// part. whole: they are all of it.
template <typename T, unsigned D, typename Rows>
__device__ __forceinline__ void run_segment(const AttnKv4Args& a, const Tile& t, unsigned seq, unsigned head,
                                            unsigned from, unsigned to, bool whole, std::size_t slot, Smem<D>& sm) {
    using S = Shape<D>;
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x / 32;

    const unsigned steps = to - from > warp ? (to - from - warp + kWarps - 1) / kWarps : 0u;
    const auto key_of = [&](unsigned i) { return (from + warp + i * kWarps) * kStep; };
    const unsigned ring = smem_addr(sm.ring[warp]);
    // page numbers, then queries, then keys: each latency starts as early as it can
    Feed<D> feed;
    feed.init(a, t, seq, head, lane);
    unsigned pages[S::stages], next_page = kKv4Padding;
#pragma unroll
    for (unsigned i = 0; i < S::stages; ++i) pages[i] = i < steps ? feed.page(a, key_of(i)) : kKv4Padding;
    float query[D / 32];
    fetch_query<T, D, Rows::ROWS>(a, t, head, query);
#pragma unroll
    for (unsigned i = 0; i < S::stages; ++i) {
        if (i < steps) feed.copy(a, key_of(i), pages[i], ring + i * S::stage, &sm.valid[warp][i]);
        cp_async_commit();
    }
    if (S::stages < steps) next_page = feed.page(a, key_of(S::stages));
    place_query<D, Rows>(a, query, sm);
    __syncthreads();  // queries

    Rows rows;
    rows.init(a, t, sm, lane);
    for (unsigned i = 0; i < steps; ++i) {
        cp_async_wait<S::stages - 1>();
        __syncwarp();
        const unsigned u0 = key_of(i), at = i % S::stages, stage = ring + at * S::stage;
        const unsigned valid = sm.valid[warp][at];
        const bool clear = valid == 0xFFFFFFFFu && u0 >= t.clear_from && u0 + kStep <= t.clear_to;
        rows.step(a, t, sm, stage, u0, valid, clear);
        __syncwarp();
        if (i + S::stages < steps) {
            feed.copy(a, key_of(i + S::stages), next_page, stage, &sm.valid[warp][at]);
            if (i + S::stages + 1 < steps) next_page = feed.page(a, key_of(i + S::stages + 1));
        }
        cp_async_commit();
    }
    cp_async_wait<0>();

    // ---- the warps' sums meet ----
    const unsigned used = min(to - from, kWarps);  // warps that had a step
    constexpr unsigned PITCH = D + 4;
    float* o = reinterpret_cast<float*>(sm.ring[0]);
    static_assert(kRows * PITCH * sizeof(float) <= sizeof(sm.ring[0]), "a warp's O fits its own ring");
    if (warp < used) {
        rows.put_sums(sm, warp);
        __syncwarp();
        // the warp's ring is drained: it becomes its O
        rows.template put_o<PITCH>(reinterpret_cast<float*>(sm.ring[warp]), t.rows);
    }
    __syncthreads();
    constexpr unsigned APART = sizeof(sm.ring[0]) / sizeof(float);
    for (unsigned i = threadIdx.x; i < t.rows * (D / 4); i += kWarps * 32) {
        const unsigned row = i / (D / 4), d = i % (D / 4) * 4;
        float m = kNegInf, l = 0.0f;
        for (unsigned w = 0; w < used; ++w) m = fmaxf(m, sm.ref[w][row]);
        float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (unsigned w = 0; w < used; ++w) {
            const float ref = sm.ref[w][row];
            const float f = ref == kNegInf ? 0.0f : exp2_approx(ref - m);
            const float4 v = *reinterpret_cast<const float4*>(o + w * APART + row * PITCH + d);
            const float mean = sm.mean[w][row][d / kKv4Group];
            l = fmaf(f, sm.sum[w][row], l);
            y.x = fmaf(f, v.x + mean, y.x);
            y.y = fmaf(f, v.y + mean, y.y);
            y.z = fmaf(f, v.z + mean, y.z);
            y.w = fmaf(f, v.w + mean, y.w);
        }
        if (whole) {
            const unsigned f = t.flat + row;
            T* out = static_cast<T*>(a.out) + (row_of(a, t, f) * a.q_heads + head * a.group + f % a.group) * D + d;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no keys: y = 0 too
            store_out(out, y.x * inv);
            store_out(out + 1, y.y * inv);
            store_out(out + 2, y.z * inv);
            store_out(out + 3, y.w * inv);
        } else {
            __stcg(reinterpret_cast<float4*>(a.part_o + (slot * kRows + row) * D + d), y);
            if (d == 0) __stcg(reinterpret_cast<float2*>(a.part_ml) + slot * kRows + row, make_float2(m, l));
        }
    }
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
template <typename T, unsigned D, unsigned ROWS>
__device__ __forceinline__ void write_blank_rows(const AttnKv4Args& a, unsigned p0) {
    const unsigned heads = a.cache.kv_heads, pairs = a.cache.seqs * a.tiles;
    const unsigned end = min(pairs, p0 + kPairCache);
    for (unsigned p = p0 + (blockIdx.x + gridDim.x - p0 % gridDim.x) % gridDim.x; p < end; p += gridDim.x) {
        const Tile t = make_tile<ROWS>(a, p / a.tiles, p % a.tiles, false);
        if (t.total != 0) continue;
        for (unsigned i = threadIdx.x; i < t.rows * heads * D; i += kWarps * 32) {
            const unsigned f = t.flat + i / D / heads, h = i / D % heads;
            store_out(static_cast<T*>(a.out) + (row_of(a, t, f) * a.q_heads + h * a.group + f % a.group) * D + i % D,
                      0.0f);
        }
    }
}

// One part of a pair: units [from, to) of (pair, head), which CTAs first ..
// first + n - 1 share.
struct Part {
    unsigned pair, head, from, to, first, n;
};

template <typename T, unsigned D, typename Rows>
__device__ __forceinline__ void run_part(const AttnKv4Args& a, const Part& p, Smem<D>& sm) {
    const unsigned seq = p.pair / a.tiles;
    const Tile t = make_tile<Rows::ROWS>(a, seq, p.pair % a.tiles, false);
    // the slot of a pair's first part is the CTA's second: it may also hold the end of another pair
    const std::size_t slot = static_cast<std::size_t>(2) * blockIdx.x + (p.from == 0 ? 1 : 0);
    run_segment<T, D, Rows>(a, t, seq, p.head, p.from, p.to, p.n == 1, slot, sm);
    if (p.n > 1) {
        // releases the CTA's parts (through the barrier), acquires the others'
        __syncthreads();
        if (threadIdx.x == 0) {
            unsigned before;
            asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(a.counters + p.first) : "memory");
            sm.last = before == p.n - 1;
            if (sm.last) a.counters[p.first] = 0;
        }
        __syncthreads();
        if (sm.last) {
            join_parts<T, D>(a, t, p.head, p.first, p.n, sm);
        }
    }
    __syncthreads();  // the next part overwrites what this one used
}

// Each pair on CTAs of its own, as few as keep every CTA at `most` units:
// the sum over pairs of ceil(units / most) * heads. Returns the least of
// kWarps candidates for `most` that fits the grid (0: none does). One warp
// tries one candidate.
template <unsigned D>
__device__ __forceinline__ unsigned fit_pairs(unsigned pairs, unsigned heads, unsigned share, Smem<D>& sm) {
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const unsigned most = share + warp * 4;
    unsigned ctas = 0;
    for (unsigned p = lane; p < pairs; p += 32) ctas += (sm.pair_units[p] + most - 1) / most;
    ctas = __reduce_add_sync(0xffffffffu, ctas) * heads;
    if (lane == 0) sm.fits[warp] = ctas <= gridDim.x;
    __syncthreads();
    for (unsigned w = 0; w < kWarps; ++w)
        if (sm.fits[w]) return share + w * 4;
    return 0;
}

template <typename T, unsigned D, typename Rows>
__global__ void __launch_bounds__(kWarps * 32, 2)
attention_kv4_shares(AttnKv4Args a) {
    extern __shared__ unsigned char smem_raw[];
    Smem<D>& sm = *reinterpret_cast<Smem<D>*>(smem_raw);
    pdl_begin();
    const unsigned heads = a.cache.kv_heads;
    const unsigned pairs = a.cache.seqs * a.tiles;
    const auto units_of = [&](unsigned pair) {
        return (make_tile<Rows::ROWS>(a, pair / a.tiles, pair % a.tiles, false).total + kStep - 1) / kStep;
    };

    if (threadIdx.x == 0) sm.found_pair = pairs;  // none yet
    // ---- sizes of all pairs; rows that see nothing are written here ----
    unsigned all_units = 0;  // the entry point sees to it that sums fit 32 bits
    unsigned units = 0, before = 0, total = 0;  // of pair threadIdx.x, when there are up to kPairCache
    for (unsigned p0 = 0; p0 < pairs; p0 += kPairCache) {
        const unsigned p = p0 + threadIdx.x;
        units = 0;
        bool blank = false;  // rows that see nothing, this CTA's to write
        if (p < pairs) {
            const bool mine = p % gridDim.x == blockIdx.x;
            const Tile t = make_tile<Rows::ROWS>(a, p / a.tiles, p % a.tiles, mine);
            units = (t.total + kStep - 1) / kStep;
            blank = mine && units == 0 && t.rows;
        }
        sm.pair_units[threadIdx.x] = units;
        if (scan_units(units, blank, sm, &before, &total)) write_blank_rows<T, D, Rows::ROWS>(a, p0);
        all_units += total;
    }
    const unsigned work = all_units * heads;
    if (work == 0) return;  // no row sees a key: their zeros are written, and nothing is to be shared out
    // short contexts: not less than a pair, up to a unit per warp, so that a
    // pair is not cut for nothing
    const unsigned share = max((work + gridDim.x - 1) / gridDim.x, min((all_units + pairs - 1) / pairs, kWarps));

    // ---- pairs on CTAs of their own, if that leaves no CTA with much more
    // than its share: a second part costs a CTA what some 28 units do ----
    Part part;
    unsigned at = 0, stop = 0;    // else: the CTA's share of the list
    unsigned pair_begin = 0;      // units of earlier pairs, one head
    unsigned block0 = 0;          // first pair of the cached block
    unsigned most = 0;
    if (pairs <= kPairCache && pairs * heads <= gridDim.x) most = fit_pairs<D>(pairs, heads, share, sm);
    if (most) {
        const unsigned n = (units + most - 1) / most;  // CTAs of this thread's pair, per head
        scan_units(n, false, sm, &before, &total);
        const unsigned b = blockIdx.x;
        if (b >= total * heads) return;
        if (n && b >= before * heads && b < (before + n) * heads) {
            sm.found_pair = threadIdx.x;
            sm.found_before = before;
        }
        __syncthreads();
        part.pair = sm.found_pair;
        const unsigned all = sm.pair_units[part.pair], cut = (all + most - 1) / most;
        const unsigned k = b - sm.found_before * heads, index = k % cut, each = (all + cut - 1) / cut;
        part.head = k / cut;
        part.n = (all + each - 1) / each;
        part.first = b - index;
        part.from = index * each;
        part.to = min(all, part.from + each);
        if (index >= part.n) return;
    } else {
        if (blockIdx.x >= (work + share - 1) / share) return;
        at = blockIdx.x * share;
        stop = min(at + share, work);
        for (unsigned p0 = 0; p0 < pairs; p0 += kPairCache) {
            const unsigned p = p0 + threadIdx.x;
            if (pairs > kPairCache) {
                units = p < pairs ? units_of(p) : 0u;
                scan_units(units, false, sm, &before, &total);
                sm.pair_units[threadIdx.x] = units;
            }
            const unsigned b = (pair_begin + before) * heads;
            if (units && at >= b && at < b + units * heads) {
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
        part.pair = sm.found_pair;
    }
    for (;;) {
        if (!most) {  // the list's part at unit `at`
            unsigned size = 0;
            for (;; ++part.pair) {  // skips pairs that see nothing
                if (part.pair >= pairs) return;  // lens changed under the call
                size = part.pair - block0 < kPairCache ? sm.pair_units[part.pair - block0] : units_of(part.pair);
                if (at < (pair_begin + size) * heads) break;
                pair_begin += size;
            }
            part.head = (at - pair_begin * heads) / size;
            const unsigned begin = pair_begin * heads + part.head * size;
            part.from = at - begin;
            part.to = min(begin + size, stop) - begin;
            part.first = begin / share;
            part.n = (begin + size - 1) / share - part.first + 1;
            at = begin + part.to;
        }
        run_part<T, D, Rows>(a, part, sm);
        if (most || at >= stop) break;
    }
}

template <typename T, unsigned D, typename Rows>
cudaError_t launch_attention(const AttnKv4Args& a, cudaStream_t s) {
    auto kernel = attention_kv4_shares<T, D, Rows>;
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
    if (!(std::fabs(scale) < INFINITY)) return invalid("b2_attention_kv4: scale must be finite");
    a.scale = scale == 0.0f ? 1.0f : std::fabs(scale);
    a.q_sign = scale > 0.0f ? 1.0f : scale < 0.0f ? -1.0f : 0.0f;
    // up to four rows of a KV head per sequence: the four-row form
    const bool narrow = max_queries * a.group <= 4;
    const std::size_t tiles = (max_queries * a.group + (narrow ? 3 : 7)) / (narrow ? 4 : 8);
    if (cache->seqs > 0x7FFFFFFFu / tiles) return invalid("b2_attention_kv4: too many row tiles");
    a.tiles = static_cast<unsigned>(tiles);
    // the kernel counts steps of 32 keys, over all pairs and heads, in 32 bits
    if ((max_len / kStep + 1) * cache->seqs > 0x3FFFFFFFu / (tiles * cache->kv_heads))
        return invalid("b2_attention_kv4: seqs * row tiles * kv_heads * max_len past 2^35 (max_len bounds the lengths)");
    a.counters = static_cast<unsigned*>(workspace);
    a.part_ml = reinterpret_cast<float*>(a.counters + kMaxGrid);
    a.part_o = a.part_ml + 2 * kMaxGrid * kRows * 2;
    // a window past every length is none; a smaller one leaves positions minus windows inside an int
    a.window = static_cast<unsigned>(window < max_len ? window : 0);
    a.sinks = static_cast<unsigned>(sinks < 0x7FFFFFFFu ? sinks : 0x7FFFFFFFu);
    cudaStream_t s = as_stream(stream);
    cudaError_t e;
    const auto run = [&](auto element) {
        using T = decltype(element);
        if (cache->head_dim == 128)
            return narrow ? launch_attention<T, 128, Narrow<128>>(a, s) : launch_attention<T, 128, Wide<128>>(a, s);
        return narrow ? launch_attention<T, 64, Narrow<64>>(a, s) : launch_attention<T, 64, Wide<64>>(a, s);
    };
    e = dtype == B2_DTYPE_F32 ? run(float()) : run(__nv_bfloat16());
    if (e != cudaSuccess) {
        cudaGetLastError();
        return set_error(B2_ERR_CUDA, std::string("b2_attention_kv4: ") + cudaGetErrorString(e));
    }
    return launch_result("b2_attention_kv4");
}

}  // extern "C"
