// Layout of the 4-bit paged KV cache (b2_kv4_cache), shared by the kernels
// that write it, read it back and attend over it.
//
// A page holds, for each KV head, one block of page_size rows of four
// sections: codes of K, codes of V, parameters of K, parameters of V. A row
// of codes is head_dim / 8 words of 32 bits, word = 8 neighbouring
// dimensions (an octet), nibble i = dimension i of the octet. The words are
// ordered for the attention's matrix instructions: a K row is cut into 4
// pieces and a V row into 8, piece i holding the words of all octets o with
// o % 4 == i (o % 8 == i) in ascending order, so each thread's operand is one
// load. A row of parameters is one word per 64 dimensions: the step s in the
// low bf16, the minimum m in the high one.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace b2 {
namespace {

constexpr unsigned kKv4Group = 64;            // dimensions that share (s, m)
constexpr unsigned kKv4Padding = 0xFFFFFFFFu;  // row_seq of a padding row

template <unsigned D>
struct Kv4Row {
    static constexpr unsigned words = D / 8;        // code words per row
    static constexpr unsigned groups = D / kKv4Group;
    static constexpr unsigned bytes = 2 * (D / 2 + 4 * groups);  // K and V of one position and head
    static __host__ __device__ constexpr unsigned k_word(unsigned octet) {
        return (octet % 4) * (words / 4) + octet / 4;
    }
    static __host__ __device__ constexpr unsigned v_word(unsigned octet) {
        return (octet % 8) * (words / 8) + octet / 8;
    }
};

// The cache as kernels take it.
struct Kv4View {
    std::uint8_t* data;
    const std::uint32_t* table;
    unsigned pages, page_shift, kv_heads, seqs, max_pages;
    unsigned head_stride, page_stride;  // bytes of a head's block, of a page
};

// Sections of the block of (page, head), in bytes from its start.
template <unsigned D>
__device__ __forceinline__ unsigned kv4_v_codes(unsigned page_shift) { return (D / 2) << page_shift; }
template <unsigned D>
__device__ __forceinline__ unsigned kv4_k_params(unsigned page_shift) { return D << page_shift; }
template <unsigned D>
__device__ __forceinline__ unsigned kv4_v_params(unsigned page_shift) {
    return (D + 4 * Kv4Row<D>::groups) << page_shift;
}

__device__ __forceinline__ std::uint8_t* kv4_block(const Kv4View& c, unsigned page, unsigned head) {
    return c.data + static_cast<std::size_t>(page) * c.page_stride + static_cast<std::size_t>(head) * c.head_stride;
}

// The page of position `pos` of sequence `seq`; false if the sequence, the
// position or the page is outside the cache.
__device__ __forceinline__ bool kv4_page(const Kv4View& c, unsigned seq, unsigned pos, unsigned* page) {
    const unsigned logical = pos >> c.page_shift;
    if (seq >= c.seqs || logical >= c.max_pages) return false;
    *page = __ldg(c.table + static_cast<std::size_t>(seq) * c.max_pages + logical);
    return *page < c.pages;
}

__device__ __forceinline__ float bf16_low(unsigned w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_high(unsigned w) { return __uint_as_float(w & 0xFFFF0000u); }
__device__ __forceinline__ unsigned bf16_pack(float lo, float hi) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&p);
}

// Checks a caller's cache description and fills *view; `what` names the entry point.
inline int kv4_view(const b2_kv4_cache* c, const char* what, Kv4View* view) {
    const std::string at(what);
    if (!c) return invalid(at + ": null cache");
    if (c->head_dim != 64 && c->head_dim != 128) return invalid(at + ": head_dim must be 64 or 128");
    if (c->page_size < 8 || (c->page_size & (c->page_size - 1)) || c->page_size > (1u << 20))
        return invalid(at + ": page_size must be a power of two, 8 to 2^20");
    if (c->kv_heads == 0 || c->kv_heads > 0xFFFF) return invalid(at + ": kv_heads out of range");
    if (c->pages > 0xFFFFFFFEu || c->seqs > 0xFFFFFFFEu || c->max_pages > 0xFFFFFFFEu)
        return invalid(at + ": cache sizes past 32 bits");
    if ((c->pages && !c->data) || (c->seqs && c->max_pages && !c->page_table)) return invalid(at + ": null cache pointer");
    if (!aligned16(c->data)) return invalid(at + ": cache data must be 16-byte aligned");
    view->data = static_cast<std::uint8_t*>(c->data);
    view->table = c->page_table;
    view->pages = static_cast<unsigned>(c->pages);
    view->page_shift = 0;
    while ((std::size_t(1) << view->page_shift) < c->page_size) ++view->page_shift;
    view->kv_heads = static_cast<unsigned>(c->kv_heads);
    view->seqs = static_cast<unsigned>(c->seqs);
    view->max_pages = static_cast<unsigned>(c->max_pages);
    const std::size_t head_bytes = c->page_size * (c->head_dim == 64 ? Kv4Row<64>::bytes : Kv4Row<128>::bytes);
    if (head_bytes > 0xFFFFFFFFu / c->kv_heads) return invalid(at + ": a page of 4 GB or more");
    view->head_stride = static_cast<unsigned>(head_bytes);
    view->page_stride = static_cast<unsigned>(head_bytes * c->kv_heads);
    return B2_OK;
}

inline bool kv4_dtype(std::uint32_t d) { return d == B2_DTYPE_F32 || d == B2_DTYPE_BF16; }

// ---- 8 neighbouring activations --------------------------------------------------

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// VEC: the 8 elements start on a 16-byte boundary.
template <bool VEC>
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
    if (VEC) {
        const float4 a = ld_plain(reinterpret_cast<const float4*>(p));
        const float4 b = ld_plain(reinterpret_cast<const float4*>(p) + 1);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = p[i];
    }
}
template <bool VEC>
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&x)[8]) {
    if (VEC) {
        const float4 a = ld_plain(reinterpret_cast<const float4*>(p));
        const unsigned w[4] = {__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(a.z), __float_as_uint(a.w)};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = bf16_low(w[i]);
            x[2 * i + 1] = bf16_high(w[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __bfloat162float(p[i]);
    }
}
// Rounded once to the element type, to 16-byte aligned global memory.
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
    st_plain(reinterpret_cast<float4*>(p), make_float4(x[0], x[1], x[2], x[3]));
    st_plain(reinterpret_cast<float4*>(p) + 1, make_float4(x[4], x[5], x[6], x[7]));
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {
    const uint4 w = make_uint4(bf16_pack(x[0], x[1]), bf16_pack(x[2], x[3]), bf16_pack(x[4], x[5]),
                               bf16_pack(x[6], x[7]));
    *reinterpret_cast<uint4*>(p) = w;
}

}  // namespace
}  // namespace b2
