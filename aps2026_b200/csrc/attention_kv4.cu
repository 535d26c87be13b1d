// Attention of each sequence's newest rows over its 4-bit paged cache
// (b2_attention_kv4).
//
// Mathematics: one pass over a row's visible keys with the running maximum M
// and sum L of its softmax: for key j with score x_j, M' = max(M, x_j),
// L' = L e^(M - M') + e^(x_j - M'), and the output sum is scaled alike.
//
// One warp per (query row, query head); each lane holds D/32 dimensions. A
// plain form that is right for every case.
#include "kv4.cuh"

namespace b2 {
namespace {

struct AttnKv4Args {
    const void* q;
    void* out;
    std::size_t q_row, q_head;
    unsigned rows, q_heads, group;      // group = q_heads / kv_heads
    const std::uint32_t* q_offsets;
    const std::uint32_t* lens;
    unsigned max_queries, max_len;
    float scale;
    unsigned window, sinks;
    Kv4View cache;
};

template <typename T, unsigned D>
__global__ void __launch_bounds__(128)
attention_kv4_rows(AttnKv4Args a) {
    pdl_begin();
    const unsigned lane = threadIdx.x & 31;
    const std::size_t units = static_cast<std::size_t>(a.cache.seqs) * a.max_queries * a.q_heads;
    for (std::size_t u = static_cast<std::size_t>(blockIdx.x) * 4 + threadIdx.x / 32; u < units;
         u += static_cast<std::size_t>(gridDim.x) * 4) {
        const unsigned h = static_cast<unsigned>(u % a.q_heads);
        const unsigned i = static_cast<unsigned>(u / a.q_heads % a.max_queries);
        const unsigned s = static_cast<unsigned>(u / a.q_heads / a.max_queries);
        const unsigned begin = a.q_offsets ? __ldg(a.q_offsets + s) : s;
        const unsigned end = a.q_offsets ? __ldg(a.q_offsets + s + 1) : s + 1;
        if (end < begin || end > a.rows || end - begin > a.max_queries) {
            if (lane == 0) flag_check(B2_CHECK_KV4);
            continue;
        }
        if (i >= end - begin) continue;
        unsigned len = __ldg(a.lens + s);
        if (len > a.max_len || len > (static_cast<std::size_t>(a.cache.max_pages) << a.cache.page_shift)) {
            if (lane == 0) flag_check(B2_CHECK_KV4);
            len = 0;
        }
        const long long pos = static_cast<long long>(len) - (end - begin) + i;
        const unsigned head = h / a.group;
        const std::size_t row = begin + i;
        // lane's dimensions: lane, lane + 32, ...
        constexpr unsigned PER = D / 32;
        float q[PER], acc[PER];
#pragma unroll
        for (unsigned e = 0; e < PER; ++e) {
            q[e] = as_float(static_cast<const T*>(a.q)[row * a.q_row + h * a.q_head + lane + 32 * e]) * a.scale;
            acc[e] = 0.0f;
        }
        float top = -INFINITY, sum = 0.0f;
        const unsigned n = pos < 0 ? 0u : static_cast<unsigned>(pos) + 1;
        const unsigned low = a.window && n > a.window ? n - a.window : 0u;
        for (unsigned j = 0; j < n; ++j) {
            if (j >= a.sinks && j < low) { j = low - 1; continue; }
            unsigned page;
            if (!kv4_page(a.cache, s, j, &page)) {
                if (lane == 0) flag_check(B2_CHECK_KV4);
                continue;
            }
            const unsigned shift = a.cache.page_shift;
            const std::size_t slot = j & ((1u << shift) - 1u);
            const std::uint8_t* block = kv4_block(a.cache, page, head);
            const unsigned* kc = reinterpret_cast<const unsigned*>(block + slot * (D / 2));
            const unsigned* vc = reinterpret_cast<const unsigned*>(block + kv4_v_codes<D>(shift) + slot * (D / 2));
            const unsigned* kp =
                reinterpret_cast<const unsigned*>(block + kv4_k_params<D>(shift)) + slot * Kv4Row<D>::groups;
            const unsigned* vp =
                reinterpret_cast<const unsigned*>(block + kv4_v_params<D>(shift)) + slot * Kv4Row<D>::groups;
            float dot = 0.0f, v[PER];
#pragma unroll
            for (unsigned e = 0; e < PER; ++e) {
                const unsigned d = lane + 32 * e, o = d / 8, sh = 4 * (d % 8);
                const unsigned pk = kp[d / kKv4Group], pv = vp[d / kKv4Group];
                const float k = static_cast<float>((kc[Kv4Row<D>::k_word(o)] >> sh) & 15u) * bf16_low(pk) + bf16_high(pk);
                v[e] = static_cast<float>((vc[Kv4Row<D>::v_word(o)] >> sh) & 15u) * bf16_low(pv) + bf16_high(pv);
                dot += q[e] * k;
            }
            dot = warp_sum(dot);
            const float m = fmaxf(top, dot), old = expf(top - m), p = expf(dot - m);
            top = m;
            sum = sum * old + p;
#pragma unroll
            for (unsigned e = 0; e < PER; ++e) acc[e] = acc[e] * old + p * v[e];
        }
#pragma unroll
        for (unsigned e = 0; e < PER; ++e) {
            const float y = sum == 0.0f ? 0.0f : acc[e] / sum;
            T* out = static_cast<T*>(a.out) + (row * a.q_heads + h) * D + lane + 32 * e;
            if constexpr (sizeof(T) == 2) *out = __float2bfloat16_rn(y);
            else *out = y;
        }
    }
}

template <typename T, unsigned D>
void launch_attention(const AttnKv4Args& a, cudaStream_t s) {
    const std::size_t units = static_cast<std::size_t>(a.cache.seqs) * a.max_queries * a.q_heads;
    auto kernel = attention_kv4_rows<T, D>;
    launch_pdl(kernel, wave_grid(reinterpret_cast<const void*>(kernel), 128, 0, (units + 3) / 4), 128, 0, s, a);
}

}  // namespace
}  // namespace b2

B2_DEFINE_CHECK_TAKER(attention_kv4)

extern "C" {

int b2_attention_kv4_workspace_size(size_t head_dim, size_t* bytes) {
    using namespace b2;
    if (!bytes) return invalid("b2_attention_kv4_workspace_size: null pointer");
    if (head_dim != 64 && head_dim != 128) return invalid("b2_attention_kv4_workspace_size: head_dim must be 64 or 128");
    *bytes = 16;
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
    if (rows > 0x7FFFFFFFu || q_heads > 0xFFFF || max_queries > 0x7FFFFFFFu || max_len > 0x7FFFFFFFu)
        return invalid("b2_attention_kv4: sizes past 31 bits");
    std::size_t need = 0;
    b2_attention_kv4_workspace_size(cache->head_dim, &need);
    if (workspace_bytes < need) return invalid("b2_attention_kv4: workspace too small");
    if (!aligned16(out) || !aligned16(workspace)) return invalid("b2_attention_kv4: out and workspace must be 16-byte aligned");
    a.q = q; a.out = out; a.q_row = q_row_stride; a.q_head = q_head_stride;
    a.rows = static_cast<unsigned>(rows); a.q_heads = static_cast<unsigned>(q_heads);
    a.group = static_cast<unsigned>(q_heads / cache->kv_heads);
    a.q_offsets = q_offsets; a.lens = lens;
    a.max_queries = static_cast<unsigned>(max_queries); a.max_len = static_cast<unsigned>(max_len);
    a.scale = scale;
    a.window = static_cast<unsigned>(window < 0x7FFFFFFFu ? window : 0);  // a window past every length: none
    a.sinks = static_cast<unsigned>(sinks < 0x7FFFFFFFu ? sinks : 0x7FFFFFFFu);
    cudaStream_t s = as_stream(stream);
    if (dtype == B2_DTYPE_F32) {
        if (cache->head_dim == 128) launch_attention<float, 128>(a, s);
        else launch_attention<float, 64>(a, s);
    } else {
        if (cache->head_dim == 128) launch_attention<__nv_bfloat16, 128>(a, s);
        else launch_attention<__nv_bfloat16, 64>(a, s);
    }
    return launch_result("b2_attention_kv4");
}

}  // extern "C"
