// Appending rows to the 4-bit paged KV cache with the rotation of keys and
// queries on the way (b2_kv4_append), and reading rows back (b2_kv4_read).
//
// Mathematics: a head's pairs (x_j, x_{j+D/2}) are rotated by their position's
// angle; then, per 64 dimensions, m = bf16(min x), s = bf16(max(max x - m, 0)
// / 15), c = clamp(rint((x - m) / s), 0, 15). m and s are rounded before the
// codes are chosen, so the codes make up for that rounding; a bf16 m is off
// by 2^-9 |m| at most, a small part of a step. Every fp32 operation is
// rounded on its own: the codes are those of the formula in plain fp32.
//
// HBM bound: each input read once, each output written once. D/16 threads own
// a head of a row, each the same octet of both halves: the rotation needs no
// exchange, and the groups' minima and maxima are shuffles inside the
// subgroup. One launch covers the row's q, k and v heads, in a grid-stride
// loop of all the CTAs that the SMs hold: 13,547 rows of 16 q and 2 x 4 kv
// heads of a fused projection appended and read back in 67 us, 356 MB at 82%
// of the measured copy rate. The append takes 46 us of it, 98%; the read 17, 57%:
// each 8 values wait for row, page and code word in turn, and a row's K and V
// look their page up separately (long_scoreboard: 23 cycles between two
// instructions of a warp). In bf16 47 us, 62% (33 and 12). For a decode step's few
// rows the two calls cost their launches: 5 to 8 us, by the host.
#include "kv4.cuh"

namespace b2 {
namespace {

// CTAs per SM that the append's registers allow without a wave of leftovers
// (4: 66.8 us for the rows above, 5: 69.0, 6 and 8, which spill: 80.6 and 87.7).
constexpr unsigned kAppendCtas = 4;

struct AppendArgs {
    const void* q;
    void* q_out;
    const void* k;
    const void* v;
    std::size_t q_row, q_head, k_row, k_head, v_row, v_head;  // strides in elements
    unsigned rows, q_heads;
    const std::uint32_t* row_seq;
    const std::uint32_t* row_pos;
    const float* cos_t;
    const float* sin_t;
    std::size_t table_rows;
    Kv4View cache;
};

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e+38f; }

// Codes of one octet, nibble i = dimension i.
__device__ __forceinline__ unsigned encode8(const float (&x)[8], float m, float inv) {
    unsigned w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        // fmaxf/fminf give a number even where x - m is NaN
        const float c = fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(x[i], m), inv)), 0.0f), 15.0f);
        w |= static_cast<unsigned>(c) << (4 * i);
    }
    return w;
}

// Quantises the subgroup's head: thread t of D/16 holds octets t (lo) and
// t + D/16 (hi). SUB = D/16 threads; lanes of a subgroup are adjacent.
template <unsigned D>
__device__ __forceinline__ void quantise(const float (&lo)[8], const float (&hi)[8], unsigned t, unsigned mask,
                                         unsigned* codes, unsigned* params, bool is_v, bool store) {
    constexpr unsigned SUB = D / 16, GROUPS = Kv4Row<D>::groups;
    // D = 128: lo is group 0, hi group 1. D = 64: both halves are group 0.
    float mn[GROUPS], mx[GROUPS];
    bool ok[GROUPS];
#pragma unroll
    for (unsigned g = 0; g < GROUPS; ++g) { mn[g] = 3.402823466e+38f; mx[g] = -3.402823466e+38f; ok[g] = true; }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        mn[0] = fminf(mn[0], lo[i]); mx[0] = fmaxf(mx[0], lo[i]); ok[0] &= finite(lo[i]);
        mn[GROUPS - 1] = fminf(mn[GROUPS - 1], hi[i]); mx[GROUPS - 1] = fmaxf(mx[GROUPS - 1], hi[i]);
        ok[GROUPS - 1] &= finite(hi[i]);
    }
#pragma unroll
    for (unsigned g = 0; g < GROUPS; ++g) {
#pragma unroll
        for (unsigned o = SUB / 2; o > 0; o >>= 1) {
            mn[g] = fminf(mn[g], __shfl_xor_sync(mask, mn[g], o));
            mx[g] = fmaxf(mx[g], __shfl_xor_sync(mask, mx[g], o));
            ok[g] = __shfl_xor_sync(mask, ok[g] ? 1 : 0, o) && ok[g];
        }
    }
    unsigned par[GROUPS], w_lo = 0, w_hi = 0;
#pragma unroll
    for (unsigned g = 0; g < GROUPS; ++g) {
        const float m = __bfloat162float(__float2bfloat16_rn(mn[g]));
        const float step = __fmul_rn(fmaxf(__fsub_rn(mx[g], m), 0.0f), 1.0f / 15.0f);
        const float s = __bfloat162float(__float2bfloat16_rn(step));
        const float inv = s < 1.17549435e-38f ? 0.0f : __frcp_rn(s);
        par[g] = ok[g] ? bf16_pack(s, m) : 0x7FFF7FFFu;  // NaN, NaN
        if (g == 0) w_lo = ok[0] ? encode8(lo, m, inv) : 0u;
        if (g == GROUPS - 1) w_hi = ok[g] ? encode8(hi, m, inv) : 0u;
    }
    if (!store) return;
    codes[is_v ? Kv4Row<D>::v_word(t) : Kv4Row<D>::k_word(t)] = w_lo;
    codes[is_v ? Kv4Row<D>::v_word(t + SUB) : Kv4Row<D>::k_word(t + SUB)] = w_hi;
#pragma unroll
    for (unsigned g = 0; g < GROUPS; ++g)
        if (t == g) params[g] = par[g];
}

// Unit = (row, head) over the q, k and v heads; D/16 threads per unit.
template <typename T, unsigned D, bool VEC>
__global__ void __launch_bounds__(256, kAppendCtas)
kv4_append_rows(AppendArgs a) {
    pdl_begin();
    constexpr unsigned SUB = D / 16, UNITS = 256 / SUB;
    const unsigned heads = a.q_heads + 2 * a.cache.kv_heads;
    const unsigned units = a.rows * heads;
    const unsigned t = threadIdx.x % SUB;
    const unsigned lane = threadIdx.x & 31;
    const unsigned mask = ((1u << SUB) - 1u) << (lane / SUB * SUB);
    for (unsigned u = blockIdx.x * UNITS + threadIdx.x / SUB; u < units; u += gridDim.x * UNITS) {
        const unsigned row = u / heads, h = u - row * heads;
        const unsigned seq = __ldg(a.row_seq + row), pos = __ldg(a.row_pos + row);
        const bool padding = seq == kKv4Padding;
        const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + a.cache.kv_heads;
        const unsigned head = is_q ? h : is_v ? h - a.q_heads - a.cache.kv_heads : h - a.q_heads;
        const T* src = is_q ? static_cast<const T*>(a.q) + row * a.q_row + head * a.q_head
                       : is_v ? static_cast<const T*>(a.v) + row * a.v_row + head * a.v_head
                              : static_cast<const T*>(a.k) + row * a.k_row + head * a.k_head;
        float lo[8], hi[8];
        load8<VEC>(src + t * 8, lo);
        load8<VEC>(src + D / 2 + t * 8, hi);
        // a row whose rotation cannot be had is skipped whole, its values too
        bool ok = !padding;
        if (a.cos_t) {
            if (pos >= a.table_rows) {
                if (!padding && t == 0) flag_check(B2_CHECK_ROPE);
                ok = false;
            } else if (!is_v) {
                const std::size_t at = static_cast<std::size_t>(pos) * (D / 2) + t * 8;
                float c[8], s[8];
                load8<VEC>(a.cos_t + at, c);
                load8<VEC>(a.sin_t + at, s);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x0 = lo[i], x1 = hi[i];
                    lo[i] = __fsub_rn(__fmul_rn(x0, c[i]), __fmul_rn(x1, s[i]));
                    hi[i] = __fadd_rn(__fmul_rn(x1, c[i]), __fmul_rn(x0, s[i]));
                }
            }
        }
        if (is_q) {
            if (!ok) {
#pragma unroll
                for (int i = 0; i < 8; ++i) lo[i] = hi[i] = 0.0f;
            }
            T* dst = static_cast<T*>(a.q_out) + (static_cast<std::size_t>(row) * a.q_heads + head) * D;
            store8(dst + t * 8, lo);
            store8(dst + D / 2 + t * 8, hi);
            continue;
        }
        unsigned page = 0;
        if (ok && !kv4_page(a.cache, seq, pos, &page)) {
            if (t == 0) flag_check(B2_CHECK_KV4);
            ok = false;
        }
        const unsigned slot = pos & ((1u << a.cache.page_shift) - 1u);
        std::uint8_t* block = kv4_block(a.cache, ok ? page : 0, head);
        const unsigned shift = a.cache.page_shift;
        std::uint8_t* codes = block + (is_v ? kv4_v_codes<D>(shift) : 0u) + static_cast<std::size_t>(slot) * (D / 2);
        std::uint8_t* params = block + (is_v ? kv4_v_params<D>(shift) : kv4_k_params<D>(shift)) +
                               static_cast<std::size_t>(slot) * 4 * Kv4Row<D>::groups;
        quantise<D>(lo, hi, t, mask, reinterpret_cast<unsigned*>(codes), reinterpret_cast<unsigned*>(params), is_v, ok);
    }
}

// Unit = (row, KV head, K or V); D/8 threads per unit, one octet each.
template <typename T, unsigned D>
__global__ void __launch_bounds__(256)
kv4_read_rows(Kv4View cache, const std::uint32_t* row_seq, const std::uint32_t* row_pos, unsigned rows, T* k_out,
              T* v_out) {
    pdl_begin();
    constexpr unsigned SUB = D / 8, UNITS = 256 / SUB;
    const unsigned per_row = 2 * cache.kv_heads, units = rows * per_row;
    const unsigned o = threadIdx.x % SUB;
    for (unsigned u = blockIdx.x * UNITS + threadIdx.x / SUB; u < units; u += gridDim.x * UNITS) {
        const unsigned row = u / per_row, h = u - row * per_row;
        const bool is_v = h >= cache.kv_heads;
        const unsigned head = is_v ? h - cache.kv_heads : h;
        const unsigned seq = __ldg(row_seq + row), pos = __ldg(row_pos + row);
        float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        unsigned page = 0;
        if (seq != kKv4Padding) {
            if (kv4_page(cache, seq, pos, &page)) {
                const unsigned shift = cache.page_shift, slot = pos & ((1u << shift) - 1u);
                const std::uint8_t* block = kv4_block(cache, page, head);
                const unsigned* codes = reinterpret_cast<const unsigned*>(
                    block + (is_v ? kv4_v_codes<D>(shift) : 0u) + static_cast<std::size_t>(slot) * (D / 2));
                const unsigned* params = reinterpret_cast<const unsigned*>(
                    block + (is_v ? kv4_v_params<D>(shift) : kv4_k_params<D>(shift)) +
                    static_cast<std::size_t>(slot) * 4 * Kv4Row<D>::groups);
                const unsigned w = codes[is_v ? Kv4Row<D>::v_word(o) : Kv4Row<D>::k_word(o)];
                const unsigned p = params[o / (kKv4Group / 8)];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    x[i] = __fmaf_rn(static_cast<float>((w >> (4 * i)) & 15u), bf16_low(p), bf16_high(p));
            } else if (o == 0) {
                flag_check(B2_CHECK_KV4);
            }
        }
        T* out = (is_v ? v_out : k_out) + (static_cast<std::size_t>(row) * cache.kv_heads + head) * D + o * 8;
        store8(out, x);
    }
}

// Grid of 256-thread CTAs for a grid-stride loop, `per_sm` of them per SM at
// most: as many as one holds (no occupancy query: it costs a call 1 us).
inline unsigned full_grid(std::size_t ctas, unsigned per_sm) {
    const std::size_t most = static_cast<std::size_t>(sm_count()) * per_sm;
    return static_cast<unsigned>(ctas < most ? ctas : most);
}

template <typename T, unsigned D>
void launch_append(const AppendArgs& a, bool vec, cudaStream_t s) {
    const std::size_t units = static_cast<std::size_t>(a.rows) * (a.q_heads + 2 * a.cache.kv_heads);
    const std::size_t ctas = (units + 256 / (D / 16) - 1) / (256 / (D / 16));
    auto kernel = vec ? kv4_append_rows<T, D, true> : kv4_append_rows<T, D, false>;
    launch_pdl(kernel, full_grid(ctas, kAppendCtas), 256, 0, s, a);
}

template <typename T, unsigned D>
void launch_read(const Kv4View& c, const std::uint32_t* seq, const std::uint32_t* pos, unsigned rows, void* k, void* v,
                 cudaStream_t s) {
    const std::size_t units = static_cast<std::size_t>(rows) * 2 * c.kv_heads;
    const std::size_t ctas = (units + 256 / (D / 8) - 1) / (256 / (D / 8));
    auto kernel = kv4_read_rows<T, D>;
    launch_pdl(kernel, full_grid(ctas, 8), 256, 0, s, c, seq, pos, rows, static_cast<T*>(k), static_cast<T*>(v));
}

}  // namespace
}  // namespace b2

B2_DEFINE_CHECK_TAKER(kv4_cache)

extern "C" {

int b2_kv4_page_bytes(size_t page_size, size_t kv_heads, size_t head_dim, size_t* bytes) {
    using namespace b2;
    if (!bytes) return invalid("b2_kv4_page_bytes: null pointer");
    b2_kv4_cache c{nullptr, 0, page_size, kv_heads, head_dim, nullptr, 0, 0};
    Kv4View view{};
    const int rc = kv4_view(&c, "b2_kv4_page_bytes", &view);
    if (rc == B2_OK) *bytes = view.page_stride;
    return rc;
}

int b2_kv4_append(const void* q, size_t q_row_stride, size_t q_head_stride, size_t q_heads, void* q_out,
                  const void* k, size_t k_row_stride, size_t k_head_stride, const void* v, size_t v_row_stride,
                  size_t v_head_stride, uint32_t dtype, size_t rows, const uint32_t* row_seq,
                  const uint32_t* row_pos, const float* cos_table, const float* sin_table, size_t table_rows,
                  const b2_kv4_cache* cache, b2_stream_t stream) {
    using namespace b2;
    AppendArgs a{};
    const int rc = kv4_view(cache, "b2_kv4_append", &a.cache);
    if (rc != B2_OK) return rc;
    if (!kv4_dtype(dtype)) return invalid("b2_kv4_append: unknown dtype");
    if ((cos_table == nullptr) != (sin_table == nullptr)) return invalid("b2_kv4_append: one rotation table without the other");
    if (rows == 0) return B2_OK;
    if (!k || !v || !row_seq || !row_pos) return invalid("b2_kv4_append: null pointer");
    if (q && (q_heads == 0 || !q_out)) return invalid("b2_kv4_append: q without q_heads / q_out");
    if (!q) q_heads = 0;
    // units and a grid's worth of slack count in 32 bits
    if (rows > 0x7FFFFFFFu || q_heads > 0xFFFF || rows * (q_heads + 2 * cache->kv_heads) > 0x7FFFFFFFu)
        return invalid("b2_kv4_append: too many rows");
    if (q_out && !aligned16(q_out)) return invalid("b2_kv4_append: q_out must be 16-byte aligned");
    a.q = q; a.q_out = q_out; a.k = k; a.v = v;
    a.q_row = q_row_stride; a.q_head = q_head_stride;
    a.k_row = k_row_stride; a.k_head = k_head_stride;
    a.v_row = v_row_stride; a.v_head = v_head_stride;
    a.rows = static_cast<unsigned>(rows); a.q_heads = static_cast<unsigned>(q_heads);
    a.row_seq = row_seq; a.row_pos = row_pos;
    a.cos_t = cos_table; a.sin_t = sin_table; a.table_rows = table_rows;
    const std::size_t per16 = dtype == B2_DTYPE_F32 ? 4 : 8;  // elements per 16 bytes
    const std::size_t strides = q_row_stride * (q ? 1 : 0) | q_head_stride * (q ? 1 : 0) | k_row_stride |
                                k_head_stride | v_row_stride | v_head_stride;
    const bool vec = strides % per16 == 0 && aligned16(q) && aligned16(k) && aligned16(v) && aligned16(cos_table) &&
                     aligned16(sin_table);
    cudaStream_t s = as_stream(stream);
    if (dtype == B2_DTYPE_F32) {
        if (cache->head_dim == 128) launch_append<float, 128>(a, vec, s);
        else launch_append<float, 64>(a, vec, s);
    } else {
        if (cache->head_dim == 128) launch_append<__nv_bfloat16, 128>(a, vec, s);
        else launch_append<__nv_bfloat16, 64>(a, vec, s);
    }
    return launch_result("b2_kv4_append");
}

int b2_kv4_read(const b2_kv4_cache* cache, const uint32_t* row_seq, const uint32_t* row_pos, size_t rows,
                void* k_out, void* v_out, uint32_t dtype, b2_stream_t stream) {
    using namespace b2;
    Kv4View c{};
    const int rc = kv4_view(cache, "b2_kv4_read", &c);
    if (rc != B2_OK) return rc;
    if (!kv4_dtype(dtype)) return invalid("b2_kv4_read: unknown dtype");
    if (rows == 0) return B2_OK;
    if (!row_seq || !row_pos || !k_out || !v_out) return invalid("b2_kv4_read: null pointer");
    if (!aligned16(k_out) || !aligned16(v_out)) return invalid("b2_kv4_read: outputs must be 16-byte aligned");
    if (rows > 0x7FFFFFFFu || rows * 2 * cache->kv_heads > 0x7FFFFFFFu) return invalid("b2_kv4_read: too many rows");
    const unsigned n = static_cast<unsigned>(rows);
    cudaStream_t s = as_stream(stream);
    if (dtype == B2_DTYPE_F32) {
        if (cache->head_dim == 128) launch_read<float, 128>(c, row_seq, row_pos, n, k_out, v_out, s);
        else launch_read<float, 64>(c, row_seq, row_pos, n, k_out, v_out, s);
    } else {
        if (cache->head_dim == 128) launch_read<__nv_bfloat16, 128>(c, row_seq, row_pos, n, k_out, v_out, s);
        else launch_read<__nv_bfloat16, 64>(c, row_seq, row_pos, n, k_out, v_out, s);
    }
    return launch_result("b2_kv4_read");
}

}  // extern "C"
