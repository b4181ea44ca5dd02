// Rows into and out of a paged cache, quantised where it has 8 bits.
//
// A row (one token's k or v of one kv head) is taken by the least power of two
// of lanes that hold it at eight elements each; its largest absolute value is
// found by exchanges among them. Bytes bound both directions.
#include <algorithm>

#include "xp_elem.hpp"

namespace xp {
namespace {

constexpr uint32_t kKvThreads = 256;

struct KvRows {
    void *         cache[2];       // k, v
    float*         scale[2];
    void*          rows[2];
    uint64_t       stride[2];
    const int32_t *cu, *kv_len;
    PageMap        map;
    uint32_t       n_seq, n_tokens, kv_heads, head_dim, lanes;
};

// The row of the cache that belongs to packed token t's head h: its index in
// rows of head_dim, or -1 (no row); `owned` says whether a sequence has t.
__device__ __forceinline__ int64_t row_in_cache(const KvRows& a, uint32_t t, uint32_t h, bool* owned) {
    const uint32_t b = seq_of_row(a.cu, a.n_seq, a.n_tokens, t);
    *owned = b < a.n_seq;
    if (!*owned) return -1;
    const RowSpan r = row_span(a.cu, a.n_tokens, b);
    const int64_t p = row_position(a.kv_len[b], r.end - r.first, t - r.first);
    *owned = p >= 0;
    const int32_t g = page_of(a.map, b, p);
    return g < 0 ? -1 : int64_t(cache_row(uint32_t(g), a.kv_heads, h, a.map.page_shift, uint32_t(p) & ((1u << a.map.page_shift) - 1u)));
}

// x / scale rounded to the nearest whole number, even on a tie, of the exact
// quotient: the rounded product with the reciprocal is off by one at most
// next to a tie, which the exact remainder (one fma) tells.
__device__ __forceinline__ int quantise1(float x, float scale, float inv) {
    float q = rintf(x * inv);
    const float r = fmaf(-q, scale, x), half = 0.5f * scale, to = r < 0.0f ? -1.0f : 1.0f;
    const bool odd = int(q) & 1;
    if (fabsf(r) > half || (fabsf(r) == half && odd)) q += to;
    return int(fminf(fmaxf(q, -127.0f), 127.0f));
}

template <int IN, int CACHE>
__global__ __launch_bounds__(kKvThreads) void paged_kv_write_kernel(KvRows a) {
    const uint32_t per = kKvThreads / a.lanes, sub = threadIdx.x / a.lanes, lane = threadIdx.x % a.lanes;
    const uint64_t n = uint64_t(a.n_tokens) * a.kv_heads * 2;
    const bool live = lane * 8 < a.head_dim;
    for (uint64_t i0 = uint64_t(blockIdx.x) * per; i0 < n; i0 += uint64_t(gridDim.x) * per) {
        const uint64_t i = i0 + sub;
        const bool in = i < n;
        const uint32_t t = uint32_t(in ? i / (a.kv_heads * 2) : 0), w = uint32_t(in ? i % (a.kv_heads * 2) : 0);
        const uint32_t kv = w / a.kv_heads, h = w % a.kv_heads;
        bool owned;
        const int64_t row = in ? row_in_cache(a, t, h, &owned) : -1;
        float x[8] = {};
        if (row >= 0 && live) load8<IN>(a.rows[kv], uint64_t(t) * a.stride[kv] + uint64_t(h) * a.head_dim + lane * 8, x);
        const uint64_t to = uint64_t(row) * a.head_dim + lane * 8;
        if constexpr (CACHE == XP_ELEM_F16 || CACHE == XP_ELEM_BF16) {
            if (row >= 0 && live) store8<CACHE>(a.cache[kv], to, x);
        } else {
            // as bit patterns an infinity is over every number and a NaN over it
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[j]) & 0x7FFFFFFFu);
            for (uint32_t o = 1; o < a.lanes; o <<= 1) top = max(top, uint32_t(__shfl_xor(int(top), int(o), kWave)));
            const bool finite = top < 0x7F800000u;
            float scale = 0.0f;
            u32x2 code{0u, 0u};
            if (!finite) {
                scale = __uint_as_float(0x7FC00000u);
            } else if (top != 0u) {
                if constexpr (CACHE == XP_ELEM_I8) {
                    // at least the least normal number, whose reciprocal is finite
                    scale = fmaxf(__uint_as_float(top) / 127.0f, 0x1p-126f);
                    const float inv = 1.0f / scale;
#pragma unroll
                    for (int j = 0; j < 8; ++j) code[j / 4] |= uint32_t(quantise1(x[j], scale, inv) & 0xFF) << (8 * (j % 4));
                } else {
                    // max <= 448 2^k = 1.75 2^(8 + k)
                    const int k = max(int(top >> 23) - 135 + ((top & 0x7FFFFFu) > 0x600000u ? 1 : 0), -126);
                    scale = __uint_as_float(uint32_t(k + 127) << 23);
                    const float inv = __uint_as_float(uint32_t(127 - k) << 23);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        int c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j] * inv, x[4 * j + 1] * inv, 0, false);
                        c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j + 2] * inv, x[4 * j + 3] * inv, c, true);
                        code[j] = uint32_t(c);
                    }
                }
            }
            if (row >= 0 && live) *reinterpret_cast<u32x2*>(static_cast<uint8_t*>(a.cache[kv]) + to) = code;
            if (row >= 0 && lane == 0) a.scale[kv][row] = scale;
        }
    }
}

template <int OUT, int CACHE>
__global__ __launch_bounds__(kKvThreads) void paged_kv_read_kernel(KvRows a) {
    const uint32_t per = kKvThreads / a.lanes, sub = threadIdx.x / a.lanes, lane = threadIdx.x % a.lanes;
    const uint64_t n = uint64_t(a.n_tokens) * a.kv_heads * 2;
    if (lane * 8 >= a.head_dim) return;
    for (uint64_t i = uint64_t(blockIdx.x) * per + sub; i < n; i += uint64_t(gridDim.x) * per) {
        const uint32_t t = uint32_t(i / (a.kv_heads * 2)), w = uint32_t(i % (a.kv_heads * 2));
        const uint32_t kv = w / a.kv_heads, h = w % a.kv_heads;
        bool owned;
        const int64_t row = row_in_cache(a, t, h, &owned);
        if (!owned) continue;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = __uint_as_float(0x7FC00000u);
        if (row >= 0) {
            load8<CACHE>(a.cache[kv], uint64_t(row) * a.head_dim + lane * 8, x);
            if constexpr (CACHE == XP_ELEM_I8 || CACHE == XP_ELEM_E4M3) {
                const float s = a.scale[kv][row];
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] *= s;
            }
        }
        store8<OUT>(a.rows[kv], uint64_t(t) * a.stride[kv] + uint64_t(h) * a.head_dim + lane * 8, x);
    }
}

// The checks and the arguments of both directions; *skip: nothing to do.
int kv_call(const char* fn, const xp_paged_kv* c, const xp_paged_seqs* s, const xp_rows* k, const xp_rows* v,
            xp_stream stream, const void* out, KvRows* a, dim3* grid, bool* skip) {
    XP_CHECK(check_cache(fn, c));
    XP_CHECK(check_seqs(fn, s));
    XP_CHECK(check_rows(fn, "k", k, c->head_dim, 16));
    XP_CHECK(check_rows(fn, "v", v, c->head_dim, 16));
    if (k->heads != c->kv_heads || v->heads != c->kv_heads)
        return set_error(XP_E_ARG, "%s: k has %u and v %u heads, the cache %u", fn, k->heads, v->heads, c->kv_heads);
    if (k->elem != v->elem) return set_error(XP_E_ARG, "%s: k and v differ in elem", fn);
    *skip = s->n_tokens == 0 || s->n_seq == 0;
    if (*skip) return XP_OK;
    XP_CHECK(check_here(fn, stream, out));
    *a = {{c->k, c->v}, {c->k_scale, c->v_scale}, {k->data, v->data}, {k->stride, v->stride}, s->cu, s->kv_len,
          page_map(c, s), s->n_seq, s->n_tokens, c->kv_heads, c->head_dim, 1};
    while (a->lanes * 8 < c->head_dim) a->lanes *= 2;
    const uint64_t rows = uint64_t(s->n_tokens) * c->kv_heads * 2, per = kKvThreads / a->lanes;
    *grid = dim3(uint32_t(std::min<uint64_t>((rows + per - 1) / per, 1u << 20)));
    return XP_OK;
}

}  // namespace
}  // namespace xp

using namespace xp;

#define XP_KV_CACHE(KERNEL, E)                                                                                           \
    switch (c->elem) {                                                                                                   \
        case XP_ELEM_F16: hipLaunchKernelGGL((KERNEL<E, XP_ELEM_F16>), grid, dim3(kKvThreads), 0, as_stream(stream), a); break;   \
        case XP_ELEM_BF16: hipLaunchKernelGGL((KERNEL<E, XP_ELEM_BF16>), grid, dim3(kKvThreads), 0, as_stream(stream), a); break; \
        case XP_ELEM_I8: hipLaunchKernelGGL((KERNEL<E, XP_ELEM_I8>), grid, dim3(kKvThreads), 0, as_stream(stream), a); break;     \
        default: hipLaunchKernelGGL((KERNEL<E, XP_ELEM_E4M3>), grid, dim3(kKvThreads), 0, as_stream(stream), a); break;           \
    }
#define XP_KV_LAUNCH(KERNEL)                                                       \
    switch (k->elem) {                                                             \
        case XP_ELEM_F32: XP_KV_CACHE(KERNEL, XP_ELEM_F32) break;                  \
        case XP_ELEM_F16: XP_KV_CACHE(KERNEL, XP_ELEM_F16) break;                  \
        default: XP_KV_CACHE(KERNEL, XP_ELEM_BF16) break;                          \
    }

extern "C" {

int xp_paged_kv_write(const xp_paged_kv* c, const xp_paged_seqs* s, const xp_rows* k, const xp_rows* v,
                      xp_stream stream) {
    KvRows a;
    dim3 grid;
    bool skip;
    XP_CHECK(kv_call(__func__, c, s, k, v, stream, c ? c->k : nullptr, &a, &grid, &skip));
    if (skip) return XP_OK;
    XP_KV_LAUNCH(paged_kv_write_kernel)
    XP_LAUNCHED();
    return XP_OK;
}

int xp_paged_kv_read(const xp_paged_kv* c, const xp_paged_seqs* s, const xp_rows* k, const xp_rows* v,
                     xp_stream stream) {
    KvRows a;
    dim3 grid;
    bool skip;
    XP_CHECK(kv_call(__func__, c, s, k, v, stream, k ? k->data : nullptr, &a, &grid, &skip));
    if (skip) return XP_OK;
    XP_KV_LAUNCH(paged_kv_read_kernel)
    XP_LAUNCHED();
    return XP_OK;
}

}  // extern "C"
