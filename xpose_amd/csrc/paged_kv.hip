// Rows into and out of a paged cache, quantised where it has 8 bits.
//
// Bytes bound both directions. A workgroup takes a few tokens, all their heads' k and
// v rows. A row is taken by the least power of two of lanes that hold it at eight elements
// each (its largest absolute value is found by exchanges among them), kKvAhead
// rows at a time, so that each lane has that many loads in flight; where the tokens'
// rows lie in the cache is found meanwhile, a lane a token, and passed through LDS.
// 32000 rows of 4 heads of 64 in f16, written and read back: 37.2 us a row at a time, 25.3
// to 27.6
// so (a copy reaches 26.7); 4700 of 8 heads of 128 from bf16 to e4m3 and back 26.6 and 19.1.
#include <algorithm>

#include "xp_elem.hpp"

namespace xp {
namespace {

constexpr uint32_t kKvThreads = 256;
constexpr uint32_t kKvAhead = 4;           // rows that a lane sends for at once
constexpr uint32_t kKvTokens = 64, kKvSeqs = 255;

struct KvRows {
    void *         cache[2];       // k, v
    float*         scale[2];
    void*          rows[2];
    uint64_t       stride[2];
    const int32_t *cu, *kv_len;
    PageMap        map;
    uint32_t       n_seq, n_tokens, kv_heads, head_dim, lanes, tokens;
};

// Where the workgroup's tokens lie: the index of head 0's row in the cache, kNoRow
// where the position has none, kNoSeq where the token belongs to no sequence.
constexpr int64_t kNoRow = -1, kNoSeq = -2;
struct KvSlots {
    int32_t cu[kKvSeqs + 1];
    int64_t at[kKvTokens];
};
__device__ __forceinline__ void find_slots(const KvRows& a, KvSlots& s, uint32_t t0) {
    const bool few = a.n_seq <= kKvSeqs;
    if (few && threadIdx.x <= a.n_seq) s.cu[threadIdx.x] = a.cu[threadIdx.x];
    __syncthreads();
    if (threadIdx.x < a.tokens) {
        const uint32_t t = t0 + threadIdx.x;
        int64_t at = kNoSeq;
        if (t < a.n_tokens) {
            const int32_t* cu = few ? s.cu : a.cu;
            const uint32_t b = seq_of_row(cu, a.n_seq, a.n_tokens, t);
            if (b < a.n_seq) {
                const RowSpan r = row_span(cu, a.n_tokens, b);
                const int64_t p = row_position(a.kv_len[b], r.end - r.first, t - r.first);
                if (p >= 0) {
                    const int32_t g = page_of(a.map, b, p);
                    at = g < 0 ? kNoRow : int64_t(cache_row(uint32_t(g), a.kv_heads, 0, a.map.page_shift, uint32_t(p) & ((1u << a.map.page_shift) - 1u)));
                }
            }
        }
        s.at[threadIdx.x] = at;
    }
    __syncthreads();
}
// Row i of the workgroup's: its token (of them), plane and head.
struct KvRow {
    uint32_t token, kv, head;
};
__device__ __forceinline__ KvRow row_of(const KvRows& a, uint32_t i) {
    const uint32_t t = i / (2u * a.kv_heads), w = i - t * 2u * a.kv_heads, kv = w >= a.kv_heads ? 1u : 0u;
    return {t, kv, w - kv * a.kv_heads};
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

// The scale and the eight codes of a row, from the largest of its absolute values'
// bit patterns (as which an infinity is over every number and a NaN over it).
template <int CACHE>
__device__ __forceinline__ float quantise8(const float (&x)[8], uint32_t top, u32x2& code) {
    code = u32x2{0u, 0u};
    if (top >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
    if (top == 0u) return 0.0f;
    if constexpr (CACHE == XP_ELEM_I8) {
        // at least the least normal number, whose reciprocal is finite
        const float scale = fmaxf(__uint_as_float(top) / 127.0f, 0x1p-126f), inv = 1.0f / scale;
#pragma unroll
        for (int j = 0; j < 8; ++j) code[j / 4] |= uint32_t(quantise1(x[j], scale, inv) & 0xFF) << (8 * (j % 4));
        return scale;
    } else {
        // max <= 448 2^k = 1.75 2^(8 + k)
        const int k = max(int(top >> 23) - 135 + ((top & 0x7FFFFFu) > 0x600000u ? 1 : 0), -126);
        const float inv = __uint_as_float(uint32_t(127 - k) << 23);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            int c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j] * inv, x[4 * j + 1] * inv, 0, false);
            c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j + 2] * inv, x[4 * j + 3] * inv, c, true);
            code[j] = uint32_t(c);
        }
        return __uint_as_float(uint32_t(k + 127) << 23);
    }
}

// The largest of a row's lanes' values, in all of them (lanes a power of two, up to 32).
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
    return max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, 0xF, 0xF, true)));
}
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t lanes) {
    if (lanes >= 2) v = dpp_max<0xB1>(v);      // quad_perm [1,0,3,2]
    if (lanes >= 4) v = dpp_max<0x4E>(v);      // quad_perm [2,3,0,1]
    if (lanes >= 8) v = dpp_max<0x141>(v);     // row_half_mirror
    if (lanes >= 16) v = dpp_max<0x140>(v);    // row_mirror
    if (lanes >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = max(uint32_t(r[0]), uint32_t(r[1]));
    }
    return v;
}

template <int IN, int CACHE>
__global__ __launch_bounds__(kKvThreads) void paged_kv_write_kernel(KvRows a) {
    __shared__ KvSlots slots;
    const uint32_t per = kKvThreads / a.lanes, sub = threadIdx.x / a.lanes, lane = threadIdx.x % a.lanes;
    const uint32_t t0 = blockIdx.x * a.tokens, nt = min(a.tokens, a.n_tokens - t0), n = nt * a.kv_heads * 2;
    const bool live = lane * 8 < a.head_dim;
    constexpr uint32_t AHEAD = kKvAhead;
    for (uint32_t i0 = 0; i0 < n; i0 += per * AHEAD) {
        Raw8<IN> raw[AHEAD];
        KvRow r[AHEAD];
#pragma unroll
        for (uint32_t j = 0; j < AHEAD; ++j) {
            const uint32_t i = i0 + j * per + sub;
            r[j] = row_of(a, min(i, n - 1u));
            raw[j].zero();
            if (i < n && live)
                raw[j].load(a.rows[r[j].kv], uint64_t(t0 + r[j].token) * a.stride[r[j].kv] + uint64_t(r[j].head) * a.head_dim + lane * 8);
        }
        if (i0 == 0) find_slots(a, slots, t0);
#pragma unroll
        for (uint32_t j = 0; j < AHEAD; ++j) {
            float x[8];
            raw[j].floats(x);
            const int64_t base = slots.at[r[j].token], row = base + (int64_t(r[j].head) << a.map.page_shift);
            const bool put = base >= 0 && i0 + j * per + sub < n;
            const uint64_t to = uint64_t(row) * a.head_dim + lane * 8;
            if constexpr (CACHE == XP_ELEM_F16 || CACHE == XP_ELEM_BF16) {
                if (put && live) store8<CACHE>(a.cache[r[j].kv], to, x);
            } else {
                uint32_t top = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7FFFFFFFu);
                top = row_max(top, a.lanes);
                u32x2 code;
                const float scale = quantise8<CACHE>(x, top, code);
                if (put && live) *reinterpret_cast<u32x2*>(static_cast<uint8_t*>(a.cache[r[j].kv]) + to) = code;
                if (put && lane == 0) a.scale[r[j].kv][row] = scale;
            }
        }
    }
}

template <int OUT, int CACHE>
__global__ __launch_bounds__(kKvThreads) void paged_kv_read_kernel(KvRows a) {
    __shared__ KvSlots slots;
    const uint32_t per = kKvThreads / a.lanes, sub = threadIdx.x / a.lanes, lane = threadIdx.x % a.lanes;
    const uint32_t t0 = blockIdx.x * a.tokens, nt = min(a.tokens, a.n_tokens - t0), n = nt * a.kv_heads * 2;
    find_slots(a, slots, t0);
    if (lane * 8 >= a.head_dim) return;
    constexpr uint32_t AHEAD = kKvAhead;
    for (uint32_t i0 = 0; i0 < n; i0 += per * AHEAD) {
        Raw8<CACHE> raw[AHEAD];
        float s[AHEAD];
        KvRow r[AHEAD];
#pragma unroll
        for (uint32_t j = 0; j < AHEAD; ++j) {
            r[j] = row_of(a, min(i0 + j * per + sub, n - 1u));
            const int64_t base = slots.at[r[j].token], row = max(base, int64_t(0)) + (int64_t(r[j].head) << a.map.page_shift);
            s[j] = 1.0f;
            raw[j].zero();
            if (base >= 0) {
                raw[j].load(a.cache[r[j].kv], uint64_t(row) * a.head_dim + lane * 8);
                if constexpr (CACHE == XP_ELEM_I8 || CACHE == XP_ELEM_E4M3) s[j] = a.scale[r[j].kv][row];
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < AHEAD; ++j) {
            const int64_t base = slots.at[r[j].token];
            if (i0 + j * per + sub >= n || base == kNoSeq) continue;
            float x[8];
            raw[j].floats(x);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = base < 0 ? __uint_as_float(0x7FC00000u) : CACHE == XP_ELEM_I8 || CACHE == XP_ELEM_E4M3 ? x[e] * s[j] : x[e];
            store8<OUT>(a.rows[r[j].kv], uint64_t(t0 + r[j].token) * a.stride[r[j].kv] + uint64_t(r[j].head) * a.head_dim + lane * 8, x);
        }
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
          page_map(c, s), s->n_seq, s->n_tokens, c->kv_heads, c->head_dim, 1, 1};
    while (a->lanes * 8 < c->head_dim) a->lanes *= 2;
    // tokens of a workgroup: as many as fill its loads once, and no fewer than 1024 workgroups
    const uint32_t at_once = kKvAhead * (kKvThreads / a->lanes) / (2 * c->kv_heads);
    a->tokens = std::max(1u, std::min({at_once, kKvTokens, s->n_tokens / 1024 + 1}));
    const uint32_t groups = (s->n_tokens + a->tokens - 1) / a->tokens;
    if (groups >= 1u << 24) return set_error(XP_E_ARG, "%s: %u tokens are over 2^24 workgroups", fn, s->n_tokens);
    *grid = dim3(groups);
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
