// Attention of packed rows: over a paged cache, and over packed prompts.
//
// out_i = sum_j p_ij v_j / sum_j p_ij, p_ij = exp(s_ij - max_j s_ij), s_ij =
// scale q_i . k_j, over the positions j that i sees. The running maximum and
// sum make it one pass over the keys: when the maximum rises from m to m', what
// has been summed is multiplied by exp(m - m').
//
// The simple form: a wave takes one query head of one token and its keys one
// by one.
#include <algorithm>

#include "xp_elem.hpp"

namespace xp {
namespace {

struct AttnRows {
    const void *q, *k, *v;         // k, v: the cache's planes, or the packed rows
    void*       out;
    const float *k_scale, *v_scale;
    uint64_t    q_stride, k_stride, v_stride, out_stride;
    const int32_t *cu, *kv_len;    // kv_len NULL: packed
    PageMap     map;
    uint32_t    n_seq, n_tokens, heads, kv_heads, head_dim, window;
    float       scale;
};
constexpr int kMostDims = 256 / kWave;

template <int Q, int KV, bool PAGED>
__global__ __launch_bounds__(kWave) void rows_attention_kernel(AttnRows a) {
    const uint32_t t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, D = a.head_dim;
    const uint32_t kvh = h / (a.heads / a.kv_heads);
    const uint32_t b = seq_of_row(a.cu, a.n_seq, a.n_tokens, t);
    if (b >= a.n_seq) return;
    const RowSpan r = row_span(a.cu, a.n_tokens, b);
    const uint32_t n = r.end - r.first;
    const int64_t p = row_position(PAGED ? a.kv_len[b] : int32_t(n), n, t - r.first);
    if (p < 0) return;
    float q[kMostDims], o[kMostDims];
    const uint64_t qi = uint64_t(t) * a.q_stride + uint64_t(h) * D;
#pragma unroll
    for (int j = 0; j < kMostDims; ++j) {
        const uint32_t d = lane + j * kWave;
        q[j] = d < D ? load1<Q>(a.q, qi + d) : 0.0f;
        o[j] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    bool whole = true;
    for (int64_t j = a.window && p >= a.window ? p - a.window + 1 : 0; j <= p; ++j) {
        uint64_t ki, vi;
        float ks = 1.0f, vs = 1.0f;
        if constexpr (PAGED) {
            const int32_t g = page_of(a.map, b, j);
            if (g < 0) {
                whole = false;
                break;
            }
            const uint64_t row = cache_row(uint32_t(g), a.kv_heads, kvh, a.map.page_shift, uint32_t(j) & ((1u << a.map.page_shift) - 1u));
            ki = vi = row * D;
            if constexpr (KV == XP_ELEM_I8 || KV == XP_ELEM_E4M3) ks = a.k_scale[row], vs = a.v_scale[row];
        } else {
            ki = uint64_t(r.first + j) * a.k_stride + uint64_t(kvh) * D;
            vi = uint64_t(r.first + j) * a.v_stride + uint64_t(kvh) * D;
        }
        float s = 0.0f, v[kMostDims];
#pragma unroll
        for (int x = 0; x < kMostDims; ++x) {
            const uint32_t d = lane + x * kWave;
            if (d < D) s = fmaf(q[x], load1<KV>(a.k, ki + d), s);
            v[x] = d < D ? load1<KV>(a.v, vi + d) : 0.0f;
        }
        s = wave_sum(s) * ks * a.scale;
        const float top = fmaxf(m, s);
        const float keep = top == m ? 1.0f : exp_hw(m - top), w = exp_hw(s - (top == -INFINITY ? 0.0f : top));
        m = top;
        l = l * keep + w;
#pragma unroll
        for (int x = 0; x < kMostDims; ++x) o[x] = o[x] * keep + w * (v[x] * vs);
    }
    const float norm = whole ? (l > 0.0f || l != l ? 1.0f / l : 0.0f) : __uint_as_float(0x7FC00000u);
    const uint64_t oi = uint64_t(t) * a.out_stride + uint64_t(h) * D;
#pragma unroll
    for (int x = 0; x < kMostDims; ++x)
        if (lane + x * kWave < D) store1<Q>(a.out, oi + lane + x * kWave, o[x] * norm);
}

int check_attention(const char* fn, const xp_rows* out, const xp_rows* q, uint32_t head_dim, uint32_t kv_heads,
                    uint32_t n_tokens, float scale, const void* workspace, size_t bytes, uint32_t n_seq) {
    XP_CHECK(check_rows(fn, "q", q, head_dim, 16));
    XP_CHECK(check_rows(fn, "out", out, head_dim, 16));
    if (out->heads != q->heads || out->elem != q->elem) return set_error(XP_E_ARG, "%s: out has not q's heads and elem", fn);
    if (out->data == q->data) return set_error(XP_E_ARG, "%s: out must not be q", fn);
    if (q->heads % kv_heads) return set_error(XP_E_ARG, "%s: %u heads are no multiple of %u kv heads", fn, q->heads, kv_heads);
    if (uint64_t(n_tokens) * q->heads > 0x7FFFFFFFull)
        return set_error(XP_E_ARG, "%s: %u tokens of %u heads are over 2^31 - 1", fn, n_tokens, q->heads);
    if (!(scale == scale) || scale - scale != 0.0f) return set_error(XP_E_ARG, "%s: scale is not finite", fn);
    if (workspace) {
        size_t need = 0;
        XP_CHECK(xp_attention_workspace(n_tokens, n_seq, q->heads, kv_heads, head_dim, &need));
        if (bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16)
            return set_error(XP_E_ARG, "%s: a workspace of %zu bytes, or not 16-byte aligned: %zu are needed", fn, bytes, need);
    }
    return XP_OK;
}

}  // namespace
}  // namespace xp

using namespace xp;

extern "C" {

int xp_attention_workspace(uint32_t n_tokens, uint32_t n_seq, uint32_t heads, uint32_t kv_heads, uint32_t head_dim,
                           size_t* bytes) {
    XP_REQUIRE(bytes, "bytes is null");
    XP_REQUIRE(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, "%u heads are no multiple of %u kv heads", heads, kv_heads);
    XP_REQUIRE(head_dim > 0 && head_dim % 16 == 0 && head_dim <= 256, "head_dim %u is not a multiple of 16 up to 256", head_dim);
    *bytes = 16;
    return XP_OK;
}

int xp_attention_paged(const xp_rows* out, const xp_rows* q, const xp_paged_kv* c, const xp_paged_seqs* s,
                       uint32_t window, float scale, void* workspace, size_t workspace_bytes, xp_stream stream) {
    XP_CHECK(check_cache(__func__, c));
    XP_CHECK(check_seqs(__func__, s));
    XP_CHECK(check_attention(__func__, out, q, c->head_dim, c->kv_heads, s->n_tokens, scale, workspace, workspace_bytes, s->n_seq));
    XP_REQUIRE(c->elem != XP_ELEM_BF16 || q->elem == XP_ELEM_BF16, "a BF16 cache takes BF16 queries");
    if (s->n_tokens == 0 || s->n_seq == 0) return XP_OK;
    XP_CHECK(check_here(__func__, stream, out->data));
    const AttnRows a{q->data, c->k, c->v, out->data, c->k_scale, c->v_scale, q->stride, 0, 0, out->stride, s->cu, s->kv_len,
                     page_map(c, s), s->n_seq, s->n_tokens, q->heads, c->kv_heads, c->head_dim, window, scale};
    const dim3 grid(s->n_tokens, q->heads);
#define XP_PAGED(Q, KV) hipLaunchKernelGGL((rows_attention_kernel<Q, KV, true>), grid, dim3(kWave), 0, as_stream(stream), a)
#define XP_PAGED_Q(KV)                                              \
    if (q->elem == XP_ELEM_F32) XP_PAGED(XP_ELEM_F32, KV);          \
    else if (q->elem == XP_ELEM_F16) XP_PAGED(XP_ELEM_F16, KV);     \
    else XP_PAGED(XP_ELEM_BF16, KV);
    if (c->elem == XP_ELEM_BF16) {
        XP_PAGED(XP_ELEM_BF16, XP_ELEM_BF16);
    } else if (c->elem == XP_ELEM_F16) {
        XP_PAGED_Q(XP_ELEM_F16)
    } else if (c->elem == XP_ELEM_I8) {
        XP_PAGED_Q(XP_ELEM_I8)
    } else {
        XP_PAGED_Q(XP_ELEM_E4M3)
    }
#undef XP_PAGED_Q
#undef XP_PAGED
    XP_LAUNCHED();
    return XP_OK;
}

int xp_attention_packed(const xp_rows* out, const xp_rows* q, const xp_rows* k, const xp_rows* v, uint32_t head_dim,
                        uint32_t n_seq, uint32_t n_tokens, const int32_t* cu, uint32_t window, float scale,
                        void* workspace, size_t workspace_bytes, xp_stream stream) {
    XP_REQUIRE(head_dim > 0 && head_dim % 16 == 0 && head_dim <= 256, "head_dim %u is not a multiple of 16 up to 256", head_dim);
    XP_REQUIRE(n_seq <= (1u << 24) && n_tokens <= 0x7FFFFFFFu, "%u sequences, %u tokens: too many", n_seq, n_tokens);
    XP_CHECK(check_rows(__func__, "k", k, head_dim, 16));
    XP_CHECK(check_rows(__func__, "v", v, head_dim, 16));
    XP_CHECK(check_attention(__func__, out, q, head_dim, k->heads, n_tokens, scale, workspace, workspace_bytes, n_seq));
    XP_REQUIRE(v->heads == k->heads, "k has %u heads, v %u", k->heads, v->heads);
    XP_REQUIRE(q->elem != XP_ELEM_F32 && k->elem == q->elem && v->elem == q->elem, "q, k and v are all F16 or all BF16");
    if (n_tokens == 0 || n_seq == 0) return XP_OK;
    XP_REQUIRE(cu, "cu is null");
    XP_CHECK(check_here(__func__, stream, out->data));
    const AttnRows a{q->data, k->data, v->data, out->data, nullptr, nullptr, q->stride, k->stride, v->stride, out->stride, cu,
                     nullptr, PageMap{}, n_seq, n_tokens, q->heads, k->heads, head_dim, window, scale};
    const dim3 grid(n_tokens, q->heads);
    if (q->elem == XP_ELEM_F16)
        hipLaunchKernelGGL((rows_attention_kernel<XP_ELEM_F16, XP_ELEM_F16, false>), grid, dim3(kWave), 0, as_stream(stream), a);
    else
        hipLaunchKernelGGL((rows_attention_kernel<XP_ELEM_BF16, XP_ELEM_BF16, false>), grid, dim3(kWave), 0, as_stream(stream), a);
    XP_LAUNCHED();
    return XP_OK;
}

}  // extern "C"
