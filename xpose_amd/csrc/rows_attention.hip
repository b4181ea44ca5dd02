// Attention of packed rows: over a paged cache, and over packed prompts.
//
// out_i = sum_j p_ij v_j / sum_j p_ij, p_ij = exp(s_ij - max_j s_ij), s_ij =
// scale q_i . k_j, over the positions j that i sees. The running maximum and
// sum make it one pass over the keys: when the maximum rises from m to m', what
// has been summed is multiplied by exp(m - m').
//
// The products are made by two kernels, for few rows a sequence
// (rows_attn_few.hip) and for many (rows_attn_tile.hip). Where the rows alone
// leave CUs without work the keys are split, and a second kernel joins the parts.
#include <algorithm>

#include "xp_rows_attn.hpp"

namespace xp {
namespace {

constexpr uint32_t kJoinThreads = 256, kJoinWaves = kJoinThreads / kWave;

// A workgroup joins the parts of one row: the sums relative to the largest
// reference, each wave every fourth part.
template <int DP>
__global__ __launch_bounds__(kJoinThreads) void rows_attn_join_kernel(AttnRows a) {
    constexpr int PER = DP / kWave;
    __shared__ float s_o[kJoinWaves][DP];
    __shared__ float s_l[kJoinWaves];
    const uint32_t t = blockIdx.x / a.heads, head = blockIdx.x % a.heads, lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave);
    const uint32_t seq = seq_of_row(a.cu, a.n_seq, a.n_tokens, t);
    if (seq >= a.n_seq) return;
    const TileSeq ts = tile_seq(a, seq);
    if (ts.past + int32_t(t - ts.first) < 0) return;
    const uint32_t group = a.heads / a.kv_heads, row = (t - ts.first) * group + head % group;
    const uint32_t tile = row >> a.row_shift, r = row & ((1u << a.row_shift) - 1u), tile_rows = 1u << a.row_shift;
    uint32_t n;
    const uint32_t first = deal_first(a, seq, tile, head / group, &n);
    if (n == 0 || uint64_t(first) + uint64_t(n - 1u) * a.kv_heads >= a.items) return;    // a cu that gives rows twice
    const float* base = a.part + uint64_t(first) * part_floats(tile_rows, DP);
    const uint64_t step = uint64_t(a.kv_heads) * part_floats(tile_rows, DP);
    auto ml = [&](uint32_t p) { return reinterpret_cast<const float2*>(base + p * step + tile_rows * DP)[r]; };
    float top = -INFINITY;
    for (uint32_t p = lane; p < n; p += kWave) top = fmaxf(top, ml(p).x);
    top = wave_max(top);
    float o[PER] = {}, l = 0.0f;
    for (uint32_t p = wave; p < n; p += kJoinWaves) {
        const float2 w = ml(p);
        if (w.x == -INFINITY) continue;            // it saw nothing
        const float f = exp2_hw(w.x - top);
        const float* x = base + p * step + r * DP + lane * PER;
        l += w.y * f;
#pragma unroll
        for (int j = 0; j < PER; ++j) o[j] += x[j] * f;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) s_o[wave][lane * PER + j] = o[j];
    if (lane == 0) s_l[wave] = l;
    __syncthreads();
    const uint32_t d = threadIdx.x * 4;
    if (d >= a.head_dim) return;
    f32x4 v{0.0f, 0.0f, 0.0f, 0.0f};
    float sum = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < kJoinWaves; ++w) {
        sum += s_l[w];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += s_o[w][d + j];
    }
    store_row4(a, t, head, d, v, sum);
}

// ---- which kernel, and whether to split ------------------------------------------
struct AttnPlan {
    bool     few;
    uint32_t row_shift, items, target;     // items: the grid; target 0: the keys are not split
    size_t   part_bytes;
};
constexpr uint32_t kCus = 256;
// The tiles of a call, at most: every sequence with rows may leave one part-filled.
uint64_t most_tiles(uint32_t n_tokens, uint32_t n_seq, uint32_t heads, uint32_t kv_heads, uint32_t rows) {
    return (uint64_t(n_tokens) * (heads / kv_heads) / rows + std::min(n_seq, n_tokens)) * kv_heads;
}
AttnPlan attn_plan(bool paged, uint32_t n_tokens, uint32_t n_seq, uint32_t heads, uint32_t kv_heads, uint32_t head_dim) {
    AttnPlan p{};
    const uint64_t rows = uint64_t(n_tokens) * (heads / kv_heads);
    p.few = paged && rows <= uint64_t(std::min(n_seq, n_tokens)) * 2 * kFewRows;
    const uint32_t tile = p.few ? kFewRows : kTileRows;
    p.row_shift = uint32_t(__builtin_ctz(tile));
    const uint64_t tiles = most_tiles(n_tokens, n_seq, heads, kv_heads, tile);
    const uint64_t enough = p.few ? 8 * kCus : 2 * kCus;
    if (tiles < enough) {
        p.target = p.few ? 4 * kCus : 2 * kCus;
        p.part_bytes = size_t((tiles + p.target) * part_floats(tile, padded_dim(head_dim)) * sizeof(float));
    }
    p.items = uint32_t(std::min<uint64_t>(tiles + p.target, 0x7FFFFFFFu));
    return p;
}

int attention_call(const char* fn, AttnRows a, const AttnPlan& plan, int cache, bool paged, void* workspace, hipStream_t st) {
    AttnPlan p = plan;
    if (!workspace) p.target = 0;
    a.target = p.target;
    a.part = static_cast<float*>(workspace);
    a.row_shift = p.row_shift;
    a.items = p.items;
    const uint32_t dp = padded_dim(a.head_dim);
    const uint32_t block = p.few ? kFewWaves * few_keys(dp, elem_bytes(cache)) : tile_keys_of(dp);
    a.block_shift = uint32_t(__builtin_ctz(block));
    XP_CHECK(p.few ? launch_few(a, cache, p.items, st) : launch_tile(a, cache, paged, p.items, st));
    if (p.target == 0) return XP_OK;
    const dim3 grid(a.n_tokens * a.heads);
    if (dp == 64) hipLaunchKernelGGL((rows_attn_join_kernel<64>), grid, dim3(kJoinThreads), 0, st, a);
    else if (dp == 128) hipLaunchKernelGGL((rows_attn_join_kernel<128>), grid, dim3(kJoinThreads), 0, st, a);
    else hipLaunchKernelGGL((rows_attn_join_kernel<256>), grid, dim3(kJoinThreads), 0, st, a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return set_error(XP_E_HIP, "%s: kernel launch -> %s", fn, hipGetErrorString(e));
    return XP_OK;
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
    if (!(scale > 0.0f) || scale - scale != 0.0f) return set_error(XP_E_ARG, "%s: scale %g is not positive and finite", fn, double(scale));
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
    *bytes = std::max<size_t>({16, attn_plan(true, n_tokens, n_seq, heads, kv_heads, head_dim).part_bytes,
                               attn_plan(false, n_tokens, n_seq, heads, kv_heads, head_dim).part_bytes});
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
    AttnRows a{};
    a.q = q->data, a.k = c->k, a.v = c->v, a.out = out->data, a.k_scale = c->k_scale, a.v_scale = c->v_scale;
    a.q_stride = q->stride, a.out_stride = out->stride;
    a.cu = s->cu, a.kv_len = s->kv_len, a.map = page_map(c, s), a.n_seq = s->n_seq, a.n_tokens = s->n_tokens;
    a.heads = q->heads, a.kv_heads = c->kv_heads, a.head_dim = c->head_dim, a.window = window, a.q_elem = q->elem, a.scale = scale;
    return attention_call(__func__, a, attn_plan(true, a.n_tokens, a.n_seq, a.heads, a.kv_heads, a.head_dim), c->elem, true, workspace,
                          as_stream(stream));
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
    AttnRows a{};
    a.q = q->data, a.k = k->data, a.v = v->data, a.out = out->data;
    a.q_stride = q->stride, a.k_stride = k->stride, a.v_stride = v->stride, a.out_stride = out->stride;
    a.cu = cu, a.n_seq = n_seq, a.n_tokens = n_tokens;
    a.heads = q->heads, a.kv_heads = k->heads, a.head_dim = head_dim, a.window = window, a.q_elem = q->elem, a.scale = scale;
    return attention_call(__func__, a, attn_plan(false, n_tokens, n_seq, a.heads, a.kv_heads, head_dim), k->elem, false, workspace,
                          as_stream(stream));
}

}  // extern "C"
