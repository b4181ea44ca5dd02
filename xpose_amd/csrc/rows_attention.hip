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
constexpr uint32_t kJoinSlices = 4;        // workgroups a tile
constexpr int kJoinBatch = 16;             // parts that a wave reads at once

// Workgroup (slice, w) joins the tile that begins in run w and ends behind it, if
// there is one: every kJoinSlices-th row: a wave a row, or, of few rows of many parts,
// all four waves, every fourth part each.
template <int DP>
__global__ __launch_bounds__(kJoinThreads) void rows_attn_join_kernel(AttnRows a) {
    constexpr int PER = DP / kWave;
    typedef float vec __attribute__((ext_vector_type(PER)));
    __shared__ float s_o[kJoinWaves][DP];
    __shared__ float2 s_ml[kJoinWaves];
    const uint32_t lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave), w0 = blockIdx.y;
    const JoinTile p = reinterpret_cast<const JoinTile*>(a.part)[w0];
    const uint32_t n = uniform(p.parts), r0 = p.r0, rows = uniform(p.rows), group = a.heads / a.kv_heads;
    if (n < 2) return;
    const uint64_t size = part_floats(1u << a.row_shift, DP);
    const float* base = part_record(a, w0, false, size);
    const bool all = n >= 2 * kJoinWaves && rows <= kJoinWaves * kJoinSlices;     // all waves a row
    const uint32_t step = all ? kJoinWaves : 1u, at = all ? wave : 0u;
    for (uint32_t r = blockIdx.x + (all ? 0u : wave * kJoinSlices); r < rows; r += kJoinSlices * (all ? 1u : kJoinWaves)) {
        const uint32_t t = by_group(a, r0 + r), head = p.kv_head * group + (r0 + r - t * group);
        float top = -INFINITY, l = 0.0f;
        vec o{};
        for (uint32_t i0 = at; i0 < n; i0 += step * kJoinBatch) {
            float2 ml[kJoinBatch];
            vec x[kJoinBatch];
#pragma unroll
            for (int j = 0; j < kJoinBatch; ++j) {
                const uint32_t i = min(i0 + j * step, n - 1u);
                const float* rec = base + (2ull * i + (i == 0 ? 1u : 0u)) * size;
                ml[j] = reinterpret_cast<const float2*>(rec + (size_t(DP) << a.row_shift))[r];
                x[j] = *reinterpret_cast<const vec*>(rec + size_t(r) * DP + lane * PER);
            }
            float most = top;
#pragma unroll
            for (int j = 0; j < kJoinBatch; ++j) {
                if (i0 + j * step >= n) ml[j] = {-INFINITY, 0.0f};
                most = fmaxf(most, ml[j].x);
            }
            const float keep = top == -INFINITY ? 0.0f : exp2_hw(top - most);
            l *= keep;
            o *= keep;
            top = most;
#pragma unroll
            for (int j = 0; j < kJoinBatch; ++j) {
                const bool in = ml[j].x != -INFINITY;                // it saw something
                const float f = in ? exp2_hw(ml[j].x - top) : 0.0f;
                l += in ? ml[j].y * f : 0.0f;
#pragma unroll
                for (int e = 0; e < PER; ++e) o[e] += in ? x[j][e] * f : 0.0f;
            }
        }
        if (all) __syncthreads();
        *reinterpret_cast<vec*>(&s_o[wave][lane * PER]) = o;
        if (lane == 0) s_ml[wave] = {top, l};
        if (all) __syncthreads();
        const uint32_t d = (all ? threadIdx.x : lane) * 4;
        if (d < a.head_dim && p.past + int32_t(t) >= 0) {
            const uint32_t v0 = all ? 0u : wave, v1 = all ? kJoinWaves : wave + 1u;
            float most = -INFINITY, sum = 0.0f;
            for (uint32_t v = v0; v < v1; ++v) most = fmaxf(most, s_ml[v].x);
            f32x4 y{0.0f, 0.0f, 0.0f, 0.0f};
            for (uint32_t v = v0; v < v1; ++v) {
                const float2 ml = s_ml[v];
                if (ml.x == -INFINITY) continue;
                const float f = exp2_hw(ml.x - most);
                sum += ml.y * f;
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] += s_o[v][d + j] * f;
            }
            store_row4(a, p.first + t, head, d, y, sum);
        }
    }
}

// ---- which kernel, and how the work is dealt ----------------------------------------
struct AttnPlan {
    bool     few;
    uint32_t row_shift, tiles, target;     // the most tiles; target 0: a workgroup for each
    size_t   part_bytes;
};
constexpr uint32_t kCus = 256;
AttnPlan attn_plan(bool paged, uint32_t n_tokens, uint32_t n_seq, uint32_t heads, uint32_t kv_heads, uint32_t head_dim) {
    AttnPlan p{};
    const uint64_t rows = uint64_t(n_tokens) * (heads / kv_heads);
    const uint32_t seqs = std::min(n_seq, n_tokens);
    p.few = paged && rows <= uint64_t(seqs) * 2 * kFewRows;
    const uint32_t tile = p.few ? kFewRows : kTileRows;
    p.row_shift = uint32_t(__builtin_ctz(tile));
    // every sequence with rows may leave one tile part filled
    const uint64_t tiles = (rows / tile + seqs) * kv_heads;
    p.tiles = uint32_t(std::min<uint64_t>(tiles, 0x7FFFFFFFu));
    if (tiles < (p.few ? 16 : 4) * kCus) {
        p.target = padded_dim(head_dim) == 256 ? kCus : 2 * kCus;          // what fits the device at once
        p.part_bytes = size_t(p.target) * (sizeof(JoinTile) + 2 * part_floats(tile, padded_dim(head_dim)) * sizeof(float));
    }
    return p;
}

int attention_call(const char* fn, AttnRows a, const AttnPlan& p, int cache, bool paged, void* workspace, hipStream_t st) {
    const uint32_t dp = padded_dim(a.head_dim);
    set_group(a);
    a.row_shift = p.row_shift;
    a.block_shift = uint32_t(__builtin_ctz(p.few ? kFewWaves * few_keys(dp, elem_bytes(cache)) : tile_keys_of(dp)));
    // what the list may hold, and 32-bit places in it
    const uint64_t most = uint64_t(p.tiles) * ((uint64_t(a.most_keys) >> a.block_shift) + 4);
    a.target = workspace && most < 0x7FFFFFFFull ? p.target : 0u;
    a.target_shift = a.target ? uint32_t(__builtin_ctz(a.target)) : 0u;
    a.most_blocks = uint32_t(std::min<uint64_t>(most, 0x7FFFFFFFu));
    a.part = static_cast<float*>(workspace);
    const uint32_t grid = a.target ? a.target : p.tiles;
    XP_CHECK(p.few ? launch_few(a, cache, grid, st) : launch_tile(a, cache, paged, grid, st));
    if (a.target == 0) return XP_OK;
    const dim3 join(kJoinSlices, a.target), block(kJoinThreads);
    if (dp == 64) hipLaunchKernelGGL((rows_attn_join_kernel<64>), join, block, 0, st, a);
    else if (dp == 128) hipLaunchKernelGGL((rows_attn_join_kernel<128>), join, block, 0, st, a);
    else hipLaunchKernelGGL((rows_attn_join_kernel<256>), join, block, 0, st, a);
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
    a.most_keys = int32_t(std::min<uint64_t>(uint64_t(s->table) * c->page_size, kMostKeys));
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
    a.most_keys = int32_t(std::min<uint32_t>(n_tokens, kMostKeys));
    return attention_call(__func__, a, attn_plan(false, n_tokens, n_seq, a.heads, a.kv_heads, head_dim), k->elem, false, workspace,
                          as_stream(stream));
}

}  // extern "C"
