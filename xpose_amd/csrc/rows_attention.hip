// Attention of packed rows: over a paged cache, and over packed prompts.
//
// out_i = sum_j p_ij v_j / sum_j p_ij, p_ij = exp(s_ij - max_j s_ij), s_ij =
// scale q_i . k_j, over the positions j that i sees. The running maximum and
// sum make it one pass over the keys: when the maximum rises from m to m', what
// has been summed is multiplied by exp(m - m').
//
// The products are made by three kernels: for few rows a sequence (rows_attn_few.hip,
// tiles of 16), for many (rows_attn_tile.hip, 128), and for prompts whose tiles of 128
// would leave CUs without work (rows_attn_mid.hip, 32). The first two may also take the
// blocks of all tiles as one list in equal runs, whose parts the kernel below joins.
#include <algorithm>
#include <cmath>

#include "xp_rows_attn.hpp"

namespace xp {
namespace {

constexpr uint32_t kJoinThreads = 256, kJoinWaves = kJoinThreads / kWave, kJoinGrid = 1024;
constexpr uint32_t kMostTarget = 512;
constexpr int kJoinBatch = 8;              // parts that a wave reads at once

// The rows of all tiles that more than one workgroup worked on, shared out evenly: a
// workgroup a row where there are no more rows than that, each wave every fourth part;
// else a wave a row.
template <int DP>
__global__ __launch_bounds__(kJoinThreads) void rows_attn_join_kernel(AttnRows a) {
    constexpr int PER = DP / kWave, TW = kMostTarget / kJoinThreads;
    typedef float vec __attribute__((ext_vector_type(PER)));
    __shared__ float s_o[kJoinWaves][DP];
    __shared__ float2 s_ml[kJoinWaves];
    __shared__ uint32_t s_up[kMostTarget], s_sum[kJoinWaves];
    const uint32_t lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave);
    const JoinTile* tiles = reinterpret_cast<const JoinTile*>(a.part);
    // the rows up to and with each workgroup's tile
    uint32_t mine[TW], sum = 0;
#pragma unroll
    for (int j = 0; j < TW; ++j) {
        const uint32_t w = threadIdx.x * TW + j;
        mine[j] = w < a.target && tiles[w].parts > 1u ? tiles[w].rows : 0u;
        sum += mine[j];
    }
    const uint32_t up = wave_scan_add(sum);
    if (lane == kWave - 1) s_sum[wave] = up;
    __syncthreads();
    uint32_t before = up - sum, total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kJoinWaves; ++w) {
        before += w < wave ? s_sum[w] : 0u;
        total += s_sum[w];
    }
#pragma unroll
    for (int j = 0; j < TW; ++j) s_up[threadIdx.x * TW + j] = before += mine[j];
    __syncthreads();
    total = uniform(total);
    const bool all = total <= kJoinGrid;
    const uint32_t group = a.heads / a.kv_heads, step = all ? kJoinWaves : 1u, at = all ? wave : 0u;
    const uint64_t size = part_floats(1u << a.row_shift, DP);
    for (uint32_t i = all ? blockIdx.x : blockIdx.x * kJoinWaves + wave; i < total; i += kJoinGrid * (all ? 1u : kJoinWaves)) {
        uint32_t w0 = 0;                   // the first tile whose sum is over i
#pragma unroll
        for (uint32_t s = kMostTarget / 2; s > 0; s /= 2) w0 += s_up[w0 + s - 1u] <= i ? s : 0u;
        w0 = uniform(w0);
        const JoinTile p = tiles[w0];
        const uint32_t n = uniform(p.parts), r = uniform(i - (s_up[w0] - p.rows));
        const uint32_t t = by_group(a, p.r0 + r), head = p.kv_head * group + (p.r0 + r - t * group);
        const float* base = part_record(a, w0, false, size);
        float top = -INFINITY, l = 0.0f;
        vec o{};
        for (uint32_t i0 = at; i0 < n; i0 += step * kJoinBatch) {
            float2 ml[kJoinBatch];
            vec x[kJoinBatch];
#pragma unroll
            for (int j = 0; j < kJoinBatch; ++j) {
                const uint32_t k = min(i0 + j * step, n - 1u);
                const float* rec = base + (2ull * k + (k == 0 ? 1u : 0u)) * size;
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
            float most = -INFINITY, s = 0.0f;
            for (uint32_t v = v0; v < v1; ++v) most = fmaxf(most, s_ml[v].x);
            f32x4 y{0.0f, 0.0f, 0.0f, 0.0f};
            for (uint32_t v = v0; v < v1; ++v) {
                const float2 ml = s_ml[v];
                if (ml.x == -INFINITY) continue;
                const float f = exp2_hw(ml.x - most);
                s += ml.y * f;
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] += s_o[v][d + j] * f;
            }
            store_row4(a, p.first + t, head, d, y, s);
        }
    }
}

// ---- which kernel, and how the work is dealt ----------------------------------------
enum class AttnKind { few, mid, tile };
struct AttnPlan {
    AttnKind kind;
    uint32_t row_shift, tiles, target, least_run;     // tiles: at most; target 0: a workgroup for each
};
constexpr uint32_t kCus = 256;
// Few rows a sequence of a cache go to rows_attn_few.hip (a tile of 16 rows reads its keys
// once, so up to 32), the others to the kernel that takes least by this estimate, in us: `keys`
// is what a sequence has, as far as the host knows (of a cache, what its tables hold;
// half of a prompt's tokens on average), a block 64 keys of 128 dims for 128 rows.
//   mid    8 for each round of workgroups, and 0.075 a key of a wave (a quarter of the keys)
//   tile   8, and the longer of the longest tile (1.75 a block, 2.4 where workgroups
//          share CUs) and all blocks at 0.005
//   list   24 (256 dims: 36) for the second piece and the join, and all blocks at 0.0055
// and of the first kernel, with all it reads, tables taken as half full, at 7 bytes a ps:
//   tiles  4.5 (7), and 0.0095 a key of 128 dims in the longest, or all, and half that
//   list   12 (13.5) with the join, 11 a tile that a workgroup takes, and all
// Measured, mid / tile / list: prompts of 2000 in 4 heads over 1 of 256 66 / 125 / 56,
// with a window of 512 36 / 47 / 48; prompts over 8 kv heads of 128 of 100 tokens 9.9 /
// 11.6 / 16, of 1000 40 / 35 / 55, of 2000 94 / 64 / 102; chunks of 512 over 1000 34 / 44 /
// 52, of 100 (four) over 1000 27 / 36 / 40, of 64 over 8000 109 / 185 / 37, of 200 over
// 30000 371 / 665 / 160.
// Of the first, single rows over 8 kv heads of 128, tiles / list: 1 sequence of 100 4.5 / 8.7,
// of 500 8.5 / 11.0, of 1000 13.8 / 11.1, of 2000 23 / 11; 16 of 500 10.5 / 16, of 2000 27 /
// 29; 64 up to 2000 55 / 63, up to 8000 197 / 179; 256 up to 2000 179 / 215; 4 heads over 1 of
// 256, F32 over F16, 1 of 130 10.1 / 13.4, of 400 15.5 / 13.8, of 2000 48 / 14.
bool few_rows(uint64_t rows, uint32_t seqs) { return rows <= uint64_t(seqs) * 2 * kFewRows; }
uint32_t slots_of(uint32_t dp) { return dp == 256 ? kCus : 2 * kCus; }      // workgroups that run at once
AttnPlan attn_plan(bool paged, uint32_t n_tokens, uint32_t n_seq, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t bytes,
                   double keys, bool may_list) {
    AttnPlan p{};
    const uint64_t rows = uint64_t(n_tokens) * (heads / kv_heads);
    const uint32_t seqs = std::min(n_seq, n_tokens), dp = padded_dim(head_dim);
    // every sequence with rows may leave one tile part filled
    auto tiles = [&](uint32_t tile) { return (rows / tile + seqs) * kv_heads; };
    const uint32_t slots = slots_of(dp);
    bool list = false;
    const double dims = dp / 128.0;
    if (paged && few_rows(rows, seqs)) {
        p.kind = AttnKind::few;
        const double n = double(tiles(kFewRows)), all = n * keys / 2 * (2.0 * dp * bytes) / 7e6, longest = 0.0095 * dims * keys;
        const double t_tiles = (dp == 256 ? 7 : 4.5) + std::max(longest, all + longest / 2);
        list = may_list && (dp == 256 ? 13.5 : 12) + 11 * n / slots + all < t_tiles;
    } else {
        const double mean = paged ? keys : keys / 2;
        const double big = double(tiles(kTileRows)), rounds = std::ceil(double(rows) * kv_heads / kMidRows / slots);
        const double t_mid = 8 * rounds + std::max(rounds * mean, keys) / 4 * 0.075 * dims;
        const double t_tile = 8 + std::max(keys / 64 * (big > kCus ? 2.4 : 1.75), big * mean / 64 * 0.005) * dims;
        const double t_list = (dp == 256 ? 36 : 24) + big * mean / 64 * 0.0055 * dims * (dp == 256 ? 2 : 1);
        list = may_list && t_list < t_mid && t_list < t_tile;
        p.kind = list || t_tile <= t_mid ? AttnKind::tile : AttnKind::mid;
    }
    const uint32_t tile = p.kind == AttnKind::few ? kFewRows : p.kind == AttnKind::mid ? kMidRows : kTileRows;
    p.row_shift = uint32_t(__builtin_ctz(tile));
    p.tiles = uint32_t(std::min<uint64_t>(tiles(tile), 0x7FFFFFFFu));
    if (list) {
        p.target = slots;
        static_assert(2 * kCus <= kMostTarget, "the join's table");
        p.least_run = p.kind == AttnKind::few ? 0 : 2;
    }
    return p;
}
size_t part_bytes(uint32_t target, uint32_t tile, uint32_t head_dim) {
    return size_t(target) * (sizeof(JoinTile) + 2 * part_floats(tile, padded_dim(head_dim)) * sizeof(float));
}

int attention_call(const char* fn, AttnRows a, bool paged, int cache, void* workspace, size_t bytes, hipStream_t st) {
    const uint32_t dp = padded_dim(a.head_dim);
    double keys = paged ? double(a.most_keys) : double(a.n_tokens) / a.n_seq;
    if (a.window) keys = std::min(keys, double(a.window) + double(kTileRows) / (a.heads / a.kv_heads));
    const AttnPlan p = attn_plan(paged, a.n_tokens, a.n_seq, a.heads, a.kv_heads, a.head_dim, elem_bytes(cache), keys, workspace != nullptr);
    set_group(a);
    a.row_shift = p.row_shift;
    a.block_shift = uint32_t(__builtin_ctz(p.kind == AttnKind::few   ? kFewWaves * few_keys(dp, elem_bytes(cache))
                                           : p.kind == AttnKind::mid ? kMidKeys
                                                                     : tile_keys_of(dp)));
    // what the list may hold, and 32-bit places in it
    const uint64_t most = uint64_t(p.tiles) * ((uint64_t(a.most_keys) >> a.block_shift) + 4);
    a.target = most < 0x7FFFFFFFull && part_bytes(p.target, 1u << p.row_shift, a.head_dim) <= bytes ? p.target : 0u;
    a.least_run = p.least_run;
    a.target_shift = a.target ? uint32_t(__builtin_ctz(a.target)) : 0u;
    a.most_blocks = uint32_t(std::min<uint64_t>(most, 0x7FFFFFFFu));
    a.part = static_cast<float*>(workspace);
    const uint32_t grid = a.target ? a.target : p.tiles;
    if (grid >= 1u << 24) return set_error(XP_E_ARG, "%s: %u tokens of %u heads are over 2^24 tiles of %u rows", fn, a.n_tokens, a.heads, 1u << p.row_shift);
    XP_CHECK(p.kind == AttnKind::few   ? launch_few(a, cache, grid, st)
             : p.kind == AttnKind::mid ? launch_mid(a, cache, paged, grid, st)
                                       : launch_tile(a, cache, paged, grid, st));
    if (a.target == 0) return XP_OK;
    const dim3 join(kJoinGrid), block(kJoinThreads);
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
    // whatever the lengths: what a list of the tiles of so many rows takes
    const bool few = few_rows(uint64_t(n_tokens) * (heads / kv_heads), std::min(n_seq, n_tokens));
    *bytes = part_bytes(slots_of(padded_dim(head_dim)), few ? kFewRows : kTileRows, head_dim);
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
    return attention_call(__func__, a, true, c->elem, workspace, workspace_bytes, as_stream(stream));
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
    return attention_call(__func__, a, false, k->elem, workspace, workspace_bytes, as_stream(stream));
}

}  // extern "C"
