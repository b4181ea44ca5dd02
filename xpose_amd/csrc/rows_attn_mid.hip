// Attention of short prompts and chunks: tiles of 32 rows, a workgroup's four waves each
// at keys of their own, so that there are four times the tiles of rows_attn_tile.hip
// where those would leave CUs without work. The 32 rows of a wave are xp_rows_attn32.hpp's.
//
// A wave's keys go through LDS of its own, 32 at a time, K and V in one buffer each: the
// next K is on its way from the end of the scores on, the next V from the end of the
// values on, and no barrier is needed until the waves' sums meet.
//
// Latency bounds it: a step of a wave's 32 keys takes 2.4 us (its products 0.25), with one wave
// a SIMD at 256 dims, two at less. A prompt of 2000 rows of 4 heads over 1 of 256 with a
// window of 512 takes 32 us; as tiles of 128 rows 47, as a list 48.
#include "xp_rows_attn32.hpp"

namespace xp {
namespace {

constexpr uint32_t kMidThreads = kMidWaves * kWave;

template <int CACHE, int DP, int TERMS, bool PAGED>
__global__ __launch_bounds__(kMidThreads, DP == 256 || TERMS == 2 ? 1 : 2) void rows_attn_mid_kernel(AttnRows a) {
    typedef Rows32<CACHE, DP, TERMS, 1> R;
    constexpr int SZ = R::SZ, RB = R::RB, NC = R::NC, RPI = R::RPI, KT = 32, OT = R::OT;
    constexpr int LOADS = KT / RPI, OPS = LOADS + (SZ == 1 ? 1 : 0);       // of K, and of V
    constexpr int STEP = int(kMidWaves) * KT;
    struct __attribute__((aligned(16))) Stage {
        unsigned char k[KT * RB], v[KT * RB];
    };
    __shared__ Stage s_kv[kMidWaves];
    __shared__ float s_scale[SZ == 1 ? kMidWaves : 1][2][KT];
    __shared__ uint32_t s_bad[kMidWaves];
    __shared__ float2 s_ml[kMidWaves][kMidRows];
    __shared__ UnitsLds s_units;

    const uint32_t group = a.heads / a.kv_heads;
    const uint32_t rowbytes = a.head_dim * SZ, pmask = (1u << a.map.page_shift) - 1u;

    Dealer<false> deal(a, s_units);
    SeqWork sw{};
    const Piece it = deal.next(a, &sw);
    if (!it.live) return;
    const uint32_t lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave);
    const uint32_t n32 = lane % 32, h = lane / 32;
    Stage& st = s_kv[wave];
    const float *k_scale = s_scale[SZ == 1 ? wave : 0][0], *v_scale = s_scale[SZ == 1 ? wave : 0][1];
    const uint32_t n_rows = sw.n_new * group, first = sw.first;
    const int32_t past = sw.past;
    const uint32_t r0 = it.tile * kMidRows, r1 = min(r0 + kMidRows, n_rows);
    const uint32_t row = min(r0 + n32, r1 - 1u), tok = by_group(a, row), head = it.kv_head * group + (row - tok * group);
    const int32_t p0 = past + int32_t(by_group(a, r0)), p1 = past + int32_t(by_group(a, r1 - 1u));   // of the first and the last row
    const KeyRange keys = seen_keys(a, p0, p1);
    const int32_t back = a.window && a.window <= uint32_t(kMostKeys) ? int32_t(a.window) - 1 : kMostKeys;
    R rows;
    rows.see1 = past + int32_t(tok), rows.see0 = min(rows.see1 - back, a.most_keys);
    rows.all0 = p1 - back, rows.all1 = p0, rows.any0 = min(p0 - back, a.most_keys), rows.any1 = p1;
    rows.lane = lane;
    rows.send(a, uint64_t(first + tok) * a.q_stride + uint64_t(head) * a.head_dim);

    const int32_t n = int32_t(it.n), k0 = (keys.lo / STEP + int32_t(it.blk)) * STEP + int32_t(wave) * KT;
    // the pages of the two groups of 16 keys of steps i .. i + 31
    int32_t lane_pages = kNoKeys;
    auto read_pages = [&](int32_t i) {
        if constexpr (PAGED) lane_pages = lane_page(a, it.seq, keys, k0 + (i + int32_t(lane / 2)) * STEP + 16 * int32_t(lane % 2));
    };
    const uint64_t kst = PAGED ? rowbytes : a.k_stride * SZ, vst = PAGED ? rowbytes : a.v_stride * SZ;
    const void* zero = &g_attn_zero;
    // the loads of K (V) of step i; the groups of 16 keys without a page as a mask
    auto issue = [&](int32_t i, bool is_v) -> uint32_t {
        const int32_t key0 = k0 + i * STEP;
        int32_t page[2] = {0, 0};
        uint32_t bad = 0;
        bool whole = key0 >= keys.lo && key0 + KT <= keys.hi && rowbytes == uint32_t(RB);
        if constexpr (PAGED) {
            if (!is_v && i != 0 && i % 32 == 0) read_pages(i);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                page[x] = __builtin_amdgcn_readlane(lane_pages, (i % 32) * 2 + x);
                if (page[x] == kNoPage) bad |= 1u << x;
                whole = whole && page[x] >= 0;
            }
        }
        const unsigned char* plane = static_cast<const unsigned char*>(is_v ? a.v : a.k);
        const uint64_t stride = is_v ? vst : kst;
        const uint32_t lds = lds_offset(is_v ? st.v : st.k), lr = lane / NC, loff = lr * uint32_t(stride);
        const uint32_t c = (lane % NC) ^ (is_v ? swizzle_v<NC, SZ == 1, 3>(lr) : swizzle_k<NC>(lr));
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            // (a swizzle takes bits of the key, and j RPI and lr share none)
            const uint32_t ch = 16u * (c ^ (is_v ? swizzle_v<NC, SZ == 1, 3>(j * RPI) : swizzle_k<NC>(j * RPI)));
            const int32_t pg = page[j * RPI / 16];
            const uint64_t at = PAGED ? cache_row(uint32_t(max(pg, 0)), a.kv_heads, it.kv_head, a.map.page_shift, (uint32_t(key0) + j * RPI) & pmask) * rowbytes
                                      : (uint64_t(first) + uint64_t(key0) + j * RPI) * stride + it.kv_head * rowbytes;
            if (whole) {
                to_lds16<false>(plane + at, loff + ch, lds + j * 1024);
            } else {
                const int32_t k = key0 + int32_t(j * RPI + lr);
                const bool in = k >= keys.lo && k < keys.hi && pg >= 0 && ch < rowbytes;
                to_lds16<false>(in ? plane + at + (loff + ch) : zero, lds + j * 1024);
            }
        }
        if constexpr (SZ == 1) {
            const int32_t p = lane % KT < 16 ? page[0] : page[1], k = key0 + int32_t(lane % KT);
            const float* sp = (is_v ? a.v_scale : a.k_scale) + cache_row(uint32_t(max(p, 0)), a.kv_heads, it.kv_head, a.map.page_shift, uint32_t(k) & pmask);
            const void* from = p >= 0 && k >= keys.lo && k < keys.hi ? static_cast<const void*>(sp) : zero;
            const uint32_t to = lds_offset(is_v ? v_scale : k_scale);
            if (lane < uint32_t(KT)) to_lds4(from, to);
        }
        return bad;
    };
    auto drained = [] { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };

    read_pages(0);
    uint32_t bad = issue(0, false);
    issue(0, true);
    rows.begin(a);
    for (int32_t i = 0; i < n; ++i) {
        const int32_t key0 = k0 + i * STEP;
        const bool none = rows.skips(key0);
        const uint32_t bad0 = bad;
        wait_loads<OPS>();
        if (!none) rows.scores(st.k, k_scale);
        drained();
        // the pages of V's step are those that K's next step may replace
        if (i + 1 < n && (i + 1) % 32 != 0) {
            bad = issue(i + 1, false);
            wait_loads<OPS>();
        } else {
            wait_loads<0>();
        }
        if (!none) {
            const bool part = SZ == 2 && (key0 < rows.all0 || key0 + KT - 1 > rows.all1);
            if (part) {
                if (lane == 0) s_bad[wave] = 0;
                drained();
#pragma unroll
                for (int j = 0; j < LOADS; ++j) rows.sieve(st.v, uint32_t(j * RPI), &s_bad[wave]);
                drained();
            }
            rows.weights(key0, bad0, v_scale);
            rows.values(st.v);
            if (part)
                rows.add_sieved(a, key0, &s_bad[wave], [&](int32_t k) -> uint64_t {
                    if constexpr (PAGED) {
                        const int32_t pg = uniform_page(a.map, it.seq, k);   // it has one: a row without is zeros
                        return cache_row(uint32_t(max(pg, 0)), a.kv_heads, it.kv_head, a.map.page_shift, uint32_t(k) & pmask) * a.head_dim;
                    } else {
                        return (uint64_t(first) + uint64_t(k)) * a.v_stride + uint64_t(it.kv_head) * a.head_dim;
                    }
                });
        }
        drained();
        if (i + 1 < n) {
            if ((i + 1) % 32 == 0) bad = issue(i + 1, false);
            issue(i + 1, true);
        }
    }

    // the waves' sums, relative to the largest reference, through the stages' memory:
    // row r's chunk of four values c in place c ^ (r % 8)
    const float l = add_xor32(rows.l);
    if (h == 0) s_ml[wave][n32] = {rows.m == -INFINITY && l == 0.0f ? -INFINITY : rows.ref, l};
    constexpr int PASSES = SZ == 1 ? 2 : 1, CH = DP / 4 / PASSES;
    static_assert(sizeof(Stage) == sizeof(float) * kMidRows * DP / PASSES, "a wave's sums fill its stage");
    float* sums = reinterpret_cast<float*>(&st);
#pragma unroll
    for (int pass = 0; pass < PASSES; ++pass) {
        __syncthreads();
#pragma unroll
        for (int t = 0; t < OT / PASSES; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<f32x4*>(sums + n32 * (4 * CH) + 4 * ((8 * t + 2 * j + h) ^ (n32 & 7u))) = rows.sums(pass * (OT / PASSES) + t, j);
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < (r1 - r0) * CH; i += kMidThreads) {
            const uint32_t r = i / CH, c = i % CH, d = 4 * (pass * CH + c);
            if (d >= a.head_dim) continue;
            float top = -INFINITY, sum = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < kMidWaves; ++w) top = fmaxf(top, s_ml[w][r].x);
            f32x4 o{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (uint32_t w = 0; w < kMidWaves; ++w) {
                const float2 ml = s_ml[w][r];
                const bool in = ml.x != -INFINITY;
                const float f = in ? exp2_hw(ml.x - top) : 0.0f;
                const f32x4 x = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(&s_kv[w]) + r * (4 * CH) + 4 * (c ^ (r & 7u)));
                sum += in ? ml.y * f : 0.0f;
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] += in ? x[j] * f : 0.0f;
            }
            const uint32_t rr = r0 + r, t = by_group(a, rr);
            if (past + int32_t(t) >= 0) store_row4(a, first + t, it.kv_head * group + (rr - t * group), d, o, sum);
        }
    }
}

template <int CACHE, int TERMS, bool PAGED>
int launch_dim(const AttnRows& a, uint32_t grid_size, hipStream_t st) {
    const dim3 grid(grid_size), block(kMidThreads);
    switch (padded_dim(a.head_dim)) {
        case 64: hipLaunchKernelGGL((rows_attn_mid_kernel<CACHE, 64, TERMS, PAGED>), grid, block, 0, st, a); break;
        case 128: hipLaunchKernelGGL((rows_attn_mid_kernel<CACHE, 128, TERMS, PAGED>), grid, block, 0, st, a); break;
        default: hipLaunchKernelGGL((rows_attn_mid_kernel<CACHE, 256, TERMS, PAGED>), grid, block, 0, st, a); break;
    }
    XP_LAUNCHED();
    return XP_OK;
}

}  // namespace

int launch_mid(const AttnRows& a, int cache, bool paged, uint32_t grid_size, hipStream_t st) {
    if (!paged) return cache == XP_ELEM_F16 ? launch_dim<XP_ELEM_F16, 1, false>(a, grid_size, st) : launch_dim<XP_ELEM_BF16, 1, false>(a, grid_size, st);
    const bool two = a.q_elem == XP_ELEM_F32;
    switch (cache) {
        case XP_ELEM_BF16: return launch_dim<XP_ELEM_BF16, 1, true>(a, grid_size, st);
        case XP_ELEM_F16: return two ? launch_dim<XP_ELEM_F16, 2, true>(a, grid_size, st) : launch_dim<XP_ELEM_F16, 1, true>(a, grid_size, st);
        case XP_ELEM_I8: return two ? launch_dim<XP_ELEM_I8, 2, true>(a, grid_size, st) : launch_dim<XP_ELEM_I8, 1, true>(a, grid_size, st);
        default: return two ? launch_dim<XP_ELEM_E4M3, 2, true>(a, grid_size, st) : launch_dim<XP_ELEM_E4M3, 1, true>(a, grid_size, st);
    }
}

}  // namespace xp
