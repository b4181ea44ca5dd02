// Attention of many rows (prompts and their chunks): a workgroup's four waves take
// 32 rows each of a tile and share the keys' tiles in LDS.
// The 32 rows of a wave are xp_rows_attn32.hpp's.
//
// 32 rows a wave, as many as two waves a SIMD have registers for at 128 dims, and four waves
// to a tile of keys: each wave reads the whole tile, 32 KB for 1024 cycles of products, which
// the LDS gives at about the rate of the products. K and V go to LDS without passing through
// registers, one tile ahead. Instruction issue bounds it: at 128 dims the products take 0.47 of
// a SIMD's cycles, what else there is for its two waves (an exponential a score, maximum,
// sum, packing) 0.46, and they hardly meet. A prompt of 16384, 16 heads over 2 of 128 in bf16,
// takes 1100 to 1180 us (930 to 1000 TFLOP/s; a library's product of 8192 1224), 8192 at 64 dims 650, at
// 256 dims (one wave a SIMD) 540 to 610; chunks of 512 over 15000 in bf16 880, f16 810, e4m3 670, i8
// 570 (each wave widens all keys itself). Tried: a wave's priority raised for its products
// or for its softmax (both 5 % slower), three waves a SIMD at 64 dims (spills; lists 20 % slower).
#include "xp_rows_attn32.hpp"

namespace xp {
namespace {

constexpr uint32_t kTileThreads = kTileWaves * kWave;

template <int CACHE, int DP>
struct KeyTile {
    typedef Rows32<CACHE, DP, 1, int(tile_keys_of(DP)) / 32> R;
    static constexpr int SZ = R::SZ, RB = R::RB, NC = R::NC, RPI = R::RPI;
    static constexpr int KT = tile_keys_of(DP), LOADS = KT / RPI / int(kTileWaves);   // of a wave
    static_assert(LOADS >= 1 && LOADS * RPI * int(kTileWaves) == KT, "every wave loads whole rows");
    struct __attribute__((aligned(16))) Stage {
        unsigned char k[KT * RB], v[KT * RB];
        float scale[SZ == 1 ? 2 * KT : 4];
    };
};

template <int CACHE, int DP, int TERMS, bool PAGED, bool LIST>
__global__ __launch_bounds__(kTileThreads, DP == 256 || TERMS == 2 ? 1 : 2) void rows_attn_tile_kernel(AttnRows a) {
    using T = KeyTile<CACHE, DP>;
    typedef Rows32<CACHE, DP, TERMS, T::KT / 32> R;
    constexpr int SZ = T::SZ, RB = T::RB, NC = T::NC, RPI = T::RPI, KT = T::KT, OT = R::OT;
    typedef typename T::Stage Stage;
    __shared__ Stage s0;
    __shared__ Stage s1;
    __shared__ uint32_t s_bad[2][KT / 32];       // keys of a tile whose V row is not finite

    const uint32_t group = a.heads / a.kv_heads;
    const uint32_t rowbytes = a.head_dim * SZ, pmask = (1u << a.map.page_shift) - 1u;

    __shared__ UnitsLds s_units;
    Dealer<LIST> deal(a, s_units);
    SeqWork sw{};
    if (LIST) deal.join(a, Piece{}, sw, 0);
    for (Piece it = deal.next(a, &sw); it.live; it = deal.next(a, &sw)) {
    // (anew for each piece, or what follows from them is kept through all, in too many registers)
    const uint32_t tid = LIST ? opaque_tid() : threadIdx.x, lane = tid % kWave, wave = uniform(tid / kWave);
    const uint32_t n32 = lane % 32, h = lane / 32;
    const uint32_t n_rows = sw.n_new * group, first = sw.first;
    const int32_t past = sw.past;
    const uint32_t r0 = it.tile * kTileRows, r1 = min(r0 + kTileRows, n_rows);
    const uint32_t wr0 = r0 + 32 * wave;                                   // this wave's rows
    const bool idle = wr0 >= r1;
    const uint32_t wr1 = min(wr0 + 32, r1), wa = idle ? r1 - 1u : wr0, wb = idle ? r1 - 1u : wr1 - 1u;
    const uint32_t row = min(wa + n32, wb), tok = by_group(a, row), head = it.kv_head * group + (row - tok * group);
    // of the tile's first and last row, and of the wave's
    const int32_t tp0 = past + int32_t(by_group(a, r0)), tp1 = past + int32_t(by_group(a, r1 - 1u));
    const int32_t p0 = past + int32_t(by_group(a, wa)), p1 = past + int32_t(by_group(a, wb));
    const KeyRange keys = seen_keys(a, tp0, tp1);
    const int32_t back = a.window && a.window <= uint32_t(kMostKeys) ? int32_t(a.window) - 1 : kMostKeys;
    R rows;
    rows.see1 = past + int32_t(tok), rows.see0 = min(rows.see1 - back, a.most_keys);
    rows.all0 = p1 - back, rows.all1 = p0, rows.any0 = min(p0 - back, a.most_keys), rows.any1 = p1;
    rows.lane = lane;
    rows.send(a, uint64_t(first + tok) * a.q_stride + uint64_t(head) * a.head_dim);

    const int32_t n = int32_t(it.n), k0 = (keys.lo / KT + int32_t(it.blk)) * KT;
    // the pages of the 64 groups of 16 keys from step i on, a lane each, and those of the steps after
    constexpr int GROUPS = KT / 16, AHEAD = 64 / GROUPS;
    int32_t lane_pages = kNoKeys, next_pages = kNoKeys;
    uint64_t no_page = 0, no_row = 0;
    auto read_pages = [&](int32_t i) { return lane_page(a, it.seq, keys, k0 + i * KT + 16 * int32_t(lane)); };
    auto set_pages = [&](int32_t pages) {
        lane_pages = pages;
        no_page = __ballot(pages == kNoPage);
        no_row = __ballot(pages < 0);
    };
    // A load takes RPI rows; this lane's 16 bytes of them, the same for all loads of a
    // wave (they are 4 RPI rows apart, in which the swizzles repeat)
    static_assert(swizzle_k<NC>(kTileWaves * RPI) == 0 && swizzle_v<NC, SZ == 1, 3>(kTileWaves * RPI) == 0);
    const uint64_t kst = PAGED ? rowbytes : a.k_stride * SZ, vst = PAGED ? rowbytes : a.v_stride * SZ;
    const uint32_t rt0 = wave * RPI + lane / NC;
    const uint32_t ck = 16u * ((lane % NC) ^ swizzle_k<NC>(rt0)), cv = 16u * ((lane % NC) ^ swizzle_v<NC, SZ == 1, 3>(rt0));
    const uint32_t koff = (lane / NC) * uint32_t(kst) + ck, voff = (lane / NC) * uint32_t(vst) + cv;
    // the loads of step i into a stage; the groups of 16 keys that have no page come back as a mask
    auto issue = [&](int32_t i, Stage& s) -> uint32_t {
        const int32_t key0 = k0 + i * KT;
        const uint32_t kl = lds_offset(s.k), vl = lds_offset(s.v);
        const void* zero = &g_attn_zero;
        uint32_t bad = 0, none = 0, at = 0;
        if constexpr (PAGED) {
            if (i != 0 && i % AHEAD == 0) {
                set_pages(next_pages);
                if (i + AHEAD < n) next_pages = read_pages(i + AHEAD);
            }
            at = uint32_t(i % AHEAD) * GROUPS;
            bad = uint32_t(no_page >> at) & ((1u << GROUPS) - 1u);
            none = uint32_t(no_row >> at) & ((1u << GROUPS) - 1u);
        }
        const bool whole = key0 >= keys.lo && key0 + KT <= keys.hi && none == 0u && rowbytes == uint32_t(RB);
        auto each = [&](auto put) {
#pragma unroll
            for (int j = 0; j < T::LOADS; ++j) {
                const uint32_t ri = (uint32_t(j) * kTileWaves + wave) * RPI;
                uint64_t kat, vat;
                int32_t pg = 0;
                if constexpr (PAGED) {
                    pg = __builtin_amdgcn_readlane(lane_pages, int(at + ri / 16));
                    kat = vat = cache_row(uint32_t(max(pg, 0)), a.kv_heads, it.kv_head, a.map.page_shift, (uint32_t(key0) + ri) & pmask) * rowbytes;
                } else {
                    const uint64_t tk = uint64_t(first) + uint64_t(key0) + ri;
                    kat = tk * kst + it.kv_head * rowbytes;
                    vat = tk * vst + it.kv_head * rowbytes;
                }
                put(ri, pg, static_cast<const unsigned char*>(a.k) + kat, static_cast<const unsigned char*>(a.v) + vat);
            }
        };
        if (whole)
            each([&](uint32_t ri, int32_t, const unsigned char* kb, const unsigned char* vb) {
                to_lds16<false>(kb, koff, kl + ri * RB);
                to_lds16<false>(vb, voff, vl + ri * RB);
            });
        else
            each([&](uint32_t ri, int32_t pg, const unsigned char* kb, const unsigned char* vb) {
                const int32_t k = key0 + int32_t(ri + lane / NC);
                const bool in = k >= keys.lo && k < keys.hi && pg >= 0;
                to_lds16<false>(in && ck < rowbytes ? kb + koff : zero, kl + ri * RB);
                to_lds16<false>(in && cv < rowbytes ? vb + voff : zero, vl + ri * RB);
            });
        if constexpr (SZ == 1) {
            // wave 0: K's scales, wave 1: V's
            if (wave < 2) {
                const int32_t p = __shfl(lane_pages, int(at + (lane % KT) / 16), kWave), k = key0 + int32_t(lane % KT);
                const float* sp = (wave == 0 ? a.k_scale : a.v_scale) + cache_row(uint32_t(max(p, 0)), a.kv_heads, it.kv_head, a.map.page_shift, uint32_t(k) & pmask);
                const void* from = p >= 0 && k >= keys.lo && k < keys.hi ? static_cast<const void*>(sp) : zero;
                if (KT == 64 || lane < uint32_t(KT)) to_lds4(from, lds_offset(s.scale) + wave * KT * 4);
            }
        }
        return bad;
    };

    // the positions that all of the tile's rows see
    const int32_t tall0 = tp1 - back, tall1 = tp0;
    auto step = [&](int32_t i, Stage& cur, Stage& next, uint32_t bad, uint32_t* flags) -> uint32_t {
        const int32_t key0 = k0 + i * KT;
        wait_loads<0>();
        if (SZ == 2 && threadIdx.x < KT / 32) flags[threadIdx.x] = 0;
        __syncthreads();
        uint32_t nbad = 0;
        if (i + 1 < n) nbad = issue(i + 1, next);
        const bool part = SZ == 2 && (key0 < tall0 || key0 + KT - 1 > tall1);
        if (part) {
#pragma unroll
            for (int j = 0; j < T::LOADS; ++j) rows.sieve(cur.v, (uint32_t(j) * kTileWaves + wave) * RPI, flags);
            __syncthreads();
        }
        if (!idle && !rows.skips(key0)) {
            rows.scores(cur.k, cur.scale);
            rows.weights(key0, bad, cur.scale + KT);
            rows.values(cur.v);
            if (part)
                rows.add_sieved(a, key0, flags, [&](int32_t k) -> uint64_t {
                    if constexpr (PAGED) {
                        const int32_t pg = uniform_page(a.map, it.seq, k);   // it has one: a row without is zeros
                        return cache_row(uint32_t(max(pg, 0)), a.kv_heads, it.kv_head, a.map.page_shift, uint32_t(k) & pmask) * a.head_dim;
                    } else {
                        return (uint64_t(first) + uint64_t(k)) * a.v_stride + uint64_t(it.kv_head) * a.head_dim;
                    }
                });
        }
        return nbad;
    };
    if constexpr (PAGED) {
        set_pages(read_pages(0));
        if (AHEAD < n) next_pages = read_pages(AHEAD);
    }
    uint32_t bad = issue(0, s0);
    rows.begin(a);
    for (int32_t i = 0; i < n; i += 2) {
        bad = step(i, s0, s1, bad, s_bad[0]);
        if (i + 1 < n) bad = step(i + 1, s1, s0, bad, s_bad[1]);
    }

    const float l = add_xor32(rows.l);
    const bool live = !idle && wr0 + n32 < r1;
    if (LIST && live && it.n < it.of) {
        float* part = part_record(a, deal.wg, it.blk == 0, part_floats(kTileRows, DP));
        const uint32_t r = row - r0;
#pragma unroll
        for (int t = 0; t < OT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) *reinterpret_cast<f32x4*>(part + r * DP + 32 * t + 8 * j + 4 * h) = rows.sums(t, j);
        if (h == 0) reinterpret_cast<float2*>(part + kTileRows * DP)[r] = {rows.m == -INFINITY && l == 0.0f ? -INFINITY : rows.ref, l};
    } else if (live && rows.see1 >= 0) {
#pragma unroll
        for (int t = 0; t < OT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t d = 32 * t + 8 * j + 4 * h;
                if (d < a.head_dim) store_row4(a, first + tok, head, d, rows.sums(t, j), l);
            }
    }
    if (LIST && it.blk == 0 && it.n < it.of) deal.join(a, it, sw, r1 - r0);
    __syncthreads();                                   // the stages are the next piece's
    }
}

template <int CACHE, int TERMS, bool PAGED, bool LIST>
int launch_dim(const AttnRows& a, uint32_t grid_size, hipStream_t st) {
    const dim3 grid(grid_size), block(kTileThreads);
    switch (padded_dim(a.head_dim)) {
        case 64: hipLaunchKernelGGL((rows_attn_tile_kernel<CACHE, 64, TERMS, PAGED, LIST>), grid, block, 0, st, a); break;
        case 128: hipLaunchKernelGGL((rows_attn_tile_kernel<CACHE, 128, TERMS, PAGED, LIST>), grid, block, 0, st, a); break;
        default: hipLaunchKernelGGL((rows_attn_tile_kernel<CACHE, 256, TERMS, PAGED, LIST>), grid, block, 0, st, a); break;
    }
    XP_LAUNCHED();
    return XP_OK;
}

}  // namespace

template <bool LIST>
static int launch_list(const AttnRows& a, int cache, bool paged, uint32_t grid_size, hipStream_t st) {
    if (!paged)
        return cache == XP_ELEM_F16 ? launch_dim<XP_ELEM_F16, 1, false, LIST>(a, grid_size, st) : launch_dim<XP_ELEM_BF16, 1, false, LIST>(a, grid_size, st);
    const bool two = a.q_elem == XP_ELEM_F32;
    switch (cache) {
        case XP_ELEM_BF16: return launch_dim<XP_ELEM_BF16, 1, true, LIST>(a, grid_size, st);
        case XP_ELEM_F16: return two ? launch_dim<XP_ELEM_F16, 2, true, LIST>(a, grid_size, st) : launch_dim<XP_ELEM_F16, 1, true, LIST>(a, grid_size, st);
        case XP_ELEM_I8: return two ? launch_dim<XP_ELEM_I8, 2, true, LIST>(a, grid_size, st) : launch_dim<XP_ELEM_I8, 1, true, LIST>(a, grid_size, st);
        default: return two ? launch_dim<XP_ELEM_E4M3, 2, true, LIST>(a, grid_size, st) : launch_dim<XP_ELEM_E4M3, 1, true, LIST>(a, grid_size, st);
    }
}
int launch_tile(const AttnRows& a, int cache, bool paged, uint32_t grid_size, hipStream_t st) {
    return a.target ? launch_list<true>(a, cache, paged, grid_size, st) : launch_list<false>(a, cache, paged, grid_size, st);
}

}  // namespace xp
