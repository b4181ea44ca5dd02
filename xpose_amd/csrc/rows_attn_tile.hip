// Attention of many rows (prompts and their chunks): a workgroup's four waves take
// 32 rows each of a tile and share the keys' tiles in LDS.
//
// As for few rows the scores are made transposed, S^T = K Q^T, on the 32-row
// matrix instruction: a lane holds scores of one row, keys 8 i + 4 (lane / 32) +
// 0..3, and the product O^T = V^T P^T takes its weights from those registers as
// they are, its 16 keys in the order 4 h + 0..3, 8 + 4 h + 0..3 (h = lane / 32), in
// which V's columns are read.
#include "xp_rows_attn.hpp"

namespace xp {
namespace {

constexpr uint32_t kTileThreads = kTileWaves * kWave;

template <int CACHE, int DP>
struct KeyTile {
    static constexpr int SZ = CACHE == XP_ELEM_F16 || CACHE == XP_ELEM_BF16 ? 2 : 1;
    static constexpr int RB = DP * SZ, NC = RB / 16, RPI = 64 / NC;
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
    constexpr int SZ = T::SZ, RB = T::RB, NC = T::NC, RPI = T::RPI, KT = T::KT, KG = KT / 32;
    constexpr bool BF16 = CACHE == XP_ELEM_BF16;
    constexpr int QS = DP / 16, OT = DP / 32;
    // F16 weights are 2^7 of their size, and the reference may lag the maximum by 2^8
    constexpr float kBias = BF16 ? 0.0f : 7.0f, kLag = 8.0f;
    typedef typename T::Stage Stage;
    __shared__ Stage s0;
    __shared__ Stage s1;
    __shared__ uint32_t s_bad[2][KT / 32];       // keys of a tile whose V row is not finite

    const uint32_t lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave);
    const uint32_t n32 = lane % 32, h = lane / 32, group = a.heads / a.kv_heads;
    const uint32_t rowbytes = a.head_dim * SZ, pmask = (1u << a.map.page_shift) - 1u;

    __shared__ UnitsLds s_units;
    Dealer<LIST> deal(a, s_units);
    SeqWork sw{};
    if (LIST) deal.join(a, Piece{}, sw, 0);
    for (Piece it = deal.next(a, &sw); it.live; it = deal.next(a, &sw)) {
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
    const int32_t see1 = past + int32_t(tok), see0 = min(see1 - back, a.most_keys);
    // the positions that all of the wave's rows see, and that any does
    const int32_t all0 = p1 - back, all1 = p0, any0 = min(p0 - back, a.most_keys), any1 = p1;

    auto dim = [&](int s) { return SZ == 2 ? uint32_t(16 * s) + 8u * h : uint32_t(32 * (s / 2)) + 16u * h + 8u * (s % 2); };
    Query<BF16, TERMS, QS, 2> q;
    q.read(a, uint64_t(first + tok) * a.q_stride + uint64_t(head) * a.head_dim, dim);

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
    // the loads of step i into a stage; the groups of 16 keys that have no page come back as a mask
    auto issue = [&](int32_t i, Stage& s) -> uint32_t {
        const int32_t key0 = k0 + i * KT;
        const uint32_t kl = lds_offset(s.k), vl = lds_offset(s.v);
        const bool inside = key0 >= keys.lo && key0 + KT <= keys.hi;
        const void* zero = &g_attn_zero;
        uint32_t bad = 0;
        if constexpr (PAGED) {
            if (i != 0 && i % AHEAD == 0) {
                set_pages(next_pages);
                if (i + AHEAD < n) next_pages = read_pages(i + AHEAD);
            }
            const uint32_t at = uint32_t(i % AHEAD) * GROUPS;
            bad = uint32_t(no_page >> at) & ((1u << GROUPS) - 1u);
            const bool whole = inside && (uint32_t(no_row >> at) & ((1u << GROUPS) - 1u)) == 0u && rowbytes == uint32_t(RB);
            const uint32_t off = (lane / NC) * rowbytes;
#pragma unroll
            for (int j = 0; j < T::LOADS; ++j) {
                const uint32_t ri = (uint32_t(j) * kTileWaves + wave) * RPI, rt = ri + lane / NC;
                const uint32_t ck = 16u * ((lane % NC) ^ swizzle_k<NC>(rt)), cv = 16u * ((lane % NC) ^ swizzle_v<NC, SZ == 1, 3>(rt));
                const int32_t pg = __builtin_amdgcn_readlane(lane_pages, int(at + ri / 16));
                const uint64_t base = cache_row(uint32_t(max(pg, 0)), a.kv_heads, it.kv_head, a.map.page_shift, (uint32_t(key0) + ri) & pmask) * rowbytes;
                const unsigned char *kb = static_cast<const unsigned char*>(a.k) + base, *vb = static_cast<const unsigned char*>(a.v) + base;
                if (whole) {
                    to_lds16<false>(kb, off + ck, kl + ri * RB);
                    to_lds16<false>(vb, off + cv, vl + ri * RB);
                } else {
                    const int32_t k = key0 + int32_t(rt);
                    const bool in = k >= keys.lo && k < keys.hi && pg >= 0;
                    to_lds16<false>(in && ck < rowbytes ? kb + (off + ck) : zero, kl + ri * RB);
                    to_lds16<false>(in && cv < rowbytes ? vb + (off + cv) : zero, vl + ri * RB);
                }
            }
            if constexpr (SZ == 1) {
                // wave 0: K's scales, wave 1: V's
                if (wave < 2) {
                    const int32_t p = __shfl(lane_pages, int(at + (lane % KT) / 16), kWave), k = key0 + int32_t(lane % KT);
                    const float* sp = (wave == 0 ? a.k_scale : a.v_scale) + cache_row(uint32_t(max(p, 0)), a.kv_heads, it.kv_head, a.map.page_shift, uint32_t(k) & pmask);
                    const void* from = p >= 0 && k >= keys.lo && k < keys.hi ? static_cast<const void*>(sp) : zero;
                    if (KT == 64 || lane < uint32_t(KT)) to_lds4(from, lds_offset(s.scale) + wave * KT * 4);
                }
            }
        } else {
            const uint32_t head_at = it.kv_head * rowbytes;
            const uint64_t kst = a.k_stride * SZ, vst = a.v_stride * SZ;
#pragma unroll
            for (int j = 0; j < T::LOADS; ++j) {
                const uint32_t ri = (uint32_t(j) * kTileWaves + wave) * RPI, rt = ri + lane / NC;
                const uint32_t ck = 16u * ((lane % NC) ^ swizzle_k<NC>(rt)), cv = 16u * ((lane % NC) ^ swizzle_v<NC, SZ == 1, 3>(rt));
                const int32_t k = key0 + int32_t(rt);
                const bool in = inside || (k >= keys.lo && k < keys.hi);
                const uint64_t tk = uint64_t(first) + uint64_t(k);
                to_lds16<false>(in && ck < rowbytes ? static_cast<const unsigned char*>(a.k) + tk * kst + (head_at + ck) : zero, kl + ri * RB);
                to_lds16<false>(in && cv < rowbytes ? static_cast<const unsigned char*>(a.v) + tk * vst + (head_at + cv) : zero, vl + ri * RB);
            }
        }
        return bad;
    };

    f32x16 acc[OT];
#pragma unroll
    for (int t = 0; t < OT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[t][i] = 0.0f;
    float m = -INFINITY, l = 0.0f, ref = 0.0f, rl = -100.0f;

    // In a tile that not all rows see, a value that is not finite would reach the
    // rows that do not, as 0 times it. Such values are taken out of the tile (zeros in
    // their place) and added for the rows that see them, from memory. Every wave looks
    // through the rows it has loaded; a barrier follows.
    auto sieve = [&](Stage& s, uint32_t* flags) {
        if constexpr (SZ == 2) {
            constexpr uint32_t kExp = BF16 ? 0x7F80u : 0x7C00u;
#pragma unroll
            for (int i = 0; i < T::LOADS; ++i) {
                const uint32_t ri = (uint32_t(i) * kTileWaves + wave) * RPI;
                u32x4* p = reinterpret_cast<u32x4*>(s.v + ri * RB) + lane;
                u32x4 w = *p;
                bool hit = false;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t lo = (w[j] & kExp) == kExp ? 0xFFFFu : 0u, hi = ((w[j] >> 16) & kExp) == kExp ? 0xFFFF0000u : 0u;
                    hit = hit || lo || hi;
                    w[j] &= ~(lo | hi);
                }
                if (hit) {
                    *p = w;
                    const uint32_t rt = ri + lane / NC;
                    atomicOr(flags + rt / 32, 1u << (rt % 32));
                }
            }
        }
    };

    auto work = [&](int32_t key0, Stage& s, uint32_t bad, const uint32_t* flags, float coef) {
        if (idle || key0 > any1 || key0 + KT <= any0) return;
        const uint32_t fk = swizzle_k<NC>(n32);
        f32x16 sc[KG];
#pragma unroll
        for (int x = 0; x < KG; ++x) {
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[x][i] = 0.0f;
            const unsigned char* kr = s.k + (32 * x + n32) * RB;
            if constexpr (SZ == 2) {
#pragma unroll
                for (int st = 0; st < QS; ++st) {
                    const u32x4 kf = *reinterpret_cast<const u32x4*>(kr + 16 * ((2 * st + h) ^ fk));
                    if constexpr (TERMS == 2) sc[x] = mfma32<BF16>(kf, q.lo[st], sc[x]);
                    sc[x] = mfma32<BF16>(kf, q.hi[st], sc[x]);
                }
            } else {
#pragma unroll
                for (int st = 0; st < QS; st += 2) {
                    const u32x4 kb = *reinterpret_cast<const u32x4*>(kr + 16 * ((st + h) ^ fk));
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const u32x2 k0 = widen4<CACHE>(kb[2 * y]), k1 = widen4<CACHE>(kb[2 * y + 1]);
                        const u32x4 kf{k0[0], k0[1], k1[0], k1[1]};
                        if constexpr (TERMS == 2) sc[x] = mfma32<BF16>(kf, q.lo[st + y], sc[x]);
                        sc[x] = mfma32<BF16>(kf, q.hi[st + y], sc[x]);
                    }
                }
                // keys 8 i + 4 h + 0..3 of the 32
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 ks = *reinterpret_cast<const f32x4*>(s.scale + 32 * x + 8 * i + 4 * h);
#pragma unroll
                    for (int j = 0; j < 4; ++j) sc[x][4 * i + j] *= ks[j];
                }
            }
        }
        const bool all = key0 >= all0 && key0 + KT - 1 <= all1;
        if (!all || bad) {
#pragma unroll
            for (int x = 0; x < KG; ++x)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int32_t kt = 32 * x + 8 * (i / 4) + i % 4, k = key0 + kt + int32_t(4 * h);
                    if (bad & (1u << (kt / 16))) sc[x][i] = __uint_as_float(0x7FC00000u);
                    if (k < see0 || k > see1) sc[x][i] = -INFINITY;
                }
        }
        float top = -INFINITY;
#pragma unroll
        for (int x = 0; x < KG; ++x)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, sc[x][i]);
        m = fmaxf(m, max_xor32(top) * coef);                               // coef > 0
        if constexpr (SZ == 1) rl = fmaxf(rl, scale_exponent(wave_max(s.scale[KT + lane % KT])));
        const float nref = (m == -INFINITY ? 0.0f : m) + (SZ == 1 ? rl : 0.0f) - kBias;
        if (__any(!(nref <= ref + kLag && m != -INFINITY) || l == 0.0f)) {
            const float keep = exp2_hw(ref - nref);
            l *= keep;
#pragma unroll
            for (int t = 0; t < OT; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[t][i] *= keep;
            ref = nref;
        }
        u32x4 ph[2 * KG], pl[TERMS == 2 ? 2 * KG : 1];
        float sum = 0.0f;
#pragma unroll
        for (int x = 0; x < KG; ++x)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                float p[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) p[j] = exp2_hw(fmaf(sc[x][i + j], coef, -ref));
                sum += (p[0] + p[1]) + (p[2] + p[3]);
                if constexpr (SZ == 1) {
                    const f32x4 vs = *reinterpret_cast<const f32x4*>(s.scale + KT + 32 * x + 2 * i + 4 * h);
#pragma unroll
                    for (int j = 0; j < 4; ++j) p[j] = !all && sc[x][i + j] == -INFINITY ? 0.0f : p[j] * vs[j];
                }
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    uint32_t hi, lo = 0;
                    pack_weights<BF16, TERMS>(p[2 * w], p[2 * w + 1], hi, lo);
                    ph[2 * x + i / 8][(i % 8) / 2 + w] = hi;
                    if constexpr (TERMS == 2) pl[2 * x + i / 8][(i % 8) / 2 + w] = lo;
                }
            }
        l += sum;
        if constexpr (SZ == 2) {
            const uint32_t kv = 4 * h + (lane % 16) / 4, fv = swizzle_v<NC, false, 3>(kv), c0 = 2 * ((lane / 16) & 1u) + ((lane >> 1) & 1u);
            const unsigned char* vr = s.v + kv * RB + 8 * (lane & 1u);
#pragma unroll
            for (int x = 0; x < 2 * KG; ++x)
#pragma unroll
                for (int t = 0; t < OT; ++t) {
                    const unsigned char* p = vr + 16 * x * RB + 16 * ((4 * t + c0) ^ fv);
                    const u32x2 v0 = lds_tr16(p), v1 = lds_tr16(p + 8 * RB);
                    const u32x4 vf{v0[0], v0[1], v1[0], v1[1]};
                    if constexpr (TERMS == 2) acc[t] = mfma32<BF16>(vf, pl[x], acc[t]);
                    acc[t] = mfma32<BF16>(vf, ph[x], acc[t]);
                }
        } else {
            const uint32_t r8 = (lane % 16) / 2, kv = (r8 / 4) * 8 + 4 * h + r8 % 4, fv = swizzle_v<NC, true, 3>(kv);
            const unsigned char* vr = s.v + kv * RB + 8 * (lane & 1u);
#pragma unroll
            for (int x = 0; x < 2 * KG; ++x)
#pragma unroll
                for (int t = 0; t < OT; ++t) {
                    const u32x2 vb = lds_tr8(vr + 16 * x * RB + 16 * ((2 * t + ((lane / 16) & 1u)) ^ fv));
                    const u32x2 v0 = widen4<CACHE>(vb[0]), v1 = widen4<CACHE>(vb[1]);
                    const u32x4 vf{v0[0], v0[1], v1[0], v1[1]};
                    if constexpr (TERMS == 2) acc[t] = mfma32<BF16>(vf, pl[x], acc[t]);
                    acc[t] = mfma32<BF16>(vf, ph[x], acc[t]);
                }
        }
        if constexpr (SZ == 2) {
            if (!flags) return;
            // what the sieve took out, a key at a time: its weight is in the half of
            // the wave that has the key
#pragma unroll
            for (int x = 0; x < KG; ++x)
                for (uint32_t left = uniform(flags[x]); left; left &= left - 1u) {
                    const uint32_t kt = uint32_t(__builtin_ctz(left)), i = (kt / 8) * 4 + kt % 4, own = (kt / 4) & 1u;
                    const int32_t k = key0 + 32 * x + int32_t(kt);
                    float score = sc[x][0];
#pragma unroll
                    for (int j = 1; j < 16; ++j) score = i == uint32_t(j) ? sc[x][j] : score;
                    float p = exp2_hw(fmaf(score, coef, -ref));
                    p = __shfl(p, int(n32 + 32 * own), kWave);
                    const bool sees = k >= see0 && k <= see1;
                    uint64_t at;
                    if constexpr (PAGED) {
                        const int32_t pg = uniform_page(a.map, it.seq, k);   // it has one: a row without is zeros
                        at = cache_row(uint32_t(max(pg, 0)), a.kv_heads, it.kv_head, a.map.page_shift, uint32_t(k) & pmask) * a.head_dim;
                    } else {
                        at = (uint64_t(first) + uint64_t(k)) * a.v_stride + uint64_t(it.kv_head) * a.head_dim;
                    }
#pragma unroll
                    for (int t = 0; t < OT; ++t)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint32_t d = 32 * t + 8 * j + 4 * h;
                            if (d >= a.head_dim) continue;
                            const u32x2 w = *reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(a.v) + at + d);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float v = BF16 ? (e % 2 ? bf16hi(w[e / 2]) : bf16lo(w[e / 2])) : (e % 2 ? f16_hi(w[e / 2]) : f16_lo(w[e / 2]));
                                if (sees && !(fabsf(v) <= 3.4e38f)) acc[t][4 * j + e] += p * v;
                            }
                        }
                }
        }
    };

    // the positions that all of the tile's rows see
    const int32_t tall0 = tp1 - back, tall1 = tp0;
    auto step = [&](int32_t i, Stage& cur, Stage& next, uint32_t bad, uint32_t* flags, float coef) -> uint32_t {
        const int32_t key0 = k0 + i * KT;
        wait_loads<0>();
        if (SZ == 2 && threadIdx.x < KT / 32) flags[threadIdx.x] = 0;
        __syncthreads();
        uint32_t nbad = 0;
        if (i + 1 < n) nbad = issue(i + 1, next);
        const bool part = SZ == 2 && (key0 < tall0 || key0 + KT - 1 > tall1);
        if (part) {
            sieve(cur, flags);
            __syncthreads();
        }
        work(key0, cur, bad, part ? flags : nullptr, coef);
        return nbad;
    };
    if constexpr (PAGED) {
        set_pages(read_pages(0));
        if (AHEAD < n) next_pages = read_pages(AHEAD);
    }
    uint32_t bad = issue(0, s0);
    q.take(a, dim);
    const float coef = a.scale * 1.4426950408889634f * q.up;
    for (int32_t i = 0; i < n; i += 2) {
        bad = step(i, s0, s1, bad, s_bad[0], coef);
        if (i + 1 < n) bad = step(i + 1, s1, s0, bad, s_bad[1], coef);
    }

    l += __shfl_xor(l, 32, kWave);
    const bool live = !idle && wr0 + n32 < r1;
    if (LIST && live && it.n < it.of) {
        float* part = part_record(a, deal.wg, it.blk == 0, part_floats(kTileRows, DP));
        const uint32_t r = row - r0;
#pragma unroll
        for (int t = 0; t < OT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<f32x4*>(part + r * DP + 32 * t + 8 * j + 4 * h) = f32x4{acc[t][4 * j], acc[t][4 * j + 1], acc[t][4 * j + 2], acc[t][4 * j + 3]};
        if (h == 0) reinterpret_cast<float2*>(part + kTileRows * DP)[r] = {m == -INFINITY && l == 0.0f ? -INFINITY : ref, l};
    } else if (live && see1 >= 0) {
#pragma unroll
        for (int t = 0; t < OT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t d = 32 * t + 8 * j + 4 * h;
                if (d < a.head_dim) store_row4(a, first + tok, head, d, f32x4{acc[t][4 * j], acc[t][4 * j + 1], acc[t][4 * j + 2], acc[t][4 * j + 3]}, l);
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
