// Attention of few rows (single tokens, short chunks) over a paged cache: tiles of
// 16 rows, a workgroup's four waves each at keys of their own.
//
// Scores are made transposed, S^T = K Q^T: a lane then holds scores of one row
// only, keys 4 (lane / 16) + 0..3 of each 16, which is as the product O^T = V^T P^T
// takes the weights. Nothing passes between lanes but a row's maximum.
//
// Bytes bound it: a wave sends its next 8 to 16 KB of K and V straight to LDS of its
// own while it works on the last, without a barrier until the waves' sums meet. 64 single
// tokens over up to 8000 positions (8 kv heads of 128 in bf16, 1.1 GB) take 180 us, 6.2 TB/s (a
// wave that only loads reaches 7.0), 16 over 32768 in 8 bits (1.1 GB) 182 us; as tiles alone,
// without the list, 194 and 329. One over 4096 positions of one head of 256 takes 15 us (86):
// launch, four dependent reads (lengths, pages, keys, and once more in the join), 4 MB.
#include "xp_rows_attn.hpp"

namespace xp {
namespace {

constexpr uint32_t kFewThreads = kFewWaves * kWave;

template <int CACHE, int DP>
struct FewTile {
    static constexpr int SZ = CACHE == XP_ELEM_F16 || CACHE == XP_ELEM_BF16 ? 2 : 1;
    static constexpr int RB = DP * SZ, NC = RB / 16, RPI = 64 / NC;       // row bytes, its chunks, rows of one load
    static constexpr int KT = few_keys(DP, SZ), LOADS = KT / RPI;
    static constexpr int SCALES = SZ == 1 ? (2 * KT + 63) / 64 : 0;       // loads
    static constexpr int OPS = 2 * LOADS + SCALES;                        // loads of a stage
    struct __attribute__((aligned(16))) Stage {
        unsigned char k[KT * RB], v[KT * RB];
        float scale[SZ == 1 ? 2 * KT : 4];                                // K's, then V's
    };
};

template <int CACHE, int DP, int TERMS, bool LIST>
__global__ __launch_bounds__(kFewThreads, DP == 256 ? 1 : 2) void rows_attn_few_kernel(AttnRows a) {
    using T = FewTile<CACHE, DP>;
    constexpr int SZ = T::SZ, RB = T::RB, NC = T::NC, RPI = T::RPI, KT = T::KT, KG = KT / 16;
    constexpr bool BF16 = CACHE == XP_ELEM_BF16;
    constexpr int QS = DP / 32, OT = DP / 16;
    constexpr float kBias = BF16 ? 0.0f : 12.0f;     // F16 weights up to 2^12: those under 2^-26 lose bits
    typedef typename T::Stage Stage;
    __shared__ Stage s0[kFewWaves];
    __shared__ Stage s1[kFewWaves];
    __shared__ float2 s_ml[kFewWaves][kFewRows];

    const uint32_t group = a.heads / a.kv_heads;
    const uint32_t rowbytes = a.head_dim * SZ, pmask = (1u << a.map.page_shift) - 1u;

    __shared__ UnitsLds s_units;
    Dealer<LIST> deal(a, s_units);
    SeqWork sw{};
    if (LIST) deal.join(a, Piece{}, sw, 0);
    for (Piece it = deal.next(a, &sw); it.live; it = deal.next(a, &sw)) {
    // (anew for each piece, or what follows from them is kept through all, in too many registers)
    const uint32_t tid = LIST ? opaque_tid() : threadIdx.x, lane = tid % kWave, wave = uniform(tid / kWave);
    const uint32_t n16 = lane % 16, g = lane / 16;
    const uint32_t n_rows = sw.n_new * group, first = sw.first;
    const int32_t past = sw.past;
    const uint32_t r0 = it.tile * kFewRows, r1 = min(r0 + kFewRows, n_rows);
    const uint32_t row = min(r0 + n16, r1 - 1u), tok = by_group(a, row), head = it.kv_head * group + (row - tok * group);
    const int32_t pos0 = past + int32_t(by_group(a, r0)), pos1 = past + int32_t(by_group(a, r1 - 1u));   // of the tile's first and last row
    const KeyRange keys = seen_keys(a, pos0, pos1);
    // the positions that this lane's row sees, and those that all of the tile's do
    const int32_t back = a.window && a.window <= uint32_t(kMostKeys) ? int32_t(a.window) - 1 : kMostKeys;
    const int32_t see1 = past + int32_t(tok), see0 = min(see1 - back, a.most_keys), all0 = pos1 - back, all1 = pos0;

    // K's chunk of a step: 16 bytes, eight dims of 16 bits, or two runs of eight of 8 bits
    auto dim = [&](int s) { return SZ == 2 ? uint32_t(32 * s) + 8u * g : uint32_t(64 * (s / 2)) + 16u * g + 8u * (s % 2); };
    Query<BF16, TERMS, QS, 4> q;
    q.read(a, uint64_t(first + tok) * a.q_stride + uint64_t(head) * a.head_dim, dim);

    constexpr int32_t STEP = kFewWaves * KT;
    const int32_t n = int32_t(it.n), k0 = (keys.lo / STEP + int32_t(it.blk)) * STEP + int32_t(wave) * KT;
    // the pages of steps i .. i + 63, a lane each
    int32_t lane_pages[KG];
    auto read_pages = [&](int32_t i) {
#pragma unroll
        for (int x = 0; x < KG; ++x) lane_pages[x] = lane_page(a, it.seq, keys, k0 + (i + int32_t(lane)) * STEP + 16 * x);
    };
    // the loads of step i into a stage; the groups of 16 keys that have no page come back as a mask
    auto issue = [&](int32_t i, Stage& s) -> uint32_t {
        const int32_t key0 = k0 + i * STEP;
        int32_t page[KG];
        uint32_t bad = 0;
        bool whole = key0 >= keys.lo && key0 + KT <= keys.hi && rowbytes == uint32_t(RB);
        if (i != 0 && i % 64 == 0) read_pages(i);
#pragma unroll
        for (int x = 0; x < KG; ++x) {
            page[x] = __builtin_amdgcn_readlane(lane_pages[x], i % 64);
            if (page[x] == kNoPage) bad |= 1u << x;
            whole = whole && page[x] >= 0;
        }
        const uint32_t kl = lds_offset(s.k), vl = lds_offset(s.v), off = (lane / NC) * rowbytes;
        const void* zero = &g_attn_zero;
        auto each = [&](auto put) {
#pragma unroll
            for (int j = 0; j < T::LOADS; ++j) {
                const uint32_t rt = uint32_t(j * RPI) + lane / NC;         // this lane's key of the tile
                const uint32_t ck = 16u * ((lane % NC) ^ swizzle_k<NC>(rt)), cv = 16u * ((lane % NC) ^ swizzle_v<NC, SZ == 1, 4>(rt));
                const int32_t pg = page[j * RPI / 16];
                const uint64_t base = cache_row(uint32_t(max(pg, 0)), a.kv_heads, it.kv_head, a.map.page_shift, (uint32_t(key0) + j * RPI) & pmask) * rowbytes;
                put(j, rt, ck, cv, pg, static_cast<const unsigned char*>(a.k) + base, static_cast<const unsigned char*>(a.v) + base);
            }
        };
        if (whole)
            each([&](int j, uint32_t, uint32_t ck, uint32_t cv, int32_t, const unsigned char* kb, const unsigned char* vb) {
                to_lds16<true>(kb, off + ck, kl + j * 1024);
                to_lds16<true>(vb, off + cv, vl + j * 1024);
            });
        else
            each([&](int j, uint32_t rt, uint32_t ck, uint32_t cv, int32_t pg, const unsigned char* kb, const unsigned char* vb) {
                const int32_t k = key0 + int32_t(rt);
                const bool in = k >= keys.lo && k < keys.hi && pg >= 0;
                to_lds16<true>(in && ck < rowbytes ? kb + (off + ck) : zero, kl + j * 1024);
                to_lds16<true>(in && cv < rowbytes ? vb + (off + cv) : zero, vl + j * 1024);
            });
        if constexpr (SZ == 1) {
            const uint32_t sl = lds_offset(s.scale);
#pragma unroll
            for (int y = 0; y < T::SCALES; ++y) {
                const uint32_t j = y * 64 + lane, kt = j % KT;             // K's KT scales, then V's
                int32_t p = page[0];
#pragma unroll
                for (int x = 1; x < KG; ++x) p = kt / 16 == uint32_t(x) ? page[x] : p;
                const int32_t k = key0 + int32_t(kt);
                const float* sp = (j < KT ? a.k_scale : a.v_scale) + cache_row(uint32_t(max(p, 0)), a.kv_heads, it.kv_head, a.map.page_shift, uint32_t(k) & pmask);
                to_lds4(p >= 0 && k >= keys.lo && k < keys.hi ? static_cast<const void*>(sp) : zero, sl + y * 256);
            }
        }
        return bad;
    };

    f32x4 acc[OT];
#pragma unroll
    for (int t = 0; t < OT; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f, ref = 0.0f, rl = -100.0f;   // ref: what the sums are relative to, m and the scales' exponent

    auto work = [&](int32_t key0, const Stage& s, uint32_t bad, float coef) {
        if (key0 >= keys.hi || key0 + KT <= keys.lo) return;
        const uint32_t fk = swizzle_k<NC>(n16);
        float sc[KG][4];
#pragma unroll
        for (int x = 0; x < KG; ++x) {
            f32x4 c{0.0f, 0.0f, 0.0f, 0.0f};
            const unsigned char* kr = s.k + (16 * x + n16) * RB;
            if constexpr (SZ == 2) {
#pragma unroll
                for (int st = 0; st < QS; ++st) {
                    const u32x4 kf = *reinterpret_cast<const u32x4*>(kr + 16 * ((4 * st + g) ^ fk));
                    if constexpr (TERMS == 2) c = mfma16<BF16>(kf, q.lo[st], c);
                    c = mfma16<BF16>(kf, q.hi[st], c);
                }
            } else {
#pragma unroll
                for (int st = 0; st < QS; st += 2) {
                    const u32x4 kb = *reinterpret_cast<const u32x4*>(kr + 16 * ((2 * st + g) ^ fk));
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const u32x2 k0 = widen4<CACHE>(kb[2 * y]), k1 = widen4<CACHE>(kb[2 * y + 1]);
                        const u32x4 kf{k0[0], k0[1], k1[0], k1[1]};
                        if constexpr (TERMS == 2) c = mfma16<BF16>(kf, q.lo[st + y], c);
                        c = mfma16<BF16>(kf, q.hi[st + y], c);
                    }
                }
            }
            f32x4 ks{1.0f, 1.0f, 1.0f, 1.0f};
            if constexpr (SZ == 1) ks = *reinterpret_cast<const f32x4*>(s.scale + 16 * x + 4 * g);
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[x][i] = SZ == 1 ? c[i] * (ks[i] * coef) : c[i] * coef;
        }
        const bool all = key0 >= all0 && key0 + KT - 1 <= all1;
        if (!all || bad) {
#pragma unroll
            for (int x = 0; x < KG; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int32_t k = key0 + int32_t(16 * x + 4 * g) + i;
                    if (bad & (1u << x)) sc[x][i] = __uint_as_float(0x7FC00000u);
                    if (k < see0 || k > see1) sc[x][i] = -INFINITY;
                }
        }
        float top = -INFINITY;
#pragma unroll
        for (int x = 0; x < KG; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, sc[x][i]);
        top = max_xor16(max_xor32(top));
        m = fmaxf(m, top);
        if constexpr (SZ == 1) rl = fmaxf(rl, scale_exponent(wave_max(lane < uint32_t(KT) ? s.scale[KT + lane] : 0.0f)));
        const float nref = (m == -INFINITY ? 0.0f : m) + (SZ == 1 ? rl : 0.0f) - kBias;
        if (__any(nref != ref)) {
            const float keep = exp2_hw(ref - nref);
            l *= keep;
#pragma unroll
            for (int t = 0; t < OT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[t][i] *= keep;
            ref = nref;
        }
        u32x2 ph[KG], pl[KG];
#pragma unroll
        for (int x = 0; x < KG; ++x) {
            f32x4 p;
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = exp2_hw(sc[x][i] - ref);
            l += (p[0] + p[1]) + (p[2] + p[3]);
            if constexpr (SZ == 1) {
                const f32x4 vs = *reinterpret_cast<const f32x4*>(s.scale + KT + 16 * x + 4 * g);
#pragma unroll
                for (int i = 0; i < 4; ++i) p[i] = sc[x][i] == -INFINITY ? 0.0f : p[i] * vs[i];
            }
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                uint32_t h, lo = 0;
                pack_weights<BF16, TERMS>(p[2 * w], p[2 * w + 1], h, lo);
                ph[x][w] = h;
                pl[x][w] = lo;
            }
        }
        if constexpr (SZ == 2) {
            const uint32_t kv = 4 * g + n16 / 4, fv = swizzle_v<NC, false, 4>(kv);
            const unsigned char* vr = s.v + kv * RB + 8 * (lane & 1u);
#pragma unroll
            for (int x = 0; x < KG; ++x)
#pragma unroll
                for (int t = 0; t < OT; ++t) {
                    const u32x2 vf = lds_tr16(vr + 16 * x * RB + 16 * ((2 * t + ((lane >> 1) & 1u)) ^ fv));
                    if constexpr (TERMS == 2) acc[t] = mfma16k16<BF16>(vf, pl[x], acc[t]);
                    acc[t] = mfma16k16<BF16>(vf, ph[x], acc[t]);
                }
        } else {
            const uint32_t r8 = n16 / 2, kv = (r8 / 4) * 16 + 4 * g + r8 % 4, fv = swizzle_v<NC, true, 4>(kv);
            const unsigned char* vr = s.v + kv * RB + 8 * (lane & 1u);
#pragma unroll
            for (int x = 0; x < KG; x += 2)
#pragma unroll
                for (int t = 0; t < OT; ++t) {
                    const u32x2 vb = lds_tr8(vr + 16 * x * RB + 16 * (uint32_t(t) ^ fv));
                    const u32x2 v0 = widen4<CACHE>(vb[0]), v1 = widen4<CACHE>(vb[1]);
                    const u32x4 vf{v0[0], v0[1], v1[0], v1[1]};
                    if constexpr (TERMS == 2) acc[t] = mfma16<BF16>(vf, u32x4{pl[x][0], pl[x][1], pl[x + 1][0], pl[x + 1][1]}, acc[t]);
                    acc[t] = mfma16<BF16>(vf, u32x4{ph[x][0], ph[x][1], ph[x + 1][0], ph[x + 1][1]}, acc[t]);
                }
        }
    };

    // two stages: the loads of one are on their way while the other is worked on
    read_pages(0);
    uint32_t bad0 = issue(0, s0[wave]), bad1 = 0;
    if (1 < n) bad1 = issue(1, s1[wave]);
    q.take(a, dim);
    const float coef = a.scale * 1.4426950408889634f * q.up;
    for (int32_t i = 0; i < n; i += 2) {
        if (i + 1 < n) wait_loads<T::OPS>();
        else wait_loads<0>();
        work(k0 + i * STEP, s0[wave], bad0, coef);
        if (i + 1 >= n) break;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (i + 2 < n) {
            bad0 = issue(i + 2, s0[wave]);
            wait_loads<T::OPS>();
        } else {
            wait_loads<0>();
        }
        work(k0 + (i + 1) * STEP, s1[wave], bad1, coef);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (i + 3 < n) bad1 = issue(i + 3, s1[wave]);
    }

    // the waves' sums, relative to the largest reference
    l = add_xor16(add_xor32(l));
    if (m == -INFINITY && l == 0.0f) ref = -INFINITY;
    __syncthreads();
    static_assert(sizeof(float) * kFewWaves * kFewRows * (DP + 4) <= 2 * sizeof(s0), "the sums fit the stages");
    // a wave's sums in its stages' memory: rows 0..7 in the first, 8..15 in the second
    auto sum_at = [&](uint32_t w, uint32_t r) -> float* {
        return reinterpret_cast<float*>(r < 8 ? &s0[w] : &s1[w]) + (r & 7u) * (DP + 4);
    };
    if (g == 0) s_ml[wave][n16] = {ref, l};
#pragma unroll
    for (int t = 0; t < OT; ++t) *reinterpret_cast<f32x4*>(sum_at(wave, n16) + 16 * t + 4 * g) = acc[t];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < (r1 - r0) * (DP / 4); i += kFewThreads) {
        const uint32_t r = i / (DP / 4), d = (i % (DP / 4)) * 4;
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kFewWaves; ++w) top = fmaxf(top, s_ml[w][r].x);
        f32x4 o{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t w = 0; w < kFewWaves; ++w) {
            const float2 ml = s_ml[w][r];
            const float f = ml.x == -INFINITY ? 0.0f : exp2_hw(ml.x - top);
            const f32x4 x = *reinterpret_cast<const f32x4*>(sum_at(w, r) + d);
            sum += ml.x == -INFINITY ? 0.0f : ml.y * f;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] += ml.x == -INFINITY ? 0.0f : x[j] * f;
        }
        if (d >= a.head_dim) continue;
        if (LIST && it.n < it.of) {
            float* part = part_record(a, deal.wg, it.blk == 0, part_floats(kFewRows, DP));
            *reinterpret_cast<f32x4*>(part + r * DP + d) = o;
            if (d == 0) reinterpret_cast<float2*>(part + kFewRows * DP)[r] = {top, sum};
            continue;
        }
        const uint32_t rr = r0 + r, t = by_group(a, rr);
        if (past + int32_t(t) < 0) continue;
        store_row4(a, first + t, it.kv_head * group + (rr - t * group), d, o, sum);
    }
    if (LIST && it.blk == 0 && it.n < it.of) deal.join(a, it, sw, r1 - r0);
    __syncthreads();                                   // the stages are the next piece's
    }
}

template <int CACHE, int TERMS, bool LIST>
int launch_dim(const AttnRows& a, uint32_t grid_size, hipStream_t st) {
    const dim3 grid(grid_size), block(kFewThreads);
    switch (padded_dim(a.head_dim)) {
        case 64: hipLaunchKernelGGL((rows_attn_few_kernel<CACHE, 64, TERMS, LIST>), grid, block, 0, st, a); break;
        case 128: hipLaunchKernelGGL((rows_attn_few_kernel<CACHE, 128, TERMS, LIST>), grid, block, 0, st, a); break;
        default: hipLaunchKernelGGL((rows_attn_few_kernel<CACHE, 256, TERMS, LIST>), grid, block, 0, st, a); break;
    }
    XP_LAUNCHED();
    return XP_OK;
}

}  // namespace

template <bool LIST>
static int launch_list(const AttnRows& a, int cache, uint32_t grid_size, hipStream_t st) {
    const bool two = a.q_elem == XP_ELEM_F32;
    switch (cache) {
        case XP_ELEM_BF16: return launch_dim<XP_ELEM_BF16, 1, LIST>(a, grid_size, st);
        case XP_ELEM_F16: return two ? launch_dim<XP_ELEM_F16, 2, LIST>(a, grid_size, st) : launch_dim<XP_ELEM_F16, 1, LIST>(a, grid_size, st);
        case XP_ELEM_I8: return two ? launch_dim<XP_ELEM_I8, 2, LIST>(a, grid_size, st) : launch_dim<XP_ELEM_I8, 1, LIST>(a, grid_size, st);
        default: return two ? launch_dim<XP_ELEM_E4M3, 2, LIST>(a, grid_size, st) : launch_dim<XP_ELEM_E4M3, 1, LIST>(a, grid_size, st);
    }
}
int launch_few(const AttnRows& a, int cache, uint32_t grid_size, hipStream_t st) {
    return a.target ? launch_list<true>(a, cache, grid_size, st) : launch_list<false>(a, cache, grid_size, st);
}

}  // namespace xp
