// 32 rows of attention in one wave, what rows_attn_tile.hip and rows_attn_mid.hip
// share.
//
// The scores are made transposed, S^T = K Q^T, on the 32-row matrix instruction: a
// lane holds scores of one row, keys 8 i + 4 (lane / 32) + 0..3 of each 32, and the
// product O^T = V^T P^T takes its weights from those registers as they are, its 16 keys
// in the order 4 h + 0..3, 8 + 4 h + 0..3 (h = lane / 32), in which V's columns are
// read. Nothing passes between lanes but a row's maximum (and at the end its sum).
#pragma once

#include "xp_rows_attn.hpp"

namespace xp {

template <int CACHE, int DP, int TERMS, int KG>
struct Rows32 {
    static constexpr bool BF16 = CACHE == XP_ELEM_BF16;
    static constexpr int SZ = CACHE == XP_ELEM_F16 || CACHE == XP_ELEM_BF16 ? 2 : 1;
    static constexpr int RB = DP * SZ, NC = RB / 16, RPI = 64 / NC;       // row bytes, its chunks, rows of one load
    static constexpr int KT = 32 * KG, QS = DP / 16, OT = DP / 32;
    // F16 weights are 2^7 of their size, and the reference may lag the maximum by 2^8
    static constexpr float kBias = BF16 ? 0.0f : 7.0f, kLag = 8.0f;

    Query<BF16, TERMS, QS, 2> q;
    f32x16 acc[OT];
    f32x16 sc[KG];                 // scores of the tile at hand
    float  m, l, ref, rl;          // maximum, sum, what they are relative to, the scales' exponent
    float  coef;
    int32_t see0, see1;            // the positions that this lane's row sees
    int32_t all0, all1;            // those that all of the wave's rows do
    int32_t any0, any1;            // and that any does
    uint32_t lane;

    // K's chunk of two steps is 16 bytes: eight dims of 16 bits, or two runs of eight of 8
    __device__ __forceinline__ uint32_t dim(int s) const {
        const uint32_t h = lane / 32;
        return SZ == 2 ? uint32_t(16 * s) + 8u * h : uint32_t(32 * (s / 2)) + 16u * h + 8u * (s % 2);
    }
    // (after this lane's row's limits and lane are set)
    __device__ __forceinline__ void send(const AttnRows& a, uint64_t at) {
        q.read(a, at, [&](int s) { return dim(s); });
    }
    __device__ __forceinline__ void begin(const AttnRows& a) {
#pragma unroll
        for (int t = 0; t < OT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[t][i] = 0.0f;
        m = -INFINITY, l = 0.0f, ref = 0.0f, rl = -100.0f;
        q.take(a, [&](int s) { return dim(s); });
        coef = a.scale * 1.4426950408889634f * q.up;
    }
    __device__ __forceinline__ bool skips(int32_t key0) const { return key0 > any1 || key0 + KT <= any0; }

    __device__ __forceinline__ void scores(const unsigned char* k, const float* k_scale) {
        const uint32_t n32 = lane % 32, h = lane / 32, fk = swizzle_k<NC>(n32);
#pragma unroll
        for (int x = 0; x < KG; ++x) {
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[x][i] = 0.0f;
            const unsigned char* kr = k + (32 * x + n32) * RB;
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
                    const f32x4 ks = *reinterpret_cast<const f32x4*>(k_scale + 32 * x + 8 * i + 4 * h);
#pragma unroll
                    for (int j = 0; j < 4; ++j) sc[x][4 * i + j] *= ks[j];
                }
            }
        }
    }

    // The softmax's step: masks, the weights as operands. bad: groups of 16 keys without
    // a page.
    u32x4 ph[2 * KG], pl[TERMS == 2 ? 2 * KG : 1];
    __device__ __forceinline__ void weights(int32_t key0, uint32_t bad, const float* v_scale) {
        const uint32_t h = lane / 32;
        const bool all = key0 >= all0 && key0 + KT - 1 <= all1;
        if (!all || bad) {
#pragma unroll
            for (int x = 0; x < KG; ++x)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int32_t kt = 32 * x + 8 * (i / 4) + i % 4, at = key0 + kt + int32_t(4 * h);
                    if (bad & (1u << (kt / 16))) sc[x][i] = __uint_as_float(0x7FC00000u);
                    if (at < see0 || at > see1) sc[x][i] = -INFINITY;
                }
        }
        float top = -INFINITY;
#pragma unroll
        for (int x = 0; x < KG; ++x)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, sc[x][i]);
        m = fmaxf(m, max_xor32(top) * coef);                               // coef > 0
        if constexpr (SZ == 1) rl = fmaxf(rl, scale_exponent(wave_max(v_scale[lane % KT])));
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
                    const f32x4 vs = *reinterpret_cast<const f32x4*>(v_scale + 32 * x + 2 * i + 4 * h);
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
    }

    __device__ __forceinline__ void values(const unsigned char* v) {
        const uint32_t h = lane / 32;
        if constexpr (SZ == 2) {
            const uint32_t kv = 4 * h + (lane % 16) / 4, fv = swizzle_v<NC, false, 3>(kv), c0 = 2 * ((lane / 16) & 1u) + ((lane >> 1) & 1u);
            const unsigned char* vr = v + kv * RB + 8 * (lane & 1u);
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
            const unsigned char* vr = v + kv * RB + 8 * (lane & 1u);
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
    }

    // In a tile that not all rows see, a value that is not finite would reach the rows
    // that do not, as 0 times it. Such values are taken out of the tile (zeros in their
    // place, flags for their keys), 1 KB that a wave has loaded at a time (row0: its first
    // row), and added afterwards for the rows that see them, from memory.
    __device__ __forceinline__ void sieve(unsigned char* v, uint32_t row0, uint32_t* flags) const {
        constexpr uint32_t kExp = BF16 ? 0x7F80u : 0x7C00u;
        u32x4* p = reinterpret_cast<u32x4*>(v + row0 * RB) + lane;
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
            const uint32_t rt = row0 + lane / NC;
            atomicOr(flags + rt / 32, 1u << (rt % 32));
        }
    }
    // at(k): the elements before the row of position k. The key's weight is in the half
    // of the wave that has the key.
    template <typename RowAt>
    __device__ __forceinline__ void add_sieved(const AttnRows& a, int32_t key0, const uint32_t* flags, RowAt row_at) {
        const uint32_t n32 = lane % 32, h = lane / 32;
#pragma unroll
        for (int x = 0; x < KG; ++x)
            for (uint32_t left = uniform(flags[x]); left; left &= left - 1u) {
                const uint32_t kt = uint32_t(__builtin_ctz(left)), i = (kt / 8) * 4 + kt % 4, own = (kt / 4) & 1u;
                const int32_t k = key0 + 32 * x + int32_t(kt);
                float score = sc[x][0];
#pragma unroll
                for (int j = 1; j < 16; ++j) score = i == uint32_t(j) ? sc[x][j] : score;
                const float p = __shfl(exp2_hw(fmaf(score, coef, -ref)), int(n32 + 32 * own), kWave);
                const bool sees = k >= see0 && k <= see1;
                const uint16_t* v = static_cast<const uint16_t*>(a.v) + row_at(k);
#pragma unroll
                for (int t = 0; t < OT; ++t) {
                    __builtin_amdgcn_sched_barrier(0);     // few registers, not few waits: this is rare
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t d = 32 * t + 8 * j + 4 * h;
                        const u32x2 w = *reinterpret_cast<const u32x2*>(v + (d < a.head_dim ? d : 0u));
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float y = BF16 ? (e % 2 ? bf16hi(w[e / 2]) : bf16lo(w[e / 2])) : (e % 2 ? f16_hi(w[e / 2]) : f16_lo(w[e / 2]));
                            if (sees && !(fabsf(y) <= 3.4e38f)) acc[t][4 * j + e] += p * y;
                        }
                    }
                }
            }
    }
    __device__ __forceinline__ f32x4 sums(int t, int j) const {              // dims 32 t + 8 j + 4 h ..
        return f32x4{acc[t][4 * j], acc[t][4 * j + 1], acc[t][4 * j + 2], acc[t][4 * j + 3]};
    }
};

}  // namespace xp
