// What the kernels of attention over packed rows share (rows_attn_few.hip,
// rows_attn_mid.hip, rows_attn_tile.hip, rows_attention.hip): their places in the deal, operands of
// the matrix instructions, tiles on their way to LDS.
#pragma once

#include "xp_elem.hpp"
#include "xp_rows_deal.hpp"

namespace xp {

#ifdef __HIPCC__
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return uint32_t(__builtin_amdgcn_readfirstlane(int(v))); }
__device__ __forceinline__ uint32_t of_lane(uint32_t v, uint32_t lane) { return uint32_t(__builtin_amdgcn_readlane(int(v), int(lane))); }
// Sums of lanes 0 .. l in lane l (row shifts, then the rows' totals).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_add(uint32_t v) {
    return v + uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_scan_add(uint32_t v) {
    v = dpp_add<0x111, 0xF>(v);    // row_shr:1
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    v = dpp_add<0x118, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);    // row_bcast:15 -> rows 1, 3
    return dpp_add<0x143, 0xC>(v); // row_bcast:31 -> rows 2, 3
}
__device__ __forceinline__ SeqWork lane_work(const AttnRows& a, uint32_t b) {
    return b < a.n_seq ? seq_work(a, b) : SeqWork{0, 0, 0, 0};
}
__device__ __forceinline__ SeqWork work_of_lane(const SeqWork& w, uint32_t l) {
    return {of_lane(w.first, l), of_lane(w.n_new, l), of_lane(w.tiles, l), int32_t(of_lane(uint32_t(w.past), l))};
}
// The tiles, and with LIST the blocks of the list, of all kv heads of up to 64
// sequences, a lane each, and their sums up to and with each lane's. (The sums of a
// cu that gives rows many times over may wrap: the callers bound what they find.)
struct LaneUnits {
    SeqWork  w;
    uint32_t own, up;
    __device__ __forceinline__ void read(const AttnRows& a, uint32_t b0, bool blocks) {
        w = lane_work(a, b0 + threadIdx.x % kWave);
        sum(a, blocks);
    }
    __device__ __forceinline__ void sum(const AttnRows& a, bool blocks) {
        own = (blocks ? head_list(a, w).blocks : w.tiles) * a.kv_heads;
        up = wave_scan_add(own);
    }
    __device__ __forceinline__ uint32_t all() const { return of_lane(up, kWave - 1); }
};
// The sequence that a unit is in, and the unit's place in it.
struct Found {
    SeqWork  w;
    uint32_t seq, at;
    bool     live;
};
// The call's units. The first 64 sequences' are kept in LDS, not in registers: every
// wave writes them there, the same, and reads what it has written.
struct UnitsLds {
    uint32_t v[6][kWave];
};
struct Units {
    UnitsLds& lds;
    uint32_t  total;
    bool      blocks;              // units are blocks of the list, not tiles
    __device__ __forceinline__ Units(const AttnRows& a, UnitsLds& s, bool list) : lds(s), total(0), blocks(list) {
        LaneUnits u;
        u.read(a, 0, list);
        count(a, u);
        if (list && total < uint64_t(a.least_run) * a.target) {
            blocks = false;
            u.sum(a, false);
            count(a, u);
        }
        const uint32_t lane = threadIdx.x % kWave;
        s.v[0][lane] = u.w.n_new, s.v[1][lane] = u.w.tiles, s.v[2][lane] = uint32_t(u.w.past), s.v[3][lane] = u.own, s.v[4][lane] = u.up;
        s.v[5][lane] = u.w.first;
    }
    __device__ __forceinline__ void count(const AttnRows& a, const LaneUnits& u) {
        total = u.all();
        for (uint32_t b0 = kWave; b0 < a.n_seq; b0 += kWave) {
            LaneUnits v;
            v.read(a, b0, blocks);
            total += v.all();
        }
        total = uniform(min(total, a.most_blocks));
    }
    __device__ __forceinline__ Found find(const AttnRows& a, uint32_t i) const {
        const uint32_t lane = threadIdx.x % kWave;
        uint32_t before = 0;
        LaneUnits v{{lds.v[5][lane], lds.v[0][lane], lds.v[1][lane], int32_t(lds.v[2][lane])}, lds.v[3][lane], lds.v[4][lane]};
        for (uint32_t b0 = 0; b0 < a.n_seq; b0 += kWave) {
            if (b0) v.read(a, b0, blocks);
            const uint64_t hit = __ballot(i < before + v.up);
            if (hit) {
                const uint32_t l = uint32_t(__ffsll(static_cast<long long>(hit))) - 1u;
                return {work_of_lane(v.w, l), uniform(b0 + l), uniform(i - before - of_lane(v.up - v.own, l)), true};
            }
            before += v.all();
        }
        return {{0, 0, 0, 0}, 0, 0, false};
    }
};
// The piece at place `at` of the list (n up to the tile's end; 0: not live, or a
// gap of `of`).
__device__ __forceinline__ Piece list_piece(const AttnRows& a, const Units& units, uint32_t at, SeqWork* work) {
    const Found f = units.find(a, at);
    Piece p{0, 0, 0, 0, 0, 0, false};
    if (!f.live) return p;
    const HeadList l = head_list(a, f.w);
    const uint32_t h = l.blocks ? f.at / l.blocks : a.kv_heads;
    if (h >= a.kv_heads) return p;
    p = head_piece(a, f.w, l, f.at - h * l.blocks);
    *work = f.w;
    return {f.seq, uniform(p.tile), uniform(h), uniform(p.blk), uniform(p.n), uniform(p.of), p.live};
}
// The call's tile i, whole.
__device__ __forceinline__ Piece whole_tile(const AttnRows& a, const Units& units, uint32_t i, SeqWork* work) {
    const Found f = units.find(a, i);
    const uint32_t tile = f.w.tiles - 1u - f.at / a.kv_heads;
    if (!f.live || tile >= f.w.tiles) return {0, 0, 0, 0, 0, 0, false};
    *work = f.w;
    const uint32_t n = tile_blocks(a, f.w, tile).n;
    return {f.seq, uniform(tile), uniform(f.at % a.kv_heads), 0, uniform(n), uniform(n), true};
}
// Workgroup `block` of the grid as one of the list: neighbours in it share keys, so
// each XCD (which takes every eighth workgroup) gets an eighth of it.
__device__ __forceinline__ uint32_t list_wg(const AttnRows& a, uint32_t blocks, uint32_t block) {
    return blocks > a.target && a.target % 8 == 0 ? (block % 8) * (a.target / 8) + block / 8 : block;
}

// The pieces of this workgroup, one after the other, with the sequence's work.
template <bool LIST>
struct Dealer {
    Units    units;
    uint32_t at, end, wg;          // places of the list, or tiles
    __device__ __forceinline__ Dealer(const AttnRows& a, UnitsLds& s) : units(a, s, LIST), at(blockIdx.x), end(units.total), wg(blockIdx.x) {
        if (LIST && units.blocks) {
            wg = uniform(list_wg(a, units.total, blockIdx.x));
            at = uniform(wg < units.total ? run_first(a, units.total, wg) : 0u);
            end = uniform(wg < units.total ? run_first(a, units.total, wg + 1) : 0u);
        }
    }
    // For the join: of the last piece that next() gave, or that there was none to join.
    __device__ __forceinline__ void join(const AttnRows& a, const Piece& p, const SeqWork& w, uint32_t rows) const {
        const uint32_t last = at - p.n - p.blk + p.of - 1u;       // the tile's last block
        const uint32_t parts = p.live && p.blk == 0 && p.n < p.of && last < units.total ? run_of(a, units.total, last) - wg + 1u : 0u;
        if (threadIdx.x == 0)
            reinterpret_cast<JoinTile*>(a.part)[wg] = {parts, p.tile << a.row_shift, rows, p.kv_head, w.first, w.past, {0, 0}};
    }
    // (not live at the end)
    __device__ __forceinline__ Piece next(const AttnRows& a, SeqWork* work) {
        if constexpr (!LIST) {
            Piece p{0, 0, 0, 0, 0, 0, false};
            if (wg == blockIdx.x) p = whole_tile(a, units, wg, work);
            wg = ~0u;                                             // one only
            p.live = p.live && p.n > 0;
            return p;
        }
        while (at < end) {
            if (units.blocks) {
                Piece p = list_piece(a, units, at, work);
                if (!p.live) break;
                if (p.n) {
                    p.n = min(p.n, end - at);
                    at += p.n;
                    return p;
                }
                at += p.of;
            } else {
                const Piece p = whole_tile(a, units, at, work);
                at += a.target;
                if (!p.live) break;
                if (p.n) return p;
            }
        }
        return {0, 0, 0, 0, 0, 0, false};
    }
};

// Uniform words of tables that no kernel changes while it runs.
__device__ __forceinline__ int32_t uniform_word(const int32_t* p, uint64_t i) {
    return ((const __attribute__((address_space(4))) int32_t*)p)[i];
}
__device__ __forceinline__ int32_t uniform_page(const PageMap& m, uint32_t b, int32_t p) {
    const uint32_t i = uint32_t(p) >> m.page_shift;
    if (p < 0 || i >= m.table) return -1;
    const int32_t g = uniform_word(m.pages, uint64_t(b) * m.table + i);
    return g >= 0 && uint32_t(g) < m.n_pages ? g : -1;
}

// The pages of the 16-key groups that lane l of a wave is asked for, in front of
// their use: kNoKeys where no row of the tile sees the group, kNoPage where it has no
// page.
constexpr int32_t kNoKeys = -1, kNoPage = -2;
__device__ __forceinline__ int32_t lane_page(const AttnRows& a, uint32_t seq, const KeyRange& keys, int32_t key) {
    if (key >= keys.hi || key + 16 <= keys.lo) return kNoKeys;
    const int32_t g = page_of(a.map, seq, key);
    return g < 0 ? kNoPage : g;
}

// ---- operands ------------------------------------------------------------------------
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <bool BF16>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <bool BF16>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// 16 keys: k = 4 (lane / 16) + 0..3
template <bool BF16>
__device__ __forceinline__ f32x4 mfma16k16(u32x2 a, u32x2 b, f32x4 c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack_op(float x, float y) {
    if constexpr (BF16) return pack_bf16(x, y);
    else return pack_f16(x, y);
}
// Four codes of 8 bits as F16 terms (exact: a whole number up to 128, or four
// bits of mantissa).
template <int CACHE>
__device__ __forceinline__ u32x2 widen4(uint32_t w) {
    if constexpr (CACHE == XP_ELEM_E4M3) {
        const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(int(w), 1.0f, false);
        const auto hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(int(w), 1.0f, true);
        return {__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
    } else {
        // the byte c + 128 in the mantissa of 1024: 1152 + c, less 1152
        const uint32_t u = w ^ 0x80808080u;
        const f16x2 bias{_Float16(1152.0f), _Float16(1152.0f)};
        const f16x2 lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias;
        const f16x2 hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias;
        return {__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
    }
}

// ---- tiles in LDS -------------------------------------------------------------------
// A tile holds keys as rows of DP elements in 16-byte chunks; chunk c of a key lies in
// place c ^ f(key), so that what a wave reads at once meets each of the 64 banks once: a
// line of 256 bytes, which holds up to four short rows. Of K a lane reads a chunk, 16
// following keys at a time (as f has it 6.7 cycles a read, with eight values of f for 16
// keys 8.3; rows of 32 chunks all the same get eight, as sixteen take more registers than
// there are: a prompt of 8192, 16 heads over 4 of 256, 892 us so, 988 with sixteen). V is
// read transposed, half a wave at a time: 16-bit elements as four following keys of 64
// bytes in the kernels of 32 rows (HI 3), eight of 32 in that of 16 (HI 4); 8-bit ones as
// keys 0..3 and 8..11 of 32 bytes, and keys 0..7 and 16..23 of 16.
template <int CHUNKS>
__device__ __forceinline__ constexpr uint32_t swizzle_k(uint32_t key) {
    return CHUNKS >= 32 ? ((key & 3u) << 1) | ((key >> 2) & 1u) : CHUNKS == 16 ? key & 15u : CHUNKS == 8 ? (key >> 1) & 7u : (key >> 2) & 3u;
}
template <int CHUNKS, bool BYTES, int HI>
__device__ __forceinline__ constexpr uint32_t swizzle_v(uint32_t key) {
    constexpr int LINE = CHUNKS >= 16 ? 0 : CHUNKS == 8 ? 1 : 2;         // log2 of the rows in 256 bytes
    if constexpr (!BYTES) return HI == 3 ? ((key & 3u) >> LINE) << 2 : ((key & 7u) >> LINE) << 1;
    const uint32_t far = (key >> HI) & 1u;
    if constexpr (HI == 3) return (((key & 3u) >> LINE) | (far << (2 - LINE))) << 1;
    else return ((key & 7u) >> LINE) | (far << (3 - LINE));
}

// Loads straight into LDS, lane l's 16 (4) bytes to lds + 16 l (4 l): from a
// lane's own address, or from an offset to a uniform one. ONCE marks them as not to be
// kept in the caches (1 GiB read so: 7.0 TB/s, without 6.2). In assembly, because the
// compiler puts a wait for every such load in flight before any read of LDS, the
// other stage's too; the kernels wait themselves (wait_loads) before they read a
// stage. No register is written, so nothing can be reused while they fly; the
// compiler's own waits only get longer by them. m0 holds the LDS address, and a
// load may follow its write after one wait state.
__device__ __forceinline__ uint32_t lds_offset(const void* p) {
    return uniform(uint32_t(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void*)p)));
}
template <bool ONCE>
__device__ __forceinline__ void to_lds16(const void* from, uint32_t lds) {
    if constexpr (ONCE)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" ::"s"(uniform(lds)), "v"(from) : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(uniform(lds)), "v"(from) : "memory", "m0");
}
template <bool ONCE>
__device__ __forceinline__ void to_lds16(const void* base, uint32_t off, uint32_t lds) {
    if constexpr (ONCE)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(uniform(lds)), "v"(off), "s"(base) : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(uniform(lds)), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void to_lds4(const void* from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(uniform(lds)), "v"(from) : "memory", "m0");
}
// Until at most N loads of this wave are in flight (they land in order).
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// Column reads: lanes 16 g .. 16 g + 15 address four rows of 16 elements (8
// bytes a lane, 4 lanes a row); lane i of them gets element i of each row.
__device__ __forceinline__ u32x2 lds_tr16(const void* p) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
}
// The same of bytes: eight rows, two lanes a row.
__device__ __forceinline__ u32x2 lds_tr8(const void* p) {
    typedef int i32x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2*)p));
}

// What lies outside of a tile is read from here.
static __device__ const u32x4 g_attn_zero = {0u, 0u, 0u, 0u};
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
// The larger of x here and 16 (32) lanes away; every lane of the four (two) gets it.
__device__ __forceinline__ float max_xor32(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_xor16(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float add_xor16(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// x and y as sums of two F16 terms of the same sign: the first rounded towards
// zero, the second, the rest rounded to nearest, at least 2^-24 where the first is
// not zero. So x times an infinity is one (a term of 0, or of the other sign, would
// make it NaN). Off by 2^-21 of the value (half a step of a rest under 2^-10 of it),
// or 2^-24.
__device__ __forceinline__ void two_terms(float x, float y, uint32_t& hi, uint32_t& lo) {
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x, y));
    const float a = f16_lo(hi), b = f16_hi(hi), u = fmaxf(fabsf(x - a), 0x1p-24f), v = fmaxf(fabsf(y - b), 0x1p-24f);
    lo = pack_f16(a == 0.0f ? x : copysignf(u, x), b == 0.0f ? y : copysignf(v, y));
}

// ---- queries ------------------------------------------------------------------------
// A query row's operands: STEPS runs of eight dims, run s from dim(s) on (past the
// head's dims: zeros). Queries of another type than the operands' (and those of
// two terms) are taken as 2^e times F16 numbers, the row's largest in [2^14, 2^15),
// so that none is out of range: BF16 ones keep all their bits down to 2^-38 of the
// largest, and F32 ones are the sum of two terms, 21 bits. GROUPS: the lanes that
// hold a row, 64 / GROUPS apart. read() only sends for them, so that the first keys'
// loads are on their way before take() waits.
template <bool BF16, int TERMS, int STEPS, int GROUPS>
struct Query {
    u32x4 hi[STEPS], lo[TERMS == 2 ? STEPS : 1];
    float up;                      // 2^e
    template <typename DimOf>
    __device__ __forceinline__ void read(const AttnRows& a, uint64_t at, DimOf dim) {
        const uint32_t D = a.head_dim;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const uint64_t i = dim(s) < D ? at + dim(s) : at;
            if constexpr (TERMS == 2) {
                const u32x4* p = reinterpret_cast<const u32x4*>(static_cast<const float*>(a.q) + i);
                hi[s] = p[0];
                lo[s] = p[1];
            } else {
                hi[s] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q) + i);
            }
        }
    }
    template <typename DimOf>
    __device__ __forceinline__ void take(const AttnRows& a, DimOf dim) {
        const uint32_t D = a.head_dim;
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
            if (dim(s) >= D) {
                hi[s] = u32x4{0u, 0u, 0u, 0u};
                if constexpr (TERMS == 2) lo[s] = hi[s];
            }
        up = 1.0f;
        if (TERMS == 1 && a.q_elem == (BF16 ? XP_ELEM_BF16 : XP_ELEM_F16)) return;
        // F32, or the other 16-bit type
        auto at = [&](int s, int j) -> float {
            if constexpr (TERMS == 2) return __uint_as_float(j < 4 ? hi[s][j] : lo[s][j - 4]);
            else if constexpr (BF16) return j % 2 ? f16_hi(hi[s][j / 2]) : f16_lo(hi[s][j / 2]);
            else return j % 2 ? bf16hi(hi[s][j / 2]) : bf16lo(hi[s][j / 2]);
        };
        float top = 0.0f;
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(at(s, j)));
        top = max_xor32(top);
        if constexpr (GROUPS == 4) top = max_xor16(top);
        const uint32_t e = __float_as_uint(top) >> 23;
        const bool fit = e >= 15u && e <= 253u;
        const float down = fit ? __uint_as_float((268u - e) << 23) : 1.0f;
        up = fit ? __uint_as_float((e - 14u) << 23) : 1.0f;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            u32x4 h{}, r{};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float u = at(s, 2 * w) * down, v = at(s, 2 * w + 1) * down;
                uint32_t p, q = 0;
                if constexpr (TERMS == 2) two_terms(u, v, p, q);
                else p = pack_op<BF16>(u, v);
                h[w] = p;
                r[w] = q;
            }
            hi[s] = h;
            if constexpr (TERMS == 2) lo[s] = r;
        }
    }
};

// Four dims of an output row: o / sum, zeros where nothing was seen.
__device__ __forceinline__ void store_row4(const AttnRows& a, uint32_t tok, uint32_t head, uint32_t d, f32x4 o, float sum) {
    const float norm = sum == 0.0f ? 0.0f : 1.0f / sum;
    const uint64_t at = uint64_t(tok) * a.out_stride + uint64_t(head) * a.head_dim + d;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] *= norm;
    if (a.q_elem == XP_ELEM_F32) *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + at) = o;
    else
        *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.out) + at) =
            a.q_elem == XP_ELEM_F16 ? u32x2{pack_f16(o[0], o[1]), pack_f16(o[2], o[3])} : u32x2{pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3])};
}

// Weights of two F16 terms, or of one.
template <bool BF16, int TERMS>
__device__ __forceinline__ void pack_weights(float x, float y, uint32_t& hi, uint32_t& lo) {
    if constexpr (TERMS == 2) two_terms(x, y, hi, lo);
    else hi = pack_op<BF16>(x, y);
}

// The power of two at or over the largest finite scale of a tile (as its
// exponent), which the weights are divided by so that weight times scale stays
// in F16's range.
__device__ __forceinline__ float scale_exponent(float largest) {
    const uint32_t u = __float_as_uint(largest);
    return fmaxf(float(int(u >> 23) - 127 + ((u & 0x7FFFFFu) != 0u)), -100.0f);
}
#endif  // __HIPCC__

// The parts: record 2 w + 1 of workgroup w for a tile that begins in its run and
// does not end there, 2 w for one that began before. A record is tile_rows sums
// of DP values, then a (reference, sum of weights) pair a row.
XP_HD uint64_t part_floats(uint32_t tile_rows, uint32_t dp) { return uint64_t(tile_rows) * (dp + 2); }

__device__ __forceinline__ float* part_record(const AttnRows& a, uint32_t wg, bool begins, uint64_t floats) {
    return a.part + size_t(a.target) * (sizeof(JoinTile) / 4) + (2ull * wg + (begins ? 1u : 0u)) * floats;
}

inline uint32_t padded_dim(uint32_t d) { return d <= 64 ? 64u : d <= 128 ? 128u : 256u; }

// The kernels' tiles: rows, and keys of a block (what a workgroup takes at a time).
constexpr uint32_t kFewRows = 16, kFewWaves = 4;
XP_HD constexpr uint32_t few_keys(uint32_t dp, uint32_t size) {    // of a wave at a time: 8 KB of K and V, 16 keys or more (32 of 8 bits)
    return size == 1 ? (dp == 64 ? 64u : 32u) : (dp == 64 ? 32u : 16u);
}
constexpr uint32_t kTileWaves = 4, kTileRows = 32 * kTileWaves;
XP_HD constexpr uint32_t tile_keys_of(uint32_t dp) { return dp == 256 ? 32u : 64u; }
constexpr uint32_t kMidWaves = 4, kMidRows = 32, kMidKeys = 32 * kMidWaves;
// Launchers; `grid` workgroups.
int launch_few(const AttnRows& a, int cache, uint32_t grid, hipStream_t st);
int launch_mid(const AttnRows& a, int cache, bool paged, uint32_t grid, hipStream_t st);
int launch_tile(const AttnRows& a, int cache, bool paged, uint32_t grid, hipStream_t st);

}  // namespace xp
