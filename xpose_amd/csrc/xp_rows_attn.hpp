// What the kernels of attention over packed rows share (rows_attn_few.hip,
// rows_attn_tile.hip, rows_attention.hip): arguments, how the work is dealt to
// workgroups, operands of the matrix instructions, tiles on their way to LDS.
#pragma once

#include "xp_elem.hpp"

namespace xp {

struct AttnRows {
    const void *q, *k, *v;         // k, v: the cache's planes, or the packed rows
    void*       out;
    const float *k_scale, *v_scale;
    uint64_t    q_stride, k_stride, v_stride, out_stride;   // elements
    const int32_t *cu, *kv_len;    // kv_len NULL: packed
    PageMap     map;
    uint32_t    n_seq, n_tokens, heads, kv_heads, head_dim, window;
    int32_t     q_elem;
    float       scale;
    // The deal (deal_item): rows of a tile and keys of a block (powers of two),
    // the items aimed at (0: the keys are not split), where the parts of split keys go
    uint32_t    row_shift, block_shift, target, items;
    float*      part;
};

// ---- how the work is dealt -------------------------------------------------------
// Row i of sequence b and kv head h is token i / group, head h group + i %
// group: the query heads of one kv head share its keys. An item is a tile of
// tile_rows such rows with a run of `chunk` blocks of the keys that the tile
// sees. Without a split there is one item a tile. With one, chunk is the same
// for all tiles and makes about `target` items of the whole call: workgroups
// with equal work, whatever the lengths. Every workgroup works that out from
// the lengths itself (64 sequences a step of a wave), as does the kernel that
// joins the parts. Items of a sequence run from its last tile, which sees the
// most keys, to its first; the kv head changes fastest, so that the tiles of a
// head meet in one XCD's L2 where kv_heads shares a factor with 8.
struct SeqWork {
    uint32_t tiles, span;          // row tiles of one kv head, most key blocks of any tile
};
constexpr int32_t kMostKeys = 1 << 30;      // of a sequence
XP_HD SeqWork seq_work(const AttnRows& a, uint32_t b) {
    const RowSpan r = row_span(a.cu, a.n_tokens, b);
    const uint32_t n = r.end - r.first, group = a.heads / a.kv_heads;
    int32_t len = a.kv_len ? a.kv_len[b] : int32_t(n);
    len = len < 0 ? 0 : (len > kMostKeys ? kMostKeys : len);
    uint32_t keys = uint32_t(len);
    if (a.window) {
        // the tokens of a tile's rows see a window before the first and
        // themselves, from anywhere in a block on
        const uint32_t seen = a.window > uint32_t(kMostKeys) ? uint32_t(kMostKeys) : a.window;
        const uint32_t most = seen + ((1u << a.row_shift) - 1u) / group + 1u + (1u << a.block_shift);
        keys = most < keys ? most : keys;
    }
    const uint32_t m = (1u << a.row_shift) - 1u, k = (1u << a.block_shift) - 1u;
    return {(n * group + m) >> a.row_shift, (keys + k) >> a.block_shift};
}
XP_HD uint32_t parts_of(const SeqWork& w, uint32_t chunk) { return w.span <= chunk ? 1u : (w.span + chunk - 1) / chunk; }

struct Item {
    uint32_t seq, tile, part, kv_head, chunk;
    bool     live;
};
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
// Blocks of a part, in a call of up to 64 sequences from w of each lane's (any
// rounding of the sum is every wave's).
__device__ __forceinline__ uint32_t chunk_of(const AttnRows& a, float blocks) {
    if (a.target == 0) return 0x7FFFFFFFu;
    return uniform(uint32_t(fminf(fmaxf(ceilf(blocks * float(a.kv_heads) / float(a.target)), 1.0f), 1e9f)));
}
__device__ __forceinline__ SeqWork lane_work(const AttnRows& a, uint32_t b) {
    return b < a.n_seq ? seq_work(a, b) : SeqWork{0, 0};
}
__device__ __forceinline__ uint32_t deal_chunk(const AttnRows& a) {
    if (a.target == 0) return 0x7FFFFFFFu;
    float blocks = 0.0f;
    for (uint32_t b0 = 0; b0 < a.n_seq; b0 += kWave) {
        const SeqWork w = lane_work(a, b0 + threadIdx.x % kWave);
        blocks += float(w.tiles) * float(w.span);
    }
    return chunk_of(a, wave_sum(blocks));
}
// Item i of the call; not live past the last one.
__device__ __forceinline__ Item deal_item(const AttnRows& a, uint32_t i) {
    const uint32_t lane = threadIdx.x % kWave;
    SeqWork w = lane_work(a, lane);
    // up to 64 sequences are read once
    const uint32_t chunk = a.n_seq <= kWave ? chunk_of(a, wave_sum(float(w.tiles) * float(w.span))) : deal_chunk(a);
    uint32_t before = 0;
    for (uint32_t b0 = 0; b0 < a.n_seq; b0 += kWave) {
        if (b0) w = lane_work(a, b0 + lane);
        const uint32_t parts = parts_of(w, chunk), own = w.tiles * parts * a.kv_heads, up = wave_scan_add(own);
        const uint64_t hit = __ballot(i < before + up);
        if (hit) {
            const uint32_t l = uint32_t(__ffsll(static_cast<long long>(hit))) - 1u;
            const uint32_t np = of_lane(parts, l), nt = of_lane(w.tiles, l);
            uint32_t j = i - before - of_lane(up - own, l);
            const uint32_t h = j % a.kv_heads;
            j /= a.kv_heads;
            // (sums of a cu that gives rows many times over may have wrapped)
            return {uniform(b0 + l), uniform(nt - 1u - j / np), uniform(j % np), uniform(h), chunk, j / np < nt};
        }
        before += of_lane(up, kWave - 1);
    }
    return {0, 0, 0, 0, chunk, false};
}
// The first item of tile `tile` of sequence `seq`, kv head `head`, and how many
// parts it has; they follow each other kv_heads apart.
__device__ __forceinline__ uint32_t deal_first(const AttnRows& a, uint32_t seq, uint32_t tile, uint32_t head, uint32_t* n_parts) {
    const uint32_t lane = threadIdx.x % kWave, chunk = deal_chunk(a);
    uint32_t before = 0;
    for (uint32_t b0 = 0; b0 < a.n_seq; b0 += kWave) {
        const SeqWork w = lane_work(a, b0 + lane);
        const uint32_t parts = parts_of(w, chunk), own = w.tiles * parts * a.kv_heads, up = wave_scan_add(own);
        if (seq < b0 + kWave) {
            const uint32_t l = seq - b0;
            *n_parts = of_lane(parts, l);
            return before + of_lane(up - own, l) + (of_lane(w.tiles, l) - 1u - tile) * *n_parts * a.kv_heads + head;
        }
        before += of_lane(up, kWave - 1);
    }
    *n_parts = 0;
    return 0;
}

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

// A tile's sequence: its packed rows and the position of its first new token.
struct TileSeq {
    uint32_t first, n_new;
    int32_t  past;                 // negative where it is shorter than its new rows
};
__device__ __forceinline__ TileSeq tile_seq(const AttnRows& a, uint32_t b) {
    const int32_t n = int32_t(a.n_tokens);
    const int32_t x = min(max(uniform_word(a.cu, b), 0), n), y = min(max(uniform_word(a.cu, b + 1), x), n);
    const int32_t len = a.kv_len ? min(max(uniform_word(a.kv_len, b), 0), kMostKeys) : y - x;
    return {uint32_t(x), uint32_t(y - x), len - (y - x)};
}
// The keys [lo, hi) that tokens at positions p0 .. p1 see, and of their blocks
// the run [first, end) of one part.
struct TileKeys {
    int32_t lo, hi, first, end;
};
__device__ __forceinline__ TileKeys tile_keys(const AttnRows& a, int32_t p0, int32_t p1, uint32_t part, uint32_t chunk) {
    TileKeys t;
    t.hi = max(p1 + 1, 0);
    t.lo = a.window && a.window <= uint32_t(kMostKeys) ? max(p0 - int32_t(a.window) + 1, 0) : 0;
    const int32_t b0 = t.lo >> a.block_shift, b1 = (t.hi + (1 << a.block_shift) - 1) >> a.block_shift;
    t.first = b0 + int32_t(part * chunk);
    t.end = b1 - t.first > int32_t(chunk) ? t.first + int32_t(chunk) : b1;
    return t;
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
// A tile holds keys as rows of DP elements in 16-byte chunks. A row is a
// multiple of 64 or 128 bytes, so the chunks of eight keys that a wave reads at
// once would meet in the same banks: chunk c of a key lies in place c ^ f(key).
// K is read a chunk a lane, eight following keys at a time. V is read
// transposed: 16 lanes take 4 keys of 32 bytes (16-bit elements) or 8 keys of 16
// bytes (8-bit ones: keys 4 h + 0..3 and, 8 or 16 on, four more), so there f takes other bits.
template <int CHUNKS>
__device__ __forceinline__ uint32_t swizzle_k(uint32_t key) {
    if constexpr (CHUNKS >= 8) return ((key & 3u) << 1) | ((key >> 2) & 1u);
    else return (key >> 1) & 3u;
}
// (HI: the bit that tells the second four of such eight keys from the first)
template <int CHUNKS, bool BYTES, int HI>
__device__ __forceinline__ uint32_t swizzle_v(uint32_t key) {
    if constexpr (!BYTES) return swizzle_k<CHUNKS>(key);
    else if constexpr (CHUNKS >= 8) return ((key & 3u) << 1) | ((key >> HI) & 1u);
    else return ((key >> 1) & 1u) | ((key >> (HI - 1)) & 2u);
}

// Loads straight into LDS, lane l's 16 (4) bytes to lds + 16 l (4 l): from a
// lane's own address, or from an offset to a uniform one. In assembly, because the
// compiler puts a wait for every such load in flight before any read of LDS, the
// other stage's too; the kernels wait themselves (wait_loads) before they read a
// stage. No register is written, so nothing can be reused while they fly; the
// compiler's own waits only get longer by them. m0 holds the LDS address, and a
// load may follow its write after one wait state.
__device__ __forceinline__ uint32_t lds_offset(const void* p) {
    return uniform(uint32_t(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void*)p)));
}
__device__ __forceinline__ void to_lds16(const void* from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(uniform(lds)), "v"(from) : "memory", "m0");
}
__device__ __forceinline__ void to_lds16(const void* base, uint32_t off, uint32_t lds) {
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
// largest, and F32 ones are the sum of two terms, 21 bits. Returns 2^e. GROUPS: the
// lanes that hold a row, 64 / GROUPS apart.
template <bool BF16, int TERMS, int STEPS, int GROUPS, typename DimOf>
__device__ __forceinline__ float load_query(u32x4 (&hi)[STEPS], u32x4 (&lo)[TERMS == 2 ? STEPS : 1], const AttnRows& a,
                                            uint64_t at, DimOf dim) {
    const uint32_t D = a.head_dim;
    if (TERMS == 1 && a.q_elem == (BF16 ? XP_ELEM_BF16 : XP_ELEM_F16)) {
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
        {
            const bool in = dim(s) < D;
            const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q) + (in ? at + dim(s) : at));
            hi[s] = in ? w : u32x4{0u, 0u, 0u, 0u};
        }
        return 1.0f;
    }
    // (of two terms: F32 alone; of one: the other 16-bit type; dims past the
    // head's: the row's first, as zeros)
    float x[STEPS][8], top = 0.0f;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const bool in = dim(s) < D;
        if constexpr (TERMS == 2) load8<XP_ELEM_F32>(a.q, in ? at + dim(s) : at, x[s]);
        else load8<BF16 ? XP_ELEM_F16 : XP_ELEM_BF16>(a.q, in ? at + dim(s) : at, x[s]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[s][j] = in ? x[s][j] : 0.0f;
            top = fmaxf(top, fabsf(x[s][j]));
        }
    }
    top = max_xor32(top);
    if constexpr (GROUPS == 4) top = max_xor16(top);
    const uint32_t e = __float_as_uint(top) >> 23;
    const bool fit = e >= 15u && e <= 253u;
    const float down = fit ? __uint_as_float((268u - e) << 23) : 1.0f, up = fit ? __uint_as_float((e - 14u) << 23) : 1.0f;
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float u = x[s][2 * w] * down, v = x[s][2 * w + 1] * down;
            if constexpr (TERMS == 2) {
                uint32_t p, r;
                two_terms(u, v, p, r);
                hi[s][w] = p;
                lo[s][w] = r;
            } else {
                hi[s][w] = pack_op<BF16>(u, v);
            }
        }
    return up;
}

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

// The parts of split keys: item i's rows, tile_rows sums of DP values each, then a
// (maximum, sum) pair a row.
XP_HD uint64_t part_floats(uint32_t tile_rows, uint32_t dp) { return uint64_t(tile_rows) * (dp + 2); }

inline uint32_t padded_dim(uint32_t d) { return d <= 64 ? 64u : d <= 128 ? 128u : 256u; }

// The kernels' tiles: rows, and keys of a block (what a workgroup takes at a time).
constexpr uint32_t kFewRows = 16, kFewWaves = 4;
XP_HD constexpr uint32_t few_keys(uint32_t dp, uint32_t size) {    // of a wave at a time: 8 KB of K and V, 16 keys or more (32 of 8 bits)
    return size == 1 ? (dp == 64 ? 64u : 32u) : (dp == 64 ? 32u : 16u);
}
constexpr uint32_t kTileWaves = 4, kTileRows = 32 * kTileWaves;
XP_HD constexpr uint32_t tile_keys_of(uint32_t dp) { return dp == 256 ? 32u : 64u; }
// Launchers; `items` workgroups.
int launch_few(const AttnRows& a, int cache, uint32_t items, hipStream_t st);
int launch_tile(const AttnRows& a, int cache, bool paged, uint32_t items, hipStream_t st);

}  // namespace xp
