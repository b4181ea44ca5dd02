// How the attention of packed rows deals its work to workgroups: arguments and plain
// index functions (host and device), so that they can be checked without a GPU.
#pragma once

#include "xp_rows.hpp"

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
    // How the work is dealt (below): rows of a tile and keys of a block (powers of
    // two), the workgroups that share the list (0: a tile each) and where their
    // parts go, the most blocks of the list, the positions of the page table
    uint32_t    row_shift, block_shift, target, target_shift, least_run, most_blocks;
    int32_t     most_keys;
    uint32_t    group_mul, group_shift;    // n / (heads / kv_heads) = n group_mul >> group_shift
    float*      part;
};

// ---- how the work is dealt -------------------------------------------------------
// Row i of sequence b and kv head h is token i / group, head h group + i %
// group: the query heads of one kv head share its keys. Rows go by tiles, keys
// by blocks; a tile's blocks are those that any of its rows sees.
//
// Where the tiles alone fill the device (target 0) a workgroup takes one whole
// tile: the longest first, the kv head changing fastest, so that the tiles of
// a head meet in one XCD's L2 where kv_heads shares a factor with 8.
//
// Otherwise `target` workgroups share the call, by its lengths, which only the
// kernel knows. Where a workgroup would get fewer than least_run blocks each takes
// whole tiles, every target-th of that order. Else all blocks, tile after tile, are one
// list that they share in equal runs. A run's first and last tile may be parts; their
// sums go to `part`, two records a workgroup, and the join kernel adds them; whole
// tiles are written at once. In the list, tile v of a head comes after tile
// tiles - 1 - v: of a causal prompt such a pair has about the same blocks
// whatever v, so a place in the list is found by a division. (One odd tile in
// the middle comes last.)
//
// Every wave finds its own place from the lengths, 64 sequences at a time.
constexpr int32_t kMostKeys = 1 << 30;      // of a sequence
struct SeqWork {
    uint32_t first, n_new, tiles;  // first packed row, new tokens, row tiles of one kv head
    int32_t  past;                 // position of the first new token (negative: the sequence is shorter)
};
struct Blocks {
    uint32_t first, n;
};
XP_HD SeqWork seq_work(const AttnRows& a, uint32_t b) {
    const RowSpan r = row_span(a.cu, a.n_tokens, b);
    const uint32_t n = r.end - r.first, m = (1u << a.row_shift) - 1u;
    int32_t len = a.kv_len ? a.kv_len[b] : int32_t(n);
    len = len < 0 ? 0 : (len > kMostKeys ? kMostKeys : len);
    return {r.first, n, (n * (a.heads / a.kv_heads) + m) >> a.row_shift, len - int32_t(n)};
}
// n / d, d = heads / kv_heads, for n below 2^31 as a product: with 2^(l - 1) < d <=
// 2^l, s = 31 + l and m = ceil(2^s / d) < 2^32, n m / 2^s is over n / d by n (m d - 2^s) /
// (d 2^s) < n / 2^s <= 2^-l <= 1 / d, not enough to reach the next whole number
// (Granlund and Montgomery, 1994).
XP_HD void set_group(AttnRows& a) {
    const uint32_t d = a.heads / a.kv_heads;
    uint32_t l = 0;
    while ((1u << l) < d) ++l;
    a.group_shift = 31 + l;
    a.group_mul = uint32_t(((1ull << a.group_shift) + d - 1) / d);
}
XP_HD uint32_t by_group(const AttnRows& a, uint32_t n) { return uint32_t((uint64_t(n) * a.group_mul) >> a.group_shift); }
// The keys [lo, hi) that tokens at positions p0 .. p1 see. Past the table one
// position is left, which has no page: who sees it or more gets NaN.
struct KeyRange {
    int32_t lo, hi;
};
XP_HD KeyRange seen_keys(const AttnRows& a, int32_t p0, int32_t p1) {
    int32_t hi = p1 + 1 < 0 ? 0 : p1 + 1, lo = a.window && a.window <= uint32_t(kMostKeys) ? p0 - int32_t(a.window) + 1 : 0;
    hi = hi > a.most_keys + 1 ? a.most_keys + 1 : hi;
    lo = lo < 0 ? 0 : (lo > a.most_keys ? a.most_keys : lo);
    return {lo, hi};
}
// The blocks of one tile.
XP_HD Blocks tile_blocks(const AttnRows& a, const SeqWork& w, uint32_t tile) {
    const uint32_t r0 = tile << a.row_shift, rows = w.n_new * (a.heads / a.kv_heads);
    const uint32_t r1 = r0 + (1u << a.row_shift) < rows ? r0 + (1u << a.row_shift) : rows;
    const KeyRange k = seen_keys(a, w.past + int32_t(by_group(a, r0)), w.past + int32_t(by_group(a, r1 - 1u)));
    const uint32_t f = uint32_t(k.lo) >> a.block_shift, e = (uint32_t(k.hi) + (1u << a.block_shift) - 1u) >> a.block_shift;
    return {f, e > f ? e - f : 0u};
}
// The list of one kv head of a sequence: `pairs` runs of `pair` blocks and the
// middle tile's. `pair` is at least what tiles v and tiles - 1 - v have together,
// for every v. A tile sees up to its last token, hi(v) = past + floor(((v + 1) rows
// - 1) / group) + 1 or 0 where that is negative (the last tile, which may be part
// filled, and any past the table, less): convex in v but for the rounding, so the
// pair of the first and the last tile has the most, less one token a rounding;
// and ceil(x / k) + ceil(y / k) <= (x + y + 2 (k - 1)) / k. With a window no tile has
// more than the window before its first token, its tokens and a block's rest on
// either side.
struct HeadList {
    uint32_t pairs, pair, blocks;
};
XP_HD HeadList head_list(const AttnRows& a, const SeqWork& w) {
    HeadList l{w.tiles / 2, 0, 0};
    if (w.tiles == 0) return l;
    if (l.pairs) {
        // (halves and rests apart: all fits 32 bits)
        const uint32_t m = (1u << a.block_shift) - 1u;
        auto hi = [&](uint32_t tiles) {
            const int32_t h = w.past + int32_t(by_group(a, (tiles << a.row_shift) - 1u));
            return uint32_t(h < -1 ? 0 : h + 1);
        };
        const uint32_t x = hi(w.tiles), y = hi(1);
        uint32_t most = (x >> a.block_shift) + (y >> a.block_shift) + (((x & m) + (y & m) + 2 + 2 * m) >> a.block_shift);
        const uint32_t table = 2 * ((uint32_t(a.most_keys) + 1 + m) >> a.block_shift);
        most = most < table ? most : table;
        if (a.window && a.window <= uint32_t(kMostKeys)) {
            const uint32_t full = 2 * ((a.window + by_group(a, (1u << a.row_shift) - 1u) + 1u + 2 * m) >> a.block_shift);
            most = most < full ? most : full;
        }
        l.pair = most;
    }
    l.blocks = l.pairs * l.pair + (w.tiles % 2 ? tile_blocks(a, w, w.tiles / 2).n : 0u);
    return l;
}
// Where tile `tile` begins in its head's list (the walk of head_piece backwards).
XP_HD uint32_t tile_place(const AttnRows& a, const SeqWork& w, const HeadList& l, uint32_t tile) {
    const uint32_t v = tile < w.tiles - 1u - tile ? tile : w.tiles - 1u - tile;
    if (tile == w.tiles - 1u - tile) return l.pairs * l.pair;
    return v * l.pair + (tile == v ? tile_blocks(a, w, w.tiles - 1u - v).n : 0u);
}
// The run of workgroup w, [run_first(w), run_first(w + 1)), of a list of `blocks`, and
// the workgroup of a block. (target is 2^target_shift.)
XP_HD uint32_t run_first(const AttnRows& a, uint32_t blocks, uint32_t w) {
    return blocks <= a.target ? w : uint32_t((uint64_t(w) * blocks) >> a.target_shift);
}
XP_HD uint32_t run_of(const AttnRows& a, uint32_t blocks, uint32_t block) {
    if (blocks <= a.target) return block;
    // a float's guess is at most one off (24 bits, target at most 2^16)
    uint32_t w = uint32_t(float(block) * (float(a.target) / float(blocks)));
    w = w < a.target ? w : a.target - 1u;
    if (run_first(a, blocks, w) > block) --w;
    else if (run_first(a, blocks, w + 1) <= block) ++w;
    return w;
}
// What a workgroup does next: blocks [blk, blk + n) of a tile's `of`.
struct Piece {
    uint32_t seq, tile, kv_head, blk, n, of;
    bool     live;
};
// The place `at` of a head's list: the tile, its block, and how many places to
// its end; n 0 in the gap behind a pair, `of` then the gap's length.
XP_HD Piece head_piece(const AttnRows& a, const SeqWork& w, const HeadList& l, uint32_t at) {
    Piece p{0, 0, 0, 0, 0, 0, true};
    const uint32_t v = l.pair ? at / l.pair : 0u;
    if (v >= l.pairs) {
        p.tile = w.tiles / 2;
        p.blk = at - l.pairs * l.pair;
        p.of = tile_blocks(a, w, p.tile).n;
    } else {
        const uint32_t off = at - v * l.pair, big = tile_blocks(a, w, w.tiles - 1u - v).n, small = tile_blocks(a, w, v).n;
        if (off < big) p.tile = w.tiles - 1u - v, p.blk = off, p.of = big;
        else if (off < big + small) p.tile = v, p.blk = off - big, p.of = small;
        else return Piece{0, 0, 0, 0, 0, l.pair - off, true};
    }
    p.n = p.of > p.blk ? p.of - p.blk : 0u;
    p.live = p.tile < w.tiles && p.n > 0;
    return p;
}

// What the join kernel has to know of the tile that begins in a workgroup's run and
// does not end there, written by that workgroup: its parts (0: there is none), its
// rows, kv head and sequence. `target` of these are in front of the parts.
struct JoinTile {
    uint32_t parts, r0, rows, kv_head, first;
    int32_t  past;
    uint32_t unused[2];
};

}  // namespace xp
