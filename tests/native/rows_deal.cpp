// The deal of xpose_amd/csrc/xp_rows_deal.hpp, walked as the kernels walk it.
#include <cstring>
#include <vector>

#include "../../xpose_amd/csrc/xp_rows_deal.hpp"

// Walks the list of a call and counts how often each block of each tile comes up.
// 0: every block once, the join finds every tile where it was dealt, and no
// workgroup writes a record twice; otherwise the number of the first thing that
// does not hold. *waste: places of the list without a block, in thousandths.
extern "C" int rd_walk(const int32_t* cu, const int32_t* kv_len, uint32_t n_seq, uint32_t n_tokens, uint32_t heads, uint32_t kv_heads,
                       uint32_t window, uint32_t row_shift, uint32_t block_shift, uint32_t target, int32_t most_keys,
                       uint32_t* blocks_out, uint32_t* waste) {
    using namespace xp;
    AttnRows a{};
    a.cu = cu, a.kv_len = kv_len, a.n_seq = n_seq, a.n_tokens = n_tokens, a.heads = heads, a.kv_heads = kv_heads, a.window = window;
    a.row_shift = row_shift, a.block_shift = block_shift, a.target = target, a.target_shift = uint32_t(__builtin_ctz(target)), a.most_keys = most_keys;
    set_group(a);
    uint32_t blocks = 0;
    std::vector<uint32_t> before;
    std::vector<std::vector<int>> seen;            // of each (sequence, head, tile)
    std::vector<std::vector<size_t>> index;
    for (uint32_t b = 0; b < n_seq; ++b) {
        const SeqWork w = seq_work(a, b);
        before.push_back(blocks);
        blocks += head_list(a, w).blocks * kv_heads;
        index.emplace_back();
        for (uint32_t h = 0; h < kv_heads; ++h)
            for (uint32_t t = 0; t < w.tiles; ++t) {
                index[b].push_back(seen.size());
                seen.emplace_back(tile_blocks(a, w, t).n, 0);
            }
    }
    *blocks_out = blocks;
    uint32_t gaps = 0, last = 0;
    for (uint32_t wg = 0; wg < target; ++wg) {
        uint32_t at = wg < blocks ? run_first(a, blocks, wg) : 0, end = wg < blocks ? run_first(a, blocks, wg + 1) : 0;
        if (wg < blocks && (at != last || end < at)) return 1;
        if (wg < blocks) last = end;
        int records[2] = {0, 0};
        while (at < end) {
            if (run_of(a, blocks, at) != wg) return 2;
            uint32_t b = 0;
            while (b + 1 < n_seq && before[b + 1] <= at) ++b;
            const SeqWork w = seq_work(a, b);
            const HeadList l = head_list(a, w);
            const uint32_t place = at - before[b], h = place / l.blocks;
            if (h >= kv_heads) return 3;
            const Piece p = head_piece(a, w, l, place - h * l.blocks);
            if (!p.live) return 4;
            if (p.n == 0) {
                if (p.of == 0) return 5;
                gaps += p.of < end - at ? p.of : end - at;
                at += p.of;
                continue;
            }
            const uint32_t n = p.n < end - at ? p.n : end - at;
            std::vector<int>& s = seen[index[b][h * w.tiles + p.tile]];
            for (uint32_t i = p.blk; i < p.blk + n; ++i) ++s.at(i);
            if (p.of != s.size()) return 6;
            const uint32_t first = before[b] + h * l.blocks + tile_place(a, w, l, p.tile);
            if (first + p.blk != at) return 7;
            const uint32_t w0 = run_of(a, blocks, first), w1 = run_of(a, blocks, first + p.of - 1);
            if ((n < p.of) != (w0 != w1)) return 8;
            if (n < p.of) {
                if (records[p.blk == 0]++) return 9;
                if ((p.blk == 0) != (wg == w0)) return 10;
            }
            at += n;
        }
    }
    if (blocks && last != blocks) return 11;
    for (const std::vector<int>& s : seen)
        for (int c : s)
            if (c != 1) return 12;
    *waste = blocks ? uint32_t(uint64_t(gaps) * 1000 / blocks) : 0;
    return 0;
}

// by_group against a division, for one number of query heads a kv head.
extern "C" int rd_by_group(uint32_t d, const uint32_t* n, uint32_t count) {
    xp::AttnRows a{};
    a.heads = d, a.kv_heads = 1;
    xp::set_group(a);
    for (uint32_t i = 0; i < count; ++i)
        if (xp::by_group(a, n[i]) != n[i] / d) return 1;
    return 0;
}
