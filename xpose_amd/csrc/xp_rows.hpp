// Packed rows and paged caches: what the operators of rope_rows.hip,
// paged_kv.hip and rows_attention.hip share. The index functions are plain
// C++ (host and device), so that they can be checked without a GPU.
#pragma once

#include <cstdint>

#include "xp_internal.hpp"

namespace xp {

#define XP_HD __host__ __device__ __forceinline__

// ---- where a packed token and a position lie ----------------------------------

// Sequence b's packed rows, bounded to [0, n_tokens] and not falling.
struct RowSpan {
    uint32_t first, end;
};
XP_HD RowSpan row_span(const int32_t* cu, uint32_t n_tokens, uint32_t b) {
    const int64_t n = n_tokens, x = cu[b], y = cu[b + 1];
    const int64_t a = x < 0 ? 0 : (x > n ? n : x);
    const int64_t e = y < a ? a : (y > n ? n : y);
    return {uint32_t(a), uint32_t(e)};
}
// The sequence that holds packed token t, or n_seq: the last one whose first
// row is not behind t (empty sequences before it share that row).
XP_HD uint32_t seq_of_row(const int32_t* cu, uint32_t n_seq, uint32_t n_tokens, uint32_t t) {
    uint32_t lo = 0, hi = n_seq;                   // cu[lo] <= t < cu[hi], as far as cu says so
    while (lo + 1 < hi) {
        const uint32_t m = (lo + hi) / 2;
        if (int64_t(cu[m]) <= int64_t(t)) lo = m; else hi = m;
    }
    const RowSpan r = row_span(cu, n_tokens, lo);
    return t >= r.first && t < r.end ? lo : n_seq;
}
// The position of row i (of n new ones) of a sequence of length len; negative
// where the sequence is shorter than its new rows.
XP_HD int64_t row_position(int32_t len, uint32_t n, uint32_t i) { return int64_t(len) - int64_t(n) + int64_t(i); }

struct PageMap {
    const int32_t* pages;
    uint32_t       table, n_pages, page_shift;
};
// The page of position p of sequence b, or -1 where it has none.
XP_HD int32_t page_of(const PageMap& m, uint32_t b, int64_t p) {
    const int64_t i = p >> m.page_shift;
    if (p < 0 || i >= int64_t(m.table)) return -1;
    const int32_t g = m.pages[uint64_t(b) * m.table + uint64_t(i)];
    return g >= 0 && uint32_t(g) < m.n_pages ? g : -1;
}
// The row (in rows of head_dim) of kv head h in slot `slot` of page g.
XP_HD uint64_t cache_row(uint32_t g, uint32_t kv_heads, uint32_t h, uint32_t page_shift, uint32_t slot) {
    return ((uint64_t(g) * kv_heads + h) << page_shift) + slot;
}

// ---- the host's checks ----------------------------------------------------------

inline uint32_t elem_bytes(int e) {
    return e == XP_ELEM_F32 ? 4u : e == XP_ELEM_F16 || e == XP_ELEM_BF16 ? 2u : 1u;
}
// Each returns XP_OK or XP_E_ARG with a message naming `fn` and `what`.
int check_rows(const char* fn, const char* what, const xp_rows* r, uint32_t head_dim, uint32_t align);
int check_cache(const char* fn, const xp_paged_kv* c);
int check_seqs(const char* fn, const xp_paged_seqs* s);
// Whether `stream` and `out` are the current device's.
int check_here(const char* fn, xp_stream stream, const void* out);
PageMap page_map(const xp_paged_kv* c, const xp_paged_seqs* s);

#define XP_CHECK(call)                            \
    do {                                          \
        if (int _rc = (call); _rc != XP_OK) return _rc; \
    } while (0)

}  // namespace xp
