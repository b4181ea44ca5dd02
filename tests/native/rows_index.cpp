// The index functions of packed rows and paged caches (xpose_amd/csrc/xp_rows.hpp),
// the ones the kernels call, for the tests of ragged, malformed and bad tables.
#include "../../xpose_amd/csrc/xp_rows.hpp"

extern "C" {

void ri_row_span(const int32_t* cu, uint32_t n_tokens, uint32_t b, uint32_t* out) {
    const xp::RowSpan r = xp::row_span(cu, n_tokens, b);
    out[0] = r.first;
    out[1] = r.end;
}
uint32_t ri_seq_of_row(const int32_t* cu, uint32_t n_seq, uint32_t n_tokens, uint32_t t) {
    return xp::seq_of_row(cu, n_seq, n_tokens, t);
}
int64_t ri_row_position(int32_t len, uint32_t n, uint32_t i) { return xp::row_position(len, n, i); }
int32_t ri_page_of(const int32_t* pages, uint32_t table, uint32_t n_pages, uint32_t shift, uint32_t b, int64_t p) {
    return xp::page_of(xp::PageMap{pages, table, n_pages, shift}, b, p);
}
uint64_t ri_cache_row(uint32_t g, uint32_t kv_heads, uint32_t h, uint32_t shift, uint32_t slot) {
    return xp::cache_row(g, kv_heads, h, shift, slot);
}

}  // extern "C"
