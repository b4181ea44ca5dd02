// Argument checks shared by the operators over packed rows and paged caches.
#include "xp_rows.hpp"

namespace xp {

int check_rows(const char* fn, const char* what, const xp_rows* r, uint32_t head_dim, uint32_t align) {
    if (!r || !r->data) return set_error(XP_E_ARG, "%s: %s is null", fn, what);
    if (r->elem != XP_ELEM_F32 && r->elem != XP_ELEM_F16 && r->elem != XP_ELEM_BF16)
        return set_error(XP_E_ARG, "%s: %s: rows are F32, F16 or BF16, not elem %d", fn, what, r->elem);
    if (r->heads == 0 || r->heads > 65535u) return set_error(XP_E_ARG, "%s: %s has %u heads (1 to 65535)", fn, what, r->heads);
    if (r->stride < uint64_t(r->heads) * head_dim)
        return set_error(XP_E_ARG, "%s: %s: stride %llu is less than %u heads of %u", fn, what,
                         static_cast<unsigned long long>(r->stride), r->heads, head_dim);
    if (r->stride > (1ull << 26)) return set_error(XP_E_ARG, "%s: %s: stride is over 2^26 elements", fn, what);
    const uint32_t size = elem_bytes(r->elem);
    if (align < size) align = size;
    if (reinterpret_cast<uintptr_t>(r->data) % align || r->stride * size % align)
        return set_error(XP_E_ARG, "%s: %s: data and stride have to be multiples of %u bytes", fn, what, align);
    return XP_OK;
}

int check_cache(const char* fn, const xp_paged_kv* c) {
    if (!c || !c->k || !c->v) return set_error(XP_E_ARG, "%s: the cache is null", fn);
    const bool scaled = c->elem == XP_ELEM_I8 || c->elem == XP_ELEM_E4M3;
    if (!scaled && c->elem != XP_ELEM_F16 && c->elem != XP_ELEM_BF16)
        return set_error(XP_E_ARG, "%s: a cache is F16, BF16, I8 or E4M3, not elem %d", fn, c->elem);
    if (scaled != (c->k_scale != nullptr) || scaled != (c->v_scale != nullptr))
        return set_error(XP_E_ARG, "%s: a cache of 8 bits has scales and one of 16 bits has none", fn);
    if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)))
        return set_error(XP_E_ARG, "%s: page_size %u is not a power of two from 16 to 1024", fn, c->page_size);
    if (c->head_dim == 0 || c->head_dim % 16 || c->head_dim > 256)
        return set_error(XP_E_ARG, "%s: head_dim %u is not a multiple of 16 up to 256", fn, c->head_dim);
    if (c->kv_heads == 0 || c->kv_heads > 65535u) return set_error(XP_E_ARG, "%s: %u kv heads (1 to 65535)", fn, c->kv_heads);
    if (c->n_pages > 0x7FFFFFFFu) return set_error(XP_E_ARG, "%s: %u pages are over 2^31 - 1", fn, c->n_pages);
    for (const void* p : {static_cast<const void*>(c->k), static_cast<const void*>(c->v), static_cast<const void*>(c->k_scale),
                          static_cast<const void*>(c->v_scale)})
        if (reinterpret_cast<uintptr_t>(p) % 16) return set_error(XP_E_ARG, "%s: the cache's planes have to be 16-byte aligned", fn);
    return XP_OK;
}

int check_seqs(const char* fn, const xp_paged_seqs* s) {
    if (!s) return set_error(XP_E_ARG, "%s: the sequences are null", fn);
    if (s->n_seq && s->n_tokens && (!s->cu || !s->kv_len || !s->pages))
        return set_error(XP_E_ARG, "%s: cu, kv_len or pages is null", fn);
    if (s->n_seq > (1u << 24)) return set_error(XP_E_ARG, "%s: %u sequences are over 2^24", fn, s->n_seq);
    if (s->n_tokens > 0x7FFFFFFFu) return set_error(XP_E_ARG, "%s: %u tokens are over 2^31 - 1", fn, s->n_tokens);
    if (s->table > (1u << 26)) return set_error(XP_E_ARG, "%s: a table of %u pages is over 2^26", fn, s->table);
    return XP_OK;
}

int check_here(const char* fn, xp_stream stream, const void* out) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return set_error(XP_E_HIP, "%s: hipGetDevice failed", fn);
    if (stream) {
        hipDevice_t d = dev;
        if (hipStreamGetDevice(as_stream(stream), &d) != hipSuccess)
            return set_error(XP_E_HIP, "%s: hipStreamGetDevice failed", fn);
        if (d != dev) return set_error(XP_E_ARG, "%s: the stream is device %d's, the current one is %d", fn, d, dev);
    }
    hipPointerAttribute_t a;
    if (hipPointerGetAttributes(&a, out) != hipSuccess || a.type == hipMemoryTypeUnregistered) {
        (void)hipGetLastError();
        return set_error(XP_E_ARG, "%s: the output is not device memory", fn);
    }
    if (a.type == hipMemoryTypeDevice && a.device != dev)
        return set_error(XP_E_ARG, "%s: the output is device %d's, the current one is %d", fn, a.device, dev);
    return XP_OK;
}

PageMap page_map(const xp_paged_kv* c, const xp_paged_seqs* s) {
    return {s->pages, s->table, c->n_pages, uint32_t(__builtin_ctz(c->page_size))};
}

}  // namespace xp
