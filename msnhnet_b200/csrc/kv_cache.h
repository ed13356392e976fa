// The paged cache as the kernels take it, and the checks its entry points share.
#pragma once
#include "token_ops.h"

namespace msnh {

struct KvParams {
    uint8_t *k, *v;
    long long k_page, k_token, k_head, v_page, v_token, v_head;     // strides in elements
    long long table_stride;
    int *table, *lengths, *refs, *refused;
    int n_pages, page_size, heads, dim, n_seqs, max_pages;
    float *k_scales, *v_scales;                                     // of 8-bit codes: [page][head][blocks]
    int block, blocks;                                              // tokens of a scale (0: no codes), scales of a page and head
};

inline KvParams kv_params(const MsnhB200KvCache &c) {
    return {static_cast<uint8_t *>(c.k_pages), static_cast<uint8_t *>(c.v_pages), c.k_page_stride, c.k_token_stride, c.k_head_stride, c.v_page_stride,
            c.v_token_stride, c.v_head_stride, c.table_stride, c.page_table, c.lengths, c.refs, c.refused, c.n_pages, c.page_size, c.n_kv_heads, c.head_dim,
            c.n_seqs, c.max_pages, c.dtype == MSNH_B200_E4M3 ? c.k_scales : nullptr, c.dtype == MSNH_B200_E4M3 ? c.v_scales : nullptr,
            c.dtype == MSNH_B200_E4M3 ? c.scale_block : 0, c.dtype == MSNH_B200_E4M3 ? c.page_size / c.scale_block : 0};
}

// Whether every row of head_dim values starts on a multiple of `bytes` and is a multiple of it long.
inline bool kv_rows_multiple_of(const MsnhB200KvCache &c, size_t bytes) {
    const size_t size = dtype_size(c.dtype);
    for (const int64_t stride : {c.k_page_stride, c.k_token_stride, c.k_head_stride, c.v_page_stride, c.v_token_stride, c.v_head_stride})
        if (stride * size % bytes) return false;
    return c.head_dim * size % bytes == 0 && reinterpret_cast<uintptr_t>(c.k_pages) % bytes == 0 && reinterpret_cast<uintptr_t>(c.v_pages) % bytes == 0;
}

// `upkeep`: the operation writes refs and counts refusals.
inline int check_cache(MsnhB200Ctx *ctx, const MsnhB200KvCache *c, bool upkeep, const char *what) {
    if (!is_float_type(c->dtype) && c->dtype != MSNH_B200_E4M3) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "%s: a cache of type %d", what, c->dtype);
    if (c->n_pages < 1 || c->page_size < 1 || c->n_kv_heads < 1 || c->head_dim < 1 || c->n_seqs < 1 || c->max_pages < 1)
        return fail(ctx, MSNH_B200_ERR_ARG, "%s: the cache's sizes must be positive", what);
    if (static_cast<int64_t>(c->max_pages) * c->page_size > 0x7fffffff || static_cast<int64_t>(c->page_size) * c->n_kv_heads * c->head_dim >= 1 << 30)
        return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "%s: 2^31 tokens of a sequence or 2^30 values of a page, and more", what);
    if (c->n_pages > 1 << 30) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "%s: %d pages (at most 2^30 are taken)", what, c->n_pages);
    if (!c->k_pages || !c->v_pages || !c->page_table || !c->lengths) return fail(ctx, MSNH_B200_ERR_ARG, "%s: null pages, table or lengths", what);
    if (c->dtype == MSNH_B200_E4M3) {
        if (!c->k_scales || !c->v_scales) return fail(ctx, MSNH_B200_ERR_ARG, "%s: null scales", what);
        if (c->scale_block < 1 || c->page_size % c->scale_block) return fail(ctx, MSNH_B200_ERR_ARG, "%s: scales of %d tokens in pages of %d", what, c->scale_block, c->page_size);
    }
    if (upkeep && (!c->refs || !c->refused)) return fail(ctx, MSNH_B200_ERR_ARG, "%s: null refs or refused", what);
    if (c->table_stride < c->max_pages) return fail(ctx, MSNH_B200_ERR_ARG, "%s: rows of the page table overlap", what);
    for (const int64_t stride : {c->k_page_stride, c->k_token_stride, c->k_head_stride, c->v_page_stride, c->v_token_stride, c->v_head_stride})
        if (stride < 0) return fail(ctx, MSNH_B200_ERR_ARG, "%s: a stride is negative", what);
    return MSNH_B200_OK;
}

}  // namespace msnh
