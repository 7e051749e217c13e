// xq_paged.h — the paged KV cache as the kernels see it, and the host's check of the
// caller's description of it.
#pragma once

#include "xq_fa_common.h"
#include "xq_host.h"

namespace xq {

struct PagesView {
    uint8_t* k;
    uint8_t* v;
    int64_t k_row, k_head, k_page, v_row, v_head, v_page;  // strides, bytes
    const int32_t* table;
    const int32_t* rows;
    int32_t table_cols, page_rows, n_pages, n_head_kv;
    int32_t row_limit;  // rows a table can address (below 2^31 - 2^8)
    UDivFlat d_page;    // by page_rows

    // Page of row r < row_limit of sequence b; not below n_pages where it is none.
    XQ_DEV uint32_t page(int64_t b, uint32_t r) const {
        return (uint32_t)table[b * table_cols + d_page.quot(r)];
    }
};

inline bool elem_aligned(const xq_tensor* t, size_t a, int from) {
    for (int i = from; i < 4; ++i)
        if (t->nb[i] % a) return false;
    return true;
}

// `kinds`: bit set over the storage types {F32, F16, BF16, E5M2, Q8_0, Q4_0} in that order.
enum : uint32_t { kF32 = 1, kF16 = 2, kBF16 = 4, kE5M2 = 8, kQ8 = 16, kQ4 = 32 };
inline uint32_t type_bit(int t) {
    switch (t) {
    case XQ_TYPE_F32: return kF32;
    case XQ_TYPE_F16: return kF16;
    case XQ_TYPE_BF16: return kBF16;
    case XQ_TYPE_E5M2: return kE5M2;
    case XQ_TYPE_Q8_0: return kQ8;
    case XQ_TYPE_Q4_0: return kQ4;
    default: return 0;
    }
}

inline xq_status pages_check(const xq_kv_pages* c, int64_t D, int64_t n_head_kv, int64_t n_seq, uint32_t kinds, PagesView* out) {
    if (!c) return failf(XQ_ERR_BAD_ARG, "null cache");
    const xq_tensor &k = c->k, &v = c->v;
    if (!(type_bit(k.type) & kinds) || k.type != v.type)
        return failf(XQ_ERR_UNSUPPORTED, "cache type %d/%d not supported", k.type, v.type);
    if (k.ne[0] != D || v.ne[0] != D) return failf(XQ_ERR_BAD_SHAPE, "cache head dim differs");
    for (int i = 1; i < 4; ++i)
        if (k.ne[i] < 1 || k.ne[i] != v.ne[i] || k.ne[i] > 0x7fffffff) return failf(XQ_ERR_BAD_SHAPE, "cache pools' shapes");
    if (n_head_kv > 0 && k.ne[2] != n_head_kv) return failf(XQ_ERR_BAD_SHAPE, "cache KV heads differ");
    if (k.nb[0] != type_size(k.type) || v.nb[0] != type_size(k.type))
        return failf(XQ_ERR_UNSUPPORTED, "cache records must be contiguous");
    const size_t a = k.type == XQ_TYPE_E5M2 ? 1 : k.type == XQ_TYPE_F32 ? 4 : 2;
    if (!elem_aligned(&k, a, 1) || !elem_aligned(&v, a, 1) || !aligned(k.data, a) || !aligned(v.data, a))
        return failf(XQ_ERR_UNSUPPORTED, "cache strides and pointers must be multiples of %zu bytes", a);
    if (c->n_seq != n_seq) return failf(XQ_ERR_BAD_SHAPE, "cache holds %d sequences, the call %lld", c->n_seq, (long long)n_seq);
    if (c->table_cols < 1) return failf(XQ_ERR_BAD_ARG, "table_cols must be at least 1");
    if (out) {
        out->k = (uint8_t*)k.data;
        out->v = (uint8_t*)v.data;
        out->k_row = (int64_t)k.nb[1], out->k_head = (int64_t)k.nb[2], out->k_page = (int64_t)k.nb[3];
        out->v_row = (int64_t)v.nb[1], out->v_head = (int64_t)v.nb[2], out->v_page = (int64_t)v.nb[3];
        out->table = c->table;
        out->rows = c->rows;
        out->table_cols = c->table_cols;
        out->page_rows = (int32_t)k.ne[1];
        out->n_pages = (int32_t)k.ne[3];
        out->n_head_kv = (int32_t)k.ne[2];
        const int64_t lim = (int64_t)c->table_cols * k.ne[1];
        out->row_limit = (int32_t)(lim < 0x7fffff00 ? lim : 0x7fffff00);
        out->d_page = UDivFlat((uint32_t)k.ne[1]);
    }
    return XQ_OK;
}

inline bool pages_null(const xq_kv_pages* c) { return !c->k.data || !c->v.data || !c->table || !c->rows; }

}  // namespace xq
