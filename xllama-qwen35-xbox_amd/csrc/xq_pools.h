// xq_pools.h — the pools that a page table addresses, as the kernels that move rows and pages see
// them, and the host's check of the caller's description.
#pragma once

#include "xq_paged.h"

namespace xq {

constexpr int kPoolsPerLaunch = 40;  // 40 bytes each: kernel arguments stay below 2 KiB

typedef uint32_t u32x4p __attribute__((ext_vector_type(4), aligned(1)));
typedef uint16_t u16p __attribute__((aligned(1)));

struct Pool {
    uint8_t* base;
    int64_t page, row, head;  // strides, bytes
    uint32_t line;            // contiguous bytes: a record, or a row's n_head_kv records (heads 1)
    uint32_t heads;           // lines per row
};

struct PoolSet {
    Pool p[kPoolsPerLaunch];
};

// 16 bytes of the run at byte off (the last piece of a run is moved up to end with it).
XQ_DEV uint32_t piece_at(uint32_t i, uint32_t run) { return min(i * 16u, run - 16u); }

inline xq_status pools_check(const xq_tensor* pools, int32_t n_pools, int32_t* page_rows, int32_t* n_pages) {
    if (!pools) return failf(XQ_ERR_BAD_ARG, "null pools");
    if (n_pools < 1 || n_pools > 1024) return failf(XQ_ERR_BAD_ARG, "n_pools must be in [1, 1024]");
    for (int32_t i = 0; i < n_pools; ++i) {
        const xq_tensor& t = pools[i];
        const size_t ts = type_size(t.type);
        if (!ts) return failf(XQ_ERR_UNSUPPORTED, "pool %d: type %d", i, t.type);
        for (int j = 0; j < 4; ++j)
            if (t.ne[j] < 1 || t.ne[j] > 0x7fffffff) return failf(XQ_ERR_BAD_SHAPE, "pool %d: bad ne", i);
        if (t.ne[0] % 32 || t.ne[0] > 65536) return failf(XQ_ERR_UNSUPPORTED, "pool %d: head dim must be a multiple of 32", i);
        if (t.nb[0] != ts) return failf(XQ_ERR_UNSUPPORTED, "pool %d: records must be contiguous", i);
        if (t.ne[1] != pools[0].ne[1] || t.ne[3] != pools[0].ne[3])
            return failf(XQ_ERR_BAD_SHAPE, "pool %d: page_rows and n_pages must be those of pool 0", i);
        if ((int64_t)record_bytes(t.type, t.ne[0]) * t.ne[2] > ((int64_t)1 << 24)) return failf(XQ_ERR_UNSUPPORTED, "pool %d: row above 2^24 bytes", i);
        if ((int64_t)record_bytes(t.type, t.ne[0]) * t.ne[2] * t.ne[1] >= ((int64_t)1 << 31))
            return failf(XQ_ERR_UNSUPPORTED, "pool %d: page of 2^31 bytes or more", i);
        if (!t.data) return failf(XQ_ERR_BAD_ARG, "pool %d: null data pointer", i);
    }
    *page_rows = (int32_t)pools[0].ne[1];
    *n_pages = (int32_t)pools[0].ne[3];
    return XQ_OK;
}

inline Pool pool_of(const xq_tensor& t) {
    Pool p{};
    const size_t rec = record_bytes(t.type, t.ne[0]);
    p.base = (uint8_t*)t.data;
    p.row = (int64_t)t.nb[1], p.head = (int64_t)t.nb[2], p.page = (int64_t)t.nb[3];
    const bool one = t.ne[2] == 1 || t.nb[2] == rec;  // a row's records lie one after another
    p.line = (uint32_t)(one ? rec * t.ne[2] : rec);
    p.heads = one ? 1u : (uint32_t)t.ne[2];
    return p;
}

inline xq_status table_check(int32_t n_seq, int32_t table_cols) {
    if (n_seq < 1 || table_cols < 1) return failf(XQ_ERR_BAD_ARG, "bad table sizes");
    return XQ_OK;
}

// (a pool's rows given twice would be moved twice, by waves that do not wait for each other)
inline xq_status pools_differ(const xq_tensor* pools, int32_t n_pools) {
    for (int32_t i = 0; i < n_pools; ++i)
        for (int32_t j = 0; j < i; ++j)
            if (pools[i].data == pools[j].data) return failf(XQ_ERR_BAD_ARG, "pools %d and %d are one", j, i);
    return XQ_OK;
}

}  // namespace xq
