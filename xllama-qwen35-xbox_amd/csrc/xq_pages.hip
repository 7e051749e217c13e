// xq_pages.hip — pages of a KV cache: copied, compacted, handed out, forked, released.
//
// Nothing is computed here: bytes move from HBM to HBM (bound by a copy's rate, and for few
// pages by the launch and a chain of dependent loads: table, then row), and small integer
// tables change. Pool records may lie anywhere (free row, head and page strides), so a
// page is `runs` of contiguous bytes: one where the page is one block, one per row or head,
// or one per record.
#include "xq_pools.h"

namespace xq {

constexpr int kMaxForks = 1024;

// ---------------------------------------------------------------- copy

// A workgroup copies kPieces x 256 pieces of one (pair, pool): every load is issued before
// the first store. live == nullptr: whole pages; else the first live[i] rows. Bound by HBM:
// 512 pages of 32 rows in 16 pools (2 x 537 MB) 207 us, 5.2 TB/s, where a 2 GiB copy reaches 4.9.
constexpr int kPieces = 4;

__global__ __launch_bounds__(256) void pages_copy_kernel(PoolSet set, const int32_t* __restrict__ src, const int32_t* __restrict__ dst,
                                                         const int32_t* __restrict__ live, uint32_t n, uint32_t page_rows,
                                                         uint32_t n_pages, uint32_t chunks) {
    const uint32_t pool = blockIdx.y, pair = blockIdx.x / chunks, chunk = blockIdx.x - pair * chunks;
    const uint32_t from = (uint32_t)src[pair], to = (uint32_t)dst[pair];
    if (from >= n_pages || to >= n_pages || from == to) return;
    const uint32_t rows = live ? (uint32_t)live[pair] : page_rows;
    const Pool p = set.p[pool];
    // runs of the rows: (outer, inner), the contiguous bytes of each
    uint32_t run = p.line, inner = rows, outer = p.heads;
    int64_t s_in = p.row, s_out = p.head;
    if (p.row == (int64_t)p.line) {  // rows of a head (or of the page) lie one after another
        run = p.line * rows;
        inner = 1;
    }
    if (rows == 0) return;
    const uint32_t pieces = (run + 15u) / 16u, total = pieces * inner * outer;
    const uint8_t* a = p.base + (int64_t)from * p.page;
    uint8_t* b = p.base + (int64_t)to * p.page;
    u32x4p v[kPieces];
    int64_t at[kPieces];
    const uint32_t i0 = chunk * (256u * kPieces) + threadIdx.x;
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
        const uint32_t i = i0 + 256u * k;
        if (i < total) {
            const uint32_t r = i / pieces;
            const uint32_t o = r / inner;
            at[k] = (int64_t)o * s_out + (int64_t)(r - o * inner) * s_in + piece_at(i - r * pieces, run);
            v[k] = *(const u32x4p*)(a + at[k]);
        }
    }
#pragma unroll
    for (int k = 0; k < kPieces; ++k)
        if (i0 + 256u * k < total) *(u32x4p*)(b + at[k]) = v[k];
}

// ---------------------------------------------------------------- compact

// One wave per (sequence, pool, 64 pieces of a row): lane l moves its 16 bytes of every
// row of the path, eight rows loaded before the first is stored. Row j is written after
// every row of index <= j has been read by the same lane, and a later entry's source lies
// past it (path[i] >= i > j), so no other lane's order matters; pieces do not overlap.
// Bound by the launch and its chain of reads (rows and path, table, records): five rows of 8
// sequences in 16 pools (2 x 1 MB) 4 us.
__global__ __launch_bounds__(64) void pages_compact_kernel(PoolSet set, const int32_t* __restrict__ table, const int32_t* __restrict__ rows,
                                                           int32_t table_cols, int32_t row_limit, UDivFlat d_page, uint32_t n_pages,
                                                           const int32_t* __restrict__ path, const int32_t* __restrict__ n_path,
                                                           int32_t path_cols, int32_t* __restrict__ rows_out) {
    const uint32_t b = blockIdx.y, pool = blockIdx.z, lane = threadIdx.x;
    const int32_t base = rows[b], n = max(0, min(n_path[b], path_cols));
    if (rows_out && pool == 0 && blockIdx.x == 0 && lane == 0) rows_out[b] = (int32_t)((uint32_t)base + (uint32_t)n);
    const Pool p = set.p[pool];
    const uint32_t per_line = (p.line + 15u) / 16u, unit = blockIdx.x * 64u + lane;
    const uint32_t h = unit / per_line, off = (unit - h * per_line) * 16u;
    const bool on = h < p.heads;
    const uint32_t len = on ? min(16u, p.line - off) : 0u;
    uint8_t* q = p.base + (int64_t)h * p.head + off;
    auto row_at = [&](int64_t r, bool& ok) -> int64_t {  // byte offset of a row in its pool
        ok = ok && r >= 0 && r < row_limit;
        const uint32_t u = ok ? (uint32_t)r : 0u;
        const uint32_t c = d_page.quot(u), page = (uint32_t)table[(int64_t)b * table_cols + c];
        ok = ok && page < n_pages;
        return ok ? (int64_t)page * p.page + (int64_t)(u - c * d_page.d) * p.row : 0;
    };
    for (int j0 = 0; j0 < n; j0 += 64) {
        // lane l looks up entry j0 + l
        const int j = j0 + (int)lane;
        const int32_t e = j < n ? path[(int64_t)b * path_cols + j] : -1;
        bool ok = j < n && e > j;
        const int64_t s = row_at((int64_t)base + e, ok), d = row_at((int64_t)base + j, ok);
        uint64_t todo = __builtin_amdgcn_ballot_w64(ok);
        while (todo) {
            u32x4p v[8];
            int64_t to[8];
            int m = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (todo) {
                    const int l = __builtin_ctzll(todo);
                    todo &= todo - 1;
                    const int64_t from = ((int64_t)__builtin_amdgcn_readlane((int)(s >> 32), l) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)s, l);
                    to[k] = ((int64_t)__builtin_amdgcn_readlane((int)(d >> 32), l) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)d, l);
                    if (len == 16u) {
                        v[k] = *(const u32x4p*)(q + from);
                    } else {  // the end of a line: whole 16-bit words
                        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
                        for (uint32_t x = 0; x < 8; ++x)
                            if (2 * x < len) w[x / 2] |= (uint32_t)*(const u16p*)(q + from + 2 * x) << (16 * (x & 1));
                        v[k] = u32x4p{w[0], w[1], w[2], w[3]};
                    }
                    ++m;
                }
            }
            // every row of the batch is in before the first is stored
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (k < m) {
                    if (len == 16u) {
                        *(u32x4p*)(q + to[k]) = v[k];
                    } else {
#pragma unroll
                        for (uint32_t x = 0; x < 8; ++x)
                            if (2 * x < len) *(u16p*)(q + to[k] + 2 * x) = (uint16_t)(v[k][x / 2] >> (16 * (x & 1)));
                    }
                }
            }
        }
    }
}

// ---------------------------------------------------------------- free pages

constexpr int kScanThreads = 1024;

// Exclusive prefix sum over the workgroup's 1024 threads; *total the sum.
XQ_DEV uint32_t block_scan(uint32_t x, uint32_t* lds, uint32_t* total) {
    const int lane = lane_id(), w = wave_id();
    uint32_t s = x;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t y = __shfl_up(s, d);
        if (lane >= d) s += y;
    }
    if (lane == 63) lds[w] = s;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kScanThreads / 64; ++i) {
        const uint32_t y = lds[i];
        before += i < w ? y : 0u;
        all += y;
    }
    __syncthreads();
    *total = all;
    return before + s - x;
}

// The first `want` free pages (refs 0), lowest first, into list; *found how many there are
// of them. Thread t looks through the t-th span of pages.
XQ_DEV void free_pages(const int32_t* refs, uint32_t n_pages, uint32_t want, int32_t* list, uint32_t* lds, uint32_t* found) {
    const uint32_t span = (n_pages + kScanThreads - 1) / kScanThreads;
    const uint32_t p0 = min(threadIdx.x * span, n_pages), p1 = min(p0 + span, n_pages);
    uint32_t mine = 0;
    for (uint32_t p = p0; p < p1; ++p) mine += refs[p] == 0;
    uint32_t at = block_scan(mine, lds, found);
    for (uint32_t p = p0; p < p1 && at < want && mine; ++p)
        if (refs[p] == 0) list[at++] = (int32_t)p;
    *found = min(*found, want);
    __syncthreads();
}

// ---------------------------------------------------------------- reserve

// One workgroup. Wave w counts the missing pages of sequences w, w + 16, ...; a scan over the
// sequences gives each its place in the list of free pages; then the waves fill the tables.
// One workgroup, since who gets which page depends on all before. It reads every page's references on
// every call, each thread a span of its own, whether a page is wanted or not, and that bounds it: 64
// sequences, 1024 pages 8 us, 8192 13, 65536 62, 262144 215 (64 pages wanted: 9, 18, 73, 227).
// list: [n_pages] free pages, then counts: [n_seq].
__global__ __launch_bounds__(kScanThreads) void pages_reserve_kernel(int32_t* table, int32_t* refs, uint32_t n_seq, uint32_t cols,
                                                                     uint32_t n_pages, uint32_t page_rows, const int32_t* __restrict__ want,
                                                                     int32_t* __restrict__ got, int32_t* list, uint32_t* counts) {
    __shared__ uint32_t lds[kScanThreads / 64];
    const int lane = lane_id(), w = wave_id();
    constexpr uint32_t W = kScanThreads / 64;
    auto need = [&](uint32_t b) -> uint32_t {
        const int32_t x = want[b];
        return x <= 0 ? 0u : min(((uint32_t)x - 1u) / page_rows + 1u, cols);
    };
    for (uint32_t b = w; b < n_seq; b += W) {
        const uint32_t c1 = need(b);
        uint32_t missing = 0;
        for (uint32_t c = 0; c < c1; c += 64) {
            const bool m = c + lane < c1 && table[(int64_t)b * cols + c + lane] == -1;
            missing += __builtin_popcountll(__builtin_amdgcn_ballot_w64(m));
        }
        if (lane == 0) counts[b] = missing;
    }
    __syncthreads();
    // counts[b] becomes the number of pages that sequences before b miss
    uint32_t wanted = 0;
    for (uint32_t b0 = 0; b0 < n_seq; b0 += kScanThreads) {
        const uint32_t b = b0 + threadIdx.x;
        uint32_t sum;
        const uint32_t before = block_scan(b < n_seq ? counts[b] : 0u, lds, &sum);
        if (b < n_seq) counts[b] = wanted + before;
        wanted += sum;
    }
    uint32_t found;
    free_pages(refs, n_pages, min(wanted, n_pages), list, lds, &found);
    for (uint32_t b = w; b < n_seq; b += W) {
        const uint32_t c1 = need(b);
        uint32_t at = counts[b];
        for (uint32_t c = 0; c < c1; c += 64) {
            const bool m = c + lane < c1 && table[(int64_t)b * cols + c + lane] == -1;
            const uint64_t all = __builtin_amdgcn_ballot_w64(m);
            const uint32_t k = at + __builtin_popcountll(all & (((uint64_t)1 << lane) - 1));
            if (m && k < found) {
                const int32_t p = list[k];
                table[(int64_t)b * cols + c + lane] = p;
                refs[p] = 1;
            }
            at += __builtin_popcountll(all);
        }
        // the unbroken first pages (this wave wrote its row of the table itself)
        uint32_t held = 0;
        for (uint32_t c = 0; c < cols; c += 64) {
            const bool m = c + lane < cols && (uint32_t)__hip_atomic_load(&table[(int64_t)b * cols + c + lane], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) < n_pages;
            const uint64_t all = ~__builtin_amdgcn_ballot_w64(m);
            held += all ? __builtin_ctzll(all) : 64;
            if (all) break;
        }
        if (lane == 0) got[b] = (int32_t)min((uint64_t)held * page_rows, (uint64_t)0x7fffffff);
    }
}

// ---------------------------------------------------------------- fork

// One workgroup; thread i is fork i. plan: [3][n] = source page, page taken, rows to copy.
// Bound by its chain of reads (ids, rows and table, references, shared pages): 16 forks 7 us;
// the last pages' rows then follow in a copy (32 pools of q8_0, 15 MB: 8 us).
__global__ __launch_bounds__(kScanThreads) void pages_fork_kernel(int32_t* table, int32_t* rows, int32_t* refs, uint32_t n_seq, uint32_t cols,
                                                                  uint32_t n_pages, uint32_t page_rows, int32_t row_limit,
                                                                  const int32_t* __restrict__ parents, const int32_t* __restrict__ children,
                                                                  uint32_t n, int32_t* __restrict__ done, int32_t* __restrict__ plan) {
    __shared__ uint32_t lds[kScanThreads / 64];
    __shared__ int32_t kids[kMaxForks], folk[kMaxForks], list[kMaxForks], full_of[kMaxForks];
    const uint32_t i = threadIdx.x;
    const bool on = i < n;
    const int32_t p = on ? parents[i] : -1, c = on ? children[i] : -1;
    if (on) {
        kids[i] = c;
        folk[i] = p;
    }
    __syncthreads();
    bool ok = on && (uint32_t)p < n_seq && (uint32_t)c < n_seq;
    // a child named before, or that is any fork's parent
    for (uint32_t j = 0; j < n; ++j) ok = ok && !(j < i && kids[j] == c) && folk[j] != c;
    int32_t held = 0;
    if (ok) {
        held = rows[p];
        ok = rows[c] == 0 && table[(int64_t)c * cols] == -1 && held >= 0 && held <= row_limit;
    }
    const uint32_t full = ok ? (uint32_t)held / page_rows : 0u, part = ok ? (uint32_t)held - full * page_rows : 0u;
    const int32_t last = ok && part ? table[(int64_t)p * cols + full] : -1;
    if (part && (uint32_t)last >= n_pages) ok = false;
    const uint32_t takes = ok && part ? 1u : 0u;
    uint32_t total, found;
    const uint32_t rank = block_scan(takes, lds, &total);
    free_pages(refs, n_pages, total, list, lds, &found);
    if (takes && rank >= found) ok = false;
    const int32_t page = takes && ok ? list[rank] : -1;
    if (on) {
        done[i] = ok ? 1 : 0;
        plan[i] = page >= 0 ? last : -1;
        plan[n + i] = page;
        plan[2 * n + i] = (int32_t)part;
        full_of[i] = ok ? (int32_t)full : -1;
        if (page >= 0) {
            refs[page] = 1;
            table[(int64_t)c * cols + full] = page;
        }
        if (ok) rows[c] = held;
    }
    __syncthreads();
    // shared full pages: one wave per fork
    const int lane = lane_id();
    for (uint32_t f = wave_id(); f < n; f += kScanThreads / 64) {
        const int32_t k = full_of[f];
        for (int32_t x = lane; x < k; x += 64) {
            const int32_t q = table[(int64_t)folk[f] * cols + x];
            table[(int64_t)kids[f] * cols + x] = q;
            if ((uint32_t)q < n_pages) atomicAdd(&refs[q], 1);
        }
    }
}

// ---------------------------------------------------------------- release

// One thread per (named sequence, column). The exchange hands each entry to one thread,
// so a sequence named twice releases its pages once.
__global__ __launch_bounds__(256) void pages_release_kernel(int32_t* table, int32_t* rows, int32_t* refs, uint32_t n_seq, uint32_t cols,
                                                            uint32_t n_pages, const int32_t* __restrict__ seqs) {
    const uint32_t b = (uint32_t)seqs[blockIdx.y], c = blockIdx.x * 256u + threadIdx.x;
    if (b >= n_seq || c >= cols) return;
    const uint32_t p = (uint32_t)atomicExch(&table[(int64_t)b * cols + c], -1);
    if (p < n_pages) atomicSub(&refs[p], 1);
    if (c == 0) rows[b] = 0;
}

// ---------------------------------------------------------------- host

// pieces of a page: a bound over the run forms (a run's last piece counts whole)
static int64_t page_pieces(const xq_tensor& t) {
    const Pool p = pool_of(t);
    return p.row == (int64_t)p.line ? cdiv((int64_t)p.line * t.ne[1], 16) * p.heads : cdiv(p.line, 16) * p.heads * t.ne[1];
}

static xq_status copy_launch(const xq_tensor* pools, int32_t n_pools, const int32_t* src, const int32_t* dst, const int32_t* live,
                             int32_t n, int32_t page_rows, int32_t n_pages, hipStream_t stream) {
    for (int32_t i0 = 0; i0 < n_pools; i0 += kPoolsPerLaunch) {
        const int32_t m = n_pools - i0 < kPoolsPerLaunch ? n_pools - i0 : kPoolsPerLaunch;
        PoolSet set{};
        int64_t pieces = 1;
        for (int32_t i = 0; i < m; ++i) {
            set.p[i] = pool_of(pools[i0 + i]);
            const int64_t x = page_pieces(pools[i0 + i]);
            if (x > pieces) pieces = x;
        }
        const int64_t chunks = cdiv(pieces, 256 * kPieces);
        // a grid holds below 2^32 threads; the pairs go in as many launches as that takes
        const int64_t most = ((int64_t)1 << 23) / chunks < 1 ? 1 : ((int64_t)1 << 23) / chunks;
        for (int64_t j = 0; j < n; j += most) {
            const int64_t k = n - j < most ? n - j : most;
            launch("kv_pages_copy", pages_copy_kernel, dim3((uint32_t)(k * chunks), (uint32_t)m), dim3(256), stream, set, src + j, dst + j,
                   live ? live + j : nullptr, (uint32_t)k, (uint32_t)page_rows, (uint32_t)n_pages, (uint32_t)chunks);
        }
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return failf(XQ_ERR_HIP, "kv_pages_copy launch: %s", hipGetErrorString(e));
    return XQ_OK;
}

}  // namespace xq

using namespace xq;

extern "C" {

xq_status xq_kv_pages_copy(const xq_tensor* pools, int32_t n_pools, const int32_t* src, const int32_t* dst, int32_t n, void* stream) {
    int32_t page_rows, n_pages;
    xq_status st = pools_check(pools, n_pools, &page_rows, &n_pages);
    if (st != XQ_OK) return st;
    if (n < 0) return failf(XQ_ERR_BAD_ARG, "bad page count");
    if (n == 0) return done_ok();
    if (!src || !dst) return failf(XQ_ERR_BAD_ARG, "null pointer");
    if (!aligned(src, 4) || !aligned(dst, 4)) return failf(XQ_ERR_UNSUPPORTED, "misaligned pointer");
    st = copy_launch(pools, n_pools, src, dst, nullptr, n, page_rows, n_pages, (hipStream_t)stream);
    return st == XQ_OK ? done_ok() : st;
}

xq_status xq_kv_pages_compact(const xq_tensor* pools, int32_t n_pools, const int32_t* table, const int32_t* rows, int32_t n_seq,
                              int32_t table_cols, const int32_t* path, const int32_t* n_path, int32_t path_cols, int32_t* rows_out,
                              void* stream) {
    int32_t page_rows, n_pages;
    xq_status st = pools_check(pools, n_pools, &page_rows, &n_pages);
    if (st == XQ_OK) st = table_check(n_seq, table_cols);
    if (st != XQ_OK) return st;
    if (path_cols < 1) return failf(XQ_ERR_BAD_ARG, "path_cols must be at least 1");
    if (n_seq > 65535) return failf(XQ_ERR_UNSUPPORTED, "more than 65535 sequences");
    if (!table || !rows || !path || !n_path || !rows_out) return failf(XQ_ERR_BAD_ARG, "null pointer");
    if (rows_out == rows) return failf(XQ_ERR_BAD_ARG, "rows_out must not be rows");
    for (const void* x : {(const void*)table, (const void*)rows, (const void*)path, (const void*)n_path, (const void*)rows_out})
        if (!aligned(x, 4)) return failf(XQ_ERR_UNSUPPORTED, "misaligned pointer");
    st = pools_differ(pools, n_pools);
    if (st != XQ_OK) return st;
    const int64_t lim = (int64_t)table_cols * page_rows;
    for (int32_t i0 = 0; i0 < n_pools; i0 += kPoolsPerLaunch) {
        const int32_t m = n_pools - i0 < kPoolsPerLaunch ? n_pools - i0 : kPoolsPerLaunch;
        PoolSet set{};
        int64_t units = 1;
        for (int32_t i = 0; i < m; ++i) {
            set.p[i] = pool_of(pools[i0 + i]);
            const int64_t x = cdiv(set.p[i].line, 16) * set.p[i].heads;
            if (x > units) units = x;
        }
        launch("kv_pages_compact", pages_compact_kernel, dim3((uint32_t)cdiv(units, 64), (uint32_t)n_seq, (uint32_t)m), dim3(64),
               (hipStream_t)stream, set, table, rows, table_cols, (int32_t)(lim < 0x7fffff00 ? lim : 0x7fffff00), UDivFlat((uint32_t)page_rows),
               (uint32_t)n_pages, path, n_path, path_cols, i0 == 0 ? rows_out : nullptr);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return failf(XQ_ERR_HIP, "kv_pages_compact launch: %s", hipGetErrorString(e));
    return done_ok();
}

xq_status xq_kv_pages_reserve_workspace(int32_t n_seq, int32_t n_pages, size_t* bytes) {
    if (!bytes || n_seq < 1 || n_pages < 1) return failf(XQ_ERR_BAD_ARG, "bad reserve arguments");
    *bytes = 4 * ((size_t)n_seq + (size_t)n_pages);
    return done_ok();
}

xq_status xq_kv_pages_reserve(int32_t* table, int32_t* refs, int32_t n_seq, int32_t table_cols, int32_t n_pages, int32_t page_rows,
                              const int32_t* want, int32_t* got, void* workspace, size_t workspace_bytes, void* stream) {
    size_t need = 0;
    xq_status st = xq_kv_pages_reserve_workspace(n_seq, n_pages, &need);
    if (st == XQ_OK) st = table_check(n_seq, table_cols);
    if (st != XQ_OK) return st;
    if (page_rows < 1) return failf(XQ_ERR_BAD_ARG, "page_rows must be at least 1");
    // (the pages that all sequences miss are counted in 32 bits)
    if ((int64_t)n_seq * table_cols >> 32) return failf(XQ_ERR_UNSUPPORTED, "a table of 2^32 entries or more");
    if (!table || !refs || !want || !got) return failf(XQ_ERR_BAD_ARG, "null pointer");
    for (const void* x : {(const void*)table, (const void*)refs, (const void*)want, (const void*)got})
        if (!aligned(x, 4)) return failf(XQ_ERR_UNSUPPORTED, "misaligned pointer");
    if (!workspace || workspace_bytes < need) return failf(XQ_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    if (!aligned(workspace, 256)) return failf(XQ_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    int32_t* list = (int32_t*)workspace;
    launch("kv_pages_reserve", pages_reserve_kernel, dim3(1), dim3(kScanThreads), (hipStream_t)stream, table, refs, (uint32_t)n_seq,
           (uint32_t)table_cols, (uint32_t)n_pages, (uint32_t)page_rows, want, got, list, (uint32_t*)(list + n_pages));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return failf(XQ_ERR_HIP, "kv_pages_reserve launch: %s", hipGetErrorString(e));
    return done_ok();
}

xq_status xq_kv_pages_fork_workspace(int32_t n, size_t* bytes) {
    if (!bytes || n < 0 || n > kMaxForks) return failf(XQ_ERR_BAD_ARG, "n must be in [0, 1024]");
    *bytes = 12 * (size_t)(n > 0 ? n : 1);
    return done_ok();
}

xq_status xq_kv_pages_fork(const xq_tensor* pools, int32_t n_pools, int32_t* table, int32_t* rows, int32_t* refs, int32_t n_seq,
                           int32_t table_cols, const int32_t* parents, const int32_t* children, int32_t n, int32_t* done,
                           void* workspace, size_t workspace_bytes, void* stream) {
    int32_t page_rows, n_pages;
    size_t need = 0;
    xq_status st = pools_check(pools, n_pools, &page_rows, &n_pages);
    if (st == XQ_OK) st = xq_kv_pages_fork_workspace(n, &need);
    if (st == XQ_OK) st = table_check(n_seq, table_cols);
    if (st != XQ_OK) return st;
    if (n == 0) return done_ok();
    if (!table || !rows || !refs || !parents || !children || !done) return failf(XQ_ERR_BAD_ARG, "null pointer");
    for (const void* x : {(const void*)table, (const void*)rows, (const void*)refs, (const void*)parents, (const void*)children, (const void*)done})
        if (!aligned(x, 4)) return failf(XQ_ERR_UNSUPPORTED, "misaligned pointer");
    if (!workspace || workspace_bytes < need) return failf(XQ_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    if (!aligned(workspace, 256)) return failf(XQ_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    int32_t* plan = (int32_t*)workspace;
    const int64_t lim = (int64_t)table_cols * page_rows;
    launch("kv_pages_fork", pages_fork_kernel, dim3(1), dim3(kScanThreads), (hipStream_t)stream, table, rows, refs, (uint32_t)n_seq,
           (uint32_t)table_cols, (uint32_t)n_pages, (uint32_t)page_rows, (int32_t)(lim < 0x7fffff00 ? lim : 0x7fffff00), parents, children,
           (uint32_t)n, done, plan);
    st = copy_launch(pools, n_pools, plan, plan + n, plan + 2 * (int64_t)n, n, page_rows, n_pages, (hipStream_t)stream);
    return st == XQ_OK ? done_ok() : st;
}

xq_status xq_kv_pages_release(int32_t* table, int32_t* rows, int32_t* refs, int32_t n_seq, int32_t table_cols, int32_t n_pages,
                              const int32_t* seqs, int32_t n, void* stream) {
    const xq_status st = table_check(n_seq, table_cols);
    if (st != XQ_OK) return st;
    if (n < 0 || n_pages < 1) return failf(XQ_ERR_BAD_ARG, "bad release arguments");
    if (n > 65535) return failf(XQ_ERR_UNSUPPORTED, "more than 65535 sequences");
    if (n == 0) return done_ok();
    if (!table || !rows || !refs || !seqs) return failf(XQ_ERR_BAD_ARG, "null pointer");
    for (const void* x : {(const void*)table, (const void*)rows, (const void*)refs, (const void*)seqs})
        if (!aligned(x, 4)) return failf(XQ_ERR_UNSUPPORTED, "misaligned pointer");
    launch("kv_pages_release", pages_release_kernel, dim3((uint32_t)cdiv(table_cols, 256), (uint32_t)n), dim3(256), (hipStream_t)stream,
           table, rows, refs, (uint32_t)n_seq, (uint32_t)table_cols, (uint32_t)n_pages, seqs);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return failf(XQ_ERR_HIP, "kv_pages_release launch: %s", hipGetErrorString(e));
    return done_ok();
}

}  // extern "C"
