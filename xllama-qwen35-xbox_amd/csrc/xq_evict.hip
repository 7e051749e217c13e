// xq_evict.hip — rows of least accumulated weight leave the paged cache.
//
// Per sequence with n rows and a budget k below n: the rows are ordered by (protected first, larger
// weight, lower index) and the first k stay. Those of them that lie at index k or behind move, in
// order, to the places below k that others leave, in order: no row is both read and written, so all
// move at once, and no more bytes than have to. One workgroup per sequence selects (its rows' keys
// in LDS: a radix search for the k-th, then ranks by ballots), and writes a list
// of (page, row) pairs; a second launch moves them in every pool and gives pages without rows back.
//
// What bounds it: the moves by their bytes, read and written (4 x 12001 rows cut to 4096 in 16 f16 pools, 0.7 GB: 151 us,
// 4.7 TB/s); the selection by its chain of passes on one CU per sequence (33 us of 12001 rows, 15 us of 2049;
// each pass 2 to 4 us, LDS and barriers), which only grows with a sequence's rows, not with the batch.
#include "xq_pools.h"
#include "xq_tile.h"

namespace xq {

struct EvictArgs {
    int32_t* table;
    const int32_t* rows;
    int32_t* refs;  // null: no page is shared, none is given back
    const int32_t* keep;
    int32_t cols, n_pages, page_rows, row_limit;
    int64_t first_rows, last_rows;  // protected: by position
    const float* scores;
    const int32_t* positions;  // null: the rows' indexes
    int32_t score_cols;
    float* scores_out;      // null: not wanted
    int32_t* positions_out;
    int32_t* rows_out;
    int32_t* count;  // [sequence] moves
    int32_t* stay;   // [sequence] rows that stay, or -1 where nothing was done
    int32_t* lists;  // [sequence][2][half] places to fill, rows that fill them
    int4* moves;     // [sequence][half] page and row from, page and row to
    int32_t half;
    UDivFlat d_page;
};

// Larger weights have larger keys; NaN the least, -0 is 0.
XQ_DEV uint32_t weight_key(float x) {
    const uint32_t u = x == 0.0f ? 0u : __float_as_uint(x);
    return x != x ? 0u : (u >> 31) ? ~u : u | 0x80000000u;
}

constexpr int kEvictThreads = 1024, kEvictWaves = kEvictThreads / 64;

// Exclusive sums over the 16 waves of each wave's number; the whole in *total.
XQ_DEV uint32_t before_wave(uint32_t mine, uint32_t* lds, uint32_t* total) {
    __syncthreads();
    if (lane_id() == 0) lds[wave_id()] = mine;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kEvictWaves; ++i) {
        before += i < wave_id() ? lds[i] : 0u;
        all += lds[i];
    }
    *total = all;
    return before;
}

// The lowest c bits.
XQ_DEV uint64_t low_bits(int c) { return c <= 0 ? 0ull : c >= 64 ? ~0ull : ((uint64_t)1 << c) - 1; }
// x of lane l, the same for all
XQ_DEV uint64_t lane_get64(uint64_t x, int l) { return ((uint64_t)lane_get((uint32_t)(x >> 32), l) << 32) | lane_get((uint32_t)x, l); }

// The keys of up to kHeldRows rows stay in LDS, and so do the lists of their moves: a pass over them costs no
// memory round trip (about 1 us each, of a lone workgroup). Longer sequences read them again in each pass.
constexpr int kHeldRows = 24576;

template <bool HELD>
__global__ __launch_bounds__(kEvictThreads) void evict_select_kernel(EvictArgs a) {
    constexpr int BINS = 2048;
    __shared__ uint32_t hist[BINS], lds[kEvictWaves], found[2];
    __shared__ uint16_t list[2][HELD ? kHeldRows / 2 + 2 : 2];
    __shared__ uint32_t keys[HELD ? kHeldRows : 1];
    __shared__ uint64_t safes[HELD ? kHeldRows / 64 : 1];
    const int b = blockIdx.x, tid = threadIdx.x, lane = lane_id(), wave = wave_id();
    const int n = a.rows[b], k = max(a.keep[b], 0);
    const float* const score = a.scores + (int64_t)b * a.score_cols;
    const int32_t* const position = a.positions ? a.positions + (int64_t)b * a.score_cols : nullptr;
    float* const score_out = a.scores_out && a.scores_out != a.scores ? a.scores_out + (int64_t)b * a.score_cols : nullptr;
    int32_t* const position_out = a.positions_out && a.positions_out != a.positions ? a.positions_out + (int64_t)b * a.score_cols : nullptr;
    const bool held = n >= 0 && n <= a.score_cols && n <= a.row_limit;
    const bool cut = held && n > k;
    // rows [w0, w0 + span) are this wave's, 64 at a time
    const int span = held ? ((n + kEvictWaves - 1) / kEvictWaves + 63) / 64 * 64 : 0, w0 = wave * span;
    int newest = position ? -0x7fffffff - 1 : n - 1;
    auto is_safe = [&](int p) { return p < a.first_rows || (int64_t)newest - p < a.last_rows; };
    // ---- keys, the newest position, and the weights and positions that stay where they are
    constexpr int U = 4;  // loads of a thread at once
    for (int r0 = w0; r0 < w0 + span; r0 += 64 * U) {
        float x[U];
        int32_t p[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = min(r0 + 64 * u + lane, n - 1);
            x[u] = score[r];
            p[u] = position ? position[r] : r;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + 64 * u + lane;
            newest = max(newest, p[u]);
            if (r >= min(n, w0 + span)) continue;
            if constexpr (HELD) keys[r] = weight_key(x[u]);
            if (cut && r >= k) continue;
            if (score_out) score_out[r] = x[u];
            if (position_out) position_out[r] = p[u];
        }
    }
    if (position) {
#pragma unroll
        for (int s = 1; s < 64; s *= 2) newest = max(newest, __shfl_xor(newest, s));
        if (lane == 0) lds[wave] = (uint32_t)newest;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kEvictWaves; ++i) newest = max(newest, (int)lds[i]);
    }
    uint32_t my_safe = 0;
    if (cut)
        for (int r0 = w0; r0 < w0 + span; r0 += 64 * U) {
            int32_t p[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = min(r0 + 64 * u + lane, n - 1);
                p[u] = position ? position[r] : r;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = r0 + 64 * u + lane;
                const uint64_t s = __builtin_amdgcn_ballot_w64(r < min(n, w0 + span) && is_safe(p[u]));
                if (HELD && lane == 0 && r0 + 64 * u < w0 + span) safes[(r0 + 64 * u) / 64] = s;
                my_safe += __builtin_popcountll(s);
            }
        }
    // f(row, whether it is one, its key, whether it is protected) of this wave's rows; all 64 lanes take part
    auto each = [&](auto f) {
        for (int r0 = w0; r0 < w0 + span; r0 += 64) {
            const int r = min(r0 + lane, n - 1);
            const bool on = r0 + lane < n;
            if constexpr (HELD) f(r0 + lane, on, keys[r], (bool)(safes[r0 / 64] >> lane & 1));
            else f(r0 + lane, on, weight_key(score[r]), on && is_safe(position ? position[r] : r));
        }
    };
    uint32_t moves = 0;
    bool done = cut;
    int32_t* const far_list = a.lists + (int64_t)b * 2 * a.half;  // (!HELD)
    auto hole_at = [&](uint32_t i) -> int { return HELD ? list[0][i] : far_list[i]; };
    auto tail_at = [&](uint32_t i) -> int { return HELD ? list[1][i] : far_list[a.half + i]; };
    if (cut) {
        uint32_t mine = 0, n_safe;
        before_wave(my_safe, lds, &n_safe);
        // the group that is cut: protected rows where those alone exceed the budget, else the others,
        // of which `want` stay: all keys above `key`, and the first `ties` that equal it
        const bool among_safe = n_safe > (uint32_t)k;
        const uint32_t want = among_safe ? (uint32_t)k : (uint32_t)k - n_safe;
        uint32_t key = 0, left = want;
        if (want) {
            // the key's 11, 11 and 10 bits from above, by the counts of each value
#pragma unroll 1
            for (int step = 0; step < 3; ++step) {
                const int shift = step == 0 ? 21 : step == 1 ? 10 : 0, seen = step == 0 ? 31 : step == 1 ? 21 : 10;
                const uint32_t mask = step == 2 ? 1023u : 2047u;
                __syncthreads();
                hist[2 * tid] = hist[2 * tid + 1] = 0;
                __syncthreads();
                each([&](int, bool on, uint32_t x, bool s) {
                    const bool counts = on && s == among_safe && (step == 0 || (x ^ key) >> seen == 0);
                    const uint32_t bin = counts ? (x >> shift) & mask : ~0u;
                    // lanes of one lane's bin as one: many rows may have the same weight
                    const uint32_t one = (uint32_t)__builtin_amdgcn_readfirstlane((int)bin);
                    const uint64_t same = __builtin_amdgcn_ballot_w64(bin == one);
                    if (counts && bin != one) atomicAdd(&hist[bin], 1u);
                    if (lane == 0 && one != ~0u) atomicAdd(&hist[one], (uint32_t)__builtin_popcountll(same));
                });
                __syncthreads();
                // thread t: bins 2t and 2t + 1; how many lie in the bins above
                const uint32_t h0 = hist[2 * tid], h1 = hist[2 * tid + 1];
                uint32_t up = h0 + h1;
#pragma unroll
                for (int s = 1; s < 64; s *= 2) {
                    const uint32_t y = __shfl_down(up, s);
                    if (lane + s < 64) up += y;
                }
                if (lane == 0) lds[wave] = up;
                __syncthreads();
                uint32_t above = up - (h0 + h1);
#pragma unroll
                for (int i = 0; i < kEvictWaves; ++i) above += i > wave ? lds[i] : 0u;
                if (above < left && above + h1 >= left) {
                    found[0] = 2 * tid + 1;
                    found[1] = left - above;
                } else if (above + h1 < left && above + h1 + h0 >= left) {
                    found[0] = 2 * tid;
                    found[1] = left - above - h1;
                }
                __syncthreads();
                key |= found[0] << shift;
                left = found[1];
            }
        }
        const uint32_t ties = want ? left : 0u;
        uint32_t total;
        if constexpr (HELD) {
            // One more pass over the keys: lane g of a wave has its g-th 64 rows as masks, and what stays, the places
            // left and the rows that fill them are a few operations of masks. (Passes over the rows for each of these: 12001
            // rows 40 us; with the masks 33 us. Keys read four groups ahead changed nothing.)
            static_assert(kHeldRows / kEvictWaves <= 64 * 64);
            uint64_t eq = 0, gt = 0;
            for (int g = 0; g < span / 64; ++g) {
                const uint32_t x = keys[min(w0 + 64 * g + lane, n - 1)];
                const uint64_t e = __builtin_amdgcn_ballot_w64(x == key), t = __builtin_amdgcn_ballot_w64(x > key);
                if (lane == g) eq = e, gt = t;
            }
            const int g0 = w0 + 64 * lane;
            const uint64_t in = lane < span / 64 ? low_bits(n - g0) : 0, safe = in ? safes[g0 / 64] & in : 0;
            const uint64_t group = among_safe ? safe : in & ~safe;
            eq &= group, gt &= group;
            const uint32_t n_eq = (uint32_t)__builtin_popcountll(eq), eq_upto = wave_scan(n_eq);
            const uint32_t tie0 = before_wave(lane_get(eq_upto, 63), lds, &total) + eq_upto - n_eq;
            // of the ties the first ones
            uint32_t few = ties > tie0 ? ties - tie0 : 0u;
            if (few < n_eq) {
                uint64_t first = 0;
                for (; few; --few) {
                    first |= eq & (~eq + 1);
                    eq &= eq - 1;
                }
                eq = first;
            }
            const uint64_t stays = (want ? eq | gt : 0ull) | (among_safe ? 0ull : safe), front = low_bits(k - g0);
            const uint64_t hole = in & ~stays & front, tail = stays & ~front;
            const uint32_t holes = (uint32_t)__builtin_popcountll(hole), tails = (uint32_t)__builtin_popcountll(tail);
            const uint32_t h_upto = wave_scan(holes), t_upto = wave_scan(tails);
            const uint32_t h0 = before_wave(lane_get(h_upto, 63), lds, &moves) + h_upto - holes;
            const uint32_t t0 = before_wave(lane_get(t_upto, 63), lds, &total) + t_upto - tails;
            const uint64_t below = ((uint64_t)1 << lane) - 1;
            for (int g = 0; g < span / 64; ++g) {
                const uint64_t h = lane_get64(hole, g), t = lane_get64(tail, g);
                const uint16_t r = (uint16_t)(w0 + 64 * g + lane);
                if (h >> lane & 1) list[0][lane_get(h0, g) + __builtin_popcountll(h & below)] = r;
                if (t >> lane & 1) list[1][lane_get(t0, g) + __builtin_popcountll(t & below)] = r;
            }
        } else {
            // ranks of the ties, in the rows' order
            mine = 0;
            each([&](int, bool on, uint32_t x, bool s) { mine += __builtin_popcountll(__builtin_amdgcn_ballot_w64(on && s == among_safe && x == key)); });
            const uint32_t tie0 = before_wave(mine, lds, &total);
            // f(row, a place that it leaves, whether it is to move)
            auto sorted = [&](auto f) {
                uint32_t tie = tie0;
                each([&](int r, bool on, uint32_t x, bool s) {
                    const bool group = on && s == among_safe;
                    const uint64_t eq = __builtin_amdgcn_ballot_w64(group && x == key);
                    const uint32_t rank = tie + __builtin_popcountll(eq & (((uint64_t)1 << lane) - 1));
                    const bool stays = on && (group ? want && (x > key || (x == key && rank < ties)) : !among_safe && s);
                    tie += __builtin_popcountll(eq);
                    f(r, __builtin_amdgcn_ballot_w64(on && !stays && r < k), __builtin_amdgcn_ballot_w64(stays && r >= k));
                });
            };
            uint32_t holes = 0, tails = 0;
            sorted([&](int, uint64_t h, uint64_t t) {
                holes += __builtin_popcountll(h);
                tails += __builtin_popcountll(t);
            });
            uint32_t hole0 = before_wave(holes, lds, &moves), tail0 = before_wave(tails, lds, &total);
            sorted([&](int r, uint64_t h, uint64_t t) {
                const uint64_t below = ((uint64_t)1 << lane) - 1;
                const uint32_t x = hole0 + __builtin_popcountll(h & below), y = tail0 + __builtin_popcountll(t & below);
                if (h >> lane & 1) far_list[x] = r;
                if (t >> lane & 1) far_list[a.half + y] = r;
                hole0 += __builtin_popcountll(h);
                tail0 += __builtin_popcountll(t);
            });
        }
        __syncthreads();
        // their places; a page that other sequences hold too is not written
        bool ok = true;
        const int32_t* const row = a.table + (int64_t)b * a.cols;
        for (uint32_t i0 = tid; i0 < moves; i0 += U * kEvictThreads) {
            uint32_t fp[U], tp[U], fi[U], ti[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t i = min(i0 + u * kEvictThreads, moves - 1);
                const uint32_t from = (uint32_t)tail_at(i), to = (uint32_t)hole_at(i);
                const uint32_t fc = a.d_page.quot(from), tc = a.d_page.quot(to);
                fp[u] = (uint32_t)row[fc], tp[u] = (uint32_t)row[tc];
                fi[u] = from - fc * a.d_page.d, ti[u] = to - tc * a.d_page.d;
            }
            int32_t shared[U];
#pragma unroll
            for (int u = 0; u < U; ++u) shared[u] = a.refs && tp[u] < (uint32_t)a.n_pages ? a.refs[tp[u]] : 0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                ok = ok && fp[u] < (uint32_t)a.n_pages && tp[u] < (uint32_t)a.n_pages && shared[u] <= 1;
                const uint32_t i = i0 + u * kEvictThreads;
                if (i < moves) a.moves[(int64_t)b * a.half + i] = make_int4((int)fp[u], (int)fi[u], (int)tp[u], (int)ti[u]);
            }
        }
        done = __syncthreads_and(ok);
        // weights and positions of the rows that move; a sequence left as it was keeps all
        if (done) {
            for (uint32_t i0 = tid; i0 < moves; i0 += U * kEvictThreads) {
                float x[U];
                int32_t p[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int from = tail_at(min(i0 + u * kEvictThreads, moves - 1));
                    x[u] = a.scores_out ? score[from] : 0.0f;
                    p[u] = position ? position[from] : from;
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const uint32_t i = i0 + u * kEvictThreads;
                    if (i >= moves) continue;
                    const int64_t to = (int64_t)b * a.score_cols + hole_at(i);
                    if (a.scores_out) a.scores_out[to] = x[u];
                    if (a.positions_out) a.positions_out[to] = p[u];
                }
            }
        } else {
            for (int r = k + tid; r < n; r += kEvictThreads) {
                if (score_out) score_out[r] = score[r];
                if (position_out) position_out[r] = position ? position[r] : r;
            }
        }
    }
    if (tid == 0) {
        a.rows_out[b] = done ? k : n;
        a.count[b] = done ? (int32_t)moves : 0;
        a.stay[b] = done ? k : -1;
    }
}

// A workgroup moves kMoveRows rows of a sequence in one pool at a time: a thread takes every 256th
// 16-byte piece of them, four loads before the first store.
constexpr int kMoveRows = 16;

__global__ __launch_bounds__(256) void evict_move_kernel(PoolSet set, EvictArgs a, int32_t chunks, int32_t gives) {
    __shared__ int64_t from[kMoveRows], to[kMoveRows];
    const uint32_t chunk = blockIdx.x, pool = blockIdx.y, b = blockIdx.z;
    const int n = a.count[b], k = a.stay[b];
    if (gives && a.refs && chunk == 0 && pool == 0 && k >= 0) {
        // pages behind the last row: the exchange hands each entry to one thread
        const uint32_t c0 = k ? a.d_page.quot((uint32_t)k - 1u) + 1u : 0u;
        for (uint32_t c = c0 + threadIdx.x; c < (uint32_t)a.cols; c += 256) {
            const uint32_t p = (uint32_t)atomicExch(&a.table[(int64_t)b * a.cols + c], -1);
            if (p < (uint32_t)a.n_pages) atomicSub(&a.refs[p], 1);
        }
    }
    const Pool p = set.p[pool];
    const uint32_t per_line = (p.line + 15u) / 16u, units = per_line * p.heads;
    for (int i0 = (int)chunk * kMoveRows; i0 < n; i0 += chunks * kMoveRows) {
        const int m = min(kMoveRows, n - i0);
        __syncthreads();
        if ((int)threadIdx.x < m) {
            const int4 e = a.moves[(int64_t)b * a.half + i0 + threadIdx.x];
            from[threadIdx.x] = (int64_t)e.x * p.page + (int64_t)e.y * p.row;
            to[threadIdx.x] = (int64_t)e.z * p.page + (int64_t)e.w * p.row;
        }
        __syncthreads();
        const uint32_t total = units * (uint32_t)m;
        for (uint32_t u0 = threadIdx.x; u0 < total; u0 += 1024) {
            u32x4p v[4];
            uint8_t* y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t u = u0 + 256u * j;
                if (u < total) {
                    const uint32_t r = u / units, x = u - r * units, h = x / per_line;
                    const int64_t off = (int64_t)h * p.head + piece_at(x - h * per_line, p.line);
                    v[j] = *(const u32x4p*)(p.base + from[r] + off);
                    y[j] = p.base + to[r] + off;
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (u0 + 256u * j < total) *(u32x4p*)y[j] = v[j];
        }
    }
}

static size_t evict_space(int32_t n_seq, int32_t score_cols, size_t* moves_at, size_t* lists_at) {
    const size_t half = (size_t)score_cols / 2 + 1;
    *moves_at = ((size_t)n_seq * 8 + 15) / 16 * 16;
    *lists_at = *moves_at + (size_t)n_seq * half * 16;
    return *lists_at + (size_t)n_seq * half * 8;
}

}  // namespace xq

using namespace xq;

extern "C" {

xq_status xq_kv_pages_evict_workspace(int32_t n_seq, int32_t score_cols, size_t* bytes) {
    if (!bytes || n_seq < 1 || score_cols < 1) return failf(XQ_ERR_BAD_ARG, "bad evict arguments");
    size_t m, l;
    *bytes = evict_space(n_seq, score_cols, &m, &l);
    return done_ok();
}

xq_status xq_kv_pages_evict(const xq_tensor* pools, int32_t n_pools, int32_t* table, const int32_t* rows, int32_t* refs,
                            int32_t n_seq, int32_t table_cols, const int32_t* keep, int32_t first_rows, int32_t last_rows,
                            const float* scores, const int32_t* positions, int32_t score_cols, float* scores_out,
                            int32_t* positions_out, int32_t* rows_out, void* workspace, size_t workspace_bytes, void* stream) {
    int32_t page_rows, n_pages;
    xq_status st = pools_check(pools, n_pools, &page_rows, &n_pages);
    if (st == XQ_OK) st = table_check(n_seq, table_cols);
    if (st == XQ_OK) st = pools_differ(pools, n_pools);
    if (st != XQ_OK) return st;
    if (n_seq > 65535) return failf(XQ_ERR_UNSUPPORTED, "more than 65535 sequences");
    if (score_cols < 1) return failf(XQ_ERR_BAD_ARG, "score_cols must be at least 1");
    if (score_cols > (1 << 30)) return failf(XQ_ERR_UNSUPPORTED, "score_cols above 2^30");
    if (first_rows < 0 || last_rows < 0) return failf(XQ_ERR_BAD_ARG, "first_rows and last_rows must not be negative");
    if (!table || !rows || !keep || !scores || !rows_out) return failf(XQ_ERR_BAD_ARG, "null pointer");
    if (rows_out == rows) return failf(XQ_ERR_BAD_ARG, "rows_out must not be rows");
    for (const void* x : {(const void*)table, (const void*)rows, (const void*)refs, (const void*)keep, (const void*)scores, (const void*)positions,
                          (const void*)scores_out, (const void*)positions_out, (const void*)rows_out})
        if (!aligned(x, 4)) return failf(XQ_ERR_UNSUPPORTED, "misaligned pointer");
    EvictArgs a{};
    size_t moves_at, lists_at;
    const size_t need = evict_space(n_seq, score_cols, &moves_at, &lists_at);
    if (!workspace || workspace_bytes < need) return failf(XQ_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    if (!aligned(workspace, 256)) return failf(XQ_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    const int64_t lim = (int64_t)table_cols * page_rows;
    a.table = table, a.rows = rows, a.refs = refs, a.keep = keep;
    a.cols = table_cols, a.n_pages = n_pages, a.page_rows = page_rows, a.row_limit = (int32_t)(lim < 0x7fffff00 ? lim : 0x7fffff00);
    a.first_rows = first_rows, a.last_rows = last_rows;
    a.scores = scores, a.positions = positions, a.score_cols = score_cols;
    a.scores_out = scores_out, a.positions_out = positions_out, a.rows_out = rows_out;
    a.count = (int32_t*)workspace, a.stay = a.count + n_seq;
    a.moves = (int4*)((uint8_t*)workspace + moves_at);
    a.lists = (int32_t*)((uint8_t*)workspace + lists_at);
    a.half = score_cols / 2 + 1;
    a.d_page = UDivFlat((uint32_t)page_rows);
    hipStream_t s = (hipStream_t)stream;
    launch("kv_pages_evict", score_cols <= kHeldRows ? evict_select_kernel<true> : evict_select_kernel<false>, dim3((uint32_t)n_seq), dim3(kEvictThreads), s, a);
    for (int32_t i0 = 0; i0 < n_pools; i0 += kPoolsPerLaunch) {
        const int32_t m = n_pools - i0 < kPoolsPerLaunch ? n_pools - i0 : kPoolsPerLaunch;
        PoolSet set{};
        for (int32_t i = 0; i < m; ++i) set.p[i] = pool_of(pools[i0 + i]);
        // workgroups for half of the rows, up to 4096 in all
        int64_t chunks = 4096 / ((int64_t)m * n_seq), most = cdiv(a.half, kMoveRows);
        chunks = chunks < 1 ? 1 : chunks > most ? most : chunks;
        launch("kv_pages_move", evict_move_kernel, dim3((uint32_t)chunks, (uint32_t)m, (uint32_t)n_seq), dim3(256), s, set, a, (int32_t)chunks, i0 == 0 ? 1 : 0);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return failf(XQ_ERR_HIP, "kv_pages_evict launch: %s", hipGetErrorString(e));
    return done_ok();
}

}  // extern "C"
