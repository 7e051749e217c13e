// xq_weights.hip — the attention weight that each cached row gets from a chunk's tokens, accumulated.
//
// With the lse of every (token, head) known, a row's weight is a plain sum,
//   w_r = sum_{pairs that see r} 2^(x_r - log2(e) lse),   x_r = log2(e) (f(scale q.k_r) - slope |r - at|),
// and nothing of V is read. A wave has 16 or 32 rows of K of one head as matrix operands and takes the
// head's pairs 16 at a time: the product leaves four rows of one pair in a lane, whose
// weights add up in the lane; the 16 lanes of a row join at the end.
//
// Rows are what is split, not pairs, so a row's sum has one owner and its order is fixed: no atomics. What bounds it:
// up to 16 pairs of a KV head (a decode step) the bytes of K and the launch: 16 f32 tokens over up to 8000 q8_0 rows
// 24 us, 7.5 at 5.0 TB/s; with many pairs the loads of K and the products, one after the other at the few waves that K in
// registers leaves: 32 tokens over 2 x 16001 f16 rows 33 us (27 here, 3 each before and after), 13 at 5.0 TB/s.
// An eight-wave form with K in halves took 33 us for 28.
#include <type_traits>

#include "xq_chunk.h"

namespace xq {

struct PairMeta {
    float factor, lse2, slope;  // base-2 score of a product (BIASED: natural), log2(e) lse, ALiBi slope
    int32_t lo, hi, at;         // rows seen, the token's own
    int32_t pad[2];             // (copied by two 16-byte halves, lo the first's last)
};

struct WeightsArgs : ChunkArgs {
    const float* lse;
    const float* scores;
    float* out;
    int32_t cols, fresh, splits, few_tiles;
    float decay;
    int64_t part_cols;
    _Float16* qh;   // [sequence][KV head][n_q G][QP][D]
    PairMeta* meta; // [sequence][KV head][n_q G]
    float* part;    // [split][sequence][part_cols]
    UDivFlat d_h, d_q;
};

// A wave per (sequence, token, head): its query as f16 (high and low parts beside f32) times a power
// of two that puts its largest element in [2^14, 2^15), and what its scores need.
template <int D, bool NARROW, bool BIASED>
__global__ __launch_bounds__(256) void weights_prep_kernel(WeightsArgs a, uint32_t rows) {
    constexpr int QP = NARROW ? 1 : 2, E = D / 64;
    const uint32_t row = uniform(blockIdx.x * 4 + threadIdx.x / 64);
    if (row >= rows) return;
    const uint32_t bt = a.d_h.quot(row), h = row - bt * (uint32_t)a.H;
    const uint32_t b = a.d_q.quot(bt), t = bt - b * (uint32_t)a.n_q;
    int held, n_tok, end;
    a.lengths((int)b, held, n_tok, end);
    if ((int)t >= n_tok) return;
    const int lane = lane_id();
    const uint8_t* q = a.q + b * a.q_nb3 + t * a.q_nb1 + h * a.q_nb2;
    float x[E], big = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        x[i] = NARROW ? bf16_bits_to_f32(*(const uint16_t*)(q + 2 * (E * lane + i))) : *(const float*)(q + 4 * (E * lane + i));
        big = fmaxf(big, fabsf(x[i]));
    }
    const int lift = 141 - min((int)(__float_as_uint(wave_max(big)) >> 23), 254);
    const uint32_t hk = a.d_g.quot(h);
    const int64_t pair = ((int64_t)b * a.pg.n_head_kv + hk) * a.n_q * a.G + (int64_t)t * a.G + (h - hk * a.G);
    _Float16* y = a.qh + pair * (QP * D) + E * lane;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const float v = ldexpf(a.scale < 0.0f ? -x[i] : x[i], lift);
        const _Float16 high = (_Float16)v;
        y[i] = high;
        if constexpr (QP == 2) y[D + i] = (_Float16)(v - (float)high);
    }
    if (lane == 0) {
        PairMeta m;
        m.factor = fminf(fmaxf(ldexpf(fabsf(a.scale), -lift) * (BIASED ? 1.0f : kLog2e), 1.17549435e-38f), 3.40282347e38f);
        m.lse2 = a.lse[(int64_t)bt * a.H + h] * kLog2e;
        m.slope = BIASED ? a.slope((int)h) : 0.0f;
        a.range((int)b, (int)t, held, end, m.at, m.lo, m.hi);
        if (m.lse2 == -INFINITY) m.lo = m.hi = 0;  // a token that saw nothing
        m.pad[0] = m.pad[1] = 0;
        a.meta[pair] = m;
    }
}

// 16 bytes of a record (EL elements), the lg-th of the g-th four, on their way. Quantized ones by whole aligned
// dwords (their blocks of 34 or 18 bytes are aligned to 2): a window from the dword of the block's scale,
// or, in a q8_0 block's second half, of the piece; every dword read holds a byte of the two.
template <int KT>
struct Piece {
    static constexpr bool QUANT = KT == XQ_TYPE_Q8_0 || KT == XQ_TYPE_Q4_0;
    static constexpr int EL = KT == XQ_TYPE_F16 ? 8 : KT == XQ_TYPE_Q4_0 ? 32 : 16, BLOCK = KT == XQ_TYPE_Q8_0 ? 34 : 18;
    u4t w;
    uint32_t w5;
    static XQ_DEV int at(int g, int lg) { return KT == XQ_TYPE_Q8_0 ? (2 * g + lg / 2) * BLOCK + 2 + lg % 2 * 16 : (4 * g + lg) * BLOCK + 2; }
    // bytes that the piece starts into its window: 0, 2 or 4
    static XQ_DEV uint32_t shift(uintptr_t rec, int g, int lg) {
        const uint32_t odd = (uint32_t)(rec + at(g, lg)) & 2u;
        return (KT == XQ_TYPE_Q4_0 || lg % 2 == 0) && !odd ? 4u : odd;
    }
    XQ_DEV void load(const uint8_t* rec, int g, int lg) {
        if constexpr (QUANT) {
            const uint32_t s = shift((uintptr_t)rec, g, lg);
            const uint8_t* q = rec + at(g, lg) - s;
            w = *(const u4dw*)q;
            w5 = *(const uint32_t*)(q + (s ? 16 : 12));
        } else {
            w = *(const u4any*)(rec + 64 * g + 16 * lg);
        }
    }
    // The piece out of its window; returns its block's scale (bits of f16).
    XQ_DEV uint32_t settle(uint32_t s, int lane) {
        const uint32_t sel = 0x03020100u + s / 2 * 0x02020202u;
        const uint32_t d = s == 4 ? w[0] >> 16 : w[0] & 0xffffu;
        w = u4t{__builtin_amdgcn_perm(w[1], w[0], sel), __builtin_amdgcn_perm(w[2], w[1], sel), __builtin_amdgcn_perm(w[3], w[2], sel),
                __builtin_amdgcn_perm(w5, w[3], sel)};
        return KT == XQ_TYPE_Q8_0 ? (uint32_t)__shfl((int)d, lane & ~16) : d;  // (of the block's first half)
    }
    // its j-th eight elements as f16; quantized: the integers
    XQ_DEV h8t f16(int j) const {
        if constexpr (KT == XQ_TYPE_F16) {
            return __builtin_bit_cast(h8t, w);
        } else if constexpr (KT == XQ_TYPE_E5M2) {
            const u4t o = {__builtin_amdgcn_perm(w[2 * j], w[2 * j], 0x010c000cu), __builtin_amdgcn_perm(w[2 * j], w[2 * j], 0x030c020cu),
                           __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j + 1], 0x010c000cu), __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j + 1], 0x030c020cu)};
            return __builtin_bit_cast(h8t, o);
        } else {
            // (1024 + n) - 1152 of n = q ^ 0x80; (1024 + n) - 1032 of the nibble: low ones are elements 0 .. 15
            constexpr bool Q8 = KT == XQ_TYPE_Q8_0;
            const _Float16 off = Q8 ? (_Float16)-1152.0f : (_Float16)-1032.0f;
            u4t o;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t x = w[Q8 ? 2 * j + i : 2 * (j % 2) + i];
                const uint32_t n = Q8 ? x ^ 0x80808080u : (j / 2 ? x >> 4 : x) & 0x0f0f0f0fu;
                o[2 * i] = __builtin_amdgcn_perm(0x64646464u, n, 0x05010500u);
                o[2 * i + 1] = __builtin_amdgcn_perm(0x64646464u, n, 0x05030502u);
            }
            return __builtin_bit_cast(h8t, o) + off;
        }
    }
};

// A row's power of two e by its blocks' scales (bits of f16, of the lane's pieces): d 2^-e in [2^7, 2^8) for the
// largest finite one, over the four lanes of the row. Then d q = hi + lo exactly in f16, hi its rounding.
template <int NG>
XQ_DEV int scale_power(const uint32_t (&d)[NG]) {
    int e = 103;  // 2^-24, the smallest f16
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        const int z = (int)((__float_as_uint(f16_bits_to_f32(d[g])) >> 23) & 255u);
        e = max(e, z == 255 ? 103 : z);
    }
    e = max(e, __shfl_xor(e, 16));
    return max(e, __shfl_xor(e, 32)) - (127 + 7);
}

// More pairs: a wave keeps 16 RT rows of K of a head as operands, a workgroup's four waves have other rows and
// share the head's pairs, CH at a time in LDS. Items (head, CH pairs) are split over blockIdx.y where few
// rows leave CUs without work.
template <int KT, int D, bool NARROW, bool BIASED, int RT, int CH>
__global__ __launch_bounds__(256, 2) void weights_kernel(WeightsArgs a) {
    constexpr bool QUANT = KT == XQ_TYPE_Q8_0 || KT == XQ_TYPE_Q4_0;
    constexpr int QP = NARROW ? 1 : 2, PARTS = QUANT ? 2 : 1, NB = D / 32, ROWS = 16 * RT;
    constexpr int EL = Piece<KT>::EL, PER = EL / 8, NG = D / (4 * EL);
    constexpr int PPP = QP * D / 8, NPT = CH * PPP / 256;  // 16-byte pieces of a pair; of a thread
    constexpr int RS = 2 * QP * D + 32;                    // a pair's bytes in LDS: 8 banks of 64 apart
    __shared__ __attribute__((aligned(16))) uint8_t sQ[CH * RS];
    __shared__ __attribute__((aligned(16))) PairMeta sMeta[CH];
    constexpr uint64_t HAS = ~0ull >> (64 - ROWS);
    const int lane = lane_id(), wave = wave_id(), tid = threadIdx.x, lr = lane & 15, lg = lane >> 4;
    const int b = blockIdx.z;
    int held, n_tok, end;
    a.lengths(b, held, n_tok, end);
    if ((int)blockIdx.x * 4 * ROWS >= end) return;
    const int first = (int)blockIdx.x * 4 * ROWS + wave * ROWS;
    const int n_pairs = n_tok * a.G, chunks = (n_pairs + CH - 1) / CH, items = chunks * a.pg.n_head_kv;
    const int it0 = (int)((int64_t)items * blockIdx.y / a.splits), it_end = (int)((int64_t)items * (blockIdx.y + 1) / a.splits);

    // lane lr (of each 16) has row 16r + lr
    uint64_t has = 0;
    const uint8_t* rec[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const uint32_t row = (uint32_t)first + 16 * r + lr;
        uint32_t page = ~0u, in = 0;
        if (row < (uint32_t)end) {
            const uint32_t c = a.pg.d_page.quot(row);
            page = (uint32_t)a.pg.table[(int64_t)b * a.pg.table_cols + c];
            in = row - c * a.pg.d_page.d;
        }
        const bool ok = page < (uint32_t)a.pg.n_pages;
        has |= (__builtin_amdgcn_ballot_w64(ok) & 0xffffull) << (16 * r);
        // (a row that is none: row 0 of the pool, whose weights are not taken)
        rec[r] = a.pg.k + (ok ? (uint64_t)page * a.k_page + (uint64_t)in * a.k_row : 0u);
    }
    f4t sum[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) sum[r] = f4t{0.0f, 0.0f, 0.0f, 0.0f};

    // a chunk's pairs on their way
    u4t piece[NPT], meta0, meta1;
    auto fetch = [&](int item) {
        const int hk = item / chunks, p0 = (item - hk * chunks) * CH;
        const int64_t head = ((int64_t)b * a.pg.n_head_kv + hk) * a.n_q * a.G;
#pragma unroll
        for (int j = 0; j < NPT; ++j) {
            const int i = tid + 256 * j;
            piece[j] = *(const u4t*)(a.qh + (head + min(p0 + i / PPP, n_pairs - 1)) * (QP * D) + 8 * (i % PPP));
        }
        // (a pair that is none sees nothing)
        const u4t* m = (const u4t*)(a.meta + head + min(p0 + tid % CH, n_pairs - 1));
        meta0 = m[0];
        meta1 = m[1];
        if (p0 + tid % CH >= n_pairs) meta0[3] = meta1[0] = 0;
    };
    if (it0 < it_end) fetch(it0);
    int hk = -1;
    h8t kh[RT][NB], kl[PARTS == 2 ? RT : 1][PARTS == 2 ? NB : 1];
    int ek[RT][4];  // QUANT: the powers of two of rows 16r + 4lg + i
    for (int it = it0; it < it_end; ++it) {
        if (it / chunks != hk) {
            hk = it / chunks;
            Piece<KT> raw[RT][NG];
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int g = 0; g < NG; ++g) raw[r][g].load(rec[r] + hk * a.pg.k_head, g, lg);
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                if constexpr (QUANT) {
                    uint32_t d[NG];
#pragma unroll
                    for (int g = 0; g < NG; ++g) d[g] = raw[r][g].settle(Piece<KT>::shift((uintptr_t)(rec[r] + hk * a.pg.k_head), g, lg), lane);
                    const int e = scale_power<NG>(d);
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        const _Float16 f = (_Float16)ldexpf(f16_bits_to_f32(d[g]), -e);
                        const h8t ff = {f, f, f, f, f, f, f, f};
#pragma unroll
                        for (int j = 0; j < PER; ++j) {
                            const h8t q = raw[r][g].f16(j);
                            kh[r][g * PER + j] = q * ff;
                            kl[r][g * PER + j] = __builtin_elementwise_fma(q, ff, -kh[r][g * PER + j]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) ek[r][i] = __shfl(e, 4 * lg + i);
                } else {
#pragma unroll
                    for (int g = 0; g < NG; ++g)
#pragma unroll
                        for (int j = 0; j < PER; ++j) kh[r][g * PER + j] = raw[r][g].f16(j);
                }
            }
        }
        __syncthreads();  // the last chunk is read
#pragma unroll
        for (int j = 0; j < NPT; ++j) {
            const int i = tid + 256 * j;
            *(u4t*)(sQ + i / PPP * RS + 16 * (i % PPP)) = piece[j];
        }
        if (tid < CH) {
            ((u4t*)(sMeta + tid))[0] = meta0;
            ((u4t*)(sMeta + tid))[1] = meta1;
        }
        __syncthreads();
        if (it + 1 < it_end) fetch(it + 1);
#pragma unroll 1
        for (int g = 0; g < CH / 16; ++g) {
            const PairMeta m = sMeta[16 * g + lr];
            if (!__builtin_amdgcn_ballot_w64(m.lo < min(m.hi, first + ROWS) && m.hi > first)) continue;
            const bool all = has == HAS && !__builtin_amdgcn_ballot_w64(m.lo > first || m.hi < first + ROWS);  // of its pairs see all rows
            const uint8_t* const q = sQ + (16 * g + lr) * RS + 2 * EL * lg;
            f4t s[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) s[r] = f4t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < NB; ++c) {
                const h8t x = *(const h8t*)(q + 2 * operand_at<EL>(c));
                h8t y;
                if constexpr (QP == 2) y = *(const h8t*)(q + 2 * D + 2 * operand_at<EL>(c));
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    s[r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[r][c], x, s[r], 0, 0, 0);
                    if constexpr (QP == 2) s[r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[r][c], y, s[r], 0, 0, 0);
                    if constexpr (PARTS == 2) s[r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl[r][c], x, s[r], 0, 0, 0);
                }
            }
            products_done();
            auto weight = [&](int r, int i) {
                float z = s[r][i];
                if constexpr (QUANT) z = ldexpf(z, ek[r][i]);
                if constexpr (BIASED) {
                    z *= m.factor;
                    if (a.cap > 0.0f) z = a.cap * capped_tanh(z * a.inv_cap);
                    z = less_distance(z, m.slope, first + 16 * r + 4 * lg + i, m.at);
                    z = fmaf(z, kLog2e, -m.lse2);
                } else {
                    z = fmaf(z, m.factor, -m.lse2);
                }
                return __builtin_amdgcn_exp2f(z);
            };
            if (all) {
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[r][i] += weight(r, i);
            } else {
                const uint64_t sees = tile_rows(first, m.lo, m.hi) & has;
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[r][i] += (sees >> (16 * r + 4 * lg + i)) & 1u ? weight(r, i) : 0.0f;
            }
        }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float w = row16_sum(sum[r][i]);
            const int row = first + 16 * r + 4 * lg + i;
            if (lr != 0) continue;
            if (a.splits > 1) {
                a.part[((int64_t)blockIdx.y * a.B + b) * a.part_cols + row] = w;
            } else if (row < min(end, a.cols)) {
                const int64_t at = (int64_t)b * a.cols + row;
                const bool old = a.scores && (row < held || !a.fresh);
                a.out[at] = (old ? a.decay * a.scores[at] : 0.0f) + w;
            }
        }
}

// Up to 16 pairs of a KV head (decode): bound by HBM and by latency. A workgroup has up to 64 rows; its units, a head's 16
// rows each, head after head, are shared out to the four waves, which hold the head's queries as operands and
// ask for the next unit's rows before they work on one.
template <int KT, int D, bool NARROW, bool BIASED>
__global__ __launch_bounds__(256, 2) void weights_few_kernel(WeightsArgs a) {
    constexpr bool QUANT = KT == XQ_TYPE_Q8_0 || KT == XQ_TYPE_Q4_0;
    constexpr int QP = NARROW ? 1 : 2, NB = D / 32, EL = Piece<KT>::EL, PER = EL / 8, NG = D / (4 * EL);
    __shared__ float sSum[4][64];
    const int lane = lane_id(), wave = wave_id(), lr = lane & 15, lg = lane >> 4;
    const int b = blockIdx.y, tiles = a.few_tiles, first = (int)blockIdx.x * 16 * tiles;
    int held, n_tok, end;
    a.lengths(b, held, n_tok, end);
    if (first >= end) return;
    const int n_pairs = n_tok * a.G, units = n_pairs ? tiles * a.pg.n_head_kv : 0;
    int u = units * wave / 4;
    const int u_end = units * (wave + 1) / 4;
    // lane l has row l of the workgroup's
    uint32_t page = ~0u, in = 0;
    if (first + lane < end && lane < 16 * tiles) {
        const uint32_t r = (uint32_t)(first + lane), c = a.pg.d_page.quot(r);
        page = (uint32_t)a.pg.table[(int64_t)b * a.pg.table_cols + c];
        in = r - c * a.pg.d_page.d;
    }
    sSum[wave][lane] = 0.0f;
    const uint64_t has = __builtin_amdgcn_ballot_w64(page < (uint32_t)a.pg.n_pages);
    // (a row that is none: row 0 of the pool, whose weights are not taken)
    if (page >= (uint32_t)a.pg.n_pages) page = in = 0;
    Piece<KT> raw[NG];
    uintptr_t from = 0;  // the record that they are of
    auto fetch = [&](int v) {
        const int hk = v / tiles, l = 16 * (v - hk * tiles) + lr;
        const uint8_t* rec = a.pg.k + hk * a.pg.k_head + (uint64_t)(uint32_t)__shfl((int)page, l) * a.k_page + (uint64_t)(uint32_t)__shfl((int)in, l) * a.k_row;
        from = (uintptr_t)rec;
#pragma unroll
        for (int g = 0; g < NG; ++g) raw[g].load(rec, g, lg);
    };
    if (u < u_end) fetch(u);
    int hk = -1, lo = 0, hi = 0, at = 0;
    float factor = 0.0f, lse2 = 0.0f, slope = 0.0f;
    h8t q[NB][QP];
    for (; u < u_end; ++u) {
        const int tile = u % tiles;
        if (u / tiles != hk) {
            hk = u / tiles;
            const int p = min(lr, n_pairs - 1), t = (int)a.d_g.quot((uint32_t)p), h = hk * a.G + p - t * a.G;
            float x[NB][8];
            query_load<NB, NARROW, EL>(a.q + b * a.q_nb3 + t * a.q_nb1 + h * a.q_nb2, lg, x);
            lse2 = a.lse[((int64_t)b * a.n_q + t) * a.H + h] * kLog2e;
            a.range(b, t, held, end, at, lo, hi);
            if (lse2 == -INFINITY || lr >= n_pairs) lo = hi = 0;  // a token that saw nothing, a pair that is none
            slope = BIASED ? a.slope(h) : 0.0f;
            factor = query_split<NB, QP>(x, a.scale, BIASED ? 1.0f : kLog2e, q);
        }
        f4t s = {0.0f, 0.0f, 0.0f, 0.0f};
        int e = 0;
        uint32_t d[NG];
        if constexpr (QUANT) {
#pragma unroll
            for (int g = 0; g < NG; ++g) d[g] = raw[g].settle(Piece<KT>::shift(from, g, lg), lane);
            e = scale_power<NG>(d);
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const _Float16 f = QUANT ? (_Float16)ldexpf(f16_bits_to_f32(d[g]), -e) : (_Float16)1.0f;
            const h8t ff = {f, f, f, f, f, f, f, f};
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const h8t k = raw[g].f16(j), high = QUANT ? k * ff : k;
                const int c = g * PER + j;
                s = __builtin_amdgcn_mfma_f32_16x16x32_f16(high, q[c][0], s, 0, 0, 0);
                if constexpr (QP == 2) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(high, q[c][QP - 1], s, 0, 0, 0);
                if constexpr (QUANT) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_elementwise_fma(k, ff, -high), q[c][0], s, 0, 0, 0);
            }
        }
        if (u + 1 < u_end) fetch(u + 1);
        products_done();
        const uint32_t sees = (uint32_t)((tile_rows(first, lo, hi) & has) >> (16 * tile + 4 * lg));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float z = s[i];
            if constexpr (QUANT) z = ldexpf(z, __shfl(e, 4 * lg + i));
            if constexpr (BIASED) {
                z *= factor;
                if (a.cap > 0.0f) z = a.cap * capped_tanh(z * a.inv_cap);
                z = less_distance(z, slope, first + 16 * tile + 4 * lg + i, at);
                z = fmaf(z, kLog2e, -lse2);
            } else {
                z = fmaf(z, factor, -lse2);
            }
            const float w = row16_sum((sees >> i) & 1u ? __builtin_amdgcn_exp2f(z) : 0.0f);
            if (lr == 0) sSum[wave][16 * tile + 4 * lg + i] += w;
        }
    }
    __syncthreads();
    const int row = first + lane;
    if (wave == 0 && lane < 16 * tiles && row < min(end, a.cols)) {
        const float w = (sSum[0][lane] + sSum[1][lane]) + (sSum[2][lane] + sSum[3][lane]);
        const int64_t y = (int64_t)b * a.cols + row;
        const bool old = a.scores && (row < held || !a.fresh);
        a.out[y] = (old ? a.decay * a.scores[y] : 0.0f) + w;
    }
}

__global__ __launch_bounds__(256) void weights_join_kernel(WeightsArgs a) {
    const int b = blockIdx.y, row = (int)(blockIdx.x * 256 + threadIdx.x);
    int held, n_tok, end;
    a.lengths(b, held, n_tok, end);
    if (row >= min(end, a.cols)) return;
    float w = 0.0f;
    for (int s = 0; s < a.splits; ++s) w += a.part[((int64_t)s * a.B + b) * a.part_cols + row];
    const int64_t at = (int64_t)b * a.cols + row;
    const bool old = a.scores && (row < held || !a.fresh);
    a.out[at] = (old ? a.decay * a.scores[at] : 0.0f) + w;
}

// ---------------------------------------------------------------- host

// Rows of a wave, in 16s (two where its K fits 256 registers beside the rest), and pairs in LDS at a time.
constexpr int weights_rt(bool quant, int64_t D) { return quant && D == 256 ? 1 : 2; }
constexpr int weights_ch(bool narrow, int64_t D) { return !narrow && D == 256 ? 32 : 64; }

struct WeightsPlan {
    bool few;  // pairs of a KV head
    int32_t few_tiles, splits;
    int64_t pairs, limit, wgs, part_cols;
    size_t meta_at, part_at, bytes;
};
static WeightsPlan weights_plan(const xq_tensor* q, const xq_kv_pages* c) {
    WeightsPlan P{};
    const int64_t D = q->ne[0], T = q->ne[1], H = q->ne[2], B = q->ne[3], Hkv = c->k.ne[2], G = H / Hkv;
    const int64_t limit = (int64_t)c->table_cols * c->k.ne[1];
    P.limit = limit < 0x7fffff00 ? limit : 0x7fffff00;
    P.pairs = B * H * T;
    P.few = T * G <= 16;
    if (P.few) {
        // 64 rows a workgroup, or fewer where that leaves CUs without one
        P.few_tiles = B * cdiv(P.limit, 64) >= 512 ? 4 : B * cdiv(P.limit, 32) >= 512 ? 2 : 1;
        P.splits = 1;
        P.wgs = cdiv(P.limit, 16 * P.few_tiles);
        return P;
    }
    const bool quant = c->k.type == XQ_TYPE_Q8_0 || c->k.type == XQ_TYPE_Q4_0, narrow = q->type == XQ_TYPE_BF16;
    const int64_t rows = 64 * weights_rt(quant, D);
    P.wgs = cdiv(P.limit, rows);
    P.part_cols = P.wgs * rows;
    const int64_t items = Hkv * cdiv(T * G, weights_ch(narrow, D));
    int64_t splits = cdiv(512, B * P.wgs);
    if (splits > items) splits = items;
    P.splits = (int32_t)(splits < 1 ? 1 : splits);
    P.meta_at = (size_t)P.pairs * D * 2 * (narrow ? 1 : 2);
    P.part_at = P.meta_at + (size_t)P.pairs * sizeof(PairMeta);
    P.bytes = P.part_at + (P.splits > 1 ? (size_t)P.splits * B * P.part_cols * 4 : 0);
    return P;
}

static xq_status weights_check(const xq_tensor* q, const xq_kv_pages* cache, PagesView* pg) {
    const xq_status st = chunk_check(q, cache, pg);
    if (st != XQ_OK) return st;
    if (q->ne[3] > 65535) return failf(XQ_ERR_UNSUPPORTED, "more than 65535 sequences");
    // (a grid's side holds below 2^32 threads: 2^24 workgroups of 16 rows)
    if ((int64_t)cache->table_cols * cache->k.ne[1] >= (int64_t)1 << 28) return failf(XQ_ERR_UNSUPPORTED, "a table of 2^28 rows or more");
    return XQ_OK;
}

template <typename F>
static void weights_variant(int kt, int64_t D, bool narrow, bool biased, F f) {
    auto bias = [&](auto k, auto d, auto n) { biased ? f(k, d, n, std::true_type{}) : f(k, d, n, std::false_type{}); };
    auto width = [&](auto k, auto d) { narrow ? bias(k, d, std::true_type{}) : bias(k, d, std::false_type{}); };
    auto dim = [&](auto k) { D == 128 ? width(k, std::integral_constant<int, 128>{}) : width(k, std::integral_constant<int, 256>{}); };
    switch (kt) {
    case XQ_TYPE_F16: dim(std::integral_constant<int, XQ_TYPE_F16>{}); break;
    case XQ_TYPE_E5M2: dim(std::integral_constant<int, XQ_TYPE_E5M2>{}); break;
    case XQ_TYPE_Q8_0: dim(std::integral_constant<int, XQ_TYPE_Q8_0>{}); break;
    default: dim(std::integral_constant<int, XQ_TYPE_Q4_0>{}); break;
    }
}

}  // namespace xq

using namespace xq;

extern "C" {

xq_status xq_kv_weights_workspace(const xq_tensor* q, const xq_kv_pages* cache, size_t* bytes) {
    if (!bytes) return failf(XQ_ERR_BAD_ARG, "bytes is null");
    const xq_status st = weights_check(q, cache, nullptr);
    if (st != XQ_OK) return st;
    *bytes = weights_plan(q, cache).bytes;
    return done_ok();
}

xq_status xq_kv_weights(const xq_tensor* q, const xq_kv_pages* cache, const xq_chunk_params* params, const int32_t* first,
                        const int32_t* prefix, const int32_t* n_tok, const float* lse, const float* scores, float* scores_out,
                        int32_t score_cols, float decay, int32_t fresh, void* workspace, size_t workspace_bytes, void* stream) {
    WeightsArgs a{};
    xq_status st = weights_check(q, cache, &a.pg);
    if (st == XQ_OK) st = chunk_params_check(params);
    if (st != XQ_OK) return st;
    if (score_cols < 1) return failf(XQ_ERR_BAD_ARG, "score_cols must be at least 1");
    if (!(fabsf(decay) < INFINITY)) return failf(XQ_ERR_BAD_ARG, "decay must be finite");
    if (fresh != 0 && fresh != 1) return failf(XQ_ERR_BAD_ARG, "fresh must be 0 or 1");
    if (!q->data || pages_null(cache) || !lse || !scores_out) return failf(XQ_ERR_BAD_ARG, "null data pointer");
    for (const void* x : {(const void*)first, (const void*)prefix, (const void*)n_tok, (const void*)lse, (const void*)scores, (const void*)scores_out,
                          (const void*)cache->table, (const void*)cache->rows})
        if (!aligned(x, 4)) return failf(XQ_ERR_UNSUPPORTED, "misaligned pointer");
    const WeightsPlan P = weights_plan(q, cache);
    if (P.bytes && (!workspace || workspace_bytes < P.bytes))
        return failf(XQ_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", P.bytes, workspace_bytes);
    if (P.bytes && !aligned(workspace, 256)) return failf(XQ_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    chunk_fill(a, q, params, first, prefix, n_tok);
    a.lse = lse, a.scores = scores, a.out = scores_out;
    a.cols = score_cols, a.decay = decay, a.fresh = fresh, a.splits = P.splits, a.part_cols = P.part_cols, a.few_tiles = P.few_tiles;
    a.qh = (_Float16*)workspace;
    a.meta = (PairMeta*)((uint8_t*)workspace + P.meta_at);
    a.part = (float*)((uint8_t*)workspace + P.part_at);
    a.d_h = UDivFlat((uint32_t)a.H), a.d_q = UDivFlat((uint32_t)a.n_q);
    const bool biased = a.cap > 0.0f || a.max_bias > 0.0f;
    hipStream_t s = (hipStream_t)stream;
    weights_variant(cache->k.type, q->ne[0], q->type == XQ_TYPE_BF16, biased, [&](auto k, auto d, auto nar, auto bi) {
        constexpr int D = decltype(d)::value;
        constexpr bool NARROW = decltype(nar)::value, BIASED = decltype(bi)::value;
        if (P.few) {
            launch("kv_weights", weights_few_kernel<decltype(k)::value, D, NARROW, BIASED>, dim3((uint32_t)P.wgs, (uint32_t)a.B), dim3(256), s, a);
            return;
        }
        launch("kv_weights_prep", weights_prep_kernel<D, NARROW, BIASED>, dim3((uint32_t)cdiv(P.pairs, 4)), dim3(256), s, a, (uint32_t)P.pairs);
        constexpr int KT = decltype(k)::value;
        const dim3 grid((uint32_t)P.wgs, (uint32_t)P.splits, (uint32_t)a.B);
        constexpr bool QUANT = KT == XQ_TYPE_Q8_0 || KT == XQ_TYPE_Q4_0;
        launch("kv_weights", weights_kernel<KT, D, NARROW, BIASED, weights_rt(QUANT, D), weights_ch(NARROW, D)>, grid, dim3(256), s, a);
    });
    if (P.splits > 1)
        launch("kv_weights_join", weights_join_kernel, dim3((uint32_t)cdiv(P.limit, 256), (uint32_t)a.B), dim3(256), s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return failf(XQ_ERR_HIP, "kv_weights launch: %s", hipGetErrorString(e));
    return done_ok();
}

}  // extern "C"
