// xq_fa_chunk.hip — attention of a chunk of new tokens (a prompt, a part of one, one token) over the
// paged cache.
//
// Pair p of a KV head is (token p / G, query head p % G of the group). A token sees the rows
// [lo, hi) (ChunkArgs::range): with x = log2(e) (f(scale q.k) + slope (r - its row)) over them, f the
// identity or cap tanh(./cap), and any m near their maximum,
//   O = sum_r 2^(x_r - m) v_r / sum_r 2^(x_r - m),    lse = (m + log2 sum) / log2(e).
// A workgroup takes PW pairs and walks the 64-row tiles that any of them sees, once.
#include <type_traits>

#include "xq_chunk.h"

namespace xq {

struct FaChunkArgs : ChunkArgs {
    uint8_t* dst;
    int64_t d_nb1, d_nb2, d_nb3;  // head, token, sequence
    float* lse;
    int32_t ptiles, splits;       // pair tiles of a sequence with n_q tokens; parts of one
    uint32_t seg_shift, seg_more; // (sequence, KV head) segments: 2^seg_shift of them times seg_more
    UDivFlat d_more, d_splits, d_hkv, d_h, d_q;
    float* part_o;                // [segment][pair tile][split][PW][D]
    float2* part_ml;              // [segment][pair tile][split][PW] reference, sum
};

constexpr float kLazy = 8.0f;   // base-2 headroom before the running reference moves
constexpr float kOff = -7.0f;   // weights are 2^(x - reference + 7), in (0, 2^15]: f16 keeps small ones normal
constexpr float kHigh = 6.0f;   // beside f32 Q the reference stays this far below the maximum it was taken from,
                                // so that a weight's two parts are off by 2^-37 of the largest, or 2^-22 of itself

template <int KT, int D, bool NARROW, int MT, int NW>
struct ChunkCfg {
    static constexpr bool QUANT = KT == XQ_TYPE_Q8_0 || KT == XQ_TYPE_Q4_0;
    static constexpr int PARTS = QUANT && !NARROW ? 2 : 1;  // f16 parts of a cached value
    static constexpr int QP = NARROW ? 1 : 2;               // f16 parts of Q and of the weights
    static constexpr int EL = KT == XQ_TYPE_F16 ? 8 : KT == XQ_TYPE_Q4_0 ? 32 : 16;  // elements of a 16-byte piece
    static constexpr int PPR = D / EL;                      // pieces per row
    static constexpr int TR = 64;                           // KV rows of a tile (a lane per row)
    static constexpr int RT = 2;                            // 16-row score tiles of a wave at a time
    static constexpr int PIECES = TR * PPR;
    static constexpr int NPT = (PIECES + 64 * NW - 1) / (64 * NW);  // per thread
    static constexpr int RS = 2 * D + 32;                   // image rows, bytes: 8 banks of 64 apart
    static constexpr int PB = TR * RS;                      // one part of K or V
    static constexpr int PW = 16 * MT * NW;                 // pairs of a workgroup
};

template <int KT, int D, bool NARROW, bool BIASED, int MT, int NW>
__global__ __launch_bounds__(64 * NW, 2) void fa_chunk_kernel(FaChunkArgs a) {
    using C = ChunkCfg<KT, D, NARROW, MT, NW>;
    constexpr int PARTS = C::PARTS, QP = C::QP, NB = D / 32, ND = D / 16, NPT = C::NPT, PPR = C::PPR, PW = C::PW, TR = C::TR, RT = C::RT;
    constexpr bool QUANT = C::QUANT, BY_V = PARTS == 2;
    constexpr int KC = PARTS == 2 ? 2 : 4, VC = PARTS == 2 ? 2 : 4;  // K chunks, V columns read at once
    __shared__ __attribute__((aligned(16))) uint8_t imgK[PARTS * C::PB], imgV[PARTS * C::PB];
    __shared__ __attribute__((aligned(16))) int sEk[PARTS == 2 ? TR : 4], sEv[PARTS == 2 ? TR : 4];
    __shared__ unsigned long long sBad[2];
    __shared__ int sRange[4][NW];
    const int lane = lane_id(), wave = wave_id(), tid = threadIdx.x, lr = lane & 15, lg = lane >> 4;
    const int r0 = tid / PPR, c0 = tid % PPR;  // row and piece of a tile that this thread brings

    // ---- the workgroup's segment, pair tile and part. A segment's workgroups share an XCD (or
    // 8 / 2^seg_shift of them): its rows stay in that L2. Late pair tiles, which see the most, go first.
    const uint32_t xcd = blockIdx.x & 7u, slot = blockIdx.x >> 3;
    const uint32_t turn = a.d_more.quot(slot);
    const uint32_t seg = (xcd & ((1u << a.seg_shift) - 1u)) + ((slot - turn * a.seg_more) << a.seg_shift);
    const uint32_t order = (xcd >> a.seg_shift) + (turn << (3 - a.seg_shift));
    const uint32_t po = a.d_splits.quot(order);
    const int part = (int)(order - po * (uint32_t)a.splits), pt = a.ptiles - 1 - (int)po;
    if (pt < 0) return;
    const int b = (int)a.d_hkv.quot(seg), hk = (int)seg - b * a.pg.n_head_kv;
    int held, n_tok, end;
    a.lengths(b, held, n_tok, end);
    const int n_pairs = n_tok * a.G;
    if (pt * PW >= n_pairs) return;
    const int p0 = pt * PW + wave * 16 * MT;  // this wave's first pair

    int tok[MT], lo[MT], hi[MT], at[MT];
    float slope[MT];
    int lo_min = 0x7fffffff, lo_max = 0, hi_min = 0x7fffffff, hi_max = 0;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int p = min(p0 + 16 * m + lr, n_pairs - 1);
        tok[m] = (int)a.d_g.quot((uint32_t)p);
        a.range(b, tok[m], held, end, at[m], lo[m], hi[m]);
        slope[m] = BIASED ? a.slope(hk * a.G + p - tok[m] * a.G) : 0.0f;
        // (what sees nothing asks for no tile)
        if (lo[m] < hi[m]) {
            lo_min = min(lo_min, lo[m]);
            hi_max = max(hi_max, hi[m]);
        }
        lo_max = max(lo_max, lo[m]);
        hi_min = min(hi_min, hi[m]);
    }
#pragma unroll
    for (int s = 1; s < 16; s *= 2) {
        lo_min = min(lo_min, __shfl_xor(lo_min, s));
        lo_max = max(lo_max, __shfl_xor(lo_max, s));
        hi_min = min(hi_min, __shfl_xor(hi_min, s));
        hi_max = max(hi_max, __shfl_xor(hi_max, s));
    }
    lo_min = (int)uniform((uint32_t)lo_min), lo_max = (int)uniform((uint32_t)lo_max);
    hi_min = (int)uniform((uint32_t)hi_min), hi_max = (int)uniform((uint32_t)hi_max);
    if (lane == 0) {
        sRange[0][wave] = lo_min;
        sRange[1][wave] = lo_max;
        sRange[2][wave] = hi_min;
        sRange[3][wave] = hi_max;
    }
    if (tid < 2) sBad[tid] = 0;
    __syncthreads();
    int wg_lo_min = sRange[0][0], wg_lo_max = sRange[1][0], wg_hi_min = sRange[2][0], wg_hi_max = sRange[3][0];
#pragma unroll
    for (int i = 1; i < NW; ++i) {
        wg_lo_min = min(wg_lo_min, sRange[0][i]);
        wg_lo_max = max(wg_lo_max, sRange[1][i]);
        wg_hi_min = min(wg_hi_min, sRange[2][i]);
        wg_hi_max = max(wg_hi_max, sRange[3][i]);
    }
    const uint32_t tile0 = wg_lo_min < wg_hi_max ? (uint32_t)wg_lo_min / TR : 0u;
    const uint32_t tiles = wg_lo_min < wg_hi_max ? ((uint32_t)wg_hi_max + TR - 1) / TR - tile0 : 0u;
    // (tiles below 2^25, parts up to 64)
    const uint32_t t_first = tile0 + uniform(a.d_splits.quot(tiles * (uint32_t)part));
    const uint32_t t_last = part + 1 == a.splits ? tile0 + tiles : tile0 + uniform(a.d_splits.quot(tiles * (uint32_t)(part + 1)));

    const uint8_t* const kb = a.pg.k + hk * a.pg.k_head;
    const uint8_t* const vb = a.pg.v + hk * a.pg.v_head;
    // row lane of tile t: its page (~0u where there is none) and its place in it
    auto lookup = [&](uint32_t t, uint32_t& page, uint32_t& in) {
        const uint32_t r = t * TR + lane;
        page = ~0u;
        in = 0;
        if (t < t_last && r < (uint32_t)end) {
            const uint32_t c = a.pg.d_page.quot(r);
            page = (uint32_t)a.pg.table[(int64_t)b * a.pg.table_cols + c];
            in = r - c * a.pg.d_page.d;
        }
    };
    struct Raw {
        u4t k[NPT], v[NPT];
        // quantized: the fifth dword of each piece's window, and the halves that the piece starts into it
        uint32_t k5[QUANT ? NPT : 1], v5[QUANT ? NPT : 1], shift;
    };
    Raw raw;  // the next tile's pieces, in flight while a tile is computed
    // a quantized piece (16 bytes behind a 2-byte scale in 34- or 18-byte blocks) by whole aligned dwords
    auto window = [&](const uint8_t* rec, u4t& x, uint32_t& x5) -> uint32_t {
        constexpr int BB = KT == XQ_TYPE_Q8_0 ? 34 : 18;
        const bool first = KT == XQ_TYPE_Q4_0 || c0 % 2 == 0;
        const uint8_t* q = rec + (KT == XQ_TYPE_Q8_0 ? c0 / 2 * BB + 2 + c0 % 2 * 16 : c0 * BB + 2);
        const uint32_t odd = (uint32_t)(uintptr_t)q & 2u, shift = first && !odd ? 4u : odd;
        const uint8_t* w = q - shift;
        x = *(const u4dw*)w;
        x5 = *(const uint32_t*)(w + (shift ? 16 : 12));
        return shift / 2;
    };
    auto fetch = [&](uint32_t page, uint32_t in) {
        if constexpr (QUANT) raw.shift = 0;
#pragma unroll
        for (int j = 0; j < NPT; ++j) {
            const int r4 = 4 * (r0 + 64 * NW / PPR * j);  // (modulo 64 lanes)
            const uint32_t p = (uint32_t)__builtin_amdgcn_ds_bpermute(r4, (int)page), x = (uint32_t)__builtin_amdgcn_ds_bpermute(r4, (int)in);
            raw.k[j] = u4t{0, 0, 0, 0};
            raw.v[j] = u4t{0, 0, 0, 0};
            if constexpr (QUANT) raw.k5[j] = raw.v5[j] = 0u;
            if (p < (uint32_t)a.pg.n_pages && (C::PIECES % (64 * NW) == 0 || tid + 64 * NW * j < C::PIECES)) {
                const uint8_t* k = kb + (uint64_t)p * a.k_page + (uint64_t)x * a.k_row;
                const uint8_t* v = vb + (uint64_t)p * a.v_page + (uint64_t)x * a.v_row;
                if constexpr (QUANT) {
                    raw.shift |= window(k, raw.k[j], raw.k5[j]) << (4 * j) | window(v, raw.v[j], raw.v5[j]) << (4 * j + 2);
                } else {
                    raw.k[j] = *(const u4any*)(k + 16 * c0);
                    raw.v[j] = *(const u4any*)(v + 16 * c0);
                }
            }
        }
    };
    // raw pieces -> image
    auto put = [&](uint8_t* image, const u4t x, uint32_t d, int r, int* exps, bool clean, uint32_t t) {
        constexpr int WORDS = C::EL / 2;
        uint32_t o[WORDS], low[WORDS];
        piece_f16<KT, WORDS>(x, o);
        if constexpr (QUANT && NARROW) {
            const uint32_t dd = d | (d << 16);
#pragma unroll
            for (int i = 0; i < WORDS; ++i) o[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2t, o[i]) * __builtin_bit_cast(h2t, dd));
        } else if constexpr (QUANT) {
            // d 2^-e in [2^7, 2^8) for the row's largest finite block scale; then d q = hi + lo exactly:
            // hi its rounding, lo the remainder of at most 8 bits
            const float df = f16_bits_to_f32(d);
            int e = (int)((__float_as_uint(df) >> 23) & 255u);
            if (e == 255 || e < 103) e = 103;  // 2^-24, the smallest f16
            e = max(e, dpp_i<0xB1>(e));
            e = max(e, dpp_i<0x4E>(e));
            if constexpr (PPR >= 8) e = max(e, dpp_i<0x141>(e));
            if constexpr (PPR >= 16) e = max(e, dpp_i<0x140>(e));
            e -= 127 + 7;
            const _Float16 f = (_Float16)ldexpf(df, -e);
            if (c0 == 0) exps[r] = e;
#pragma unroll
            for (int i = 0; i < WORDS; ++i) {
                const h2t q = __builtin_bit_cast(h2t, o[i]), ff = {f, f};
                const h2t high = q * ff;
                o[i] = __builtin_bit_cast(uint32_t, high);
                low[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(q, ff, -high));
            }
        }
        if (clean) {
            uint32_t bad = 0;
#pragma unroll
            for (int i = 0; i < WORDS; ++i) {
                bad |= bad_halves(o[i]);
                if constexpr (PARTS == 2) low[i] &= ~((bad_halves(o[i]) >> 15) * 0xffffu);
                o[i] = without_bad(o[i]);
            }
            if (bad) {
                int row = r;
                asm volatile("" : "+v"(row));  // (its bit is formed here, not kept over the tiles)
                atomicOr(&sBad[t & 1], 1ull << row);
            }
        }
        uint8_t* y = image + r * C::RS + c0 * (2 * C::EL);
#pragma unroll
        for (int i = 0; i < WORDS; i += 4) {
            *(u4t*)(y + 4 * i) = u4t{o[i], o[i + 1], o[i + 2], o[i + 3]};
            if constexpr (PARTS == 2) *(u4t*)(y + C::PB + 4 * i) = u4t{low[i], low[i + 1], low[i + 2], low[i + 3]};
        }
    };
    // the piece from its window; returns its block's scale
    auto realign = [&](u4t& x, uint32_t x5, uint32_t half) -> uint32_t {
        const uint32_t sel = 0x03020100u + half * 0x02020202u;
        const uint32_t d = half == 2 ? x[0] >> 16 : x[0] & 0xffffu;
        x = u4t{__builtin_amdgcn_perm(x[1], x[0], sel), __builtin_amdgcn_perm(x[2], x[1], sel),
                __builtin_amdgcn_perm(x[3], x[2], sel), __builtin_amdgcn_perm(x5, x[3], sel)};
        // q8_0: the odd lane's scale is its even neighbour's (quad_perm 0, 0, 2, 2)
        return KT == XQ_TYPE_Q8_0 ? (uint32_t)dpp_i<0xA0>((int)d) : d;
    };
    auto commit = [&](uint32_t t, bool clean) {
#pragma unroll
        for (int j = 0; j < NPT; ++j) {
            const int r = r0 + 64 * NW / PPR * j;
            if (C::PIECES % (64 * NW) && tid + 64 * NW * j >= C::PIECES) break;  // (whole waves: PIECES is a multiple of 64)
            u4t k = raw.k[j], v = raw.v[j];
            uint32_t dk = 0u, dv = 0u;
            if constexpr (QUANT) {
                dk = realign(k, raw.k5[j], (raw.shift >> (4 * j)) & 3u);
                dv = realign(v, raw.v5[j], (raw.shift >> (4 * j + 2)) & 3u);
            }
            put(imgK, k, dk, r, sEk, false, t);
            put(imgV, v, dv, r, sEv, clean, t);
        }
    };

    uint32_t page, in;
    lookup(t_first, page, in);

    // ---- Q operands: pair 16m + lr
    h8t qo[MT][NB][QP];
    float qf[MT];
    {
        float x[MT][NB][8];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int p = min(p0 + 16 * m + lr, n_pairs - 1);
            query_load<NB, NARROW>(a.q + b * a.q_nb3 + tok[m] * a.q_nb1 + (hk * a.G + p - tok[m] * a.G) * a.q_nb2, lg, x[m]);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) qf[m] = query_split<NB, QP>(x[m], a.scale, BIASED ? 1.0f : kLog2e, qo[m]);
    }
    fetch(page, in);
    uint64_t valid = __builtin_amdgcn_ballot_w64(page < (uint32_t)a.pg.n_pages);  // rows of raw's tile that have a page
    lookup(t_first + 1, page, in);

    f4t acc[MT][ND];
    float m_run[MT], l_run[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        m_run[m] = -INFINITY;
        l_run[m] = 0.0f;
#pragma unroll
        for (int n = 0; n < ND; ++n) acc[m][n] = f4t{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const float inv_cap = a.cap > 0.0f ? 1.0f / a.cap : 0.0f;

    for (uint32_t t = t_first; t < t_last; ++t) {
        const int first = (int)(t * TR);
        __syncthreads();  // the image is free, the flags are zero
        commit(t, first < wg_lo_max || first + TR > wg_hi_min);
        __syncthreads();
        const uint64_t now = valid;
        if (t + 1 < t_last) {
            fetch(page, in);
            valid = __builtin_amdgcn_ballot_w64(page < (uint32_t)a.pg.n_pages);
            lookup(t + 2, page, in);
        }
        if (tid == 0) sBad[(t + 1) & 1] = 0;
        if (p0 >= n_pairs || first >= hi_max || first + TR <= lo_min) continue;  // (a wave without pairs that see the tile)

        // which of the tile's rows each pair sees
        const bool careful = first < lo_max || first + TR > hi_min || now != ~0ull;
        uint64_t sees[MT];
        if (careful) {
#pragma unroll
            for (int m = 0; m < MT; ++m) sees[m] = tile_rows(first, lo[m], hi[m]) & now;
        }
#pragma unroll 1
        for (int sub = 0; sub < TR / (16 * RT); ++sub) {
            const int row0 = 16 * RT * sub;
            f4t s[MT][RT];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int r = 0; r < RT; ++r) s[m][r] = f4t{0.0f, 0.0f, 0.0f, 0.0f};
            // K rows, a batch of chunks at a time: all of its reads before its products
            const uint8_t* const krow = imgK + (row0 + lr) * C::RS + 16 * lg;
#pragma unroll
            for (int k0 = 0; k0 < NB; k0 += KC) {
                h8t kh[KC][RT], kl[PARTS == 2 ? KC : 1][PARTS == 2 ? RT : 1];
#pragma unroll
                for (int c = 0; c < KC; ++c)
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        const uint8_t* k = krow + 16 * r * C::RS + 64 * (k0 + c);
                        kh[c][r] = *(const h8t*)k;
                        if constexpr (PARTS == 2) kl[c][r] = *(const h8t*)(k + C::PB);
                    }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int c = 0; c < KC; ++c)
#pragma unroll
                    for (int r = 0; r < RT; ++r)
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            s[m][r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[c][r], qo[m][k0 + c][0], s[m][r], 0, 0, 0);
                            if constexpr (QP == 2) s[m][r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[c][r], qo[m][k0 + c][1], s[m][r], 0, 0, 0);
                            if constexpr (PARTS == 2) s[m][r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl[c][r], qo[m][k0 + c][0], s[m][r], 0, 0, 0);
                        }
            }
            // the first V columns come while the softmax runs
            const uint8_t* const vrow = imgV + (row0 + 4 * lg + (lr >> 2)) * C::RS + 8 * (lr & 3);
            h4t vh[2][VC][RT], vl[PARTS == 2 ? 2 : 1][PARTS == 2 ? VC : 1][PARTS == 2 ? RT : 1];
            auto columns = [&](int n0, int x) {
#pragma unroll
                for (int n = 0; n < VC; ++n)
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        const uint8_t* v = vrow + 32 * (n0 + n) + 16 * r * C::RS;
                        vh[x][n][r] = __builtin_bit_cast(h4t, column4(v));
                        if constexpr (PARTS == 2) vl[x][n][r] = __builtin_bit_cast(h4t, column4(v + C::PB));
                    }
            };
            columns(0, 0);
            products_done();
            // the lane's rows are row0 + 16r + 4lg + i; s * qf are base-2 scores (BIASED: natural ones)
            if constexpr (PARTS == 2) {
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const int4 e = *(const int4*)(sEk + row0 + 16 * r + 4 * lg);
#pragma unroll
                    for (int m = 0; m < MT; ++m)
                        s[m][r] = f4t{ldexpf(s[m][r][0], e.x), ldexpf(s[m][r][1], e.y), ldexpf(s[m][r][2], e.z), ldexpf(s[m][r][3], e.w)};
                }
            }
            if constexpr (BIASED) {
                // to final base-2 scores; their factor is 1 from here on
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int r = 0; r < RT; ++r)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float x = s[m][r][i] * qf[m];
                            if (a.cap > 0.0f) x = a.cap * capped_tanh(x * inv_cap);
                            x = fmaf(slope[m], (float)(first + row0 + 16 * r + 4 * lg + i - at[m]), x);
                            s[m][r][i] = x * kLog2e;
                        }
            }
            const auto factor = [&](int m) { return BIASED ? 1.0f : qf[m]; };
            if (careful) {
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        const uint32_t bits = (uint32_t)(sees[m] >> (row0 + 16 * r + 4 * lg));
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[m][r][i] = (bits >> i) & 1u ? s[m][r][i] : -INFINITY;
                    }
            }
            bool over = false;
            float top[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) top[m] = -INFINITY;
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                int4 e;
                if constexpr (BY_V) e = *(const int4*)(sEv + row0 + 16 * r + 4 * lg);
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        top[m] = fmaxf(top[m], BY_V ? fmaf(s[m][r][i], factor(m), (float)(i == 0 ? e.x : i == 1 ? e.y : i == 2 ? e.z : e.w)) : s[m][r][i]);
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                if constexpr (!BY_V) top[m] *= factor(m);
                over |= top[m] > m_run[m] + kLazy;
            }
            if (__builtin_amdgcn_ballot_w64(over)) {
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const float mt = across_rows_max(top[m]);
                    const float mn = mt > m_run[m] + kLazy ? ceilf(mt) - (QP == 2 ? kHigh : 0.0f) : m_run[m];
                    const float f = mn == m_run[m] ? 1.0f : __builtin_amdgcn_exp2f(m_run[m] - mn);
                    l_run[m] *= f;
#pragma unroll
                    for (int n = 0; n < ND; ++n) acc[m][n] *= f;
                    m_run[m] = mn;
                }
            }
            // weights
            h4t ph[MT][RT], pl[QP == 2 ? MT : 1][QP == 2 ? RT : 1];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const float mu = m_run[m] == -INFINITY ? 0.0f : -(m_run[m] + kOff);
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    f4t p;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        p[i] = __builtin_amdgcn_exp2f(fmaf(s[m][r][i], factor(m), mu));
                        l_run[m] += p[i];
                    }
                    if constexpr (PARTS == 2) {
                        const int4 e = *(const int4*)(sEv + row0 + 16 * r + 4 * lg);
                        p = f4t{ldexpf(p[0], e.x), ldexpf(p[1], e.y), ldexpf(p[2], e.z), ldexpf(p[3], e.w)};
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        ph[m][r][i] = (_Float16)p[i];
                        if constexpr (QP == 2) pl[m][r][i] = (_Float16)(p[i] - (float)ph[m][r][i]);
                    }
                }
            }
            // O^T += V^T P^T
            auto product = [&](const h4t (&x)[RT], const h4t (&p)[RT], f4t& o) {
                o = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7),
                                                          __builtin_shufflevector(p[0], p[1], 0, 1, 2, 3, 4, 5, 6, 7), o, 0, 0, 0);
            };
#pragma unroll
            for (int n0 = 0; n0 < ND; n0 += VC) {
                const int x = n0 / VC % 2;
                if (n0 + VC < ND) columns(n0 + VC, 1 - x);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int n = 0; n < VC; ++n)
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        product(vh[x][n], ph[m], acc[m][n0 + n]);
                        if constexpr (QP == 2) product(vh[x][n], pl[m], acc[m][n0 + n]);
                        if constexpr (PARTS == 2) product(vl[x][n], ph[m], acc[m][n0 + n]);
                    }
            }
        }
        products_done();
        // non-finite values of rows that not every pair sees: to the pairs that do
        if (careful) {
            uint64_t bad = sBad[t & 1];
            bad = ((uint64_t)__builtin_amdgcn_readfirstlane((int)(bad >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)bad);
            while (bad) {
                const int r = __builtin_ctzll(bad);
                bad &= bad - 1;
                const uint32_t row = t * TR + r, c = a.pg.d_page.quot(row);
                const uint8_t* v = vb + (uint64_t)(uint32_t)a.pg.table[(int64_t)b * a.pg.table_cols + c] * a.v_page + (uint64_t)(row - c * a.pg.d_page.d) * a.v_row;
#pragma unroll 1
                for (int d = 0; d < D; d += 16)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float x = kv_element<KT>(v, d + 4 * lg + i);
                        const bool inf = PARTS == 2 ? !__builtin_isfinite(x) : !(fabsf(x) < 65520.0f);
                        if (!__builtin_amdgcn_ballot_w64(inf)) continue;
                        const float y = __builtin_isfinite(x) ? copysignf(INFINITY, x) : x;
#pragma unroll
                        for (int m = 0; m < MT; ++m)
#pragma unroll
                            for (int n = 0; n < ND; ++n)
                                if (16 * n == d && inf && (sees[m] >> r) & 1) acc[m][n][i] += y;
                    }
            }
        }
    }

    // ---- the pairs' results, or this workgroup's part of them
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int p = p0 + 16 * m + lr;
        const float l = across_rows_sum(l_run[m]);
        if (p >= n_pairs) continue;
        if (a.splits > 1) {
            const int64_t y = (((int64_t)seg * a.ptiles + pt) * a.splits + part) * PW + (p - pt * PW);
#pragma unroll
            for (int n = 0; n < ND; ++n) *(f4t*)(a.part_o + y * D + 16 * n + 4 * lg) = acc[m][n];
            if (lg == 0) a.part_ml[y] = make_float2(m_run[m], l);
            continue;
        }
        const int h = hk * a.G + p - tok[m] * a.G;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint8_t* y = a.dst + b * a.d_nb3 + tok[m] * a.d_nb2 + h * a.d_nb1;
#pragma unroll
        for (int n = 0; n < ND; ++n) {
            const f4t o = acc[m][n] * inv;
            if constexpr (NARROW)
                *(uint2*)(y + 2 * (16 * n + 4 * lg)) = make_uint2(f32_to_bf16_bits(o[0]) | (f32_to_bf16_bits(o[1]) << 16), f32_to_bf16_bits(o[2]) | (f32_to_bf16_bits(o[3]) << 16));
            else
                *(f4t*)(y + 4 * (16 * n + 4 * lg)) = o;
        }
        if (a.lse && lg == 0) a.lse[((int64_t)b * a.n_q + tok[m]) * a.H + h] = l == 0.0f ? -INFINITY : (m_run[m] + kOff) * kLn2 + logf(l);
    }
}

// Joins the parts of each (sequence, token, head): a wave per row, D / 4 lanes a part.
template <int D, bool NARROW>
__global__ __launch_bounds__(256) void fa_chunk_join(FaChunkArgs a, uint32_t rows, int32_t PW) {
    constexpr int L = D / 4, NG = 64 / L;
    const uint32_t row = uniform(blockIdx.x * 4 + threadIdx.x / 64);
    if (row >= rows) return;
    const uint32_t bt = a.d_h.quot(row), h = row - bt * (uint32_t)a.H;
    const uint32_t b = a.d_q.quot(bt), t = bt - b * (uint32_t)a.n_q;
    int held, n_tok, end;
    a.lengths((int)b, held, n_tok, end);
    if ((int)t >= n_tok) return;
    const uint32_t hk = a.d_g.quot(h), pair = t * (uint32_t)a.G + h - hk * (uint32_t)a.G, pt = pair / (uint32_t)PW;
    const int64_t y0 = (((int64_t)(b * a.pg.n_head_kv + hk) * a.ptiles + pt) * a.splits) * PW + (pair - pt * PW);
    const int lane = lane_id(), g = lane / L, d = 4 * (lane % L);
    f4t o = {0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    for (int s = g; s < a.splits; s += NG) {
        const float2 ml = a.part_ml[y0 + (int64_t)s * PW];
        const f4t v = *(const f4t*)(a.part_o + (y0 + (int64_t)s * PW) * D + d);
        const float top = fmaxf(m, ml.x);
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top), w = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - top);
        l = fmaf(ml.y, w, l * f);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(v[e], w, o[e] * f);
        m = top;
    }
    if constexpr (NG == 2) {  // the other half of the wave has the other parts
        const float om = __shfl_xor(m, 32), ol = __shfl_xor(l, 32);
        const float top = fmaxf(m, om);
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top), w = om == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(om - top);
        l = l * f + ol * w;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = o[e] * f + __shfl_xor(o[e], 32) * w;
        m = top;
    }
    if (g) return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint8_t* y = a.dst + b * a.d_nb3 + t * a.d_nb2 + h * a.d_nb1;
    o *= inv;
    if constexpr (NARROW)
        *(uint2*)(y + 2 * d) = make_uint2(f32_to_bf16_bits(o[0]) | (f32_to_bf16_bits(o[1]) << 16), f32_to_bf16_bits(o[2]) | (f32_to_bf16_bits(o[3]) << 16));
    else
        *(f4t*)(y + 4 * d) = o;
    if (a.lse && d == 0) a.lse[(int64_t)bt * a.H + h] = l == 0.0f ? -INFINITY : (m + kOff) * kLn2 + logf(l);
}

// ---------------------------------------------------------------- host

template <int MT_, int NW_> struct ChunkForm { static constexpr int MT = MT_, NW = NW_; };

// f(KT, D, NARROW, BIASED, form) of the call
template <typename F>
static void chunk_variant(int kt, int64_t D, bool narrow, bool biased, bool large, F f) {
    auto with = [&](auto k, auto d, auto n, auto bi) {
        constexpr int DD = decltype(d)::value;
        if (large) f(k, d, n, bi, ChunkForm<DD == 128 ? 2 : 1, 8>{});
        else f(k, d, n, bi, ChunkForm<1, 4>{});
    };
    auto bias = [&](auto k, auto d, auto n) { biased ? with(k, d, n, std::true_type{}) : with(k, d, n, std::false_type{}); };
    auto width = [&](auto k, auto d) { narrow ? bias(k, d, std::true_type{}) : bias(k, d, std::false_type{}); };
    auto dim = [&](auto k) { D == 128 ? width(k, std::integral_constant<int, 128>{}) : width(k, std::integral_constant<int, 256>{}); };
    switch (kt) {
    case XQ_TYPE_F16: dim(std::integral_constant<int, XQ_TYPE_F16>{}); break;
    case XQ_TYPE_E5M2: dim(std::integral_constant<int, XQ_TYPE_E5M2>{}); break;
    case XQ_TYPE_Q8_0: dim(std::integral_constant<int, XQ_TYPE_Q8_0>{}); break;
    default: dim(std::integral_constant<int, XQ_TYPE_Q4_0>{}); break;
    }
}

// The form, parts and workspace of a call: of its shapes alone.
struct ChunkPlan {
    bool large;
    int32_t pw, ptiles, splits;
    uint32_t seg_shift, seg_more;
    int64_t wgs;
    size_t ml_at, bytes;
};
static ChunkPlan chunk_plan(const xq_tensor* q, const xq_kv_pages* c) {
    ChunkPlan P{};
    const int64_t D = q->ne[0], Hkv = c->k.ne[2], B = q->ne[3], pairs = q->ne[1] * (q->ne[2] / Hkv);
    P.large = pairs > 64;
    P.pw = !P.large ? 64 : D == 128 ? 256 : 128;
    P.ptiles = (int32_t)cdiv(pairs, P.pw);
    const int64_t segs = B * Hkv, base = segs * P.ptiles;
    int64_t limit = (int64_t)c->table_cols * c->k.ne[1];
    int64_t splits = cdiv(P.large ? 512 : 1024, base);
    const int64_t most = cdiv(limit, 256);
    if (splits > most) splits = most;
    if (splits > 64) splits = 64;
    P.splits = (int32_t)(splits < 1 ? 1 : splits);
    P.seg_shift = segs % 8 == 0 ? 3 : segs % 4 == 0 ? 2 : segs % 2 == 0 ? 1 : 0;
    P.seg_more = (uint32_t)(segs >> P.seg_shift);
    P.wgs = 8 * (int64_t)P.seg_more * cdiv((int64_t)P.ptiles * P.splits, 8 >> P.seg_shift);
    if (P.splits > 1) {
        const size_t rows = (size_t)base * P.splits * P.pw;
        P.ml_at = rows * D * 4;
        P.bytes = P.ml_at + rows * 8;
    }
    return P;
}

static xq_status fa_chunk_check(const xq_tensor* q, const xq_kv_pages* cache, const xq_tensor* dst, PagesView* pg) {
    if (!q || !cache || !dst) return failf(XQ_ERR_BAD_ARG, "null argument");
    const xq_status st = chunk_check(q, cache, pg);
    if (st != XQ_OK) return st;
    if (dst->type != q->type) return failf(XQ_ERR_UNSUPPORTED, "dst must have q's type");
    if (dst->ne[0] != q->ne[0] || dst->ne[1] != q->ne[2] || dst->ne[2] != q->ne[1] || dst->ne[3] != q->ne[3])
        return failf(XQ_ERR_BAD_SHAPE, "dst must be [D, n_head, n_q, n_seq]");
    if (dst->nb[0] != type_size(q->type)) return failf(XQ_ERR_UNSUPPORTED, "dst elements must be contiguous");
    if (!elem_aligned(dst, 16, 1) || !aligned(dst->data, 16))
        return failf(XQ_ERR_UNSUPPORTED, "dst strides and pointer must be multiples of 16 bytes");
    // (a grid holds below 2^32 threads)
    if (chunk_plan(q, cache).wgs >= (int64_t)1 << 22) return failf(XQ_ERR_UNSUPPORTED, "2^22 workgroups or more");
    return XQ_OK;
}

}  // namespace xq

using namespace xq;

extern "C" {

int xq_supports_fa_chunk(const xq_tensor* q, const xq_kv_pages* cache, const xq_tensor* dst) {
    return fa_chunk_check(q, cache, dst, nullptr) == XQ_OK;
}

xq_status xq_fa_chunk_workspace(const xq_tensor* q, const xq_kv_pages* cache, const xq_tensor* dst, size_t* bytes) {
    if (!bytes) return failf(XQ_ERR_BAD_ARG, "bytes is null");
    const xq_status st = fa_chunk_check(q, cache, dst, nullptr);
    if (st != XQ_OK) return st;
    *bytes = chunk_plan(q, cache).bytes;
    return done_ok();
}

xq_status xq_fa_chunk(const xq_tensor* q, const xq_kv_pages* cache, const xq_chunk_params* params, const int32_t* first,
                      const int32_t* prefix, const int32_t* n_tok, xq_tensor* dst, float* lse, void* workspace,
                      size_t workspace_bytes, void* stream) {
    FaChunkArgs a{};
    xq_status st = fa_chunk_check(q, cache, dst, &a.pg);
    if (st == XQ_OK) st = chunk_params_check(params);
    if (st != XQ_OK) return st;
    if (!q->data || !dst->data || pages_null(cache)) return failf(XQ_ERR_BAD_ARG, "null data pointer");
    for (const void* x : {(const void*)first, (const void*)prefix, (const void*)n_tok, (const void*)lse, (const void*)cache->table, (const void*)cache->rows})
        if (!aligned(x, 4)) return failf(XQ_ERR_UNSUPPORTED, "misaligned pointer");
    const ChunkPlan P = chunk_plan(q, cache);
    if (P.bytes && (!workspace || workspace_bytes < P.bytes))
        return failf(XQ_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", P.bytes, workspace_bytes);
    if (P.bytes && !aligned(workspace, 256)) return failf(XQ_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    chunk_fill(a, q, params, first, prefix, n_tok);
    a.dst = (uint8_t*)dst->data;
    a.d_nb1 = (int64_t)dst->nb[1], a.d_nb2 = (int64_t)dst->nb[2], a.d_nb3 = (int64_t)dst->nb[3];
    a.lse = lse;
    a.ptiles = P.ptiles, a.splits = P.splits;
    a.seg_shift = P.seg_shift, a.seg_more = P.seg_more;
    a.d_more = UDivFlat(P.seg_more), a.d_splits = UDivFlat((uint32_t)P.splits), a.d_hkv = UDivFlat((uint32_t)a.pg.n_head_kv);
    a.d_h = UDivFlat((uint32_t)a.H), a.d_q = UDivFlat((uint32_t)a.n_q);
    a.part_o = (float*)workspace, a.part_ml = (float2*)((uint8_t*)workspace + P.ml_at);
    const bool biased = a.cap > 0.0f || a.max_bias > 0.0f;
    hipStream_t s = (hipStream_t)stream;
    chunk_variant(cache->k.type, q->ne[0], q->type == XQ_TYPE_BF16, biased, P.large, [&](auto k, auto d, auto nar, auto bi, auto fm) {
        using F = decltype(fm);
        constexpr int D = decltype(d)::value;
        constexpr bool NARROW = decltype(nar)::value;
        launch("fa_chunk", fa_chunk_kernel<decltype(k)::value, D, NARROW, decltype(bi)::value, F::MT, F::NW>, dim3((uint32_t)P.wgs), dim3(64 * F::NW), s, a);
        if (P.splits > 1) {
            const uint32_t rows = (uint32_t)((int64_t)a.B * a.n_q * a.H);
            launch("fa_chunk_join", fa_chunk_join<D, NARROW>, dim3((rows + 3) / 4), dim3(256), s, a, rows, P.pw);
        }
    });
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return failf(XQ_ERR_HIP, "fa_chunk launch: %s", hipGetErrorString(e));
    return done_ok();
}

}  // extern "C"
