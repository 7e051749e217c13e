// xq_fa_chunk.hip — attention of a chunk of new tokens (a prompt, a part of one, one token) over the
// paged cache.
//
// Pair p of a KV head is (token p / G, query head p % G of the group). A token sees the rows
// [lo, hi) (ChunkArgs::range): with x = log2(e) (f(scale q.k) - slope |r - its row|) over them, f the
// identity or cap tanh(./cap), and any m near their maximum,
//   O = sum_r 2^(x_r - m) v_r / sum_r 2^(x_r - m),    lse = (m + log2 sum) / log2(e).
// A workgroup takes PW pairs and walks the 64-row tiles that any of them sees, once: K and V as f16 images in LDS,
// S = K Q^T and O^T = V^T P^T on the matrix cores, so that a lane's four scores are four rows of one pair and become
// the second product's operand where they stand. Beside f32 Q, Q and the weights are two f16 parts, and so are
// quantized values (exact integers times a scale's upper bits, and the remainder).
//
// What bounds it. Chunks: matrix products and vector issue, which overlap little: two prompts of 8191 bf16 tokens, f16 rows
// of 128, 1.1 TFLOP: 1169 to 1280 us, 0.86 to 0.94 PFLOP/s of the 1.22 of a large library product; the matrix cores are busy
// 38 % of the time and vector issue 48 %. Without any staging or barrier it would be 1003 us, so a second image buys
// little (32x32x16 products, two images and the stages interleaved by hand: 1187 us for 1185 of the 16x16x32
// form as it then was). Few tokens: the rows' bytes where there are many (32 chats of up to 8000 fp8 rows 39 us, 28 at
// 5.0 TB/s); else the two launches and a workgroup's chain of reads (lengths, table, rows, 20 us in all).
#include <type_traits>

#include "xq_chunk.h"

namespace xq {

struct FaChunkArgs : ChunkArgs {
    uint8_t* dst;
    int64_t d_nb1, d_nb2, d_nb3;  // head, token, sequence
    float* lse;
    uint32_t target;              // above 0: parts dealt by the sequences' lengths, about so many
    int32_t ptiles, splits;       // pair tiles of a sequence with n_q tokens; parts of one
    uint32_t head_shift;          // 2^head_shift KV heads side by side on the XCDs
    UDivFlat d_seq, d_more, d_splits, d_h, d_q;  // by a sequence's workgroups (of an XCD); by the heads one after another; ...
    float* part_o;                // [segment][pair tile][split][PW][D]
    float2* part_ml;              // [segment][pair tile][split][PW] reference, sum
};

constexpr float kLazy = 8.0f;   // base-2 headroom before the running reference moves
constexpr float kOff = -7.0f;   // weights are 2^(x - reference + 7), in (0, 2^15]: f16 keeps small ones normal
constexpr float kHigh = 6.0f;   // beside f32 Q the reference stays this far below the maximum it was taken from,
                                // so that a weight's two parts are off by 2^-37 of the largest, or 2^-22 of itself

// To nearest, ties to even, by the two-value conversion.
XQ_DEV uint2 bf16x4(f4t o) {
    typedef __bf16 b4t __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(uint2, __builtin_convertvector(o, b4t));
}

// A wave has 16 MT pairs and a WR-th of a tile's rows: WR waves share pairs where there are few.
template <int KT, int D, bool NARROW, int MT, int WR, int NW>
struct ChunkCfg {
    static constexpr bool QUANT = KT == XQ_TYPE_Q8_0 || KT == XQ_TYPE_Q4_0;
    static constexpr int PARTS = QUANT && !NARROW ? 2 : 1;  // f16 parts of a cached value
    static constexpr int QP = NARROW ? 1 : 2;               // f16 parts of Q and of the weights
    static constexpr int EL = KT == XQ_TYPE_F16 ? 8 : KT == XQ_TYPE_Q4_0 ? 32 : 16;  // elements of a 16-byte piece
    static constexpr int PPR = D / EL;                      // pieces per row
    static constexpr int TR = 64;                           // KV rows of a tile (a lane per row)
    static constexpr int RW = TR / WR;                      // of a wave
    static constexpr int RT = RW >= 32 ? 2 : 1;             // 16-row score tiles of a wave at a time
    static constexpr int PIECES = TR * PPR;
    static constexpr int NPT = (PIECES + 64 * NW - 1) / (64 * NW);  // per thread
    static constexpr int RS = 2 * D + 32;                   // image rows, bytes: 8 banks of 64 apart
    static constexpr int PB = TR * RS;                      // one part of K or V
    static constexpr int PW = 16 * MT * (NW / WR);          // pairs of a workgroup
    static constexpr int IMG = 2 * PARTS * PB, MS = D + 4, MERGE = WR > 1 ? NW * 16 * MS * 4 : 0, SMEM = IMG > MERGE ? IMG : MERGE;  // (MS: floats of a merged row)
};

// The workgroup's sequence, KV head, pair tile and part; false where there is none. Workgroups go out in order of their
// numbers, to the eight XCDs in turn: those of one sequence after another, late pair tiles first, which see the most,
// the heads (and, for fewer than eight, neighbouring pair tiles) over the XCDs. So those that run at one time cost
// about the same and a head's rows stay in an XCD's L2. (Sequences over the XCDs instead, eight prompts of up to 777 tokens
// with 78 to 3001 rows before them: 233 us for 129. Two prompts of 8191 tokens are 3 % the slower for it.)
XQ_DEV bool chunk_place(const FaChunkArgs& a, int& b, int& hk, int& pt, int& part) {
    const uint32_t xcd = blockIdx.x & 7u, slot = blockIdx.x >> 3;
    b = (int)a.d_seq.quot(slot);
    const uint32_t in_b = slot - (uint32_t)b * a.d_seq.d, turn = a.d_more.quot(in_b);
    hk = (int)((xcd & ((1u << a.head_shift) - 1u)) + ((in_b - turn * a.d_more.d) << a.head_shift));
    const uint32_t order = (xcd >> a.head_shift) + (turn << (3 - a.head_shift));
    const uint32_t po = a.d_splits.quot(order);
    part = (int)(order - po * (uint32_t)a.splits), pt = a.ptiles - 1 - (int)po;
    return pt >= 0;
}

// One pair tile per segment (few tokens): the rows' tiles of all sequences are dealt out in parts of `per`, sequence after
// sequence, so that a batch of all lengths has parts of one size. From the device's lengths, so a captured graph
// follows them. (Equal numbers of parts per sequence: a decode of 16 chats of up to 6001 rows 37 us; dealt 31.)
struct ChunkDeal {
    uint32_t per;
    int b0;
    uint32_t tiles, parts, upto;  // of sequence b0 + lane; parts up to and with its
    // the tiles that some token of sequence b may see: first one, number
    static XQ_DEV uint32_t tiles_of(const FaChunkArgs& a, int b, uint32_t& first) {
        int held, n_tok, end;
        a.lengths(b, held, n_tok, end);
        first = a.window ? (uint32_t)max(held + 1 - a.window, 0) / 64u : 0u;
        return n_tok ? ((uint32_t)end + 63u) / 64u - min(first, ((uint32_t)end + 63u) / 64u) : 0u;
    }
    XQ_DEV void load(const FaChunkArgs& a, int first, uint32_t before) {
        b0 = first;
        uint32_t t0;
        tiles = b0 + lane_id() < a.B ? tiles_of(a, b0 + lane_id(), t0) : 0u;
        parts = b0 + lane_id() < a.B ? max((tiles + per - 1) / per, 1u) * (uint32_t)a.pg.n_head_kv : 0u;
        upto = before + wave_scan(parts);
    }
    XQ_DEV explicit ChunkDeal(const FaChunkArgs& a) : per(1) {
        uint64_t all = 0;
        for (int b = 0; b < a.B; b += 64) {
            load(a, b, 0);
            all += lane_get(wave_scan(tiles), 63);
        }
        per = uniform((uint32_t)max((all * (uint32_t)a.pg.n_head_kv + a.target - 1) / a.target, (uint64_t)1));
        load(a, 0, 0);
    }
    XQ_DEV uint32_t last() const { return lane_get(upto, 63); }
};

// Rows that some of several tokens see, and those that all do.
struct Range {
    int lo_min = 0x7fffffff, lo_max = 0, hi_min = 0x7fffffff, hi_max = 0;
    XQ_DEV void of(int lo, int hi) {
        if (lo < hi) {  // (what sees nothing asks for no tile)
            lo_min = min(lo_min, lo);
            hi_max = max(hi_max, hi);
        }
        lo_max = max(lo_max, lo);
        hi_min = min(hi_min, hi);
    }
    XQ_DEV void with(const Range& o) {
        lo_min = min(lo_min, o.lo_min), lo_max = max(lo_max, o.lo_max);
        hi_min = min(hi_min, o.hi_min), hi_max = max(hi_max, o.hi_max);
    }
    XQ_DEV void wave() {  // over its lanes, in scalar registers
#pragma unroll
        for (int s = 1; s < 64; s *= 2) with(Range{__shfl_xor(lo_min, s), __shfl_xor(lo_max, s), __shfl_xor(hi_min, s), __shfl_xor(hi_max, s)});
        lo_min = (int)uniform((uint32_t)lo_min), lo_max = (int)uniform((uint32_t)lo_max);
        hi_min = (int)uniform((uint32_t)hi_min), hi_max = (int)uniform((uint32_t)hi_max);
    }
    template <int NW>
    XQ_DEV Range group(int (*lds)[NW], int wave) const {  // over the workgroup's waves
        if (lane_id() == 0) lds[0][wave] = lo_min, lds[1][wave] = lo_max, lds[2][wave] = hi_min, lds[3][wave] = hi_max;
        __syncthreads();
        Range r;
#pragma unroll
        for (int i = 0; i < NW; ++i) r.with(Range{lds[0][i], lds[1][i], lds[2][i], lds[3][i]});
        return r;
    }
};

// The tiles of a workgroup's part of what its pairs see (below 2^25 tiles, up to 64 parts).
template <int TR>
XQ_DEV void chunk_tiles(const FaChunkArgs& a, const Range& r, int part, uint32_t& t_first, uint32_t& t_last) {
    const uint32_t tile0 = r.lo_min < r.hi_max ? (uint32_t)r.lo_min / TR : 0u;
    const uint32_t tiles = r.lo_min < r.hi_max ? ((uint32_t)r.hi_max + TR - 1) / TR - tile0 : 0u;
    t_first = tile0 + uniform(a.d_splits.quot(tiles * (uint32_t)part));
    t_last = part + 1 == a.splits ? tile0 + tiles : tile0 + uniform(a.d_splits.quot(tiles * (uint32_t)(part + 1)));
}

template <int KT, int D, bool NARROW, bool BIASED, int MT, int WR, int NW>
__global__ __launch_bounds__(64 * NW, 2) void fa_chunk_kernel(FaChunkArgs a) {
    static_assert(MT == 1 || WR == 1);
    using C = ChunkCfg<KT, D, NARROW, MT, WR, NW>;
    constexpr int PARTS = C::PARTS, QP = C::QP, NB = D / 32, ND = D / 16, NPT = C::NPT, PPR = C::PPR, PW = C::PW, TR = C::TR, RT = C::RT;
    constexpr bool QUANT = C::QUANT, BY_V = PARTS == 2;
    constexpr int KC = PARTS == 2 ? 2 : 4, VC = PARTS == 2 ? 2 : 4;  // K chunks, V columns read at once
    __shared__ __attribute__((aligned(16))) uint8_t img[C::SMEM];
    uint8_t* const imgK = img;
    uint8_t* const imgV = img + PARTS * C::PB;
    __shared__ float sM[WR > 1 ? NW : 1][16], sL[WR > 1 ? NW : 1][16];
    __shared__ __attribute__((aligned(16))) int sEk[PARTS == 2 ? TR : 4], sEv[PARTS == 2 ? TR : 4];
    __shared__ unsigned long long sBad[2];
    __shared__ int sRange[4][NW];
    const int lane = lane_id(), wave = wave_id(), tid = threadIdx.x, lr = lane & 15, lg = lane >> 4;
    const int r0 = tid / PPR, c0 = tid % PPR;  // row and piece of a tile that this thread brings

    int b, hk, pt = 0, part;
    int n_parts = a.splits;
    int64_t piece;
    uint32_t dealt = 0;  // its tiles of a part, or 0
    constexpr bool FEW = NW == 4;
    if (FEW && a.target) {
        ChunkDeal d(a);
        while (blockIdx.x >= d.last() && d.b0 + 64 < a.B) d.load(a, d.b0 + 64, d.last());
        if (blockIdx.x >= d.last()) return;
        const int sl = __builtin_ctzll(__builtin_amdgcn_ballot_w64(blockIdx.x < d.upto));
        const uint32_t mine = lane_get(d.parts, sl), in_b = blockIdx.x - (lane_get(d.upto, sl) - mine), of_head = mine / (uint32_t)a.pg.n_head_kv;
        b = d.b0 + sl;
        hk = (int)uniform(in_b / of_head), part = (int)(in_b - (uint32_t)hk * of_head);
        n_parts = (int)of_head;
        piece = blockIdx.x;
        dealt = d.per;
    } else {
        if (!chunk_place(a, b, hk, pt, part)) return;
        piece = ((int64_t)(b * a.pg.n_head_kv + hk) * a.ptiles + pt) * a.splits + part;
    }
    int held, n_tok, end;
    a.lengths(b, held, n_tok, end);
    const int n_pairs = n_tok * a.G;
    if (pt * PW >= n_pairs) return;
    const int wp = wave / WR, row_first = wave % WR * C::RW;  // the wave's pairs, and rows of a tile
    const int p0 = pt * PW + wp * 16 * MT;

    int tok[MT], lo[MT], hi[MT], at[MT];
    float slope[MT];
    Range wr;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int p = min(p0 + 16 * m + lr, n_pairs - 1);
        tok[m] = (int)a.d_g.quot((uint32_t)p);
        a.range(b, tok[m], held, end, at[m], lo[m], hi[m]);
        slope[m] = BIASED ? a.slope(hk * a.G + p - tok[m] * a.G) : 0.0f;
        wr.of(lo[m], hi[m]);
    }
    wr.wave();
    if (tid < 2) sBad[tid] = 0;
    const Range wg = wr.group<NW>(sRange, wave);
    uint32_t t_first, t_last;
    if (FEW && dealt) {
        uint32_t t0;
        const uint32_t tiles = ChunkDeal::tiles_of(a, b, t0);
        const bool any = wg.lo_min < wg.hi_max;
        t_first = max(uniform(t0 + (uint32_t)part * dealt), any ? (uint32_t)wg.lo_min / TR : 0u);
        t_last = any ? min(uniform(t0 + min((uint32_t)(part + 1) * dealt, tiles)), ((uint32_t)wg.hi_max + TR - 1) / TR) : t_first;
    } else {
        chunk_tiles<TR>(a, wg, part, t_first, t_last);
    }

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

    for (uint32_t t = t_first; t < t_last; ++t) {
        const int first = (int)(t * TR);
        // where some pair of the workgroup does not see all rows, non-finite values stay out of the image that all share
        const bool clean = first < wg.lo_max || first + TR > wg.hi_min;
        __syncthreads();  // the image is free, the flags are zero
        commit(t, clean);
        __syncthreads();
        const uint64_t now = valid;
        if (t + 1 < t_last) {
            fetch(page, in);
            valid = __builtin_amdgcn_ballot_w64(page < (uint32_t)a.pg.n_pages);
            lookup(t + 2, page, in);
        }
        if (tid == 0) sBad[(t + 1) & 1] = 0;
        if (p0 >= n_pairs || first >= wr.hi_max || first + TR <= wr.lo_min) continue;  // (a wave without pairs that see the tile)

        // which of the tile's rows each pair sees
        const bool careful = first < wr.lo_max || first + TR > wr.hi_min || now != ~0ull;
        uint64_t sees[MT];
        if (careful || clean) {
#pragma unroll
            for (int m = 0; m < MT; ++m) sees[m] = tile_rows(first, lo[m], hi[m]) & now;
        }
#pragma unroll 1
        for (int sub = 0; sub < C::RW / (16 * RT); ++sub) {
            const int row0 = row_first + 16 * RT * sub;
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
                            if (a.cap > 0.0f) x = a.cap * capped_tanh(x * a.inv_cap);
                            x = less_distance(x, slope[m], first + row0 + 16 * r + 4 * lg + i, at[m]);
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
                if constexpr (RT == 2)
                    o = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_shufflevector(x[0], x[RT - 1], 0, 1, 2, 3, 4, 5, 6, 7),
                                                              __builtin_shufflevector(p[0], p[RT - 1], 0, 1, 2, 3, 4, 5, 6, 7), o, 0, 0, 0);
                else
                    o = __builtin_amdgcn_mfma_f32_16x16x16f16(x[0], p[0], o, 0, 0, 0);
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
        // the values that the image was cleaned of, to the pairs that see them (all of a wave's may)
        if (clean) {
            uint64_t bad = sBad[t & 1];
            if constexpr (WR > 1) bad &= (~0ull >> (64 - C::RW)) << row_first;
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
    auto emit = [&](int p, int d, f4t o, float mm, float l, bool first) {  // pair p, dims d..d+3
        const int tk = (int)a.d_g.quot((uint32_t)p), h = hk * a.G + p - tk * a.G;
        if (n_parts > 1) {
            const int64_t y = piece * PW + (p - pt * PW);
            *(f4t*)(a.part_o + y * D + d) = o;
            if (first) a.part_ml[y] = make_float2(mm, l);
            return;
        }
        o *= l == 0.0f ? 0.0f : 1.0f / l;
        uint8_t* y = a.dst + b * a.d_nb3 + tk * a.d_nb2 + h * a.d_nb1;
        if constexpr (NARROW) *(uint2*)(y + 2 * d) = bf16x4(o);
        else *(f4t*)(y + 4 * d) = o;
        if (first && a.lse) a.lse[((int64_t)b * a.n_q + tk) * a.H + h] = l == 0.0f ? -INFINITY : (mm + kOff) * kLn2 + logf(l);
    };
#pragma unroll
    for (int m = 0; m < MT; ++m) l_run[m] = across_rows_sum(l_run[m]);
    if constexpr (WR > 1) {
        if (lg == 0) {
            sM[wave][lr] = m_run[0];
            sL[wave][lr] = l_run[0];
        }
        __syncthreads();  // the last tile is read, the states are there
        float* const mg = (float*)img;
        // the waves of a pair group bring their sums to their largest reference
        auto largest = [&](int w0, int q) {
            float x = sM[w0][q];
#pragma unroll
            for (int i = 1; i < WR; ++i) x = fmaxf(x, sM[w0 + i][q]);
            return x;
        };
        const float f = m_run[0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run[0] - largest(wp * WR, lr));
#pragma unroll
        for (int n = 0; n < ND; ++n) *(f4t*)(mg + (16 * wave + lr) * C::MS + 16 * n + 4 * lg) = acc[0][n] * f;
        __syncthreads();
        for (int i = tid; i < PW * D / 4; i += 64 * NW) {
            const int q = i / (D / 4), d = 4 * (i % (D / 4)), w0 = q / 16 * WR;
            if (pt * PW + q >= n_pairs) continue;
            const float mm = largest(w0, q % 16);
            float l = 0.0f;
            f4t o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int x = w0; x < w0 + WR; ++x) {
                // (a wave without a reference: its sum is 0, or NaN by a NaN score)
                l = fmaf(sL[x][q % 16], sM[x][q % 16] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sM[x][q % 16] - mm), l);
                o += *(const f4t*)(mg + (16 * x + q % 16) * C::MS + d);
            }
            emit(pt * PW + q, d, o, mm, l, d == 0);
        }
    } else {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            if (p0 + 16 * m + lr >= n_pairs) continue;
#pragma unroll
            for (int n = 0; n < ND; ++n) emit(p0 + 16 * m + lr, 16 * n + 4 * lg, acc[m][n], m_run[m], l_run[m], n == 0 && lg == 0);
        }
    }
}

// Joins the parts of each row (sequence, token, head). NWR waves a row: D / 4 lanes read a part's dims, NG parts at a time and
// four of those in flight, each group of lanes with a running reference of its own.
template <int D, bool NARROW, int NWR>
__global__ __launch_bounds__(256) void fa_chunk_join(FaChunkArgs a, uint32_t rows, int32_t PW) {
    constexpr int L = D / 4, NG = 64 * NWR / L, UN = 4, RB = 4 / NWR;
    __shared__ __attribute__((aligned(16))) float sO[RB][NG][D], sM[RB][NG], sL[RB][NG];
    const int rb = RB == 1 ? 0 : wave_id(), tid = threadIdx.x % (64 * NWR);
    const uint32_t row = uniform(blockIdx.x * RB + rb);
    const bool real = row < rows;
    const uint32_t bt = a.d_h.quot(real ? row : 0u), h = (real ? row : 0u) - bt * (uint32_t)a.H;
    const uint32_t b = a.d_q.quot(bt), t = bt - b * (uint32_t)a.n_q;
    int held, n_tok, end;
    a.lengths((int)b, held, n_tok, end);
    const uint32_t hk = a.d_g.quot(h), pair = t * (uint32_t)a.G + h - hk * (uint32_t)a.G, pt = pair / (uint32_t)PW;
    int n_parts = a.splits;
    int64_t piece = ((int64_t)(b * a.pg.n_head_kv + hk) * a.ptiles + pt) * a.splits;
    if (a.target) {
        ChunkDeal deal(a);
        while ((uint32_t)deal.b0 + 64 <= b) deal.load(a, deal.b0 + 64, deal.last());
        const int sl = (int)b - deal.b0;
        const uint32_t mine = lane_get(deal.parts, sl);
        n_parts = (int)(mine / (uint32_t)a.pg.n_head_kv);
        piece = (int64_t)(lane_get(deal.upto, sl) - mine) + hk * n_parts;
    }
    const bool on = real && (int)t < n_tok && n_parts > 1;  // (one part: its workgroup has written the row)
    const int64_t y0 = piece * PW + (pair - pt * PW);
    const int g = tid / L, d = 4 * (tid % L);
    f4t o = {0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    for (int s0 = g; on && s0 < n_parts; s0 += NG * UN) {
        f4t y[UN];
        float2 ml[UN];
#pragma unroll
        for (int i = 0; i < UN; ++i) {
            const int64_t at = y0 + (int64_t)min(s0 + NG * i, n_parts - 1) * PW;
            ml[i] = a.part_ml[at];
            y[i] = *(const f4t*)(a.part_o + at * D + d);
            if (s0 + NG * i >= n_parts) {  // not a part: no weight, and nothing that a product could make NaN
                ml[i] = make_float2(-INFINITY, 0.0f);
                y[i] = f4t{0.0f, 0.0f, 0.0f, 0.0f};
            }
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < UN; ++i) top = fmaxf(top, ml[i].x);
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
        o *= f;
        l *= f;
        m = top;
#pragma unroll
        for (int i = 0; i < UN; ++i) {
            const float w = ml[i].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml[i].x - top);
            l = fmaf(ml[i].y, w, l);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(y[i][e], w, o[e]);
        }
    }
    *(f4t*)&sO[rb][g][d] = o;
    if (d == 0) {
        sM[rb][g] = m;
        sL[rb][g] = l;
    }
    __syncthreads();
    if (!on || g) return;
    float top = sM[rb][0], sum = 0.0f;
#pragma unroll
    for (int i = 1; i < NG; ++i) top = fmaxf(top, sM[rb][i]);
    o = f4t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NG; ++i) {
        const float w = sM[rb][i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sM[rb][i] - top);
        sum = fmaf(sL[rb][i], w, sum);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(sO[rb][i][d + e], w, o[e]);
    }
    o *= sum == 0.0f ? 0.0f : 1.0f / sum;
    uint8_t* y = a.dst + b * a.d_nb3 + t * a.d_nb2 + h * a.d_nb1;
    if constexpr (NARROW) *(uint2*)(y + 2 * d) = bf16x4(o);
    else *(f4t*)(y + 4 * d) = o;
    if (a.lse && d == 0) a.lse[(int64_t)bt * a.H + h] = sum == 0.0f ? -INFINITY : (top + kOff) * kLn2 + logf(sum);
}

// ---------------------------------------------------------------- host

// f(KT, D, NARROW, BIASED) of the call
template <typename F>
static void chunk_variant(int kt, int64_t D, bool narrow, bool biased, F f) {
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

// The form, parts and workspace of a call: of its shapes alone.
struct ChunkPlan {
    int32_t form, pw, ptiles, splits;
    uint32_t head_shift, target;
    int64_t more, per_seq, wgs;
    size_t ml_at, bytes;
};
static ChunkPlan chunk_plan(const xq_tensor* q, const xq_kv_pages* c) {
    ChunkPlan P{};
    const int64_t D = q->ne[0], Hkv = c->k.ne[2], B = q->ne[3], pairs = q->ne[1] * (q->ne[2] / Hkv);
    // As many waves share a tile's rows as the pairs leave without: all four waves on one pair group's 16 rows each
    // (decode of 16 chats of fp8 rows 37 us, with three waves idle 45), up to 64 pairs a wave for each 16; above, eight waves
    // with all pairs that the registers hold (32 each of D 128, 16 of 256), for a tile staged is then used most.
    P.form = pairs <= 16 ? 0 : pairs <= 32 ? 1 : pairs <= 64 ? 2 : 3;
    const int64_t segs = B * Hkv, tiles = cdiv((int64_t)c->table_cols * c->k.ne[1], 64);
    const auto pw = [&](int form) { return form < 3 ? 16 << form : D == 128 ? 256 : 128; };
    // Smaller ones where parts of a tile each would not be one for each CU (us by this rule and without: 17 f32 tokens on 500 q8_0
    // rows of 256 18.7 and 20.6; 200 bf16 tokens alone, f16 rows of 128, 14.1 and 18.3; 64 on 2000 f16 rows 18.5 and 18.7).
    while (P.form > 0 && segs * cdiv(pairs, pw(P.form)) * tiles < 256) --P.form;
    P.pw = pw(P.form);
    P.ptiles = (int32_t)cdiv(pairs, P.pw);
    const int64_t base = segs * P.ptiles;
    // A part costs its workgroup a start and a state written (131 KB of 256 pairs of 128): one part for each CU (512 tokens on
    // 4096 rows: 68 us, with two 81), of a tile at least.
    int64_t splits = cdiv(256, base);
    if (splits > tiles) splits = tiles;
    if (splits > 64) splits = 64;
    P.splits = (int32_t)(splits < 1 ? 1 : splits);
    if (P.form < 3 && P.ptiles == 1) {
        // two workgroups for each CU; one of 140 KB of LDS (f32 beside quantized rows of 256)
        const bool big = D == 256 && q->type == XQ_TYPE_F32 && (c->k.type == XQ_TYPE_Q8_0 || c->k.type == XQ_TYPE_Q4_0);
        const int64_t target = big ? 256 : 512;
        if (tiles > 1 && segs < 2 * target) P.target = (uint32_t)target;
    }
    P.head_shift = Hkv % 8 == 0 ? 3 : Hkv % 4 == 0 ? 2 : Hkv % 2 == 0 ? 1 : 0;
    P.more = Hkv >> P.head_shift;
    P.per_seq = P.more * cdiv((int64_t)P.ptiles * P.splits, 8 >> P.head_shift);
    P.wgs = 8 * B * P.per_seq;
    if (P.target) P.wgs = P.target + segs;
    if (P.splits > 1 || P.target) {
        const size_t rows = (size_t)(P.target ? P.wgs : base * P.splits) * P.pw;
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
    a.ptiles = P.ptiles, a.splits = P.splits, a.target = P.target;
    a.head_shift = P.head_shift;
    a.d_seq = UDivFlat((uint32_t)P.per_seq), a.d_more = UDivFlat((uint32_t)P.more), a.d_splits = UDivFlat((uint32_t)P.splits);
    a.d_h = UDivFlat((uint32_t)a.H), a.d_q = UDivFlat((uint32_t)a.n_q);
    a.part_o = (float*)workspace, a.part_ml = (float2*)((uint8_t*)workspace + P.ml_at);
    const bool biased = a.cap > 0.0f || a.max_bias > 0.0f;
    hipStream_t s = (hipStream_t)stream;
    chunk_variant(cache->k.type, q->ne[0], q->type == XQ_TYPE_BF16, biased, [&](auto k, auto d, auto nar, auto bi) {
        constexpr int KT = decltype(k)::value, D = decltype(d)::value;
        constexpr bool NARROW = decltype(nar)::value, BIASED = decltype(bi)::value;
        const dim3 grid((uint32_t)P.wgs);
        switch (P.form) {
        case 0: launch("fa_chunk", fa_chunk_kernel<KT, D, NARROW, BIASED, 1, 4, 4>, grid, dim3(256), s, a); break;
        case 1: launch("fa_chunk", fa_chunk_kernel<KT, D, NARROW, BIASED, 1, 2, 4>, grid, dim3(256), s, a); break;
        case 2: launch("fa_chunk", fa_chunk_kernel<KT, D, NARROW, BIASED, 1, 1, 4>, grid, dim3(256), s, a); break;
        default: launch("fa_chunk", fa_chunk_kernel<KT, D, NARROW, BIASED, D == 128 ? 2 : 1, 1, 8>, grid, dim3(512), s, a); break;
        }
        if (P.splits > 1 || P.target) {
            const uint32_t rows = (uint32_t)((int64_t)a.B * a.n_q * a.H);
            if (rows <= 2048) launch("fa_chunk_join", fa_chunk_join<D, NARROW, 4>, dim3(rows), dim3(256), s, a, rows, P.pw);
            else launch("fa_chunk_join", fa_chunk_join<D, NARROW, 1>, dim3((rows + 3) / 4), dim3(256), s, a, rows, P.pw);
        }
    });
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return failf(XQ_ERR_HIP, "fa_chunk launch: %s", hipGetErrorString(e));
    return done_ok();
}

}  // extern "C"
