// xq_fa_tree.hip — attention of drafted tokens (a tree, a chain, one token) over the paged cache.
//
// Pair p of a KV head is (token p / G, query head p % G of the group): all pairs of a sequence
// and KV head read the same rows, so one workgroup takes up to 16..256 of them and a row leaves
// HBM once. With x = scale log2(e) q.k over the rows that a pair sees and any m near their
// maximum,
//   O = sum_r 2^(x_r - m) v_r / sum_r 2^(x_r - m),    lse = (m + log2 sum) / log2(e):
// the sums run over the rows tile by tile, and sums with another m join by the factor 2^(m' - m).
//
// A tile is 64 rows. Its pieces (16 bytes a thread) are asked for one tile ahead into registers,
// become f16 in an LDS image [row][D], and go through 16x16x32 matrix products: scores as
// K Q^T (a lane then holds four rows of one pair, as the second product wants its weights),
// O^T as V^T P^T with V's columns read transposed from the image. The visible own rows are a
// 64-bit ancestor mask per token, formed by pointer doubling in the tiles that hold own rows;
// all other tiles carry no mask. A sequence's tiles are dealt to a fixed number of workgroups
// (SeqWork, Deal: from the device's rows and token counts, so a captured graph follows them); a
// segment that several workgroups shared leaves parts that fa_tree_join adds up.
//
// Bound by: HBM while few pairs share a row (decode of 32 x up to 8000 f16 rows, 16/8 heads of
// 128, 281 MB, two input sets in turn: 61 us, 4.6 TB/s of the 4.9 of a large copy); vector issue (conversion, softmax) between;
// matrix and vector issue together at 256 pairs (64 tokens, 4 x 32768 f16 rows, 32/8 heads, 541 MB and 138 GFLOP: 184 us,
// 2.9 TB/s and 0.75 PFLOP/s of the 1.22 of a large f16 matrix product). A second LDS image, so that
// one barrier per tile is enough, gave nothing there (188 us for 188; f32 Q 102 for 92), nor did
// wave priorities that hold the waves of a SIMD apart (188). Small calls cost 14 us: two launches
// and the five dependent reads (arguments, rows, table with Q, K with V, parts) of a lone tile.
//
// Roundings: scores, maxima, sums, accumulators f32. The matrix cores take f16 operands: BF16 Q
// goes in exactly (8 bits, scaled into range by a power of two per row), F16 and E5M2 rows
// exactly; beside BF16 Q, d * q of q8_0 / q4_0 rows and the weights are rounded to f16's 11 bits
// (2^-11 relative each, below the 2^-8 of the bf16 result, for half or a third of the products;
// d * q below f16's normal range is exact, as d is a multiple of 2^-24);
// beside F32 Q every operand is a high and a low f16, 22 bits. f16's subnormal step, 2^-24, is
// what a small operand loses: the powers of two that bring Q's rows, block scales and weights into
// range set how far below the largest that begins.
#include <type_traits>

#include "xq_kv_codec.h"
#include "xq_paged.h"

namespace xq {

constexpr int kTreeMax = 64;  // drafted tokens of a sequence: one 64-bit ancestor mask each

struct TreeArgs {
    const uint8_t* q;
    int64_t q_nb1, q_nb2, q_nb3;  // token, head, sequence
    uint8_t* dst;
    int64_t d_nb1, d_nb2, d_nb3;  // head, token, sequence
    float* lse;
    PagesView pg;
    const int32_t* parents;
    const int32_t* n_tok;
    int32_t n_q, H, G, B;
    float scale;
    uint32_t k_page, k_row, v_page, v_row;  // strides, below 2^32
    UDivFlat d_g, d_wgs, d_h, d_q;  // by the group, the workgroups, the heads, the tokens
    int32_t max_ptiles;       // pair tiles of a sequence with n_q tokens
    int32_t part_pairs;       // pairs of a part
    float* part_o;            // [parts][part_pairs][D]
    float2* part_ml;          // [parts][part_pairs] maximum, sum
};

typedef _Float16 h2t __attribute__((ext_vector_type(2)));
typedef _Float16 h4t __attribute__((ext_vector_type(4)));
typedef _Float16 h8t __attribute__((ext_vector_type(8)));
typedef float f4t __attribute__((ext_vector_type(4)));
typedef uint32_t u4t __attribute__((ext_vector_type(4)));
typedef uint32_t u4any __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t u4dw __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16any __attribute__((aligned(1)));
typedef uint32_t u4half __attribute__((ext_vector_type(4), aligned(2)));
typedef float f4el __attribute__((ext_vector_type(4), aligned(4)));

constexpr float kTreeLog2e = 1.4426950408889634f, kTreeLn2 = 0.6931471805599453f;
constexpr float kTreeLazy = 8.0f;      // base-2 headroom before the running maximum moves
constexpr float kTreeOff = -7.0f;      // weights are 2^(x - max + 7), in (0, 2^15]: f16 keeps small ones normal
constexpr float kTreeHigh = 6.0f;      // and beside f32 Q the largest lies above 2^12 (SCALED, with its block scale: 2^11):
                                       // the reference stays this far below the maximum it was taken from, so that
                                       // a weight's two parts are off by 2^-37 of the largest, or 2^-22 of itself

template <int KT, int D, bool NARROW, int MT, int WR, int NW>
struct TreeCfg {
    static constexpr bool QUANT = KT == XQ_TYPE_Q8_0 || KT == XQ_TYPE_Q4_0;
    // f32 Q on quantized K and V. Where few pairs share a row: the image holds the integers (exact
    // in f16), the block scales join in f32 (scores, and weights before their split in two).
    // That takes 5 vector instructions per weight and block, so where the waves share
    // the pairs the image holds d * q in two f16 parts instead, at three products for two.
    static constexpr bool SCALED = QUANT && !NARROW && WR > 1;
    static constexpr int PARTS = QUANT && !NARROW && !SCALED ? 2 : 1;       // f16 parts of a cached value
    static constexpr int QP = NARROW ? 1 : 2;                               // f16 parts of Q and of the weights
    // The weights become f16 parts times a power of two of V's row, that of its largest block scale. The
    // reference that keeps them in f16's range is then a maximum of x plus that power over the rows that
    // the pair sees: a row of which it sees nothing, or next to nothing, costs the others no bits,
    // whatever its scales.
    static constexpr bool BY_V = PARTS == 2 || SCALED;
    static constexpr int EL = KT == XQ_TYPE_F16 ? 8 : KT == XQ_TYPE_Q4_0 ? 32 : 16;  // elements of a 16-byte piece
    static constexpr int PPR = D / EL;                                      // pieces per row
    static constexpr int TR = 64;                                           // KV rows of a tile (a lane per row)
    static constexpr int RW = TR / WR;                                      // of a wave
    static constexpr int RT = RW >= 32 ? 2 : 1;                             // 16-row score tiles of a wave at a time
    static constexpr int PIECES = TR * PPR;                                 // of a tile and tensor
    static constexpr int NPT = (PIECES + 64 * NW - 1) / (64 * NW);          // per thread
    static constexpr int RS = 2 * D + 32;                                   // image rows, bytes: 8 banks of 64 apart, so that 16 rows' operand reads meet no bank twice at a time
    static constexpr int PB = TR * RS;                                      // one part of K or V
    static constexpr int IMG = 2 * PARTS * PB;
    static constexpr int PW = 16 * MT * (NW / WR);                          // pairs of a workgroup
    static constexpr int MS = D + 4;                                        // merge row stride, floats
    static constexpr int MERGE = WR > 1 ? NW * 16 * MS * 4 : 0;
    static constexpr int SMEM = IMG > MERGE ? IMG : MERGE;
    // Waves per SIMD: two (256 registers each); three for the E5M2 and Q4_0 forms that fit 168 registers
    // (32 fp8 chats of up to 8000 rows: 32.2 us, with two 32.5; 32 q4_0 chats 34.8, 37.9; 4 x 32000 q4_0
    // rows 52, 62). 32 f16 chats, whose form spills there, take 70.1 with three, 59.4 with two. Q8_0's form
    // fits too (163 registers) and is left at two: three take 47.1 for 49.3 (32 chats), 73.5 for 84.3
    // (4 x 32000 rows).
    // Spills: 29 of the 72 forms keep 3 to 74 registers in scratch, some of them read in the tile loop:
    // of f32 Q, all at head dim 256 but the two of one wave per SIMD (139 KB of LDS), and those of 128
    // and 256 pairs at 128; of bf16 Q, f16 rows at 256, E5M2 and Q8_0 rows of 64 pairs at 256, f16 rows of
    // 128 pairs at 128.
    static constexpr int WAVES = NARROW && D == 128 && WR == 4 && (KT == XQ_TYPE_E5M2 || KT == XQ_TYPE_Q4_0) ? 3 : 2;
    // workgroups that a CU holds
    static constexpr int BY_LDS = 160 * 1024 / (SMEM + 2048), BY_WAVES = WAVES * 4 / NW;
    static constexpr int PER_CU = BY_LDS < BY_WAVES ? BY_LDS : BY_WAVES;
};

// Element d of a record in f32 (rows with a non-finite value only).
template <int KT>
XQ_DEV float kv_element(const uint8_t* rec, int d) {
    if constexpr (KT == XQ_TYPE_F16) {
        return f16_bits_to_f32(*(const u16any*)(rec + 2 * d));
    } else if constexpr (KT == XQ_TYPE_E5M2) {
        return e5m2_to_f32(rec[d]);
    } else if constexpr (KT == XQ_TYPE_Q8_0) {
        const uint8_t* b = rec + d / 32 * 34;
        return f16_bits_to_f32(*(const u16any*)b) * (float)(int8_t)b[2 + d % 32];
    } else {
        const uint8_t* b = rec + d / 32 * 18;
        const int n = d % 32 < 16 ? b[2 + d % 16] & 15 : b[2 + d % 16] >> 4;
        return f16_bits_to_f32(*(const u16any*)b) * (float)(n - 8);
    }
}

XQ_DEV float across_rows_max(float x) {  // over lanes l, l^16, l^32, l^48
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
XQ_DEV float across_rows_sum(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}

// Nonzero halves (0x8000 each) of w that are Inf or NaN.
XQ_DEV uint32_t bad_halves(uint32_t w) { return ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u; }
XQ_DEV uint32_t without_bad(uint32_t w) { return w & ~((bad_halves(w) >> 15) * 0xffffu); }

// 16 bytes of a record as f16 pairs, exact: NW words. q8_0 / q4_0: the integers.
template <int KT, int NW>
XQ_DEV void piece_f16(const u4t raw, uint32_t (&o)[NW]) {
    if constexpr (KT == XQ_TYPE_F16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = raw[i];
    } else if constexpr (KT == XQ_TYPE_E5M2) {  // byte b -> f16 bits b << 8
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o[2 * i] = __builtin_amdgcn_perm(raw[i], raw[i], 0x010c000cu);
            o[2 * i + 1] = __builtin_amdgcn_perm(raw[i], raw[i], 0x030c020cu);
        }
    } else if constexpr (KT == XQ_TYPE_Q8_0) {  // (1024 + (q ^ 0x80)) - 1152
        const h2t k = {(_Float16)-1152.0f, (_Float16)-1152.0f};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = raw[i] ^ 0x80808080u;
            o[2 * i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2t, __builtin_amdgcn_perm(0x64646464u, w, 0x05010500u)) + k);
            o[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2t, __builtin_amdgcn_perm(0x64646464u, w, 0x05030502u)) + k);
        }
    } else {  // low nibbles n (elements 0..15), then high ones: (1024 + n) - 1032
        const h2t k = {(_Float16)-1032.0f, (_Float16)-1032.0f};
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t w = h ? (raw[i] >> 4) & 0x0f0f0f0fu : raw[i] & 0x0f0f0f0fu;
                o[8 * h + 2 * i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2t, __builtin_amdgcn_perm(0x64646464u, w, 0x05010500u)) + k);
                o[8 * h + 2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2t, __builtin_amdgcn_perm(0x64646464u, w, 0x05030502u)) + k);
            }
    }
}

// Four rows of one column (rows 4lg.. of the 16 at p's row, column lr of 16) from the image.
XQ_DEV uint2 column4(const uint8_t* p) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4 lds_s4;
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(__attribute__((address_space(3))) uint8_t*)p));
}

// Wait states between a group of matrix products and the first vector instruction that reads
// them (eight on gfx950); nothing moves across this. The compiler inserts such waits itself, but AMD
// clang 22 (ROCm 7.2) once did so an instruction late: with the accumulators in AGPRs, the last
// score product ended a block and a branch round the masking led to
//     v_accvgpr_read_b32 v2, a27 / s_nop 5 / v_accvgpr_read_b32 v3, a26 ...
// where a27 was the product's, so that one register in four held the score from before it. In the
// present forms the compiler's own waits reach eight without this.
XQ_DEV void products_done() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 7\n\ts_nop 1");
    __builtin_amdgcn_sched_barrier(0);
}

// A segment is one (sequence, KV head, pair tile); its units of work are its row tiles after
// kStart units that stand for what a workgroup spends on it before its first tile (three
// dependent loads, Q, and the state written at the end: the time of two to four tiles).
// Dealing by tiles alone (0): 32 fp8 chats 37.7 us against 32.4, 16 sequences of 25 tokens 79
// against 66; 2, 4 and 5 are within 1 % of 3 over 40 calls of all sizes.
constexpr uint32_t kStart = 3;

// Work of sequence b: its rows, tokens, row tiles, pair tiles and units.
struct SeqWork {
    int32_t held, n_tok, end;
    uint32_t tiles, ptiles, units;
};
template <int PW, int TR>
XQ_DEV SeqWork seq_work(const TreeArgs& a, int b) {
    SeqWork s;
    s.held = min(max(a.pg.rows[b], 0), a.pg.row_limit);
    s.n_tok = a.n_tok ? min(max(a.n_tok[b], 0), a.n_q) : a.n_q;
    s.end = (int32_t)min((uint32_t)s.held + (uint32_t)s.n_tok, (uint32_t)a.pg.row_limit);
    s.tiles = s.n_tok ? ((uint32_t)s.end + TR - 1) / TR : 0u;
    s.ptiles = (uint32_t)(s.n_tok * a.G + PW - 1) / PW;
    s.units = s.tiles ? (kStart + s.tiles) * s.ptiles * (uint32_t)a.pg.n_head_kv : 0u;
    return s;
}

// A number that every lane has, in a scalar register: what is formed from it stays scalar.
XQ_DEV uint32_t uniform(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }

// The units of all sequences dealt to the workgroups in order, `per` each.
struct Deal {
    uint32_t units, per;
    XQ_DEV Deal(uint32_t n, const UDivFlat& d_wgs) : units(n), per(uniform(max(d_wgs.quot(n + d_wgs.d - 1), 1u))) {}
    XQ_DEV uint32_t first(uint32_t w) const { return uniform((uint32_t)min((uint64_t)w * per, (uint64_t)units)); }
    XQ_DEV uint32_t owner(uint32_t u) const { return u / per; }  // the workgroup that has unit u
};

// Inclusive sum over the 64 lanes: inside rows of 16, then from row to row.
template <int CTRL, int ROWS>
XQ_DEV uint32_t dpp_add(uint32_t x) {
    return x + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
XQ_DEV uint32_t wave_scan(uint32_t x) {
    x = dpp_add<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8
    x = dpp_add<0x112, 0xf>(x);
    x = dpp_add<0x114, 0xf>(x);
    x = dpp_add<0x118, 0xf>(x);
    x = dpp_add<0x142, 0xa>(x);  // row_bcast 15 into rows 1 and 3
    return dpp_add<0x143, 0xc>(x);  // row_bcast 31 into rows 2 and 3
}
XQ_DEV uint32_t lane_get(uint32_t x, int l) { return (uint32_t)__builtin_amdgcn_readlane((int)x, l); }

// 64 sequences at a time, a lane each: their work and the units up to and with each.
template <int PW, int TR>
struct SeqChunk {
    int b0;
    uint32_t before, upto;  // units of the sequences before b0; up to this lane's
    SeqWork mine;
    XQ_DEV void load(const TreeArgs& a, int first, uint32_t units_before) {
        b0 = first;
        before = units_before;
        mine = SeqWork{};
        if (b0 + lane_id() < a.B) mine = seq_work<PW, TR>(a, b0 + lane_id());
        upto = before + wave_scan(mine.units);
    }
    XQ_DEV uint32_t last() const { return lane_get(upto, 63); }
    // All sequences' units; the first chunk is loaded after it.
    XQ_DEV uint32_t total(const TreeArgs& a) {
        load(a, 0, 0);
        uint32_t n = last();
        if (a.B > 64) {
            while (b0 + 64 < a.B) {
                load(a, b0 + 64, n);
                n = last();
            }
            load(a, 0, 0);
        }
        return uniform(n);
    }
};

template <int KT, int D, bool NARROW, int MT, int WR, int NW>
__global__ __launch_bounds__(64 * NW, (TreeCfg<KT, D, NARROW, MT, WR, NW>::WAVES)) void fa_tree_kernel(TreeArgs a) {
    using C = TreeCfg<KT, D, NARROW, MT, WR, NW>;
    constexpr int PARTS = C::PARTS, QP = C::QP, NB = D / 32, ND = D / 16, NPT = C::NPT, PPR = C::PPR, PW = C::PW, TR = C::TR, RT = C::RT;
    constexpr bool QUANT = C::QUANT, SCALED = C::SCALED, BY_V = C::BY_V;
    constexpr int KC = PARTS == 2 ? 2 : 4;  // 32-element chunks of K read at once
    constexpr int VC = PARTS == 2 ? 2 : 4;  // 16-element columns of V
    __shared__ __attribute__((aligned(16))) uint8_t img[C::SMEM];
    __shared__ float sM[WR > 1 ? NW : 1][16 * MT], sL[WR > 1 ? NW : 1][16 * MT];
    __shared__ __attribute__((aligned(16))) int sEk[PARTS == 2 ? TR : 4], sEv[PARTS == 2 || SCALED ? TR : 4];
    __shared__ __attribute__((aligned(16))) float sDk[SCALED ? NB : 1][SCALED ? TR : 4], sDv[SCALED ? NB : 1][SCALED ? TR : 4];
    __shared__ unsigned long long sBad[2];
    const int lane = lane_id(), wave = wave_id(), tid = threadIdx.x, lr = lane & 15, lg = lane >> 4;
    const int wr = wave % WR, pg = wave / WR;  // the wave's rows and pairs of a tile
    const int r0 = tid / PPR, c0 = tid % PPR;  // row and piece of a tile that this thread brings (64 NW / PPR rows apart)
    uint8_t* const imgK = img;
    uint8_t* const imgV = img + PARTS * C::PB;

    // every argument the prologue needs, asked for at once: left to their uses, the scalar
    // loads go out one dependent group after another
    asm volatile("" ::"s"(a.pg.rows), "s"(a.n_tok), "s"(a.pg.table), "s"(a.parents), "s"(a.q), "s"(a.pg.k), "s"(a.pg.v), "s"(a.pg.k_head),
                 "s"(a.pg.v_head), "s"(a.q_nb1), "s"(a.q_nb2), "s"(a.q_nb3), "s"(a.pg.table_cols), "s"(a.pg.n_pages), "s"(a.pg.row_limit),
                 "s"(a.pg.n_head_kv), "s"(a.pg.d_page.m), "s"(a.n_q), "s"(a.G), "s"(a.B), "s"(a.scale), "s"(a.k_page), "s"(a.v_row),
                 "s"(a.d_g.m), "s"(a.d_wgs.m));
    const uint32_t w = xcd_remap(blockIdx.x, a.d_wgs.d);
    SeqChunk<PW, TR> seqs;
    const Deal deal(seqs.total(a), a.d_wgs);
    uint32_t u = deal.first(w);
    const uint32_t u_end = deal.first(w + 1);
    while (u < u_end) {
        // ---- the segment (sequence, KV head, pair tile) that unit u belongs to
        while (u >= seqs.last()) seqs.load(a, seqs.b0 + 64, seqs.last());
        const int sl = __builtin_ctzll(__builtin_amdgcn_ballot_w64(u < seqs.upto));
        const int b = seqs.b0 + sl;
        const int held = (int)lane_get((uint32_t)seqs.mine.held, sl), n_tok = (int)lane_get((uint32_t)seqs.mine.n_tok, sl);
        const int end = (int)lane_get((uint32_t)seqs.mine.end, sl);
        const uint32_t tiles = lane_get(seqs.mine.tiles, sl), ptiles = lane_get(seqs.mine.ptiles, sl);
        const uint32_t in_b = u - (lane_get(seqs.upto, sl) - lane_get(seqs.mine.units, sl));
        const uint32_t seg_units = kStart + tiles, seg = uniform(in_b / seg_units), v0 = in_b - seg * seg_units;
        const uint32_t v1 = min(seg_units, v0 + (u_end - u));
        u += v1 - v0;
        if (v1 <= kStart) continue;  // no tile of it
        const uint32_t t_first = max(v0, kStart) - kStart, t_last = v1 - kStart;
        const int hk = (int)uniform(seg / ptiles), pt = (int)(seg - (uint32_t)hk * ptiles);
        const bool whole = t_first == 0 && t_last == tiles;
        const int n_pairs = n_tok * a.G;
        const int p0 = pt * PW + pg * 16 * MT;  // this wave's first pair

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
            // quantized: the fifth dword of each piece's window, and the bytes (0, 2 or 4, in
            // halves, two bits each) that the piece starts into its window
            uint32_t k5[QUANT ? NPT : 1], v5[QUANT ? NPT : 1], shift;
        };
        Raw raw;  // the next tile's pieces, in flight while a tile is computed
        // A quantized piece (16 bytes behind a 2-byte scale in 34- or 18-byte blocks) by whole
        // aligned dwords: 16-byte loads at 2-byte addresses took twice the time of a decode.
        // The window starts at the dword of the block's scale, or (q8_0's second pieces) of the
        // piece; every dword read holds a byte of the two.
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
        auto fetch = [&](Raw& set, uint32_t page, uint32_t in) {
            if constexpr (QUANT) set.shift = 0;
#pragma unroll
            for (int j = 0; j < NPT; ++j) {
                const int r4 = 4 * (r0 + 64 * NW / PPR * j);  // (modulo 64 lanes)
                const uint32_t p = (uint32_t)__builtin_amdgcn_ds_bpermute(r4, (int)page), x = (uint32_t)__builtin_amdgcn_ds_bpermute(r4, (int)in);
                set.k[j] = u4t{0, 0, 0, 0};
                set.v[j] = u4t{0, 0, 0, 0};
                if constexpr (QUANT) set.k5[j] = set.v5[j] = 0u;
                if (p < (uint32_t)a.pg.n_pages && (C::PIECES % (64 * NW) == 0 || tid + 64 * NW * j < C::PIECES)) {
                    const uint8_t* k = kb + (uint64_t)p * a.k_page + (uint64_t)x * a.k_row;
                    const uint8_t* v = vb + (uint64_t)p * a.v_page + (uint64_t)x * a.v_row;
                    if constexpr (QUANT) {
                        set.shift |= window(k, set.k[j], set.k5[j]) << (4 * j) | window(v, set.v[j], set.v5[j]) << (4 * j + 2);
                    } else {
                        set.k[j] = *(const u4any*)(k + 16 * c0);
                        set.v[j] = *(const u4any*)(v + 16 * c0);
                    }
                }
            }
        };
        // raw pieces -> image
        auto put = [&](uint8_t* image, int rs, int part_bytes, const u4t raw, uint32_t d, int r, int c, int* exps, float* scales, bool clean, uint32_t t) {
            constexpr int WORDS = C::EL / 2;
            uint32_t o[WORDS], lo[WORDS];
            piece_f16<KT, WORDS>(raw, o);
            if constexpr (QUANT && NARROW) {
                const uint32_t dd = d | (d << 16);
#pragma unroll
                for (int i = 0; i < WORDS; ++i) o[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2t, o[i]) * __builtin_bit_cast(h2t, dd));
            } else if constexpr (QUANT) {
                // the exponent of the row's largest finite block scale, over the row's PPR (4, 8
                // or 16) lanes
                const float df = f16_bits_to_f32(d);
                int e = (int)((__float_as_uint(df) >> 23) & 255u);
                if (e == 255 || e < 103) e = 103;  // 2^-24, the smallest f16: a zero scale asks for no larger power
                e = max(e, dpp_i<0xB1>(e));
                e = max(e, dpp_i<0x4E>(e));
                if constexpr (PPR >= 8) e = max(e, dpp_i<0x141>(e));
                if constexpr (PPR >= 16) e = max(e, dpp_i<0x140>(e));
                if constexpr (SCALED) {
                    constexpr int PB = 32 / C::EL;  // pieces of a block
                    if (c % PB == 0) scales[(c / PB) * TR + r] = df;
                    if (exps && c == 0) exps[r] = e - 126;  // d 2^-e below 1
                } else {
                    // to [2^7, 2^8); then d q = hi + lo exactly: hi its rounding, lo the remainder
                    // of at most 8 bits
                    e -= 127 + 7;
                    const _Float16 f = (_Float16)ldexpf(df, -e);
                    if (c == 0) exps[r] = e;
#pragma unroll
                    for (int i = 0; i < WORDS; ++i) {
                        const h2t q = __builtin_bit_cast(h2t, o[i]), ff = {f, f};
                        const h2t hi = q * ff;
                        o[i] = __builtin_bit_cast(uint32_t, hi);
                        lo[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(q, ff, -hi));
                    }
                }
            }
            if (!SCALED && clean) {
                uint32_t bad = 0;
#pragma unroll
                for (int i = 0; i < WORDS; ++i) {
                    bad |= bad_halves(o[i]);
                    if constexpr (PARTS == 2) lo[i] &= ~((bad_halves(o[i]) >> 15) * 0xffffu);
                    o[i] = without_bad(o[i]);
                }
                if (bad) {
                    int row = r;
                    asm volatile("" : "+v"(row));  // (its bit is formed here, not kept over the tiles)
                    atomicOr(&sBad[t & 1], 1ull << row);
                }
            }
            uint8_t* y = image + r * rs + c * (2 * C::EL);
#pragma unroll
            for (int i = 0; i < WORDS; i += 4) {
                *(u4t*)(y + 4 * i) = u4t{o[i], o[i + 1], o[i + 2], o[i + 3]};
                if constexpr (PARTS == 2) *(u4t*)(y + part_bytes + 4 * i) = u4t{lo[i], lo[i + 1], lo[i + 2], lo[i + 3]};
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
        auto commit = [&](const Raw& set, uint32_t t) {
            const bool clean = (t + 1) * TR > (uint32_t)held;  // holds rows that only some tokens see
#pragma unroll
            for (int j = 0; j < NPT; ++j) {
                const int r = r0 + 64 * NW / PPR * j, c = c0;
                if (C::PIECES % (64 * NW) && tid + 64 * NW * j >= C::PIECES) break;  // (whole waves: PIECES is a multiple of 64)
                u4t k = set.k[j], v = set.v[j];
                uint32_t dk = 0u, dv = 0u;
                if constexpr (QUANT) {
                    dk = realign(k, set.k5[j], (set.shift >> (4 * j)) & 3u);
                    dv = realign(v, set.v5[j], (set.shift >> (4 * j + 2)) & 3u);
                }
                put(imgK, C::RS, C::PB, k, dk, r, c, SCALED ? nullptr : sEk, &sDk[0][0], false, t);
                put(imgV, C::RS, C::PB, v, dv, r, c, sEv, &sDv[0][0], clean, t);
            }
        };

        uint32_t page, in;
        lookup(t_first, page, in);
        const int32_t up = a.parents && lane < n_tok ? a.parents[(int64_t)b * a.n_q + lane] : lane - 1;

        // ---- Q operands: pair 16m + lr, elements 8lg.. of each 32, times a power of two that
        //      puts the row's largest element in [2^14, 2^15)
        h8t qo[MT][NB][QP];
        float qf[MT];
        int tok[MT];
        {
            float xq[MT][NB][8];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const int p = min(p0 + 16 * m + lr, n_pairs - 1);
                tok[m] = (int)a.d_g.quot((uint32_t)p);
                const uint8_t* q = a.q + b * a.q_nb3 + tok[m] * a.q_nb1 + (hk * a.G + p - tok[m] * a.G) * a.q_nb2;
#pragma unroll
                for (int c = 0; c < NB; ++c) {
                    const int e = 32 * c + 8 * lg;
                    if constexpr (NARROW) {
                        const u4half x = *(const u4half*)(q + 2 * e);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            xq[m][c][2 * i] = __uint_as_float(x[i] << 16);
                            xq[m][c][2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u);
                        }
                    } else {
                        const f4el x = *(const f4el*)(q + 4 * e), y = *(const f4el*)(q + 4 * e + 16);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            xq[m][c][i] = x[i];
                            xq[m][c][4 + i] = y[i];
                        }
                    }
                }
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                float big = 0.0f;
#pragma unroll
                for (int c = 0; c < NB; ++c)
#pragma unroll
                    for (int j = 0; j < 8; ++j) big = fmaxf(big, fabsf(xq[m][c][j]));
                const int lift = 141 - min((int)(__float_as_uint(across_rows_max(big)) >> 23), 254);
                // (a normal number: an unseen score's -inf stays one, and a score of 0 too)
                qf[m] = fminf(fmaxf(ldexpf(fabsf(a.scale), -lift) * kTreeLog2e, 1.17549435e-38f), 3.40282347e38f);
#pragma unroll
                for (int c = 0; c < NB; ++c)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float x = ldexpf(a.scale < 0.0f ? -xq[m][c][j] : xq[m][c][j], lift);
                        const _Float16 hi = (_Float16)x;
                        qo[m][c][0][j] = hi;
                        if constexpr (QP == 2) qo[m][c][1][j] = (_Float16)(x - (float)hi);
                    }
            }
        }
        fetch(raw, page, in);
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
        if (tid < 2) sBad[tid] = 0;

        for (uint32_t t = t_first; t < t_last; ++t) {
            __syncthreads();  // the image is free, the flags are zero
            commit(raw, t);
            __syncthreads();
            const uint64_t now = valid;
            if (t + 1 < t_last) {
                fetch(raw, page, in);
                valid = __builtin_amdgcn_ballot_w64(page < (uint32_t)a.pg.n_pages);
                lookup(t + 2, page, in);
            }
            if (tid == 0) sBad[(t + 1) & 1] = 0;

            // which of the tile's rows each pair sees
            const bool careful = (t + 1) * TR > (uint32_t)held || now != ~0ull;
            uint64_t sees[MT];
            if (careful) {
                // ancestors by doubling: lane i is token i
                const int first = (int)(t * TR);
                uint64_t anc = 0;
                if (first + TR > held) {
                    int32_t p = up >= 0 && up < lane ? up : -1;
                    anc = 1ull << lane;
#pragma unroll
                    for (int d = 0; d < 6; ++d) {
                        const int from = p < 0 ? lane : p;
                        const uint32_t x = (uint32_t)__shfl((int)(uint32_t)anc, from), y = (uint32_t)__shfl((int)(uint32_t)(anc >> 32), from);
                        anc |= ((uint64_t)y << 32) | x;
                        const int32_t q = __shfl(p, from);
                        p = p < 0 ? -1 : q;
                    }
                }
                const int sh = held - first;  // rows of the tile that every token sees, below 0: of the tokens passed
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const uint64_t x = ((uint64_t)(uint32_t)__shfl((int)(uint32_t)(anc >> 32), tok[m]) << 32) | (uint32_t)__shfl((int)(uint32_t)anc, tok[m]);
                    uint64_t s = sh >= 64 ? ~0ull : sh >= 0 ? (x << sh) | ((1ull << sh) - 1) : sh > -64 ? x >> -sh : 0ull;
                    sees[m] = s & now;
                }
            }
#pragma unroll 1
            for (int sub = 0; sub < (p0 < n_pairs ? C::RW / (16 * RT) : 0); ++sub) {  // (a wave without pairs only brings tiles)
                const int row0 = C::RW * wr + 16 * RT * sub;  // the first of the wave's rows at this step
                f4t s[MT][RT];
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int r = 0; r < RT; ++r) s[m][r] = f4t{0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (SCALED) {
                    // a block's integer products, times its scales of the lane's rows
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        const uint8_t* const k = imgK + (row0 + 16 * r + lr) * C::RS + 16 * lg;
#pragma unroll
                        for (int c0 = 0; c0 < NB; c0 += 4) {
                            f4t z[4];
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                const h8t kh = *(const h8t*)(k + 64 * (c0 + c));
                                z[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qo[0][c0 + c][0], f4t{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
                                z[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qo[0][c0 + c][QP - 1], z[c], 0, 0, 0);
                            }
                            products_done();
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                const f4t d = *(const f4t*)&sDk[c0 + c][row0 + 16 * r + 4 * lg];
#pragma unroll
                                for (int i = 0; i < 4; ++i) s[0][r][i] = fmaf(z[c][i], d[i], s[0][r][i]);
                            }
                        }
                    }
                } else {
                // K rows, a batch of chunks at a time: all of its reads before its products
                const uint8_t* const krow = imgK + (row0 + lr) * C::RS + 16 * lg;
#pragma unroll
                for (int c0 = 0; c0 < NB; c0 += KC) {
                    h8t kh[KC][RT], kl[PARTS == 2 ? KC : 1][PARTS == 2 ? RT : 1];
#pragma unroll
                    for (int c = 0; c < KC; ++c)
#pragma unroll
                        for (int r = 0; r < RT; ++r) {
                            const uint8_t* k = krow + 16 * r * C::RS + 64 * (c0 + c);
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
                                s[m][r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[c][r], qo[m][c0 + c][0], s[m][r], 0, 0, 0);
                                if constexpr (QP == 2) s[m][r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[c][r], qo[m][c0 + c][1], s[m][r], 0, 0, 0);
                                if constexpr (PARTS == 2) s[m][r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl[c][r], qo[m][c0 + c][0], s[m][r], 0, 0, 0);
                            }
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
                // the lane's rows are row0 + 16r + 4lg + i; s * qf are base-2 scores
                if constexpr (PARTS == 2) {
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        const int4 e = *(const int4*)(sEk + row0 + 16 * r + 4 * lg);
#pragma unroll
                        for (int m = 0; m < MT; ++m)
                            s[m][r] = f4t{ldexpf(s[m][r][0], e.x), ldexpf(s[m][r][1], e.y), ldexpf(s[m][r][2], e.z), ldexpf(s[m][r][3], e.w)};
                    }
                }
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
                            top[m] = fmaxf(top[m], BY_V ? fmaf(s[m][r][i], qf[m], (float)(i == 0 ? e.x : i == 1 ? e.y : i == 2 ? e.z : e.w)) : s[m][r][i]);
                }
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    if constexpr (!BY_V) top[m] *= qf[m];
                    over |= top[m] > m_run[m] + kTreeLazy;
                }
                if (__builtin_amdgcn_ballot_w64(over)) {
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        const float mt = across_rows_max(top[m]);
                        const float mn = mt > m_run[m] + kTreeLazy ? ceilf(mt) - (QP == 2 ? kTreeHigh : 0.0f) : m_run[m];
                        const float f = mn == m_run[m] ? 1.0f : __builtin_amdgcn_exp2f(m_run[m] - mn);
                        l_run[m] *= f;
#pragma unroll
                        for (int n = 0; n < ND; ++n) acc[m][n] *= f;
                        m_run[m] = mn;
                    }
                }
                // weights
                h4t ph[MT][RT], pl[QP == 2 ? MT : 1][QP == 2 ? RT : 1];
                f4t pw[SCALED ? RT : 1];  // SCALED: the weights, before their block scales
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const float mu = m_run[m] == -INFINITY ? 0.0f : -(m_run[m] + kTreeOff);
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        f4t p;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            p[i] = __builtin_amdgcn_exp2f(fmaf(s[m][r][i], qf[m], mu));
                            l_run[m] += p[i];
                        }
                        if constexpr (SCALED) {
                            pw[r] = p;
                            continue;
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
                    for (int n = 0; n < VC; ++n) {
                        if constexpr (SCALED) {
                            // the weights times the block's scales, as f16 high and low parts
                            if (n % 2 == 0) {
#pragma unroll
                                for (int r = 0; r < RT; ++r) {
                                    const f4t d = *(const f4t*)&sDv[(n0 + n) / 2][row0 + 16 * r + 4 * lg];
                                    f4t w = pw[r] * d;
                                    if (careful) {  // (an unseen row's scale may be anything)
                                        const uint32_t bits = (uint32_t)(sees[0] >> (row0 + 16 * r + 4 * lg));
#pragma unroll
                                        for (int i = 0; i < 4; ++i) w[i] = (bits >> i) & 1u ? w[i] : 0.0f;
                                    }
#pragma unroll
                                    for (int i = 0; i < 4; ++i) {
                                        ph[0][r][i] = (_Float16)w[i];
                                        pl[0][r][i] = (_Float16)(w[i] - (float)ph[0][r][i]);
                                    }
                                }
                            }
                        }
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            product(vh[x][n], ph[m], acc[m][n0 + n]);
                            if constexpr (QP == 2) product(vh[x][n], pl[m], acc[m][n0 + n]);
                            if constexpr (PARTS == 2) product(vl[x][n], ph[m], acc[m][n0 + n]);
                        }
                    }
                }
            }
            products_done();
            // non-finite values of rows that not every token sees: to the tokens that do
            if (!SCALED && careful) {
                uint64_t bad = sBad[t & 1];
                if constexpr (WR > 1) bad &= (~0ull >> (64 - C::RW)) << (C::RW * wr);
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
        if (u < u_end) seqs.load(a, seqs.b0, seqs.before);  // again: not held in registers meanwhile

        // ---- the segment's result, or this workgroup's part of it
        const uint32_t piece = w + (uint32_t)((b * a.pg.n_head_kv + hk) * a.max_ptiles + pt);
        auto emit = [&](int p, int d, f4t o, float mm, float l, bool first) {  // pair p of the segment's tile, dims d..d+3
            if (whole) {
                const int q = pt * PW + p, t = (int)a.d_g.quot((uint32_t)q), h = hk * a.G + q - t * a.G;
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                uint8_t* y = a.dst + b * a.d_nb3 + t * a.d_nb2 + h * a.d_nb1;
                if constexpr (NARROW) {
                    const uint32_t w0 = f32_to_bf16_bits(o[0] * inv) | (f32_to_bf16_bits(o[1] * inv) << 16);
                    const uint32_t w1 = f32_to_bf16_bits(o[2] * inv) | (f32_to_bf16_bits(o[3] * inv) << 16);
                    *(uint2*)(y + 2 * d) = make_uint2(w0, w1);
                } else {
                    *(f4t*)(y + 4 * d) = o * inv;
                }
                if (first && a.lse) a.lse[((int64_t)b * a.n_q + t) * a.H + h] = l == 0.0f ? -INFINITY : (mm + kTreeOff) * kTreeLn2 + logf(l);
            } else {
                const int64_t at = (int64_t)piece * a.part_pairs + p;
                *(f4t*)(a.part_o + at * D + d) = o;
                if (first) a.part_ml[at] = make_float2(mm, l);
            }
        };
        if constexpr (WR > 1) {
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                l_run[m] = across_rows_sum(l_run[m]);
                if (lg == 0) {
                    sM[wave][16 * m + lr] = m_run[m];
                    sL[wave][16 * m + lr] = l_run[m];
                }
            }
            __syncthreads();  // the last tile is read, the states are there
            float* const mg = (float*)img;
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                // the waves of a pair group bring their sums to their largest maximum
                auto largest = [&](int first, int q) {
                    float x = sM[first][q];
#pragma unroll
                    for (int i = 1; i < WR; ++i) x = fmaxf(x, sM[first + i][q]);
                    return x;
                };
                const float top = largest(pg * WR, 16 * m + lr);
                const float f = m_run[m] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run[m] - top);
#pragma unroll
                for (int n = 0; n < ND; ++n) *(f4t*)(mg + (16 * wave + lr) * C::MS + 16 * n + 4 * lg) = acc[m][n] * f;
                __syncthreads();
                for (int i = tid; i < NW / WR * 16 * D / 4; i += 64 * NW) {
                    const int g = i / (16 * D / 4), p = i / (D / 4) % 16, d = 4 * (i % (D / 4)), q = 16 * m + p;
                    const int pair = g * 16 * MT + q;
                    if (pt * PW + pair < n_pairs) {
                        const float mm = largest(g * WR, q);
                        float l = 0.0f;
                        f4t o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int x = g * WR; x < g * WR + WR; ++x) {
                            // (a wave without a maximum: its sum is 0, or NaN by a NaN score)
                            l = fmaf(sL[x][q], sM[x][q] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sM[x][q] - mm), l);
                            o += *(const f4t*)(mg + (16 * x + p) * C::MS + d);
                        }
                        emit(pair, d, o, mm, l, d == 0);
                    }
                }
                __syncthreads();
            }
        } else {
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const int p = p0 - pt * PW + 16 * m + lr;
                const float l = across_rows_sum(l_run[m]);
                if (p0 + 16 * m + lr < n_pairs) {
#pragma unroll
                    for (int n = 0; n < ND; ++n) emit(p, 16 * n + 4 * lg, acc[m][n], m_run[m], l, n == 0 && lg == 0);
                }
            }
            __syncthreads();  // every wave has read the last tile's flags before the next segment clears them
        }
    }
}

// Joins the parts of the segments that more than one workgroup had. NWR waves per row
// (sequence, token, head): D / 4 lanes read a part's dims, NG parts at a time and
// four of those in flight, each group of lanes with a running maximum of its own.
// Bound by the launch and two memory round trips (4 us of a small call).
template <int D, bool NARROW, int PW, int TR, int NWR>
__global__ __launch_bounds__(256) void fa_tree_join(TreeArgs a) {
    constexpr int L = D / 4, NG = 64 * NWR / L, UN = 4, RB = 4 / NWR;
    __shared__ float sO[RB][NG][D], sM[RB][NG], sL[RB][NG];
    const int rb = RB == 1 ? 0 : wave_id(), tid = threadIdx.x % (64 * NWR);
    const uint32_t row = uniform(blockIdx.x * RB + rb);
    const uint32_t bt = a.d_h.quot(row), h = row - bt * a.d_h.d;
    const uint32_t b = a.d_q.quot(bt), t = bt - b * a.d_q.d;
    SeqChunk<PW, TR> seqs;
    const Deal deal(seqs.total(a), a.d_wgs);
    const bool real = b < (uint32_t)a.B;
    while (real && (uint32_t)seqs.b0 + 64 <= b) seqs.load(a, seqs.b0 + 64, seqs.last());
    const int sl = real ? (int)b - seqs.b0 : 0;
    const bool live = real && t < lane_get((uint32_t)seqs.mine.n_tok, sl);
    const uint32_t tiles = lane_get(seqs.mine.tiles, sl), ptiles = lane_get(seqs.mine.ptiles, sl);
    const uint32_t hk = a.d_g.quot(h), pair = t * a.G + h - hk * a.G, pt = pair / PW;
    const uint32_t u0 = lane_get(seqs.upto, sl) - lane_get(seqs.mine.units, sl) + (hk * ptiles + pt) * (kStart + tiles) + kStart;  // its first tile
    // (one part: its workgroup has written the row)
    const uint32_t w0 = live ? deal.owner(u0) : 0u, n = live ? deal.owner(u0 + tiles - 1) - w0 + 1 : 1u;
    const bool on = n > 1;
    const int64_t part0 = ((int64_t)w0 + ((int64_t)b * a.pg.n_head_kv + hk) * a.max_ptiles + pt) * a.part_pairs + (pair - pt * PW);
    const int g = tid / L, d = 4 * (tid % L);
    f4t o = {0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    for (uint32_t x0 = g; on && x0 < n; x0 += NG * UN) {
        f4t y[UN];
        float2 ml[UN];
#pragma unroll
        for (int i = 0; i < UN; ++i) {
            const int64_t at = part0 + (int64_t)min(x0 + NG * i, n - 1) * a.part_pairs;
            ml[i] = a.part_ml[at];
            y[i] = *(const f4t*)(a.part_o + at * D + d);
            if (x0 + NG * i >= n) {  // not a part: no weight, and nothing that a product could make NaN
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
    if (!on) return;
    float top = sM[rb][0], sum = 0.0f;
#pragma unroll
    for (int i = 1; i < NG; ++i) top = fmaxf(top, sM[rb][i]);
#pragma unroll
    for (int e0 = 0; e0 < D; e0 += 64 * NWR) {
        const int e = e0 + tid;
        if (e >= D) break;
        float v = 0.0f;
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const float w = sM[rb][i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sM[rb][i] - top);
            sum = fmaf(sL[rb][i], w, sum);
            v = fmaf(sO[rb][i][e], w, v);
        }
        v *= sum == 0.0f ? 0.0f : 1.0f / sum;
        uint8_t* y = a.dst + b * a.d_nb3 + t * a.d_nb2 + h * a.d_nb1;
        if constexpr (NARROW)
            ((uint16_t*)y)[e] = (uint16_t)f32_to_bf16_bits(v);
        else
            ((float*)y)[e] = v;
        if (a.lse && e == 0) a.lse[(int64_t)bt * a.H + h] = sum == 0.0f ? -INFINITY : (top + kTreeOff) * kTreeLn2 + logf(sum);
    }
}

// The kernel variant, workgroups and workspace of a call: of its shapes alone.
struct TreePlan {
    int form;                 // index into the forms below
    int pw, tr;               // pairs of a workgroup, KV rows of a tile
    uint32_t wgs;
    int32_t max_ptiles, part_pairs;
    int64_t units, parts;     // units: those that the table could hold, at most
    size_t ml_at, bytes;
};
// Forms by the pairs (tokens x group) of a KV head: up to 16, 32: the waves share the rows;
// above: they share the pairs, up to 64, 128, 256 of a workgroup. The smallest that holds the
// pairs, as products of absent pairs cost as much as others, and the most that share a row.
// Decode of 24/4 heads of 256, 8 x 16000 q8_0 rows: 73 us in the form of 16, 81 in that of 64
// (f32 Q, 4 x 32000 rows: 118; 175 in that of 32; 194); 64 pairs over f16 rows: 36 us, 40 in the
// form of 128 (f32 Q over q4_0: 52, 69); 256 pairs: 186 us, 218 in two tiles of 128.
template <int MT_, int WR_, int NW_> struct TreeForm { static constexpr int MT = MT_, WR = WR_, NW = NW_; };
template <int D, bool NARROW, typename F>
static void tree_form(int form, F f) {
    switch (form) {
    case 0: f(TreeForm<1, 4, 4>{}); break;
    case 1: f(TreeForm<1, 2, 4>{}); break;
    case 2: f(TreeForm<1, 1, 4>{}); break;
    case 3:
        if constexpr (D == 128) f(TreeForm<2, 1, 4>{});
        else f(TreeForm<1, 1, 8>{});
        break;
    default:
        if constexpr (D == 128) f(TreeForm<2, 1, 8>{});
        break;
    }
}
template <int KT, typename F>
static void tree_types(int64_t D, bool narrow, F f) {
    if (D == 128) narrow ? f(std::integral_constant<int, 128>{}, std::true_type{}) : f(std::integral_constant<int, 128>{}, std::false_type{});
    else narrow ? f(std::integral_constant<int, 256>{}, std::true_type{}) : f(std::integral_constant<int, 256>{}, std::false_type{});
}
// f(KT, D, NARROW, form) of the call
template <typename F>
static void tree_variant(int kt, int64_t D, bool narrow, int form, F f) {
    auto at = [&](auto k) {
        tree_types<decltype(k)::value>(D, narrow, [&](auto d, auto nar) {
            tree_form<decltype(d)::value, decltype(nar)::value>(form, [&](auto fm) { f(k, d, nar, fm); });
        });
    };
    switch (kt) {
    case XQ_TYPE_F16: at(std::integral_constant<int, XQ_TYPE_F16>{}); break;
    case XQ_TYPE_E5M2: at(std::integral_constant<int, XQ_TYPE_E5M2>{}); break;
    case XQ_TYPE_Q8_0: at(std::integral_constant<int, XQ_TYPE_Q8_0>{}); break;
    default: at(std::integral_constant<int, XQ_TYPE_Q4_0>{}); break;
    }
}
static TreePlan tree_plan(const xq_tensor* q, const xq_kv_pages* c) {
    TreePlan P{};
    const int64_t D = q->ne[0], Hkv = c->k.ne[2], B = q->ne[3], pairs = q->ne[1] * (q->ne[2] / Hkv);
    P.form = pairs <= 16 ? 0 : pairs <= 32 ? 1 : pairs <= 64 ? 2 : pairs <= 128 || D == 256 ? 3 : 4;
    int per_cu = 1;
    tree_variant(c->k.type, D, q->type == XQ_TYPE_BF16, P.form, [&](auto k, auto d, auto nar, auto fm) {
        using F = decltype(fm);
        using C = TreeCfg<decltype(k)::value, decltype(d)::value, decltype(nar)::value, F::MT, F::WR, F::NW>;
        P.pw = C::PW;
        P.tr = C::TR;
        per_cu = C::PER_CU;
    });
    P.max_ptiles = (int32_t)cdiv(pairs, P.pw);
    P.part_pairs = (int32_t)(pairs < P.pw ? pairs : P.pw);
    const int64_t segs = B * Hkv * P.max_ptiles;
    const int64_t limit = (int64_t)c->table_cols * c->k.ne[1];
    P.units = (cdiv(limit < 0x7fffff00 ? limit : 0x7fffff00, P.tr) + kStart) * segs;
    int64_t wgs = 256 * per_cu;
    if (wgs > P.units) wgs = P.units;
    P.wgs = (uint32_t)wgs;
    P.parts = wgs + segs;
    const size_t o = (size_t)P.parts * P.part_pairs * D * 4;
    P.ml_at = (o + 255) / 256 * 256;
    P.bytes = P.ml_at + (size_t)P.parts * P.part_pairs * 8;
    return P;
}

static xq_status tree_check(const xq_tensor* q, const xq_kv_pages* cache, const xq_tensor* dst, PagesView* pg) {
    if (!q || !cache || !dst) return failf(XQ_ERR_BAD_ARG, "null argument");
    if (q->type != XQ_TYPE_F32 && q->type != XQ_TYPE_BF16) return failf(XQ_ERR_UNSUPPORTED, "q must be F32 or BF16");
    if (dst->type != q->type) return failf(XQ_ERR_UNSUPPORTED, "dst must have q's type");
    const int64_t D = q->ne[0];
    if (D != 128 && D != 256) return failf(XQ_ERR_UNSUPPORTED, "head dim %lld not in {128, 256}", (long long)D);
    for (int i = 1; i < 4; ++i)
        if (q->ne[i] < 1 || q->ne[i] > 0x7fffffff) return failf(XQ_ERR_BAD_SHAPE, "bad ne");
    const int64_t T = q->ne[1], H = q->ne[2], B = q->ne[3];
    if (T > kTreeMax) return failf(XQ_ERR_UNSUPPORTED, "more than 64 tokens of a sequence");
    if (dst->ne[0] != D || dst->ne[1] != H || dst->ne[2] != T || dst->ne[3] != B)
        return failf(XQ_ERR_BAD_SHAPE, "dst must be [D, n_head, n_q, n_seq]");
    const size_t es = type_size(q->type);
    if (q->nb[0] != es || dst->nb[0] != es) return failf(XQ_ERR_UNSUPPORTED, "q/dst elements must be contiguous");
    if (!elem_aligned(q, es, 1) || !aligned(q->data, es)) return failf(XQ_ERR_UNSUPPORTED, "misaligned q");
    if (!elem_aligned(dst, 16, 1) || !aligned(dst->data, 16))
        return failf(XQ_ERR_UNSUPPORTED, "dst strides and pointer must be multiples of 16 bytes");
    const xq_status st = pages_check(cache, D, 0, B, kF16 | kE5M2 | kQ8 | kQ4, pg);
    if (st != XQ_OK) return st;
    for (const xq_tensor* t : {&cache->k, &cache->v})
        if (t->nb[1] >> 32 || t->nb[3] >> 32) return failf(XQ_ERR_UNSUPPORTED, "row and page strides must be below 2^32 bytes");
    const int64_t Hkv = cache->k.ne[2];
    if (H % Hkv) return failf(XQ_ERR_BAD_SHAPE, "n_head %% n_head_kv != 0");
    if (H / Hkv > 32) return failf(XQ_ERR_UNSUPPORTED, "GQA group above 32");
    if (B >> 23 || H >> 23 || B * T * H >= (int64_t)1 << 23) return failf(XQ_ERR_UNSUPPORTED, "2^23 query rows or more");
    // numbers of units are 32-bit (and divided as 31-bit ones)
    if (tree_plan(q, cache).units >= (int64_t)1 << 30) return failf(XQ_ERR_UNSUPPORTED, "a table of 2^30 tiles of work or more");
    return XQ_OK;
}

}  // namespace xq

using namespace xq;

extern "C" {

int xq_supports_fa_tree(const xq_tensor* q, const xq_kv_pages* cache, const xq_tensor* dst) {
    return tree_check(q, cache, dst, nullptr) == XQ_OK;
}

xq_status xq_fa_tree_workspace(const xq_tensor* q, const xq_kv_pages* cache, const xq_tensor* dst, size_t* bytes) {
    if (!bytes) return failf(XQ_ERR_BAD_ARG, "bytes is null");
    const xq_status st = tree_check(q, cache, dst, nullptr);
    if (st != XQ_OK) return st;
    *bytes = tree_plan(q, cache).bytes;
    return done_ok();
}

xq_status xq_fa_tree(const xq_tensor* q, const xq_kv_pages* cache, const int32_t* parents, const int32_t* n_tok, xq_tensor* dst,
                     float* lse, float scale, void* workspace, size_t workspace_bytes, void* stream) {
    TreeArgs a{};
    const xq_status st = tree_check(q, cache, dst, &a.pg);
    if (st != XQ_OK) return st;
    if (!(fabsf(scale) < INFINITY)) return failf(XQ_ERR_BAD_ARG, "scale must be finite");
    if (!q->data || !dst->data || pages_null(cache)) return failf(XQ_ERR_BAD_ARG, "null data pointer");
    for (const void* x : {(const void*)parents, (const void*)n_tok, (const void*)lse, (const void*)cache->table, (const void*)cache->rows})
        if (!aligned(x, 4)) return failf(XQ_ERR_UNSUPPORTED, "misaligned pointer");
    const TreePlan P = tree_plan(q, cache);
    const size_t need = P.bytes;
    if (!workspace || workspace_bytes < need) return failf(XQ_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    if (!aligned(workspace, 256)) return failf(XQ_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    a.q = (const uint8_t*)q->data;
    a.q_nb1 = (int64_t)q->nb[1], a.q_nb2 = (int64_t)q->nb[2], a.q_nb3 = (int64_t)q->nb[3];
    a.dst = (uint8_t*)dst->data;
    a.d_nb1 = (int64_t)dst->nb[1], a.d_nb2 = (int64_t)dst->nb[2], a.d_nb3 = (int64_t)dst->nb[3];
    a.k_page = (uint32_t)a.pg.k_page, a.k_row = (uint32_t)a.pg.k_row, a.v_page = (uint32_t)a.pg.v_page, a.v_row = (uint32_t)a.pg.v_row;
    a.lse = lse, a.parents = parents, a.n_tok = n_tok, a.scale = scale;
    a.n_q = (int32_t)q->ne[1], a.H = (int32_t)q->ne[2], a.B = (int32_t)q->ne[3];
    a.G = a.H / a.pg.n_head_kv;
    a.d_g = UDivFlat((uint32_t)a.G), a.d_wgs = UDivFlat(P.wgs), a.d_h = UDivFlat((uint32_t)a.H), a.d_q = UDivFlat((uint32_t)a.n_q);
    a.max_ptiles = P.max_ptiles, a.part_pairs = P.part_pairs;
    a.part_o = (float*)workspace, a.part_ml = (float2*)((uint8_t*)workspace + P.ml_at);
    const bool narrow = q->type == XQ_TYPE_BF16;
    hipStream_t s = (hipStream_t)stream;
    tree_variant(cache->k.type, q->ne[0], narrow, P.form, [&](auto k, auto d, auto nar, auto fm) {
        using F = decltype(fm);
        constexpr int KT = decltype(k)::value, D = decltype(d)::value;
        constexpr bool NARROW = decltype(nar)::value;
        using C = TreeCfg<KT, D, NARROW, F::MT, F::WR, F::NW>;
        launch("fa_tree", fa_tree_kernel<KT, D, NARROW, F::MT, F::WR, F::NW>, dim3(P.wgs), dim3(64 * F::NW), s, a);
        // four waves per row while those find room together: 768 rows of 256 38.7 us (one wave each
        // 42.5), 1024 rows of 128 alike, 4096 rows 20.2 (16.2), 12800 rows 75 (66)
        const uint32_t rows = (uint32_t)((int64_t)a.B * a.n_q * a.H);
        if (rows <= 2048)
            launch("fa_tree_join", fa_tree_join<D, NARROW, C::PW, C::TR, 4>, dim3(rows), dim3(256), s, a);
        else
            launch("fa_tree_join", fa_tree_join<D, NARROW, C::PW, C::TR, 1>, dim3((rows + 3) / 4), dim3(256), s, a);
    });
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return failf(XQ_ERR_HIP, "fa_tree launch: %s", hipGetErrorString(e));
    return done_ok();
}

}  // extern "C"
