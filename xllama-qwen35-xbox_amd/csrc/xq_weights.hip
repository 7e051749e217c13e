// xq_weights.hip — the attention weight that each cached row gets from a chunk's tokens, accumulated.
//
// With the lse of every (token, head) known, a row's weight is a plain sum,
//   w_r = sum_{pairs that see r} 2^(x_r - log2(e) lse),   x_r = log2(e) (f(scale q.k_r) + slope (r - at)),
// and nothing of V is read. A wave keeps 32 rows of K of one head in registers as matrix operands and
// takes the head's pairs 16 at a time: the product leaves four rows of one pair in a lane, whose
// weights add up in the lane; the 16 lanes of a row join at the end.
#include <type_traits>

#include "xq_chunk.h"

namespace xq {

constexpr int kWtRows = 32;            // rows of a wave
constexpr int kWtTile = 4 * kWtRows;   // of a workgroup

struct PairMeta {
    float factor, lse2, slope;  // base-2 score of a product (BIASED: natural), log2(e) lse, ALiBi slope
    int32_t lo, hi, at;         // rows seen, the token's own
    int32_t pad[2];
};

struct WeightsArgs : ChunkArgs {
    const float* lse;
    const float* scores;
    float* out;
    int32_t cols, fresh, splits, row_tiles;
    float decay;
    _Float16* qh;   // [sequence][KV head][n_q G][QP][D]
    PairMeta* meta; // [sequence][KV head][n_q G]
    float* part;    // [split][sequence][row_tiles kWtTile]
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

// Elements 32c + 8lg .. + 7 of a record as f16: the values, or q8_0 / q4_0's integers with the
// block's scale.
template <int KT>
XQ_DEV h8t operand8(const uint8_t* rec, int c, int lg, float& scale) {
    if constexpr (KT == XQ_TYPE_F16) {
        return __builtin_bit_cast(h8t, *(const u4half*)(rec + 64 * c + 16 * lg));
    } else if constexpr (KT == XQ_TYPE_E5M2) {
        const u32x2u w = *(const u32x2u*)(rec + 32 * c + 8 * lg);
        const u4t o = {__builtin_amdgcn_perm(w[0], w[0], 0x010c000cu), __builtin_amdgcn_perm(w[0], w[0], 0x030c020cu),
                       __builtin_amdgcn_perm(w[1], w[1], 0x010c000cu), __builtin_amdgcn_perm(w[1], w[1], 0x030c020cu)};
        return __builtin_bit_cast(h8t, o);
    } else {
        constexpr bool Q8 = KT == XQ_TYPE_Q8_0;
        const uint8_t* blk = rec + c * (Q8 ? 34 : 18);
        scale = f16_bits_to_f32(*(const u16any*)blk);
        u32x2u w = *(const u32x2u*)(blk + 2 + 8 * (Q8 ? lg : lg & 1));
        // (1024 + n) - 1152 of n = q ^ 0x80; (1024 + n) - 1032 of the nibble
        const _Float16 off = Q8 ? (_Float16)-1152.0f : (_Float16)-1032.0f;
        u4t o;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t n = Q8 ? w[i] ^ 0x80808080u : (lg & 2 ? w[i] >> 4 : w[i]) & 0x0f0f0f0fu;
            o[2 * i] = __builtin_amdgcn_perm(0x64646464u, n, 0x05010500u);
            o[2 * i + 1] = __builtin_amdgcn_perm(0x64646464u, n, 0x05030502u);
        }
        return __builtin_bit_cast(h8t, o) + off;
    }
}

template <int KT, int D, bool NARROW, bool BIASED>
__global__ __launch_bounds__(256, 2) void weights_kernel(WeightsArgs a) {
    constexpr bool QUANT = KT == XQ_TYPE_Q8_0 || KT == XQ_TYPE_Q4_0;
    constexpr int QP = NARROW ? 1 : 2, PARTS = QUANT ? 2 : 1, NB = D / 32, RT = kWtRows / 16;
    const int lane = lane_id(), wave = wave_id(), lr = lane & 15, lg = lane >> 4;
    const int b = blockIdx.z;
    int held, n_tok, end;
    a.lengths(b, held, n_tok, end);
    const int first = (int)(blockIdx.x * kWtTile) + wave * kWtRows;
    if (first >= end) return;
    const int n_pairs = n_tok * a.G, groups = (n_pairs + 15) / 16, items = groups * a.pg.n_head_kv;
    int it = (int)((int64_t)items * blockIdx.y / a.splits);
    const int it_end = (int)((int64_t)items * (blockIdx.y + 1) / a.splits);

    // the wave's rows: lane lr (of each 16) has row 16r + lr
    uint64_t has = 0;  // of the 32 rows
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
        rec[r] = ok ? a.pg.k + (uint64_t)page * a.k_page + (uint64_t)in * a.k_row : nullptr;
    }
    f4t sum[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) sum[r] = f4t{0.0f, 0.0f, 0.0f, 0.0f};
    const float inv_cap = a.cap > 0.0f ? 1.0f / a.cap : 0.0f;

    while (it < it_end) {
        const int hk = (int)uniform((uint32_t)(it / groups)), g_end = min(groups, it_end - hk * groups);
        // ---- K of this head
        h8t kh[RT][NB], kl[PARTS == 2 ? RT : 1][PARTS == 2 ? NB : 1];
        int ek[RT][4];  // QUANT: the powers of two of rows 16r + 4lg + i
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            float d[NB];
            const h8t zero = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < NB; ++c) {
                kh[r][c] = zero;
                d[c] = 0.0f;
                if (rec[r]) kh[r][c] = operand8<KT>(rec[r] + hk * a.pg.k_head, c, lg, d[c]);
            }
            if constexpr (QUANT) {
                // d 2^-e in [2^7, 2^8) for the row's largest finite block scale; then d q = hi + lo exactly
                int e = 103;  // 2^-24, the smallest f16
#pragma unroll
                for (int c = 0; c < NB; ++c) {
                    const int x = (int)((__float_as_uint(d[c]) >> 23) & 255u);
                    e = max(e, x == 255 ? 103 : x);
                }
                e -= 127 + 7;
#pragma unroll
                for (int c = 0; c < NB; ++c) {
                    const _Float16 f = (_Float16)ldexpf(d[c], -e);
                    const h8t ff = {f, f, f, f, f, f, f, f}, q = kh[r][c];
                    kh[r][c] = q * ff;
                    kl[r][c] = __builtin_elementwise_fma(q, ff, -kh[r][c]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) ek[r][i] = __shfl(e, 4 * lg + i);
            }
        }
        // ---- the pairs
        const int64_t head = ((int64_t)b * a.pg.n_head_kv + hk) * a.n_q * a.G;
        for (int g = it - hk * groups; g < g_end; ++g) {
            const int p = 16 * g + lr;
            const int64_t pair = head + min(p, n_pairs - 1);
            const PairMeta m = a.meta[pair];
            uint32_t sees = (uint32_t)(tile_rows(first, m.lo, m.hi) & has);
            if (p >= n_pairs) sees = 0;
            if (!__builtin_amdgcn_ballot_w64(sees != 0)) continue;
            const _Float16* q = a.qh + pair * (QP * D) + 8 * lg;
            f4t s[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) s[r] = f4t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < NB; ++c) {
                const h8t x = *(const h8t*)(q + 32 * c);
                h8t y;
                if constexpr (QP == 2) y = *(const h8t*)(q + D + 32 * c);
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    s[r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[r][c], x, s[r], 0, 0, 0);
                    if constexpr (QP == 2) s[r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[r][c], y, s[r], 0, 0, 0);
                    if constexpr (PARTS == 2) s[r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl[r][c], x, s[r], 0, 0, 0);
                }
            }
            products_done();
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x = s[r][i];
                    if constexpr (QUANT) x = ldexpf(x, ek[r][i]);
                    if constexpr (BIASED) {
                        x *= m.factor;
                        if (a.cap > 0.0f) x = a.cap * capped_tanh(x * inv_cap);
                        x = fmaf(m.slope, (float)(first + 16 * r + 4 * lg + i - m.at), x);
                        x = fmaf(x, kLog2e, -m.lse2);
                    } else {
                        x = fmaf(x, m.factor, -m.lse2);
                    }
                    const float w = __builtin_amdgcn_exp2f(x);
                    sum[r][i] += (sees >> (16 * r + 4 * lg + i)) & 1u ? w : 0.0f;
                }
        }
        it = (hk + 1) * groups;
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float w = row16_sum(sum[r][i]);
            const int row = first + 16 * r + 4 * lg + i;
            if (lr != 0) continue;
            if (a.splits > 1) {
                a.part[((int64_t)blockIdx.y * a.B + b) * ((int64_t)a.row_tiles * kWtTile) + row] = w;
            } else if (row < min(end, a.cols)) {
                const int64_t at = (int64_t)b * a.cols + row;
                const bool old = a.scores && (row < held || !a.fresh);
                a.out[at] = (old ? a.decay * a.scores[at] : 0.0f) + w;
            }
        }
}

__global__ __launch_bounds__(256) void weights_join_kernel(WeightsArgs a) {
    const int b = blockIdx.y, row = (int)(blockIdx.x * 256 + threadIdx.x);
    int held, n_tok, end;
    a.lengths(b, held, n_tok, end);
    if (row >= min(end, a.cols)) return;
    float w = 0.0f;
    for (int s = 0; s < a.splits; ++s) w += a.part[((int64_t)s * a.B + b) * ((int64_t)a.row_tiles * kWtTile) + row];
    const int64_t at = (int64_t)b * a.cols + row;
    const bool old = a.scores && (row < held || !a.fresh);
    a.out[at] = (old ? a.decay * a.scores[at] : 0.0f) + w;
}

// ---------------------------------------------------------------- host

struct WeightsPlan {
    int64_t pairs, row_tiles;
    int32_t splits;
    size_t meta_at, part_at, bytes;
};
static WeightsPlan weights_plan(const xq_tensor* q, const xq_kv_pages* c) {
    WeightsPlan P{};
    const int64_t D = q->ne[0], T = q->ne[1], H = q->ne[2], B = q->ne[3], Hkv = c->k.ne[2], G = H / Hkv;
    P.pairs = B * H * T;
    int64_t limit = (int64_t)c->table_cols * c->k.ne[1];
    if (limit > 0x7fffff00) limit = 0x7fffff00;
    P.row_tiles = cdiv(limit, kWtTile);
    const int64_t items = Hkv * cdiv(T * G, 16);
    int64_t splits = cdiv(512, B * P.row_tiles);
    if (splits > items) splits = items;
    P.splits = (int32_t)(splits < 1 ? 1 : splits);
    P.meta_at = (size_t)P.pairs * D * 2 * (q->type == XQ_TYPE_BF16 ? 1 : 2);
    P.part_at = P.meta_at + (size_t)P.pairs * sizeof(PairMeta);
    P.bytes = P.part_at + (P.splits > 1 ? (size_t)P.splits * B * P.row_tiles * kWtTile * 4 : 0);
    return P;
}

static xq_status weights_check(const xq_tensor* q, const xq_kv_pages* cache, PagesView* pg) {
    const xq_status st = chunk_check(q, cache, pg);
    if (st != XQ_OK) return st;
    if (q->ne[3] > 65535) return failf(XQ_ERR_UNSUPPORTED, "more than 65535 sequences");
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
    if (!workspace || workspace_bytes < P.bytes) return failf(XQ_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", P.bytes, workspace_bytes);
    if (!aligned(workspace, 256)) return failf(XQ_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    chunk_fill(a, q, params, first, prefix, n_tok);
    a.lse = lse, a.scores = scores, a.out = scores_out;
    a.cols = score_cols, a.decay = decay, a.fresh = fresh, a.splits = P.splits, a.row_tiles = (int32_t)P.row_tiles;
    a.qh = (_Float16*)workspace;
    a.meta = (PairMeta*)((uint8_t*)workspace + P.meta_at);
    a.part = (float*)((uint8_t*)workspace + P.part_at);
    a.d_h = UDivFlat((uint32_t)a.H), a.d_q = UDivFlat((uint32_t)a.n_q);
    const bool biased = a.cap > 0.0f || a.max_bias > 0.0f;
    hipStream_t s = (hipStream_t)stream;
    weights_variant(cache->k.type, q->ne[0], q->type == XQ_TYPE_BF16, biased, [&](auto k, auto d, auto nar, auto bi) {
        constexpr int D = decltype(d)::value;
        constexpr bool NARROW = decltype(nar)::value, BIASED = decltype(bi)::value;
        launch("kv_weights_prep", weights_prep_kernel<D, NARROW, BIASED>, dim3((uint32_t)cdiv(P.pairs, 4)), dim3(256), s, a, (uint32_t)P.pairs);
        launch("kv_weights", weights_kernel<decltype(k)::value, D, NARROW, BIASED>, dim3((uint32_t)P.row_tiles, (uint32_t)P.splits, (uint32_t)a.B), dim3(256), s, a);
    });
    if (P.splits > 1)
        launch("kv_weights_join", weights_join_kernel, dim3((uint32_t)cdiv(P.row_tiles * kWtTile, 256), (uint32_t)a.B), dim3(256), s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return failf(XQ_ERR_HIP, "kv_weights launch: %s", hipGetErrorString(e));
    return done_ok();
}

}  // extern "C"
