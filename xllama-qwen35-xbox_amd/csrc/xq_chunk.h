// xq_chunk.h — a chunk of new tokens over the paged cache as its kernels see it: which rows a
// token sees, the scores' transformation, and the host's check of the caller's description.
#pragma once

#include <math.h>

#include "xq_tile.h"

namespace xq {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct ChunkArgs {
    const uint8_t* q;
    int64_t q_nb1, q_nb2, q_nb3;  // token, head, sequence
    PagesView pg;
    const int32_t *first, *prefix, *n_tok;
    int32_t n_q, H, G, B, window;
    float scale, cap, inv_cap, max_bias, m0, m1;
    int32_t n_head_log2;
    uint32_t k_page, k_row, v_page, v_row;  // strides, below 2^32
    UDivFlat d_g;                           // by the group

    // Rows that sequence b holds, its new tokens, the row behind its last one.
    XQ_DEV void lengths(int b, int& held, int& tokens, int& end) const {
        held = min(max(pg.rows[b], 0), pg.row_limit);
        tokens = n_tok ? min(max(n_tok[b], 0), n_q) : n_q;
        end = (int)min((uint32_t)held + (uint32_t)tokens, (uint32_t)pg.row_limit);
    }
    // Token t's row, and the rows [lo, hi) that it sees.
    XQ_DEV void range(int b, int t, int held, int end, int& at, int& lo, int& hi) const {
        at = (int)min((uint32_t)held + (uint32_t)t, (uint32_t)pg.row_limit);
        hi = min(at + 1, end);
        if (prefix) hi = max(hi, min(prefix[b], end));
        lo = window ? max(at + 1 - window, 0) : 0;
        if (first) lo = max(lo, first[(int64_t)b * n_q + t]);
    }
    XQ_DEV float slope(int h) const {
        if (!(max_bias > 0.0f)) return 0.0f;
        return h < n_head_log2 ? powf(m0, (float)(h + 1)) : powf(m1, (float)(2 * (h - n_head_log2) + 1));
    }
};

// ALiBi: a score less the slope times the distance, on both sides of the token (a prefix shows it rows behind its own).
XQ_DEV float less_distance(float x, float slope, int row, int at) { return fmaf(-slope, fabsf((float)(row - at)), x); }

// tanh: below 0.2 its series (the next term is 5.6e-8 of it there, a step of f32), above by the exponential, whose
// difference from 1 keeps all but 2 bits.
XQ_DEV float capped_tanh(float z) {
    const float zz = z * z;
    const float near = z * fmaf(zz, fmaf(zz, fmaf(zz, -17.0f / 315.0f, 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
    const float y = z > 10.0f ? 10.0f : z < -10.0f ? -10.0f : z;  // (NaN stays)
    const float e = __builtin_amdgcn_exp2f(y * (2.0f * kLog2e));
    const float far = (e - 1.0f) * __builtin_amdgcn_rcpf(e + 1.0f);
    return fabsf(z) < 0.2f ? near : far;
}

// A query as matrix operands, which may have the inner elements in any order that the keys have too: with
// EL 8, operand c takes elements 8lg .. + 7 of the c-th 32; else a lane has EL neighbours of each 4 EL, eight at
// a time. First as they lie in memory,
template <int EL>
constexpr int operand_at(int c) {
    return c / (EL / 8) * 4 * EL + c % (EL / 8) * 8;
}
template <int NB, bool NARROW, int EL = 8>
XQ_DEV void query_load(const uint8_t* q, int lg, float (&x)[NB][8]) {
#pragma unroll
    for (int c = 0; c < NB; ++c) {
        const int e = operand_at<EL>(c) + EL * lg;
        if constexpr (NARROW) {
            const u4half y = *(const u4half*)(q + 2 * e);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[c][2 * i] = __uint_as_float(y[i] << 16);
                x[c][2 * i + 1] = __uint_as_float(y[i] & 0xffff0000u);
            }
        } else {
            const f4el y = *(const f4el*)(q + 4 * e), z = *(const f4el*)(q + 4 * e + 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[c][i] = y[i];
                x[c][4 + i] = z[i];
            }
        }
    }
}
// then in f16 (QP 2: high and low part) times 2^lift, which puts the row's largest element in [2^14, 2^15),
// and the sign of the scale. Returns the factor that makes scores of the products: |scale| 2^-lift times `unit`,
// a normal number: an unseen score's -inf stays one, and a score of 0 too.
template <int NB, int QP>
XQ_DEV float query_split(const float (&x)[NB][8], float scale, float unit, h8t (&o)[NB][QP]) {
    float big = 0.0f;
#pragma unroll
    for (int c = 0; c < NB; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) big = fmaxf(big, fabsf(x[c][j]));
    const int lift = 141 - min((int)(__float_as_uint(across_rows_max(big)) >> 23), 254);
#pragma unroll
    for (int c = 0; c < NB; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float y = ldexpf(scale < 0.0f ? -x[c][j] : x[c][j], lift);
            const _Float16 high = (_Float16)y;
            o[c][0][j] = high;
            if constexpr (QP == 2) o[c][1][j] = (_Float16)(y - (float)high);
        }
    return fminf(fmaxf(ldexpf(fabsf(scale), -lift) * unit, 1.17549435e-38f), 3.40282347e38f);
}

// The bits of a 64-row tile from row r0 on that lie in [lo, hi).
XQ_DEV uint64_t tile_rows(int r0, int lo, int hi) {
    const int a = min(max(lo - r0, 0), 64), b = min(max(hi - r0, 0), 64);
    const uint64_t below_b = b == 64 ? ~0ull : (1ull << b) - 1, below_a = a == 64 ? ~0ull : (1ull << a) - 1;
    return below_b & ~below_a;
}

inline xq_status chunk_check(const xq_tensor* q, const xq_kv_pages* cache, PagesView* pg) {
    if (!q || !cache) return failf(XQ_ERR_BAD_ARG, "null argument");
    if (q->type != XQ_TYPE_F32 && q->type != XQ_TYPE_BF16) return failf(XQ_ERR_UNSUPPORTED, "q must be F32 or BF16");
    const int64_t D = q->ne[0];
    if (D != 128 && D != 256) return failf(XQ_ERR_UNSUPPORTED, "head dim %lld not in {128, 256}", (long long)D);
    for (int i = 1; i < 4; ++i)
        if (q->ne[i] < 1 || q->ne[i] > 0x7fffffff) return failf(XQ_ERR_BAD_SHAPE, "bad ne");
    const int64_t T = q->ne[1], H = q->ne[2], B = q->ne[3];
    const size_t es = type_size(q->type);
    if (q->nb[0] != es) return failf(XQ_ERR_UNSUPPORTED, "q elements must be contiguous");
    if (!elem_aligned(q, es, 1) || !aligned(q->data, es)) return failf(XQ_ERR_UNSUPPORTED, "misaligned q");
    const xq_status st = pages_check(cache, D, 0, B, kF16 | kE5M2 | kQ8 | kQ4, pg);
    if (st != XQ_OK) return st;
    for (const xq_tensor* t : {&cache->k, &cache->v})
        if (t->nb[1] >> 32 || t->nb[3] >> 32) return failf(XQ_ERR_UNSUPPORTED, "row and page strides must be below 2^32 bytes");
    const int64_t Hkv = cache->k.ne[2];
    if (H % Hkv) return failf(XQ_ERR_BAD_SHAPE, "n_head %% n_head_kv != 0");
    if (H / Hkv > 32) return failf(XQ_ERR_UNSUPPORTED, "GQA group above 32");
    if (T >> 25 || B >> 25 || H >> 25 || B * T >= (int64_t)1 << 25 || B * T * H >= (int64_t)1 << 25)
        return failf(XQ_ERR_UNSUPPORTED, "2^25 query rows or more");
    return XQ_OK;
}

inline xq_status chunk_params_check(const xq_chunk_params* p) {
    if (!p) return failf(XQ_ERR_BAD_ARG, "null params");
    if (!(fabsf(p->scale) < INFINITY)) return failf(XQ_ERR_BAD_ARG, "scale must be finite");
    if (!(p->logit_softcap >= 0.0f && p->logit_softcap < INFINITY)) return failf(XQ_ERR_BAD_ARG, "logit_softcap must be finite and not negative");
    if (!(p->max_bias >= 0.0f && p->max_bias < INFINITY)) return failf(XQ_ERR_BAD_ARG, "max_bias must be finite and not negative");
    if (p->window < 0) return failf(XQ_ERR_BAD_ARG, "window must not be negative");
    for (int i = 0; i < 4; ++i)
        if (p->reserved[i]) return failf(XQ_ERR_BAD_ARG, "reserved fields must be 0");
    return XQ_OK;
}

// The arguments of a checked call (a.pg is filled).
inline void chunk_fill(ChunkArgs& a, const xq_tensor* q, const xq_chunk_params* p, const int32_t* first, const int32_t* prefix,
                       const int32_t* n_tok) {
    a.q = (const uint8_t*)q->data;
    a.q_nb1 = (int64_t)q->nb[1], a.q_nb2 = (int64_t)q->nb[2], a.q_nb3 = (int64_t)q->nb[3];
    a.first = first, a.prefix = prefix, a.n_tok = n_tok;
    a.n_q = (int32_t)q->ne[1], a.H = (int32_t)q->ne[2], a.B = (int32_t)q->ne[3];
    a.G = a.H / a.pg.n_head_kv;
    a.window = p->window, a.scale = p->scale, a.cap = p->logit_softcap, a.max_bias = p->max_bias;
    // (finite, so that a score of 0 stays 0 under a subnormal cap; what that makes of others is below 2^-126)
    a.inv_cap = p->logit_softcap > 0.0f ? fminf(1.0f / p->logit_softcap, 3.40282347e38f) : 0.0f;
    a.n_head_log2 = 1;
    while (2 * a.n_head_log2 <= a.H) a.n_head_log2 *= 2;
    a.m0 = powf(2.0f, -p->max_bias / (float)a.n_head_log2);
    a.m1 = powf(2.0f, -p->max_bias / 2.0f / (float)a.n_head_log2);
    a.k_page = (uint32_t)a.pg.k_page, a.k_row = (uint32_t)a.pg.k_row, a.v_page = (uint32_t)a.pg.v_page, a.v_row = (uint32_t)a.pg.v_row;
    a.d_g = UDivFlat((uint32_t)a.G);
}

}  // namespace xq
