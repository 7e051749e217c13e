// xq_rope.hip — norms of queries and keys for each head and the position rotation in one
// pass, keys and values stored into the paged cache.
//
// Per head row x of D elements: y = x * w / sqrt(mean(x^2) + eps), then for rotary index i
// with elements (a, b) and angle t = position * freq_scale * base^(-2i/n_rot) / ff[i]:
// (a cos t - b sin t, a sin t + b cos t). Each row is read once and written once: bound by
// HBM, and by the launch and one memory round trip for few tokens.
//
// A lane holds four consecutive elements, so a wave's load is 256 elements: one, two or four
// heads of a token. The sum of squares runs over the row's lanes by DPP and permlane swaps,
// the partner half of a rotated element comes from its lane by one shuffle. A wave takes
// several such units of one token, whose angles it forms once.
// The angle is formed in f64 as revolutions, reduced to (-1/2, 1/2] there, and only then goes
// to f32: at position 2^20 a f32 angle would be off by 2^-5 rad.
#include "xq_kv_codec.h"
#include "xq_paged.h"

namespace xq {

struct RopeArgs {
    const uint8_t *q, *k, *v;
    int64_t q_nb1, q_nb2, q_nb3, k_nb1, k_nb2, k_nb3, v_nb1, v_nb2, v_nb3;  // token, head, sequence
    uint8_t* out;
    int64_t o_nb1, o_nb2, o_nb3;
    const int32_t* positions;
    const int32_t* n_tok;
    const float *qw, *kw, *ff;
    PagesView pg;
    int32_t kt, q8_variant, mode, n_rot, n_q, H, Hkv;
    int32_t units_q, units_kv;    // 256-element units of a token's queries; of its keys
    int32_t parts, units_part;    // waves per token, units per wave
    int64_t n_waves;
    double rev0, rate;            // revolutions per position of index 0; factor from an index to the next
    double log2_rate;
    float attn, eps;
};

constexpr int kRopeBatch = 4;  // units whose loads a wave has in flight

typedef uint16_t u16e __attribute__((aligned(2)));
typedef uint32_t u32x2e __attribute__((ext_vector_type(2), aligned(2)));
typedef float f4e __attribute__((ext_vector_type(4), aligned(4)));

template <int T>
XQ_DEV f4e load4(const uint8_t* p) {
    if constexpr (T == XQ_TYPE_F32) {
        return *(const f4e*)p;
    } else {
        const u32x2e w = *(const u32x2e*)p;
        return f4e{bf16_bits_to_f32(w.x & 0xffffu), __uint_as_float(w.x & 0xffff0000u), bf16_bits_to_f32(w.y & 0xffffu),
                   __uint_as_float(w.y & 0xffff0000u)};
    }
}

template <int T>
XQ_DEV void store4(uint8_t* p, f4e x) {
    if constexpr (T == XQ_TYPE_F32) {
        *(f4e*)p = x;
    } else {
        *(u32x2e*)p = u32x2e{f32_to_bf16_bits(x[0]) | (f32_to_bf16_bits(x[1]) << 16),
                             f32_to_bf16_bits(x[2]) | (f32_to_bf16_bits(x[3]) << 16)};
    }
}

// Sum over the D / 4 lanes of a row, in every lane of it.
template <int D>
XQ_DEV float head_sum(float x) {
    x = row16_sum(x);
    if constexpr (D >= 128) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if constexpr (D >= 256) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return x;
}

template <int TI, int TO, int D>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(RopeArgs a) {
    constexpr int RPU = 256 / D, LPR = D / 4, ES = TI == XQ_TYPE_F32 ? 4 : 2, EO = TO == XQ_TYPE_F32 ? 4 : 2;
    const int64_t w = (int64_t)blockIdx.x * 4 + wave_id();
    if (w >= a.n_waves) return;
    const int64_t tok = w / a.parts;
    const int part = (int)(w - tok * a.parts);
    const int b = (int)(tok / a.n_q), t = (int)(tok - (int64_t)b * a.n_q);
    if (a.n_tok && t >= a.n_tok[b]) return;
    const int lane = lane_id(), sub = lane / LPR, e0 = 4 * (lane % LPR);
    const int u_end = min((part + 1) * a.units_part, a.units_q + 2 * a.units_kv);

    // the row of the cache that takes this token's key and value
    const int64_t row = (int64_t)a.pg.rows[b] + t;
    const bool in = row >= 0 && row < a.pg.row_limit;
    const uint32_t r = in ? (uint32_t)row : 0u;
    const uint32_t page = a.pg.page(b, r), off = r - a.pg.d_page.quot(r) * (uint32_t)a.pg.page_rows;
    const bool kept = in && page < (uint32_t)a.pg.n_pages;

    // cos and sin of this lane's four elements (an element past n_rot is not turned)
    const int half = a.n_rot / 2;
    const bool halves = a.mode == XQ_ROPE_HALVES;
    const bool turned = e0 < a.n_rot;
    float cs[4], sn[4];
    {
        const int i0 = halves ? (e0 >= half ? e0 - half : e0) : e0 / 2;  // first index of the lane
        const double pos = (double)a.positions[(int64_t)b * a.n_q + t];
        double rev = pos * a.rev0 * exp2(a.log2_rate * i0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (!halves && j >= 2) break;
            const int i = i0 + j;
            double x = rev;
            if (a.ff && i < half) x /= (double)a.ff[i];
            x -= rint(x);
            float s, c;
            sincospif(2.0f * (float)x, &s, &c);
            cs[j] = c * a.attn;
            sn[j] = s * a.attn;
            rev *= a.rate;
        }
    }
    const int shift = half / 4;  // lanes from an element to its partner
    const bool low = e0 < half;
    const int partner = !turned ? lane : low ? lane + shift : lane - shift;

    f4e wq = {1.0f, 1.0f, 1.0f, 1.0f}, wk = wq;
    if (a.qw) wq = *(const f4e*)(a.qw + e0);
    if (a.kw) wk = *(const f4e*)(a.kw + e0);

    for (int u0 = part * a.units_part; u0 < u_end; u0 += kRopeBatch) {
        f4e x[kRopeBatch];
        int head[kRopeBatch];
#pragma unroll
        for (int i = 0; i < kRopeBatch; ++i) {
            const int u = min(u0 + i, u_end - 1);
            const bool is_q = u < a.units_q, is_k = u < a.units_q + a.units_kv;
            head[i] = (u - (is_q ? 0 : is_k ? a.units_q : a.units_q + a.units_kv)) * RPU + sub;
            const uint8_t* p = is_q ? a.q + b * a.q_nb3 + t * a.q_nb1 : is_k ? a.k + b * a.k_nb3 + t * a.k_nb1 : a.v + b * a.v_nb3 + t * a.v_nb1;
            const int64_t nb2 = is_q ? a.q_nb2 : is_k ? a.k_nb2 : a.v_nb2;
            const int last = (is_q ? a.H : a.Hkv) - 1;
            x[i] = load4<TI>(p + min(head[i], last) * nb2 + e0 * ES);
        }
#pragma unroll
        for (int i = 0; i < kRopeBatch; ++i) {
            const int u = u0 + i;
            if (u >= u_end) break;
            const bool is_q = u < a.units_q, is_v = u >= a.units_q + a.units_kv;
            f4e y = x[i];
            if (!is_v) {
                if (is_q ? a.qw : a.kw) {
                    const float ss = head_sum<D>(fmaf(y[3], y[3], fmaf(y[2], y[2], fmaf(y[1], y[1], y[0] * y[0]))));
                    const float inv = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
                    const f4e g = is_q ? wq : wk;
#pragma unroll
                    for (int j = 0; j < 4; ++j) y[j] = y[j] * inv * g[j];
                }
                if (halves) {
                    f4e z;
#pragma unroll
                    for (int j = 0; j < 4; ++j) z[j] = __shfl(y[j], partner);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float turn = low ? fmaf(y[j], cs[j], -(z[j] * sn[j])) : fmaf(y[j], cs[j], z[j] * sn[j]);
                        y[j] = turned ? turn : y[j];
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float p = y[2 * j], q = y[2 * j + 1];
                        if (e0 + 2 * j < a.n_rot) {
                            y[2 * j] = fmaf(p, cs[j], -(q * sn[j]));
                            y[2 * j + 1] = fmaf(p, sn[j], q * cs[j]);
                        }
                    }
                }
            }
            if (is_q) {
                if (head[i] < a.H) store4<TO>(a.out + b * a.o_nb3 + t * a.o_nb1 + head[i] * a.o_nb2 + e0 * EO, y);
                continue;
            }
            const bool live = kept && head[i] < a.Hkv;
            uint8_t* y0 = is_v ? a.pg.v + page * a.pg.v_page + off * a.pg.v_row + head[i] * a.pg.v_head
                               : a.pg.k + page * a.pg.k_page + off * a.pg.k_row + head[i] * a.pg.k_head;
            const f4u yy = {y[0], y[1], y[2], y[3]};
            switch (a.kt) {
            case XQ_TYPE_F32: kv_put4<XQ_TYPE_F32>(yy, lane, e0, a.q8_variant, y0, live); break;
            case XQ_TYPE_F16: kv_put4<XQ_TYPE_F16>(yy, lane, e0, a.q8_variant, y0, live); break;
            case XQ_TYPE_BF16: kv_put4<XQ_TYPE_BF16>(yy, lane, e0, a.q8_variant, y0, live); break;
            case XQ_TYPE_E5M2: kv_put4<XQ_TYPE_E5M2>(yy, lane, e0, a.q8_variant, y0, live); break;
            case XQ_TYPE_Q8_0: kv_put4<XQ_TYPE_Q8_0>(yy, lane, e0, a.q8_variant, y0, live); break;
            default: kv_put4<XQ_TYPE_Q4_0>(yy, lane, e0, a.q8_variant, y0, live); break;
            }
        }
    }
}

static xq_status rope_check(const xq_tensor* q, const xq_tensor* k, const xq_tensor* v, const xq_rope_params* p,
                            const xq_tensor* o, const xq_kv_pages* cache, PagesView* pg) {
    if (!q || !k || !v || !p || !o || !cache) return failf(XQ_ERR_BAD_ARG, "null argument");
    if ((q->type != XQ_TYPE_F32 && q->type != XQ_TYPE_BF16) || k->type != q->type || v->type != q->type)
        return failf(XQ_ERR_UNSUPPORTED, "q/k/v must share type F32 or BF16");
    if (o->type != XQ_TYPE_F32 && o->type != XQ_TYPE_BF16) return failf(XQ_ERR_UNSUPPORTED, "q_out must be F32 or BF16");
    const int64_t D = q->ne[0];
    if (D != 64 && D != 128 && D != 256) return failf(XQ_ERR_UNSUPPORTED, "head dim %lld not in {64, 128, 256}", (long long)D);
    for (int i = 1; i < 4; ++i)
        if (q->ne[i] < 1 || q->ne[i] > 0x7fffffff) return failf(XQ_ERR_BAD_SHAPE, "bad ne");
    const int64_t T = q->ne[1], H = q->ne[2], B = q->ne[3], Hkv = k->ne[2];
    if (Hkv < 1 || Hkv > 0x7fffff || H > 0x7fffff) return failf(XQ_ERR_BAD_SHAPE, "bad head counts");
    for (const xq_tensor* t : {k, v})
        if (t->ne[0] != D || t->ne[1] != T || t->ne[2] != Hkv || t->ne[3] != B)
            return failf(XQ_ERR_BAD_SHAPE, "k/v must be [D, n_q, n_head_kv, n_seq]");
    if (o->ne[0] != D || o->ne[1] != T || o->ne[2] != H || o->ne[3] != B)
        return failf(XQ_ERR_BAD_SHAPE, "q_out must be [D, n_q, n_head, n_seq]");
    for (const xq_tensor* t : {q, k, v, o}) {
        const size_t es = type_size(t->type);
        if (t->nb[0] != es) return failf(XQ_ERR_UNSUPPORTED, "elements must be contiguous");
        if (!elem_aligned(t, es, 1) || !aligned(t->data, es)) return failf(XQ_ERR_UNSUPPORTED, "misaligned tensor");
    }
    if (p->mode != XQ_ROPE_HALVES && p->mode != XQ_ROPE_PAIRS) return failf(XQ_ERR_BAD_ARG, "bad rope mode %d", p->mode);
    if (p->n_rot < 0 || p->n_rot > D || p->n_rot % 2) return failf(XQ_ERR_BAD_ARG, "n_rot must be even and in [0, head dim]");
    if (p->mode == XQ_ROPE_HALVES && p->n_rot % 8) return failf(XQ_ERR_UNSUPPORTED, "n_rot must be a multiple of 8 for halves");
    if (!(p->freq_base > 0.0f) || !(p->freq_base < INFINITY) || !(fabsf(p->freq_scale) < INFINITY) ||
        !(fabsf(p->attn_factor) < INFINITY) || !(p->eps >= 0.0f) || !(p->eps < INFINITY))
        return failf(XQ_ERR_BAD_ARG, "bad rope parameters");
    if (p->q8_variant != 0 && p->q8_variant != 1) return failf(XQ_ERR_BAD_ARG, "q8_variant must be 0 or 1");
    return pages_check(cache, D, Hkv, B, kF32 | kF16 | kBF16 | kE5M2 | kQ8 | kQ4, pg);
}

template <int TI, int TO>
static hipError_t rope_launch(const RopeArgs& a, int64_t D, hipStream_t stream) {
    const dim3 grid((uint32_t)((a.n_waves + 3) / 4)), block(256);
    switch (D) {
    case 64: launch("qk_norm_rope", qk_norm_rope_kernel<TI, TO, 64>, grid, block, stream, a); break;
    case 128: launch("qk_norm_rope", qk_norm_rope_kernel<TI, TO, 128>, grid, block, stream, a); break;
    default: launch("qk_norm_rope", qk_norm_rope_kernel<TI, TO, 256>, grid, block, stream, a); break;
    }
    return hipGetLastError();
}

}  // namespace xq

using namespace xq;

extern "C" {

int xq_supports_qk_norm_rope(const xq_tensor* q, const xq_tensor* k, const xq_tensor* v, const xq_rope_params* params,
                             const xq_tensor* q_out, const xq_kv_pages* cache) {
    return rope_check(q, k, v, params, q_out, cache, nullptr) == XQ_OK;
}

xq_status xq_qk_norm_rope(const xq_tensor* q, const xq_tensor* k, const xq_tensor* v, const int32_t* positions,
                          const int32_t* n_tok, const float* q_weight, const float* k_weight, const float* freq_factors,
                          const xq_rope_params* p, xq_tensor* q_out, const xq_kv_pages* cache, void* stream) {
    RopeArgs a{};
    const xq_status st = rope_check(q, k, v, p, q_out, cache, &a.pg);
    if (st != XQ_OK) return st;
    if (!q->data || !k->data || !v->data || !q_out->data || !positions || pages_null(cache))
        return failf(XQ_ERR_BAD_ARG, "null data pointer");
    for (const void* x : {(const void*)positions, (const void*)n_tok, (const void*)q_weight, (const void*)k_weight,
                          (const void*)freq_factors, (const void*)cache->table, (const void*)cache->rows})
        if (!aligned(x, 4)) return failf(XQ_ERR_UNSUPPORTED, "misaligned pointer");
    const int64_t D = q->ne[0], rpu = 256 / D;
    a.q = (const uint8_t*)q->data, a.k = (const uint8_t*)k->data, a.v = (const uint8_t*)v->data;
    a.q_nb1 = (int64_t)q->nb[1], a.q_nb2 = (int64_t)q->nb[2], a.q_nb3 = (int64_t)q->nb[3];
    a.k_nb1 = (int64_t)k->nb[1], a.k_nb2 = (int64_t)k->nb[2], a.k_nb3 = (int64_t)k->nb[3];
    a.v_nb1 = (int64_t)v->nb[1], a.v_nb2 = (int64_t)v->nb[2], a.v_nb3 = (int64_t)v->nb[3];
    a.out = (uint8_t*)q_out->data;
    a.o_nb1 = (int64_t)q_out->nb[1], a.o_nb2 = (int64_t)q_out->nb[2], a.o_nb3 = (int64_t)q_out->nb[3];
    a.positions = positions, a.n_tok = n_tok, a.qw = q_weight, a.kw = k_weight, a.ff = freq_factors;
    a.kt = cache->k.type, a.q8_variant = p->q8_variant, a.mode = p->mode, a.n_rot = p->n_rot;
    a.n_q = (int32_t)q->ne[1], a.H = (int32_t)q->ne[2], a.Hkv = (int32_t)k->ne[2];
    a.units_q = (int32_t)cdiv(a.H, rpu), a.units_kv = (int32_t)cdiv(a.Hkv, rpu);
    const int64_t tokens = q->ne[1] * q->ne[3], units = a.units_q + 2 * (int64_t)a.units_kv;
    // one unit per wave while that leaves CUs without a wave, then up to all of a token's
    int64_t upw = tokens * units / 8192;
    if (upw < 1) upw = 1;
    if (upw > units) upw = units;
    a.units_part = (int32_t)upw;
    a.parts = (int32_t)cdiv(units, upw);
    a.n_waves = tokens * a.parts;
    if (a.n_waves > (int64_t)0x7fffffff) return failf(XQ_ERR_UNSUPPORTED, "too many tokens for one call");
    a.log2_rate = p->n_rot ? -2.0 / p->n_rot * log2((double)p->freq_base) : 0.0;
    a.rate = exp2(a.log2_rate);
    a.rev0 = (double)p->freq_scale / 6.283185307179586476925286766559;
    a.attn = p->attn_factor, a.eps = p->eps;
    const bool fi = q->type == XQ_TYPE_F32, fo = q_out->type == XQ_TYPE_F32;
    hipStream_t s = (hipStream_t)stream;
    const hipError_t e = fi ? fo ? rope_launch<XQ_TYPE_F32, XQ_TYPE_F32>(a, D, s) : rope_launch<XQ_TYPE_F32, XQ_TYPE_BF16>(a, D, s)
                            : fo ? rope_launch<XQ_TYPE_BF16, XQ_TYPE_F32>(a, D, s) : rope_launch<XQ_TYPE_BF16, XQ_TYPE_BF16>(a, D, s);
    if (e != hipSuccess) return failf(XQ_ERR_HIP, "qk_norm_rope launch: %s", hipGetErrorString(e));
    return done_ok();
}

}  // extern "C"
