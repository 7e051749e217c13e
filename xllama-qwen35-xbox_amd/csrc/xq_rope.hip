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
// to f32: at position 2^20 a f32 angle would be off by 2^-5 rad. The power of the base is an f64
// exp2 per lane: as a product of powers that the host hands over, prompts took 60 us for 65, but
// one token 5.0 for 4.3 and 8 trees of 25 7.5 for 6.3 (device time): two more lines of arguments.
//
// Two prompts of 4097 bf16 tokens, 24/4 heads of 256 (2 x 134 MB): 64 us with two input sets in
// turn, 69 with more than the Infinity Cache holds: 3.9 to 4.2 TB/s where a large copy reaches
// 4.9; 67 into q8_0, q4_0 or E5M2 pools; one prompt of f32 tokens 48. One token: 4.6 to 5.8 us on the
// device, a chain of dependent reads. 200 bf16 tokens, 32/8 heads of 128: 7.0 us, of which the angles
// that every wave of a token forms for itself are the part that one token does not have.
#include "xq_kv_codec.h"
#include "xq_paged.h"

namespace xq {

struct RopeArgs {
    const uint8_t *q, *k, *v;
    int64_t q_nb1, q_nb3, k_nb1, k_nb3, v_nb1, v_nb3;  // token, sequence
    uint32_t q_nb2, k_nb2, v_nb2, o_nb2;               // head, below 2^32
    uint8_t* out;
    int64_t o_nb1, o_nb3;
    const int32_t* positions;
    const int32_t* n_tok;
    const float *qw, *kw, *ff;
    PagesView pg;
    int32_t kt, q8_variant, mode, n_rot, n_q, H, Hkv;
    int32_t units_q, units_kv;    // 256-element units of a token's queries; of its keys
    int32_t units_part;           // units of a wave
    uint32_t n_waves;
    UDivFlat d_parts, d_q;        // by the waves per token; by the tokens per sequence
    double rev0, rate;            // revolutions per position of index 0; factor from an index to the next
    double log2_rate;
    float attn, eps;
};

constexpr int kRopeBatch = 4;  // units whose loads a wave has in flight

typedef uint32_t u32x2e __attribute__((ext_vector_type(2), aligned(2)));
typedef float f4e __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4f __attribute__((ext_vector_type(4), aligned(4)));

// Four neighbouring elements as they lie in memory, and as f32.
template <int T> struct Quad;
template <> struct Quad<XQ_TYPE_F32> { using Raw = u32x4f; static constexpr int W = 4; };
template <> struct Quad<XQ_TYPE_BF16> { using Raw = u32x2e; static constexpr int W = 2; };
template <int T>
XQ_DEV f4e quad_f32(const typename Quad<T>::Raw w) {
    if constexpr (T == XQ_TYPE_F32)
        return __builtin_bit_cast(f4e, w);
    else
        return f4e{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u)};
}

template <int T>
XQ_DEV void store4(uint8_t* p, f4e x) {
    if constexpr (T == XQ_TYPE_F32) {
        *(f4e*)p = x;
    } else {
        typedef float f2 __attribute__((ext_vector_type(2)));
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        *(u32x2e*)p = u32x2e{__builtin_bit_cast(uint32_t, __builtin_convertvector((f2{x[0], x[1]}), b2)),
                             __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{x[2], x[3]}), b2))};
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
    using Raw = typename Quad<TI>::Raw;
    constexpr int W = Quad<TI>::W;
    const uint32_t w = blockIdx.x * 4u + wave_id();
    if (w >= a.n_waves) return;
    const uint32_t tok = a.d_parts.quot(w);
    const int part = (int)(w - tok * a.d_parts.d);
    const int b = (int)a.d_q.quot(tok), t = (int)(tok - b * a.d_q.d);
    if (a.n_tok && t >= a.n_tok[b]) return;
    const int lane = lane_id(), sub = lane / LPR, e0 = 4 * (lane % LPR);
    const int u_first = part * a.units_part, u_end = min(u_first + a.units_part, a.units_q + 2 * a.units_kv);
    const int32_t position = a.positions[(int64_t)b * a.n_q + t];
    const int64_t row = (int64_t)a.pg.rows[b] + t;

    // A kind's units [u0, u1) in batches: every load of a batch before its first use.
    auto stream = [&](const uint8_t* base, uint32_t nb2, int heads, int u0, int u1, auto use) {
        for (int u = u0; u < u1; u += kRopeBatch) {
            Raw x[kRopeBatch];
#pragma unroll
            for (int i = 0; i < kRopeBatch; ++i) {
                const uint32_t h = (uint32_t)min(min(u + i, u1 - 1) * RPU + sub, heads - 1);
                // read once: past the caches (8194 tokens of 24 + 8 heads of 256 bf16: 65.7 us, with
                // ordinary loads 71.9)
                x[i] = __builtin_nontemporal_load((const Raw*)(base + (uint64_t)h * nb2 + e0 * ES));
            }
#pragma unroll
            for (int i = 0; i < kRopeBatch; ++i)
                if (u + i < u1) use(x[i], (u + i) * RPU + sub);
        }
    };
    const int uq1 = min(u_end, a.units_q), uk0 = max(u_first, a.units_q), uk1 = min(u_end, a.units_q + a.units_kv);
    const int uv0 = max(u_first, a.units_q + a.units_kv);

    if (u_first < a.units_q + a.units_kv) {
        // cos and sin of this lane's four elements: an element past n_rot does not turn
        const int half = a.n_rot / 2;
        const bool halves = a.mode == XQ_ROPE_HALVES;
        const bool turned = e0 < a.n_rot, low = e0 < half;
        f4e cs = {1.0f, 1.0f, 1.0f, 1.0f}, sn = {0.0f, 0.0f, 0.0f, 0.0f};
        {
            const int i0 = halves ? (low ? e0 : e0 - half) : e0 / 2;  // first index of the lane
            double rev = (double)position * a.rev0 * exp2(a.log2_rate * i0);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (!halves && j >= 2) break;
                double x = rev;
                if (a.ff && i0 + j < half) x /= (double)a.ff[i0 + j];
                x -= rint(x);
                float s, c;
                sincospif(2.0f * (float)x, &s, &c);
                c *= a.attn;
                s *= a.attn;
                if (halves) {
                    cs[j] = turned ? c : 1.0f;
                    sn[j] = turned ? (low ? -s : s) : 0.0f;
                } else if (e0 + 2 * j < a.n_rot) {
                    cs[2 * j] = cs[2 * j + 1] = c;
                    sn[2 * j] = -s;
                    sn[2 * j + 1] = s;
                }
                rev *= a.rate;
            }
        }
        const int shift = half / 4;  // lanes from an element to its partner
        const int partner = low ? lane + shift : lane - shift;
        // y cos +- z sin with y = x w / norm, z = the partner: x (w cos) / norm + x' (w' sin) / norm
        f4e qc = cs, qs = sn, kc = cs, ks = sn;
        auto weigh = [&](const float* g, f4e& c, f4e& s) {
            if (!g) return;
            const f4e own = *(const f4e*)(g + e0);
            f4e other = own;
            if (halves) {
                if (turned) other = *(const f4e*)(g + (low ? e0 + half : e0 - half));
            } else {
                other = f4e{own[1], own[0], own[3], own[2]};
            }
            c *= own;
            s *= other;
        };
        weigh(a.qw, qc, qs);
        weigh(a.kw, kc, ks);
        auto turn = [&](const Raw x, const f4e c, const f4e s, bool norm) -> f4e {
            const f4e y = quad_f32<TI>(x);
            f4e z;
            if (halves) {
                Raw other;
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    const uint32_t o = (uint32_t)__shfl((int)x[j], partner);
                    other[j] = turned ? o : 0u;  // what does not turn takes nothing, whatever is there
                }
                z = quad_f32<TI>(other);
            } else {
                z = f4e{e0 < a.n_rot ? y[1] : 0.0f, e0 < a.n_rot ? y[0] : 0.0f, e0 + 2 < a.n_rot ? y[3] : 0.0f, e0 + 2 < a.n_rot ? y[2] : 0.0f};
            }
            f4e r;
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = fmaf(y[j], c[j], z[j] * s[j]);
            if (norm) {
                const float ss = head_sum<D>(fmaf(y[3], y[3], fmaf(y[2], y[2], fmaf(y[1], y[1], y[0] * y[0]))));
                r *= __builtin_amdgcn_rsqf(fmaf(ss, 1.0f / D, a.eps));  // 1 ulp
            }
            return r;
        };
        uint8_t* const out = a.out + b * a.o_nb3 + t * a.o_nb1;
        stream(a.q + b * a.q_nb3 + t * a.q_nb1, a.q_nb2, a.H, u_first, uq1, [&](const Raw x, int head) {
            const f4e y = turn(x, qc, qs, a.qw != nullptr);
            if (head < a.H) store4<TO>(out + (uint64_t)(uint32_t)head * a.o_nb2 + e0 * EO, y);
        });
        // the row of the cache that takes this token's key
        const bool in = row >= 0 && row < a.pg.row_limit;
        const uint32_t r = in ? (uint32_t)row : 0u;
        const uint32_t page = a.pg.page(b, r), off = r - a.pg.d_page.quot(r) * a.pg.d_page.d;
        const bool kept = in && page < (uint32_t)a.pg.n_pages;
        uint8_t* const to = a.pg.k + page * a.pg.k_page + off * a.pg.k_row;
        stream(a.k + b * a.k_nb3 + t * a.k_nb1, a.k_nb2, a.Hkv, uk0 - a.units_q, uk1 - a.units_q, [&](const Raw x, int head) {
            const f4e y = turn(x, kc, ks, a.kw != nullptr);
            kv_put4_any(a.kt, f4u{y[0], y[1], y[2], y[3]}, lane, e0, a.q8_variant, to + head * a.pg.k_head, kept && head < a.Hkv);
        });
    }
    if (uv0 < u_end) {
        const bool in = row >= 0 && row < a.pg.row_limit;
        const uint32_t r = in ? (uint32_t)row : 0u;
        const uint32_t page = a.pg.page(b, r), off = r - a.pg.d_page.quot(r) * a.pg.d_page.d;
        const bool kept = in && page < (uint32_t)a.pg.n_pages;
        uint8_t* const to = a.pg.v + page * a.pg.v_page + off * a.pg.v_row;
        const int before = a.units_q + a.units_kv;
        stream(a.v + b * a.v_nb3 + t * a.v_nb1, a.v_nb2, a.Hkv, uv0 - before, u_end - before, [&](const Raw x, int head) {
            const f4e y = quad_f32<TI>(x);
            kv_put4_any(a.kt, f4u{y[0], y[1], y[2], y[3]}, lane, e0, a.q8_variant, to + head * a.pg.v_head, kept && head < a.Hkv);
        });
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
    // (a wave each at least; a grid holds below 2^32 threads)
    if (T * B >= (int64_t)1 << 26) return failf(XQ_ERR_UNSUPPORTED, "2^26 tokens or more");
    for (const xq_tensor* t : {k, v})
        if (t->ne[0] != D || t->ne[1] != T || t->ne[2] != Hkv || t->ne[3] != B)
            return failf(XQ_ERR_BAD_SHAPE, "k/v must be [D, n_q, n_head_kv, n_seq]");
    if (o->ne[0] != D || o->ne[1] != T || o->ne[2] != H || o->ne[3] != B)
        return failf(XQ_ERR_BAD_SHAPE, "q_out must be [D, n_q, n_head, n_seq]");
    for (const xq_tensor* t : {q, k, v, o}) {
        const size_t es = type_size(t->type);
        if (t->nb[0] != es) return failf(XQ_ERR_UNSUPPORTED, "elements must be contiguous");
        if (!elem_aligned(t, es, 1) || !aligned(t->data, es)) return failf(XQ_ERR_UNSUPPORTED, "misaligned tensor");
        if (t->nb[2] >> 32) return failf(XQ_ERR_UNSUPPORTED, "head strides must be below 2^32 bytes");
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
    const dim3 grid((a.n_waves + 3) / 4), block(256);
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
    a.q_nb1 = (int64_t)q->nb[1], a.q_nb2 = (uint32_t)q->nb[2], a.q_nb3 = (int64_t)q->nb[3];
    a.k_nb1 = (int64_t)k->nb[1], a.k_nb2 = (uint32_t)k->nb[2], a.k_nb3 = (int64_t)k->nb[3];
    a.v_nb1 = (int64_t)v->nb[1], a.v_nb2 = (uint32_t)v->nb[2], a.v_nb3 = (int64_t)v->nb[3];
    a.out = (uint8_t*)q_out->data;
    a.o_nb1 = (int64_t)q_out->nb[1], a.o_nb2 = (uint32_t)q_out->nb[2], a.o_nb3 = (int64_t)q_out->nb[3];
    a.positions = positions, a.n_tok = n_tok, a.qw = q_weight, a.kw = k_weight, a.ff = freq_factors;
    a.kt = cache->k.type, a.q8_variant = p->q8_variant, a.mode = p->mode, a.n_rot = p->n_rot;
    a.n_q = (int32_t)q->ne[1], a.H = (int32_t)q->ne[2], a.Hkv = (int32_t)k->ne[2];
    a.units_q = (int32_t)cdiv(a.H, rpu), a.units_kv = (int32_t)cdiv(a.Hkv, rpu);
    const int64_t tokens = q->ne[1] * q->ne[3], units = a.units_q + 2 * (int64_t)a.units_kv;
    // one unit per wave while that leaves CUs without a wave, then up to all of a token's: a wave
    // forms the angles once, but needs company. 2 x 4097 bf16 prompt tokens of 24/4 heads of 256, shared
    // out to about 8192 waves 65.7 us, 16384 64.4, 32768 70.2, 65536 84.3
    int64_t upw = tokens * units / 16384;
    if (upw < 1) upw = 1;
    if (upw > units) upw = units;
    a.units_part = (int32_t)upw;
    const int64_t parts = cdiv(units, upw);
    a.n_waves = (uint32_t)(tokens * parts);
    a.d_parts = UDivFlat((uint32_t)parts), a.d_q = UDivFlat((uint32_t)a.n_q);
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
