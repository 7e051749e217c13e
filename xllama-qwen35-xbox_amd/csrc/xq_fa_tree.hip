// xq_fa_tree.hip — attention of drafted tokens (a tree, a chain, one token) over the paged cache.
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
    int32_t n_q, H, G, B, kt, bf16;
    float scale;
};

template <int KT>
XQ_DEV float kv_element(const uint8_t* rec, int d) {
    if constexpr (KT == XQ_TYPE_F16) return f16_bits_to_f32(*(const uint16_t*)(rec + 2 * d));
    if constexpr (KT == XQ_TYPE_E5M2) return e5m2_to_f32(rec[d]);
    if constexpr (KT == XQ_TYPE_Q8_0) {
        const uint8_t* b = rec + d / 32 * 34;
        return f16_bits_to_f32(*(const uint16_t*)b) * (float)(int8_t)b[2 + d % 32];
    }
    const uint8_t* b = rec + d / 32 * 18;
    const int n = d % 32 < 16 ? b[2 + d % 16] & 15 : b[2 + d % 16] >> 4;
    return f16_bits_to_f32(*(const uint16_t*)b) * (float)(n - 8);
}

// One wave per (sequence, token, head), one row after another.
template <int KT, int D>
__global__ __launch_bounds__(64) void fa_tree_plain(TreeArgs a) {
    const int lane = threadIdx.x;
    const int h = blockIdx.x, t = blockIdx.y, b = blockIdx.z;
    const int n_tok = a.n_tok ? min(a.n_tok[b], a.n_q) : a.n_q;
    if (t >= n_tok) return;
    const int64_t held = max(0, a.pg.rows[b]);
    const int hk = h / a.G;
    uint64_t seen = 0;
    for (int j = t; j >= 0;) {
        seen |= (uint64_t)1 << j;
        const int p = a.parents ? a.parents[(int64_t)b * a.n_q + j] : j - 1;
        j = p < j ? p : -1;
    }
    constexpr int E = D / 64;
    float q[E], o[E], m = -INFINITY, l = 0.0f;
    const uint8_t* qp = a.q + b * a.q_nb3 + t * a.q_nb1 + h * a.q_nb2;
    for (int i = 0; i < E; ++i) {
        const int d = lane * E + i;
        q[i] = a.bf16 ? bf16_bits_to_f32(*(const uint16_t*)(qp + 2 * d)) : *(const float*)(qp + 4 * d);
        o[i] = 0.0f;
    }
    for (int64_t r = 0; r < held + n_tok && r < a.pg.row_limit; ++r) {
        if (r >= held && !(seen >> (r - held) & 1)) continue;
        const uint32_t page = a.pg.page(b, (uint32_t)r);
        if (page >= (uint32_t)a.pg.n_pages) continue;
        const int64_t in = r % a.pg.page_rows;
        const uint8_t* k = a.pg.k + page * a.pg.k_page + in * a.pg.k_row + hk * a.pg.k_head;
        const uint8_t* v = a.pg.v + page * a.pg.v_page + in * a.pg.v_row + hk * a.pg.v_head;
        float s = 0.0f;
        for (int i = 0; i < E; ++i) s = fmaf(q[i], kv_element<KT>(k, lane * E + i), s);
        s = wave_sum(s) * a.scale;
        const float mn = fmaxf(m, s), f = m == mn ? 1.0f : expf(m - mn), w = expf(s - mn);
        m = mn;
        l = fmaf(l, f, w);
        for (int i = 0; i < E; ++i) o[i] = fmaf(w, kv_element<KT>(v, lane * E + i), o[i] * f);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint8_t* dp = a.dst + b * a.d_nb3 + t * a.d_nb2 + h * a.d_nb1;
    for (int i = 0; i < E; ++i) {
        const int d = lane * E + i;
        if (a.bf16) *(__bf16*)(dp + 2 * d) = (__bf16)(o[i] * inv);
        else *(float*)(dp + 4 * d) = o[i] * inv;
    }
    if (a.lse && lane == 0) a.lse[((int64_t)b * a.n_q + t) * a.H + h] = l > 0.0f ? m + logf(l) : -INFINITY;
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
    const int64_t Hkv = cache->k.ne[2];
    if (H % Hkv) return failf(XQ_ERR_BAD_SHAPE, "n_head %% n_head_kv != 0");
    if (H / Hkv > 32) return failf(XQ_ERR_UNSUPPORTED, "GQA group above 32");
    if (B > 65535 || H > 65535) return failf(XQ_ERR_UNSUPPORTED, "more than 65535 sequences or heads");
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
    *bytes = 256;
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
    const size_t need = 256;
    if (!workspace || workspace_bytes < need) return failf(XQ_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    if (!aligned(workspace, 256)) return failf(XQ_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    a.q = (const uint8_t*)q->data;
    a.q_nb1 = (int64_t)q->nb[1], a.q_nb2 = (int64_t)q->nb[2], a.q_nb3 = (int64_t)q->nb[3];
    a.dst = (uint8_t*)dst->data;
    a.d_nb1 = (int64_t)dst->nb[1], a.d_nb2 = (int64_t)dst->nb[2], a.d_nb3 = (int64_t)dst->nb[3];
    a.lse = lse, a.parents = parents, a.n_tok = n_tok, a.scale = scale;
    a.n_q = (int32_t)q->ne[1], a.H = (int32_t)q->ne[2], a.B = (int32_t)q->ne[3];
    a.G = a.H / a.pg.n_head_kv;
    a.kt = cache->k.type, a.bf16 = q->type == XQ_TYPE_BF16;
    const dim3 grid((uint32_t)a.H, (uint32_t)a.n_q, (uint32_t)a.B), block(64);
    hipStream_t s = (hipStream_t)stream;
    const bool wide = q->ne[0] == 256;
    switch (a.kt) {
    case XQ_TYPE_F16: launch("fa_tree", wide ? fa_tree_plain<XQ_TYPE_F16, 256> : fa_tree_plain<XQ_TYPE_F16, 128>, grid, block, s, a); break;
    case XQ_TYPE_E5M2: launch("fa_tree", wide ? fa_tree_plain<XQ_TYPE_E5M2, 256> : fa_tree_plain<XQ_TYPE_E5M2, 128>, grid, block, s, a); break;
    case XQ_TYPE_Q8_0: launch("fa_tree", wide ? fa_tree_plain<XQ_TYPE_Q8_0, 256> : fa_tree_plain<XQ_TYPE_Q8_0, 128>, grid, block, s, a); break;
    default: launch("fa_tree", wide ? fa_tree_plain<XQ_TYPE_Q4_0, 256> : fa_tree_plain<XQ_TYPE_Q4_0, 128>, grid, block, s, a); break;
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return failf(XQ_ERR_HIP, "fa_tree launch: %s", hipGetErrorString(e));
    return done_ok();
}

}  // extern "C"
