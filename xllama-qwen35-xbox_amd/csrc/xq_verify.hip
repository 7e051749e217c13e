// xq_verify.hip — drafted tokens against the target's logits, from given random numbers.
//
// p_i = softmax(logits_i / temperature) is the target's distribution after token i. From token 0, which
// is decided, the children of the token reached are tried in order of index: child c with token x is
// accepted if u_c R < p(x), R = 1 - the p of the children's tokens rejected before (a token tried
// twice has no mass left), or, along a chain drawn from a draft's distributions q, if u_c q(x) < p(x).
// The next token is drawn from what is left: p without the rejected tokens, or max(p - q, 0): the lowest v
// whose running sum exceeds u times the whole.
//
// Whether a child would be accepted if its parent were reached does not depend on the walk: all rows'
// maxima and sums are formed at once (one pass over the logits, bound by HBM), then one wave has
// the path by ballots and pointer doubling, a lane a token. Only the next token needs sums that hold
// next to a border: those of one row per sequence, in f64 throughout. A row's sum for the tests is of f32
// exponentials joined in f64: a weight e^-d is off by up to (4 d + 2) 2^-24 of itself (the difference, two roundings of its
// factor, their product, the exponential's step), the sum by the mean of that over its mass.
//
// What bounds it: the one pass over the logits (16 x 16 rows of 128000 f32, 131 MB: 24 us, 5.5 TB/s, some of it from the
// Infinity Cache), then two launches of one row per sequence, 12 and 6 us, each a chain of dependent reads
// (statistics, path, row; sums, part, row) before its f64 arithmetic. The drawn token's place by a workgroup of 16 waves took
// 17 us, with sums kept for every 512 elements one wave has it. Loops in place of unrolled f64 code, a third of
// its size, changed nothing; the drawn row's sums in the first launch would have to be formed of all rows.
#include "xq_tile.h"

namespace xq {

constexpr int kVerifyMax = 64;    // tokens of a sequence: a lane each
constexpr int kVChunk = 8192;     // elements of a row that a workgroup takes
constexpr float kVLog2e = 1.4426950408889634f;

struct RowStat {
    float max, sum;  // of a chunk; the sum relative to its maximum
    int32_t arg;
    int32_t pad;
};
struct Walk {
    int32_t at, n;  // the last token of the path, its length; at -1: nothing left to draw
    uint64_t kids;  // its children
    double max, cool, whole;  // of row `at`: its maximum, 1 / temperature, the stats' sum
};

struct VerifyArgs {
    const uint8_t* logits;
    int64_t l_nb1, l_nb2;  // token, sequence
    const uint8_t* draft;
    int64_t q_nb1, q_nb2;
    const int32_t *tokens, *parents, *n_tok;
    const float *temperature, *uniform;
    int32_t *path, *n_path, *next;
    float* logp;
    int32_t V, n_q, B, chunks, sum_chunks;
    RowStat* stats;  // [sequence][token][chunk]
    Walk* walk;      // [sequence]
    double* sums;    // [2][sequence][sum chunk]: of p's weights; of what is left
    double* parts;   // [2][sequence][sum chunk][kVParts]: the same

    XQ_DEV int tokens_of(int b) const { return n_tok ? min(max(n_tok[b], 0), n_q) : n_q; }
    // the temperature of a sequence; 0: greedy. (Any above 1e30 leaves all finite logits the same mass.)
    XQ_DEV float heat(int b) const {
        const float t = !uniform ? 0.0f : temperature ? temperature[b] : 1.0f;
        return t > 0.0f ? fminf(t, 1e30f) : 0.0f;
    }
};

template <bool WIDE>
XQ_DEV float element(const uint8_t* row, int64_t v) {
    const float x = WIDE ? *(const float*)(row + 4 * v) : bf16_bits_to_f32(*(const uint16_t*)(row + 2 * v));
    return x == x ? x : -INFINITY;
}
// Elements v .. v + N - 1 (4 of f32, 8 of bf16); -inf from V on and for NaN.
template <bool WIDE, int N>
XQ_DEV void elements(const uint8_t* row, int v, int V, float (&x)[N]) {
    static_assert(N == (WIDE ? 4 : 8));
    if (v + N <= V) {
        if constexpr (WIDE) {
            const f4el y = *(const f4el*)(row + 4 * (int64_t)v);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = y[i];
        } else {
            const u4half y = *(const u4half*)(row + 2 * (int64_t)v);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[2 * i] = __uint_as_float(y[i] << 16);
                x[2 * i + 1] = __uint_as_float(y[i] & 0xffff0000u);
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = x[i] == x[i] ? x[i] : -INFINITY;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = v + i < V ? element<WIDE>(row, v + i) : -INFINITY;
    }
}

// A weight relative to the maximum; +inf shares the mass where it is the maximum.
XQ_DEV float weight_f32(float x, float max, float c) { return x == max ? 1.0f : __builtin_amdgcn_exp2f((x - max) * c); }
// e^d for d <= 0, off by less than 2^-51 of itself: d = k ln 2 + r, |r| <= ln 2 / 2, in two parts of ln 2; r's
// series to the 13th power (the next term is 4e-18); 0 below 2^-1074. NaN (of +inf less itself) does not come here.
XQ_DEV double exp_f64(double d) {
    d = fmax(d, -1100.0);
    const double k = rint(d * 1.4426950408889634);
    const double r = fma(-k, 2.3190468138462996e-17, fma(-k, 0.6931471805599453, d));
    double p = 1.0 / 6227020800.0;
    p = fma(p, r, 1.0 / 479001600.0);
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return ldexp(p, (int)k);
}
// `cool`: 1 / temperature
XQ_DEV double weight_f64(double x, double max, double cool) { return exp_f64(x == max ? 0.0 : (x - max) * cool); }

XQ_DEV float exponent_factor(float heat) { return fminf(kVLog2e / (heat > 0.0f ? heat : 1.0f), 3.40282347e38f); }

// Maximum, first index of it and sum of exponentials of a chunk of a row.
template <bool WIDE>
__global__ __launch_bounds__(256) void verify_stats_kernel(VerifyArgs a) {
    constexpr int N = WIDE ? 4 : 8, S = kVChunk / 256 / N;
    __shared__ float sMax[4], sSum[4];
    __shared__ int sArg[4];
    const int j = blockIdx.x, i = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    if (i >= a.tokens_of(b)) return;
    const uint8_t* row = a.logits + b * a.l_nb2 + i * a.l_nb1;
    const float c = exponent_factor(a.heat(b));
    float x[S][N];
    float top = -INFINITY;
#pragma unroll
    for (int s = 0; s < S; ++s) elements<WIDE, N>(row, j * kVChunk + (s * 256 + tid) * N, a.V, x[s]);
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
        for (int e = 0; e < N; ++e) top = fmaxf(top, x[s][e]);
    top = wave_max(top);
    if (lane_id() == 0) sMax[wave_id()] = top;
    __syncthreads();
    top = fmaxf(fmaxf(sMax[0], sMax[1]), fmaxf(sMax[2], sMax[3]));
    float sum = 0.0f;
    int arg = 0x7fffffff;
#pragma unroll
    for (int s = S - 1; s >= 0; --s)
#pragma unroll
        for (int e = N - 1; e >= 0; --e) {
            sum += weight_f32(x[s][e], top, c);
            arg = x[s][e] == top ? j * kVChunk + (s * 256 + tid) * N + e : arg;
        }
    sum = wave_sum(sum);
#pragma unroll
    for (int s = 1; s < 64; s *= 2) arg = min(arg, __shfl_xor(arg, s));
    if (lane_id() == 0) {
        sSum[wave_id()] = sum;
        sArg[wave_id()] = arg;
    }
    __syncthreads();
    if (tid == 0) {
        RowStat r;
        r.max = top;
        r.sum = top == -INFINITY ? 0.0f : (sSum[0] + sSum[1]) + (sSum[2] + sSum[3]);
        r.arg = min(min(sArg[0], sArg[1]), min(sArg[2], sArg[3]));
        r.pad = 0;
        a.stats[((int64_t)b * a.n_q + i) * a.chunks + j] = r;
    }
}

XQ_DEV uint64_t shfl64(uint64_t x, int l) { return ((uint64_t)(uint32_t)__shfl((int)(x >> 32), l) << 32) | (uint32_t)__shfl((int)(uint32_t)x, l); }
XQ_DEV double shfl_f64(double x, int l) { return __builtin_bit_cast(double, shfl64(__builtin_bit_cast(uint64_t, x), l)); }
// of a lane that is the same for all
XQ_DEV double lane_f64(double x, int l) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    return __builtin_bit_cast(double, ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), l) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)u, l));
}

// The sums of the drawn row: a workgroup has 2048 elements, a wave 512. (f64 is what they cost: 16 waves of a workgroup
// on one CU take longer than four on each of four.)
constexpr int kSumThreads = 256, kSumEach = 8, kVSum = kSumThreads * kSumEach;

constexpr int kVParts = kSumThreads / 64, kVPart = kVSum / kVParts;  // a workgroup's parts are its waves' elements

// Sum over the workgroup's threads, the same in all; the order is fixed. Each wave's own goes to parts[wave] too.
XQ_DEV double block_sum(double x, double* lds, double* parts) {
#pragma unroll
    for (int s = 1; s < 64; s *= 2) x += shfl_f64(x, lane_id() ^ s);
    __syncthreads();
    if (lane_id() == 0) lds[wave_id()] = x;
    if (lane_id() == 0 && parts) parts[wave_id()] = x;
    __syncthreads();
    x = 0.0;
#pragma unroll
    for (int i = 0; i < kVParts; ++i) x += lds[i];
    return x;
}
// Elements v .. v + 7 of a row.
template <bool WIDE>
XQ_DEV void eight(const uint8_t* row, int v, int V, float (&x)[kSumEach]) {
    constexpr int N = WIDE ? 4 : 8;
#pragma unroll
    for (int i = 0; i < kSumEach; i += N) elements<WIDE, N>(row, v + i, V, *(float(*)[N])(x + i));
}

// The path, by one wave; a lane is a token. Every lane gets the same result.
template <bool WIDE>
XQ_DEV Walk walk_path(const VerifyArgs& a, int b, bool write) {
    const int c = lane_id(), n = a.tokens_of(b);
    const float heat = a.heat(b), f = exponent_factor(heat);
    const double cool = heat > 0.0f ? 1.0 / (double)heat : 1.0;
    const bool live = c < n;
    // row c's maximum, sum and first index of the maximum
    float top = -INFINITY;
    double whole = 0.0;
    int arg = -1;
    if (live) {
        const RowStat* r = a.stats + ((int64_t)b * a.n_q + c) * a.chunks;
        // (eight chunks in flight at a time: 16 sequences of 19 chunks 11.6 us, one after another 12.5)
        constexpr int UN = 8;
        for (int j = 0; j < a.chunks; j += UN) {
            float x[UN];
#pragma unroll
            for (int i = 0; i < UN; ++i) x[i] = r[min(j + i, a.chunks - 1)].max;
#pragma unroll
            for (int i = 0; i < UN; ++i) top = fmaxf(top, x[i]);
        }
        for (int j = 0; j < a.chunks && top > -INFINITY; j += UN) {
            RowStat x[UN];
#pragma unroll
            for (int i = 0; i < UN; ++i) x[i] = r[min(j + i, a.chunks - 1)];
#pragma unroll
            for (int i = 0; i < UN; ++i) {
                if (j + i >= a.chunks) break;
                whole += (double)x[i].sum * (double)weight_f32(x[i].max, top, f);
                if (arg < 0 && x[i].max == top) arg = x[i].arg;
            }
        }
    }
    const int tok = live ? a.tokens[(int64_t)b * a.n_q + c] : -1;
    int up = !live || c == 0 ? -1 : a.parents ? a.parents[(int64_t)b * a.n_q + c] : c - 1;
    if (up < 0 || up >= c) up = -1;
    const int from = up < 0 ? c : up;
    const float p_top = __shfl(top, from);
    const double p_whole = shfl_f64(whole, from);
    const int p_arg = __shfl(arg, from);
    const bool known = up >= 0 && tok >= 0 && tok < a.V && p_top > -INFINITY;
    double p = 0.0, lp = -INFINITY;
    if (known) {
        const double x = element<WIDE>(a.logits + b * a.l_nb2 + up * a.l_nb1, tok);
        p = weight_f64(x, p_top, cool) / p_whole;
        if (write && a.logp) lp = (x == (double)p_top ? 0.0 : (x - (double)p_top) * cool) - log(p_whole);
    }
    // earlier children of the same token: whether one has the same token; the mass of the others
    bool twice = false;
    double gone = 0.0;
    uint64_t before = 0;
    if (a.parents)
        for (int i = 1; i < n - 1; ++i) {
            const int iu = __builtin_amdgcn_readlane(up, i), it = __builtin_amdgcn_readlane(tok, i);
            const double ip = lane_f64(twice ? 0.0 : p, i);  // (lane i is through with its own: i' < i)
            if (c > i && up >= 0 && iu == up) {
                before |= 1ull << i;
                gone += ip;
                twice = twice || it == tok;
            }
        }
    bool ok;
    if (heat == 0.0f) {
        ok = known && tok == p_arg;
    } else {
        const double u = live ? (double)a.uniform[(int64_t)b * (a.n_q + 1) + c] : 0.0;
        if (a.draft)
            ok = known && u * (double)fmaxf(element<WIDE>(a.draft + b * a.q_nb2 + up * a.q_nb1, tok), 0.0f) < p;
        else
            ok = known && !twice && u * (1.0 - gone) < p;
    }
    if (c == 0) ok = live;
    const uint64_t oks = __builtin_amdgcn_ballot_w64(ok);
    const uint64_t chosen = __builtin_amdgcn_ballot_w64(ok && !(before & oks));
    // on the path: chosen, and so are all tokens above
    uint64_t above = 1ull << c;
    int at = up;
#pragma unroll
    for (int d = 0; d < 6; ++d) {
        const int l = at < 0 ? c : at;
        above |= shfl64(above, l);
        const int q = __shfl(at, l);
        at = at < 0 ? -1 : q;
    }
    const uint64_t on = __builtin_amdgcn_ballot_w64(live && (above & 1) && !(above & ~chosen));
    const int len = __builtin_popcountll(on), last = on ? 63 - __builtin_clzll(on) : 0;
    Walk w;
    w.n = len;
    w.at = len ? last : -1;
    w.kids = __builtin_amdgcn_ballot_w64(live && up >= 0 && up == last) & (len ? ~0ull : 0ull);
    w.max = (double)__shfl(top, last);
    w.cool = cool;
    w.whole = shfl_f64(whole, last);
    const int last_arg = __shfl(arg, last);
    if (write) {
        const int64_t r = (int64_t)b * a.n_q;
        if (c < a.n_q) {
            const int rank = __builtin_popcountll(on & ((1ull << c) - 1));
            if (c >= len) a.path[r + c] = -1;
            if (on >> c & 1) a.path[r + rank] = c;
            if (a.logp) a.logp[(int64_t)b * (a.n_q + 1) + c] = live && up >= 0 ? (float)lp : 0.0f;
        }
        if (c == 0) a.n_path[b] = len;
    }
    if (heat == 0.0f || !len || !(w.max > -INFINITY)) {
        // nothing is drawn
        const int v = len && heat == 0.0f ? last_arg : -1;
        if (write && c == 0) {
            a.next[b] = v;
            if (a.logp) a.logp[(int64_t)b * (a.n_q + 1) + a.n_q] = v >= 0 ? (float)-log(w.whole) : len ? -INFINITY : 0.0f;
        }
        w.at = -1;
    }
    return w;
}

// Whether element i of the chunk is none of the rejected tokens.
XQ_DEV bool kept(const uint32_t* hit, int i) { return !(hit[i >> 5] >> (i & 31) & 1u); }

// The sum of n numbers, the same in all lanes; the order is fixed.
XQ_DEV double wave_total(const double* x, int n) {
    double s = 0.0;
    for (int i = lane_id(); i < n; i += 64) s += x[i];
#pragma unroll
    for (int d = 1; d < 64; d *= 2) s += shfl_f64(s, lane_id() ^ d);
    return s;
}
// Sums of this lane's and all lower lanes' numbers.
XQ_DEV double wave_upto(double x) {
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
        const double y = shfl_f64(x, lane_id() >= s ? lane_id() - s : lane_id());
        if (lane_id() >= s) x += y;
    }
    return x;
}

// The tokens (`tok`, of thread i's child i) of `kids` among the N elements from v0 on, as bits.
template <int N>
XQ_DEV void mark_kids(uint64_t kids, int tok, int v0, uint32_t* hit) {
    for (int i = threadIdx.x; i < N / 32; i += blockDim.x) hit[i] = 0;
    __syncthreads();
    if (threadIdx.x < 64 && (kids >> threadIdx.x & 1)) {
        const int64_t t = (int64_t)tok - v0;
        if (t >= 0 && t < N) atomicOr(&hit[t >> 5], 1u << (t & 31));
    }
    __syncthreads();
}

// PART 0: the path, and the sums of a chunk of the row that the next token is drawn from: of its weights
// and, without a draft, of what is left of them. PART 1: with a draft, the sum of what is left.
template <bool WIDE, int PART>
__global__ __launch_bounds__(kSumThreads) void verify_sums_kernel(VerifyArgs a) {
    __shared__ Walk shared;
    __shared__ double lds[kVParts];
    __shared__ uint32_t hit[kVSum / 32];
    const int j = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, v0 = j * kVSum;
    if constexpr (PART == 0) {
        if (wave_id() == 0) {
            const Walk w = walk_path<WIDE>(a, b, j == 0);
            if (tid == 0) shared = w;
            if (tid == 0 && j == 0) a.walk[b] = w;
        }
    } else {
        if (tid == 0) shared = a.walk[b];
    }
    __syncthreads();
    const Walk w = shared;
    if (w.at < 0) return;
    const uint8_t* row = a.logits + b * a.l_nb2 + w.at * a.l_nb1;
    const uint8_t* q = a.draft && w.kids ? a.draft + b * a.q_nb2 + w.at * a.q_nb1 : nullptr;
    if (PART == 1 && !q) return;
    double sum = 0.0;
    if constexpr (PART == 1) sum = wave_total(a.sums + (int64_t)b * a.sum_chunks, a.sum_chunks);
    const int v = v0 + tid * kSumEach;
    float x[kSumEach], y[kSumEach];
    eight<WIDE>(row, v, a.V, x);
    if constexpr (PART == 1) eight<WIDE>(q, v, a.V, y);
    else mark_kids<kVSum>(w.kids, tid < a.n_q ? a.tokens[(int64_t)b * a.n_q + tid] : -1, v0, hit);
    double all = 0.0, left = 0.0;
#pragma unroll
    for (int i = 0; i < kSumEach; ++i) {
        const double p = weight_f64(x[i], w.max, w.cool);
        if constexpr (PART == 0) {
            all += p;
            left += kept(hit, v - v0 + i) ? p : 0.0;
        } else if (v + i < a.V) {
            left += fmax(p / sum - (double)fmaxf(y[i], 0.0f), 0.0);
        }
    }
    const int64_t of_p = (int64_t)b * a.sum_chunks + j, of_rest = ((int64_t)a.B + b) * a.sum_chunks + j;
    if constexpr (PART == 0) {
        all = block_sum(all, lds, a.parts + of_p * kVParts);
        if (tid == 0) a.sums[of_p] = all;
    }
    if (PART == 1 || !q) {
        left = block_sum(left, lds, a.parts + of_rest * kVParts);
        if (tid == 0) a.sums[of_rest] = left;
    }
}

// The next token, by one wave: its chunk by the chunks' sums, its part by the parts', then its place in the part.
template <bool WIDE>
__global__ __launch_bounds__(64) void verify_pick_kernel(VerifyArgs a) {
    constexpr int E = kVPart / 64;
    __shared__ uint32_t hit[kVPart / 32];
    const int b = blockIdx.x, lane = lane_id();
    Walk w = a.walk[b];
    const float uf = a.uniform[(int64_t)b * (a.n_q + 1) + a.n_q];
    const int tok = lane < a.n_q ? a.tokens[(int64_t)b * a.n_q + lane] : -1;
    int64_t at = (int64_t)b * a.sum_chunks;
    const int64_t rest = (int64_t)a.B * a.sum_chunks;
    const double sum = wave_total(a.sums + at, a.sum_chunks);
    if (w.at < 0) return;
    double whole = wave_total(a.sums + rest + at, a.sum_chunks);
    const uint8_t* row = a.logits + b * a.l_nb2 + w.at * a.l_nb1;
    const uint8_t* q = a.draft && w.kids ? a.draft + b * a.q_nb2 + w.at * a.q_nb1 : nullptr;
    if (whole > 0.0) {
        at += rest;
    } else {  // nothing is left: the target's distribution
        whole = sum;
        q = nullptr;
        w.kids = 0;
    }
    const double aim = (uf > 0.0f ? (double)uf : 0.0) * whole;
    // the first of n numbers whose running sum exceeds the aim, else the last one with a mass; `run`: the sum before it
    double run = 0.0;
    auto reach = [&](const double* x, int n) {
        int found = 0;
        double next = run;
        for (int j0 = 0; j0 < n; j0 += 64) {
            const double mine = j0 + lane < n ? x[j0 + lane] : 0.0, upto = next + wave_upto(mine);
            const uint64_t massy = __builtin_amdgcn_ballot_w64(mine > 0.0), beyond = __builtin_amdgcn_ballot_w64(mine > 0.0 && upto > aim);
            if (massy) {
                const int l = beyond ? __builtin_ctzll(beyond) : 63 - __builtin_clzll(massy);
                found = j0 + l;
                run = l ? lane_f64(upto, l - 1) : next;
            }
            if (beyond) break;
            next = lane_f64(upto, 63);
        }
        return found;
    };
    const int chunk = reach(a.sums + at, a.sum_chunks);
    const int part = reach(a.parts + (at + chunk) * kVParts, kVParts);
    const int v0 = chunk * kVSum + part * kVPart, v = v0 + lane * E;
    float x[E], y[E];
    eight<WIDE>(row, v, a.V, x);
    if (q) eight<WIDE>(q, v, a.V, y);
    const double log_sum = a.logp ? log(sum) : 0.0;  // (while the row comes)
    mark_kids<kVPart>(w.kids, tok, v0, hit);
    double r[E], mine = 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const double p = weight_f64(x[e], w.max, w.cool);
        r[e] = q ? (v + e < a.V ? fmax(p / sum - (double)fmaxf(y[e], 0.0f), 0.0) : 0.0) : kept(hit, lane * E + e) ? p : 0.0;
        mine += r[e];
    }
    run += wave_upto(mine) - mine;
    int found = -1, any = -1;  // the lane's first element beyond the aim, its last one with a mass
#pragma unroll
    for (int e = 0; e < E; ++e) {
        run += r[e];
        if (r[e] > 0.0) {
            any = e;
            if (found < 0 && run > aim) found = e;
        }
    }
    const uint64_t beyond = __builtin_amdgcn_ballot_w64(found >= 0), massy = __builtin_amdgcn_ballot_w64(any >= 0);
    // (where the sums were rounded up: the last one)
    const int who = beyond ? __builtin_ctzll(beyond) : massy ? 63 - __builtin_clzll(massy) : 0;
    if (lane != who) return;
    const int e = beyond ? found : any;
    a.next[b] = e < 0 ? -1 : v + e;
    if (a.logp) {
        float l = -INFINITY;
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (i == e) l = x[i];
        const double d = l;
        a.logp[(int64_t)b * (a.n_q + 1) + a.n_q] = (float)((d == w.max ? 0.0 : (d - w.max) * w.cool) - log_sum);
    }
}

// ---------------------------------------------------------------- host

static xq_status verify_check(const xq_tensor* logits, const char* what) {
    if (!logits) return failf(XQ_ERR_BAD_ARG, "null %s", what);
    if (logits->type != XQ_TYPE_F32 && logits->type != XQ_TYPE_BF16) return failf(XQ_ERR_UNSUPPORTED, "%s must be F32 or BF16", what);
    for (int i = 0; i < 4; ++i)
        if (logits->ne[i] < 1 || logits->ne[i] > 0x7fffffff) return failf(XQ_ERR_BAD_SHAPE, "%s: bad ne", what);
    if (logits->ne[3] != 1) return failf(XQ_ERR_BAD_SHAPE, "%s must be [vocabulary, n_q, n_seq]", what);
    if (logits->ne[0] > (1 << 24)) return failf(XQ_ERR_UNSUPPORTED, "a vocabulary above 2^24");
    if (logits->ne[1] > kVerifyMax) return failf(XQ_ERR_UNSUPPORTED, "more than 64 tokens of a sequence");
    if (logits->ne[2] > 65535) return failf(XQ_ERR_UNSUPPORTED, "more than 65535 sequences");
    const size_t es = type_size(logits->type);
    if (logits->nb[0] != es) return failf(XQ_ERR_UNSUPPORTED, "%s: elements must be contiguous", what);
    if (logits->nb[1] % es || logits->nb[2] % es || !aligned(logits->data, es)) return failf(XQ_ERR_UNSUPPORTED, "misaligned %s", what);
    return XQ_OK;
}

static size_t verify_space(const xq_tensor* l, size_t* walk_at, size_t* sums_at) {
    const size_t chunks = (size_t)cdiv(l->ne[0], kVChunk), sums = (size_t)cdiv(l->ne[0], kVSum), B = (size_t)l->ne[2];
    *walk_at = B * (size_t)l->ne[1] * chunks * sizeof(RowStat);
    *sums_at = *walk_at + B * sizeof(Walk);
    return *sums_at + 2 * B * sums * (1 + kVParts) * 8;
}

template <bool WIDE>
static void verify_launch(const VerifyArgs& a, hipStream_t s) {
    launch("verify_stats", verify_stats_kernel<WIDE>, dim3((uint32_t)a.chunks, (uint32_t)a.n_q, (uint32_t)a.B), dim3(256), s, a);
    // (all greedy: the path and the maxima are the whole answer)
    launch("verify_sums", verify_sums_kernel<WIDE, 0>, dim3(a.uniform ? (uint32_t)a.sum_chunks : 1u, (uint32_t)a.B), dim3(kSumThreads), s, a);
    if (!a.uniform) return;
    if (a.draft) launch("verify_left", verify_sums_kernel<WIDE, 1>, dim3((uint32_t)a.sum_chunks, (uint32_t)a.B), dim3(kSumThreads), s, a);
    launch("verify_pick", verify_pick_kernel<WIDE>, dim3((uint32_t)a.B), dim3(64), s, a);
}

}  // namespace xq

using namespace xq;

extern "C" {

xq_status xq_verify_tokens_workspace(const xq_tensor* logits, size_t* bytes) {
    if (!bytes) return failf(XQ_ERR_BAD_ARG, "bytes is null");
    const xq_status st = verify_check(logits, "logits");
    if (st != XQ_OK) return st;
    size_t w, s;
    *bytes = verify_space(logits, &w, &s);
    return done_ok();
}

xq_status xq_verify_tokens(const xq_tensor* logits, const xq_tensor* draft, const int32_t* tokens, const int32_t* parents,
                           const int32_t* n_tok, const float* temperature, const float* uniform, int32_t* path, int32_t* n_path,
                           int32_t* next, float* logp, void* workspace, size_t workspace_bytes, void* stream) {
    xq_status st = verify_check(logits, "logits");
    if (st == XQ_OK && draft) st = verify_check(draft, "draft");
    if (st != XQ_OK) return st;
    if (draft) {
        if (draft->type != logits->type) return failf(XQ_ERR_UNSUPPORTED, "draft must have logits' type");
        for (int i = 0; i < 3; ++i)
            if (draft->ne[i] != logits->ne[i]) return failf(XQ_ERR_BAD_SHAPE, "draft must have logits' shape");
        if (parents) return failf(XQ_ERR_UNSUPPORTED, "a draft's distributions go with a chain: parents must be NULL");
        if (!uniform) return failf(XQ_ERR_BAD_ARG, "a draft's distributions need random numbers");
    }
    if (!logits->data || (draft && !draft->data) || !tokens || !path || !n_path || !next) return failf(XQ_ERR_BAD_ARG, "null pointer");
    for (const void* x : {(const void*)tokens, (const void*)parents, (const void*)n_tok, (const void*)temperature, (const void*)uniform,
                          (const void*)path, (const void*)n_path, (const void*)next, (const void*)logp})
        if (!aligned(x, 4)) return failf(XQ_ERR_UNSUPPORTED, "misaligned pointer");
    size_t walk_at, sums_at;
    const size_t need = verify_space(logits, &walk_at, &sums_at);
    if (!workspace || workspace_bytes < need) return failf(XQ_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    if (!aligned(workspace, 256)) return failf(XQ_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    VerifyArgs a{};
    a.logits = (const uint8_t*)logits->data;
    a.l_nb1 = (int64_t)logits->nb[1], a.l_nb2 = (int64_t)logits->nb[2];
    if (draft) {
        a.draft = (const uint8_t*)draft->data;
        a.q_nb1 = (int64_t)draft->nb[1], a.q_nb2 = (int64_t)draft->nb[2];
    }
    a.tokens = tokens, a.parents = parents, a.n_tok = n_tok, a.temperature = temperature, a.uniform = uniform;
    a.path = path, a.n_path = n_path, a.next = next, a.logp = logp;
    a.V = (int32_t)logits->ne[0], a.n_q = (int32_t)logits->ne[1], a.B = (int32_t)logits->ne[2];
    a.chunks = (int32_t)cdiv(a.V, kVChunk), a.sum_chunks = (int32_t)cdiv(a.V, kVSum);
    a.stats = (RowStat*)workspace;
    a.walk = (Walk*)((uint8_t*)workspace + walk_at);
    a.sums = (double*)((uint8_t*)workspace + sums_at);
    a.parts = a.sums + 2 * (size_t)a.B * (size_t)a.sum_chunks;
    hipStream_t s = (hipStream_t)stream;
    logits->type == XQ_TYPE_F32 ? verify_launch<true>(a, s) : verify_launch<false>(a, s);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return failf(XQ_ERR_HIP, "verify_tokens launch: %s", hipGetErrorString(e));
    return done_ok();
}

}  // extern "C"
