// xq_tile.h — pieces of a cached row as f16 matrix operands, and what the kernels over the paged
// cache share on the way there.
#pragma once

#include "xq_kv_codec.h"
#include "xq_paged.h"

namespace xq {

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

// A number that every lane has, in a scalar register: what is formed from it stays scalar.
XQ_DEV uint32_t uniform(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }

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

}  // namespace xq
