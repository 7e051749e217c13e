// xq_kv_codec.h — four f32 elements of a KV record per lane into the record's storage
// format, ggml's block quantizers bit for bit (shared by the KV append and the
// norm-and-rotation kernel). The including file is built with -ffp-contract=off.
#pragma once

#include "xq_kernels.h"

namespace xq {

XQ_DEV uint32_t f16_to_e5m2(uint32_t h) {
    const uint32_t sign = (h >> 8) & 0x80u;
    if ((h & 0x7c00u) == 0x7c00u) {
        if (!(h & 0x03ffu)) return sign | 0x7cu;
        const uint32_t top = (h >> 8) & 3u;
        return sign | 0x7cu | (top ? top : 1u);
    }
    uint32_t mag = h & 0x7fffu;
    if (mag > 0x7b00u) mag = 0x7b00u;
    return sign | ((mag + 0x7fu + ((mag >> 8) & 1u)) >> 8);
}

XQ_DEV uint32_t f32_to_bf16_bits(float x) {
    const uint32_t u = __float_as_uint(x);
    if ((u & 0x7fffffffu) > 0x7f800000u) return ((u >> 16) | 64u) & 0xffffu;
    return ((u + (0x7fffu + ((u >> 16) & 1u))) >> 16) & 0xffffu;
}

// Unaligned-tolerant vectors: the caller's rows and planes need not be aligned
// beyond their elements (gfx950 global accesses take any alignment).
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32u __attribute__((aligned(1)));
typedef uint16_t u16u __attribute__((aligned(1)));
typedef uint32_t u32x2u __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(1)));

// Lane `lane` holds elements el .. el + 3 (el = 4 * its place in its record; eight
// neighbouring lanes, aligned to eight, hold a 32-element block) of the record at y;
// `live` lanes store. Every lane of the wave takes part (DPP, shuffle).
template <int KT>
XQ_DEV void kv_put4(const f4u x, uint32_t lane, uint32_t el, int32_t q8_variant, uint8_t* y, bool live) {
    float amax = 0.0f, vmax = 0.0f;
    if constexpr (KT == XQ_TYPE_Q8_0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) amax = fabsf(x[j]) > amax ? fabsf(x[j]) : amax;  // skips every NaN
        amax = fmaxf(amax, dpp<0xB1>(amax));
        amax = fmaxf(amax, dpp<0x4E>(amax));
        amax = fmaxf(amax, dpp<0x141>(amax));
    } else if constexpr (KT == XQ_TYPE_Q4_0) {
        // the first element of the largest magnitude: of two halves the later
        // one wins only when it is strictly larger
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float m = fabsf(x[j]);
            if (amax < m) {
                amax = m;
                vmax = x[j];
            }
        }
        auto fold = [&](float oa, float ov, bool first) {  // first: this lane's half comes first
            const bool take = first ? amax < oa : !(oa < amax);
            amax = take ? oa : amax;
            vmax = take ? ov : vmax;
        };
        fold(dpp<0xB1>(amax), dpp<0xB1>(vmax), !(lane & 1u));
        fold(dpp<0x4E>(amax), dpp<0x4E>(vmax), !(lane & 2u));
        fold(dpp<0x141>(amax), dpp<0x141>(vmax), !(lane & 4u));
    }
    if constexpr (KT == XQ_TYPE_F32) {
        if (live) *(u32x4u*)(y + 4 * el) = __builtin_bit_cast(u32x4u, x);
    } else if constexpr (KT == XQ_TYPE_F16 || KT == XQ_TYPE_BF16) {
        uint32_t h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = KT == XQ_TYPE_F16 ? f32_to_f16_bits(x[j]) : f32_to_bf16_bits(x[j]);
        if (live) *(u32x2u*)(y + 2 * el) = u32x2u{h[0] | (h[1] << 16), h[2] | (h[3] << 16)};
    } else if constexpr (KT == XQ_TYPE_E5M2) {
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) w |= f16_to_e5m2(f32_to_f16_bits(x[j])) << (8 * j);
        if (live) *(u32u*)(y + el) = w;
    } else if constexpr (KT == XQ_TYPE_Q8_0) {
        const float d = amax / 127.0f;
        float id;
        if (q8_variant == 0)
            id = amax != 0.0f ? 127.0f / amax : 0.0f;
        else
            id = d != 0.0f ? 1.0f / d : 0.0f;
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float tq = x[j] * id;
            const float r = q8_variant == 0 ? rintf(tq) : roundf(tq);
            w |= (uint32_t)(uint8_t)(int8_t)(int)r << (8 * j);
        }
        uint8_t* yb = y + el / kQK * 34;
        if (live) {
            *(u32u*)(yb + 2 + el % kQK) = w;
            if (!(lane & 7u)) *(u16u*)yb = (uint16_t)f32_to_f16_bits(d);
        }
    } else {
        const float d = vmax / -8.0f;
        const float id = d != 0.0f ? 1.0f / d : 0.0f;
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            int n = (int8_t)(x[j] * id + 8.5f);
            n = n > 15 ? 15 : n;
            w |= (uint32_t)(uint8_t)n << (8 * j);
        }
        // byte j of the block holds element j low and element 16 + j high: lanes
        // 0..3 of a block take their partner's (lane + 4) nibbles
        const uint32_t hi = (uint32_t)__shfl_xor((int)w, 4);
        uint8_t* yb = y + el / kQK * 18;
        if (live && !(lane & 4u)) {
            *(u32u*)(yb + 2 + el % kQK) = w | ((hi & 0x0f0f0f0fu) << 4);
            if (!(lane & 7u)) *(u16u*)yb = (uint16_t)f32_to_f16_bits(d);
        }
    }
}

// The same with the type known at run time (the same for the whole wave).
XQ_DEV void kv_put4_any(int32_t kt, const f4u x, uint32_t lane, uint32_t el, int32_t q8_variant, uint8_t* y, bool live) {
    switch (kt) {
    case XQ_TYPE_F32: kv_put4<XQ_TYPE_F32>(x, lane, el, q8_variant, y, live); break;
    case XQ_TYPE_F16: kv_put4<XQ_TYPE_F16>(x, lane, el, q8_variant, y, live); break;
    case XQ_TYPE_BF16: kv_put4<XQ_TYPE_BF16>(x, lane, el, q8_variant, y, live); break;
    case XQ_TYPE_E5M2: kv_put4<XQ_TYPE_E5M2>(x, lane, el, q8_variant, y, live); break;
    case XQ_TYPE_Q8_0: kv_put4<XQ_TYPE_Q8_0>(x, lane, el, q8_variant, y, live); break;
    default: kv_put4<XQ_TYPE_Q4_0>(x, lane, el, q8_variant, y, live); break;
    }
}

}  // namespace xq
