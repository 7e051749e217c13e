// xq_kv.hip — KV append: F32 rows -> KV cache records at row positions.
//
// The scatter of shaders/rkva/rkva_store_f16.hlsl:63-85 (F32 -> ggml F16 RNE at
// absolute positions) widened to every KV storage type of this path, with
// ggml's block quantizers reproduced bit for bit:
//   Q8_0  quantize_row_q8_0 (x86: id = 127/amax, round half to even) or
//         quantize_row_q8_0_ref (id = 1/d, roundf);
//   Q4_0  quantize_row_q4_0_ref (d = max/-8 with max the first element of
//         largest magnitude, q = min(15, (int8)(x*id + 8.5)));
//   E5M2  f16 RNE then E5M2 RNE with finite saturation (the Q/OUT wire codec of
//         shaders/rkva/rkva_range_bulk_f16.hlsl:156-167).
// Built with -ffp-contract=off so the q4_0 "x*id + 8.5" rounds twice, as the CPU
// reference does.
#include "xq_kv_codec.h"

namespace xq {

// Bound by HBM: 5/4 of the f32 source for q8_0. One lane converts four
// consecutive elements: a wave's load is 1 KiB of contiguous source, and a
// 32-element block is eight lanes, whose maximum takes three DPP steps and no
// LDS. UN such 256-element units per wave, every load issued before the first is
// used. 8192 tokens x 4 heads x 256 to q8_0 (42.5 MB): 9.2 us per launch (4.6
// TB/s), against 30 us with one lane per 32-element block behind an LDS copy of
// the record (one record per wave, eight of its 64 lanes at work).
template <int KT, int D, int UN>
__global__ __launch_bounds__(256) void kv_store_kernel(const float* __restrict__ src,
                                                       const int32_t* __restrict__ positions,
                                                       uint32_t n_rec, uint32_t n_head_kv,
                                                       int32_t q8_variant, uint8_t* __restrict__ dst,
                                                       int32_t capacity) {
    constexpr int REC = KT == XQ_TYPE_BF16 ? 2 * D : rec_bytes(KT, D);
    constexpr uint32_t RPU = 256 / D;  // records per unit
    constexpr uint32_t LPR = D / 4;    // lanes per record
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t unit0 = (blockIdx.x * 4u + threadIdx.x / 64u) * UN;
    const uint32_t el = 4u * (lane % LPR);  // first element in the record
    f4u x[UN];
    int32_t pos[UN];
    uint32_t head[UN];
#pragma unroll
    for (int i = 0; i < UN; ++i) {
        const uint32_t rec = (unit0 + i) * RPU + lane / LPR;
        const bool ok = rec < n_rec;
        const uint32_t t = ok ? rec / n_head_kv : 0u;
        head[i] = ok ? rec - t * n_head_kv : 0u;
        x[i] = *(const f4u*)(src + (int64_t)(ok ? rec : 0u) * D + el);
        pos[i] = ok ? positions[t] : -1;
    }
#pragma unroll
    for (int i = 0; i < UN; ++i) {
        const bool live = pos[i] >= 0 && pos[i] < capacity;
        uint8_t* y = dst + ((int64_t)pos[i] * n_head_kv + head[i]) * REC;
        kv_put4<KT>(x[i], lane, el, q8_variant, y, live);
    }
}

template <int KT, int D>
static void kv_store_dispatch(const float* src, const int32_t* positions, int64_t n_rec, int32_t n_head_kv,
                              int32_t q8_variant, uint8_t* dst, int32_t capacity, hipStream_t stream) {
    const int64_t units = (n_rec + 256 / D - 1) / (256 / D);
    // Records of 16 and 32 bits per element: four units per wave once that still gives
    // every CU four workgroups. The narrower ones, whose conversion takes longer than
    // their loads, one unit whatever the size: more waves hide it better. us per append
    // of K and V, 4 heads x 256, with 1 / 2 / 4 units:
    //   tokens       f16               f32               e5m2              q8_0              q4_0
    //   3000    8.2  8.5  8.6   10.1 10.4 10.3    9.4  9.8 10.4    9.2  9.3 10.1    9.1  9.3  9.7
    //   6000   15.8 15.5 15.5   18.7 18.1 17.3   15.8 17.2 17.9   15.2 16.6 17.8   15.4 16.3 17.1
    //   8192   20.8 19.8 18.9   23.7 23.0 22.1   19.7 20.7 22.4   19.0 20.2 21.6   18.8 19.6 20.9
    //   16384  35.2 33.1 33.2   43.2 41.3 45.4   32.8 34.0 35.4   31.4 32.7 34.2   31.7 32.5 31.7
    constexpr bool wide = KT == XQ_TYPE_F32 || KT == XQ_TYPE_F16 || KT == XQ_TYPE_BF16;
    if constexpr (wide) {
        if (units >= 256 * 4 * 4 * 4) {
            launch("kv_store", kv_store_kernel<KT, D, 4>, dim3((uint32_t)((units + 15) / 16)), dim3(256), stream, src,
                   positions, (uint32_t)n_rec, (uint32_t)n_head_kv, q8_variant, dst, capacity);
            return;
        }
    }
    launch("kv_store", kv_store_kernel<KT, D, 1>, dim3((uint32_t)((units + 3) / 4)), dim3(256), stream, src,
           positions, (uint32_t)n_rec, (uint32_t)n_head_kv, q8_variant, dst, capacity);
}

template <int KT>
static hipError_t kv_store_type(int32_t head_dim, const float* src, const int32_t* positions, int64_t n_rec,
                                int32_t n_head_kv, int32_t q8_variant, uint8_t* dst, int32_t capacity,
                                hipStream_t stream) {
    switch (head_dim) {
    case 64: kv_store_dispatch<KT, 64>(src, positions, n_rec, n_head_kv, q8_variant, dst, capacity, stream); break;
    case 128: kv_store_dispatch<KT, 128>(src, positions, n_rec, n_head_kv, q8_variant, dst, capacity, stream); break;
    case 256: kv_store_dispatch<KT, 256>(src, positions, n_rec, n_head_kv, q8_variant, dst, capacity, stream); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t kv_store_launch(const float* src, const int32_t* positions, int32_t n_tokens,
                           int32_t n_head_kv, int32_t head_dim, int32_t kv_type,
                           int32_t q8_variant, void* dst, int32_t capacity, hipStream_t stream) {
    const int64_t n_rec = (int64_t)n_tokens * n_head_kv;
    if (n_rec == 0) return hipSuccess;
    uint8_t* y = (uint8_t*)dst;
    switch (kv_type) {
    case XQ_TYPE_F32: return kv_store_type<XQ_TYPE_F32>(head_dim, src, positions, n_rec, n_head_kv, q8_variant, y, capacity, stream);
    case XQ_TYPE_F16: return kv_store_type<XQ_TYPE_F16>(head_dim, src, positions, n_rec, n_head_kv, q8_variant, y, capacity, stream);
    case XQ_TYPE_BF16: return kv_store_type<XQ_TYPE_BF16>(head_dim, src, positions, n_rec, n_head_kv, q8_variant, y, capacity, stream);
    case XQ_TYPE_E5M2: return kv_store_type<XQ_TYPE_E5M2>(head_dim, src, positions, n_rec, n_head_kv, q8_variant, y, capacity, stream);
    case XQ_TYPE_Q8_0: return kv_store_type<XQ_TYPE_Q8_0>(head_dim, src, positions, n_rec, n_head_kv, q8_variant, y, capacity, stream);
    case XQ_TYPE_Q4_0: return kv_store_type<XQ_TYPE_Q4_0>(head_dim, src, positions, n_rec, n_head_kv, q8_variant, y, capacity, stream);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace xq
