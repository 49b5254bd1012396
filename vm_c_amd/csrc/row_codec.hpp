// row_codec.hpp -- device pieces of the kernels that keep a K or V row in
// registers, 8 values a lane, and append it to the paged cache: 16-bit packing
// and the GGUF block encoders over 4 lanes.
#pragma once

#include "kv_quant.hpp"

namespace vmc {
namespace {

// The fp32 result is materialised before the conversion (opaque): otherwise
// fp16(u * w) becomes one v_fma_mix, a single rounding of the exact product
// where the declared order rounds to fp32 first.
template <bool BF16>
__device__ __forceinline__ float round_half(float x) {
    return half_to_f32<BF16>(f32_to_half<BF16>(opaque(x)));
}

template <bool BF16>
__device__ __forceinline__ u32x4 pack8(const float* x) {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        w[e] = (uint32_t)f32_to_half<BF16>(opaque(x[2 * e])) |
               ((uint32_t)f32_to_half<BF16>(opaque(x[2 * e + 1])) << 16);
    return w;
}

// q8_0 / q4_0 block of 32 values held by lanes 4b .. 4b+3 (lane l: values
// 8l .. 8l+7); the encoders of kv_quant.hpp, element for element
template <int FMT>
__device__ __forceinline__ void gguf_block4(const float* x, int j, uint8_t* entry, bool write) {
    const int l = j & 3, ib = j >> 2;
    if constexpr (FMT == VMC_KV_Q8_0) {
        float amax = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x[e]));
        amax = fmaxf(amax, row_xor<1>(amax, j));
        amax = fmaxf(amax, row_xor<2>(amax, j));
        const float d = opaque(amax / 127.0f);
        const float id = d != 0.0f ? 1.0f / d : 0.0f;
        if (write) {
            uint16_t* d16 = reinterpret_cast<uint16_t*>(entry + 34 * ib);
            if (l == 0) d16[0] = f32_to_f16_bits(d);
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const int q0 = (int)roundf(x[e] * id);
                const int q1 = (int)roundf(x[e + 1] * id);
                d16[1 + 4 * l + e / 2] = (uint16_t)((q0 & 0xff) | ((q1 & 0xff) << 8));
            }
        }
    } else {
        // signed value of the first largest |x| (index order)
        float amax = 0.0f, mx = 0.0f;
        int idx = 1 << 20;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float a = fabsf(x[e]);
            if (amax < a) {
                amax = a;
                mx = x[e];
                idx = 8 * l + e;
            }
        }
        static_for<2>([&](auto m) {
            constexpr int M = 1 << decltype(m)::value;
            const float a2 = row_xor<M>(amax, j);
            const float x2 = row_xor<M>(mx, j);
            const int i2 = row_xor<M>(idx, j);
            if (a2 > amax || (a2 == amax && i2 < idx)) {
                amax = a2;
                mx = x2;
                idx = i2;
            }
        });
        const float d = opaque(mx / -8.0f);
        const float id = d != 0.0f ? 1.0f / d : 0.0f;
        uint32_t q[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x0 = __fmul_rn(x[e], id);
            const int t0 = (int)(int8_t)(int)__fadd_rn(x0, 8.5f);
            q[e] = (uint32_t)(t0 < 15 ? t0 : 15);
        }
        // byte i = value i | value i + 16 << 4: lanes 0, 1 take lanes 2, 3's codes
        uint32_t lo = 0, hi = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            lo |= q[e] << (8 * e);
            hi |= q[e + 4] << (8 * e);
        }
        const uint32_t plo = row_xor_u32<2>(lo, j);
        const uint32_t phi = row_xor_u32<2>(hi, j);
        if (write) {
            uint16_t* d16 = reinterpret_cast<uint16_t*>(entry + 18 * ib);
            if (l == 0) d16[0] = f32_to_f16_bits(d);
            if (l < 2) {
                const uint32_t w0 = lo | (plo << 4), w1 = hi | (phi << 4);
                d16[1 + 4 * l] = (uint16_t)(w0 & 0xffffu);
                d16[2 + 4 * l] = (uint16_t)(w0 >> 16);
                d16[3 + 4 * l] = (uint16_t)(w1 & 0xffffu);
                d16[4 + 4 * l] = (uint16_t)(w1 >> 16);
            }
        }
    }
}

template <bool BF16>
__device__ __forceinline__ void unpack8(const u32x4 w, float* x) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x[2 * e] = half_to_f32<BF16>((uint16_t)(w[e] & 0xffffu));
        x[2 * e + 1] = half_to_f32<BF16>((uint16_t)(w[e] >> 16));
    }
}

}  // namespace
}  // namespace vmc
