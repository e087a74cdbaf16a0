// kv_common.cuh -- the 8-bit paged key/value cache shared by its kernels.
//
// Cache layout: codes [pages][kv_heads][page][dim], one byte each (e4m3 or
// int8), and one power-of-two scale per (page, kv head): value = code * scale.
// A (page, head) tile is page * dim contiguous bytes.
//
// Scale of a tile with largest magnitude a: the smallest 2^e with
// a <= QMAX * 2^e (QMAX = 448 for e4m3, 127 for int8), e kept in
// [kScaleExpLo, kScaleExpHi].  A power of two costs at most one bit of the
// 8-bit range, and buys this: a code is x * 2^-e rounded ONCE (the product is
// exact), and when a later token raises the scale of a part-filled page, the
// page's e4m3 codes move to the new scale exactly unless they become
// subnormal (int8 codes are rounded once more).
#pragma once

#include <cuda_fp8.h>

#include "exl3_common.cuh"

namespace exl3 {

constexpr int kScaleExpLo = -40, kScaleExpHi = 40;

template <bool E4M3>
__device__ __forceinline__ int scale_exponent(float amax) {
    // amax = 1.m * 2^ex; 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6
    const int bits = __float_as_int(amax);
    const int ex = (bits >> 23) - 127, m = bits & 0x7fffff;
    const int e = E4M3 ? (m <= 0x600000 ? ex - 8 : ex - 7) : (m <= 0x7e0000 ? ex - 6 : ex - 5);
    return amax > 0.f ? min(max(e, kScaleExpLo), kScaleExpHi) : kScaleExpLo;
}

__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

// exponent of a stored scale; anything a cache cannot hold is brought into range
__device__ __forceinline__ int stored_exponent(float scale) {
    return min(max(((__float_as_int(scale) >> 23) & 0xff) - 127, kScaleExpLo), kScaleExpHi);
}

// Four values to four codes (to nearest, ties to even; beyond the range to
// the range's end).  NaN stays NaN in e4m3; int8 has none and takes 0.
template <bool E4M3>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    if constexpr (E4M3) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
        return lo | (hi << 16);
    } else {
        auto q = [](float v) { return uint32_t(__float2int_rn(fminf(fmaxf(v == v ? v : 0.f, -127.f), 127.f))) & 0xffu; };
        return q(a) | (q(b) << 8) | (q(c) << 16) | (q(d) << 24);
    }
}

// two e4m3 codes (the low, the high 16 bits) as f16x2, exact
__device__ __forceinline__ uint32_t e4m3x2_lo(uint32_t v) {
    uint32_t r;
    asm("{\n .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %1;\n cvt.rn.f16x2.e4m3x2 %0, lo;\n}\n" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t e4m3x2_hi(uint32_t v) {
    uint32_t r;
    asm("{\n .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %1;\n cvt.rn.f16x2.e4m3x2 %0, hi;\n}\n" : "=r"(r) : "r"(v));
    return r;
}

template <bool E4M3>
__device__ __forceinline__ void decode4(uint32_t w, float (&v)[4]) {
    if constexpr (E4M3) {
        const uint32_t lo = e4m3x2_lo(w), hi = e4m3x2_hi(w);
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
    } else {
        #pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = float(int8_t(w >> (8 * i)));
    }
}

}  // namespace exl3
