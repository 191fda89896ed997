// e4m3 helpers: group scales as powers of two, packing, unpacking.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace moe {

// Bits of the largest finite |f| of eight values (0 if there is none); special: an infinity or NaN is among them.
__device__ __forceinline__ uint32_t f8_top(const float (&f)[8], bool& special) {
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 8; k++) top = max(top, __float_as_uint(f[k]) & 0x7fffffffu);
    special = top >= 0x7f800000u;
    if (special) {
        top = 0;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const uint32_t a = __float_as_uint(f[k]) & 0x7fffffffu;
            if (a < 0x7f800000u) top = max(top, a);
        }
    }
    return top;
}
// The same of eight bf16 values, two at a time.
__device__ __forceinline__ uint32_t f8_top(uint4 v, bool& special) {
    const uint32_t w[4] = {v.x & 0x7fff7fffu, v.y & 0x7fff7fffu, v.z & 0x7fff7fffu, v.w & 0x7fff7fffu};
    const uint32_t m = __vmaxu2(__vmaxu2(w[0], w[1]), __vmaxu2(w[2], w[3]));
    uint32_t top = max(m >> 16, m & 0xffffu);
    special = top >= 0x7f80u;
    if (special) {
        top = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t lo = w[k] & 0xffffu, hi = w[k] >> 16;
            if (lo < 0x7f80u) top = max(top, lo);
            if (hi < 0x7f80u) top = max(top, hi);
        }
    }
    return top << 16;
}

// Biased exponent of the smallest power of two s >= 2^-126 with the value of bits `top` <= 448 s
// (448 = 1.75 * 2^8); s = 1 for zero.
__device__ __forceinline__ uint32_t f8_scale_exp(uint32_t top) {
    const int e = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    return top == 0 ? 127u : (uint32_t)max(e, 1);
}
// 1 / s, exact (the exponent of s is at most 247, so 1 / s is a normal number).
__device__ __forceinline__ float f8_inverse(uint32_t se) { return __uint_as_float((254u - se) << 23); }

// e4m3(lo) in the low byte, e4m3(hi) in the high byte; finite values beyond the range saturate.
__device__ __forceinline__ uint32_t f8_pack2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// x * inv rounded to e4m3; where `special`, an infinity becomes NaN instead of saturating.
__device__ __forceinline__ uint2 f8_pack8(const float (&f)[8], float inv, bool special) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = f[k] * inv;
    if (special)
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (fabsf(v[k]) == __int_as_float(0x7f800000)) v[k] = __int_as_float(0x7fffffff);
    return make_uint2(f8_pack2(v[0], v[1]) | f8_pack2(v[2], v[3]) << 16, f8_pack2(v[4], v[5]) | f8_pack2(v[6], v[7]) << 16);
}
__device__ __forceinline__ uint32_t f8_pack1(float f, float inv) {
    float v = f * inv;
    if (fabsf(v) == __int_as_float(0x7f800000)) v = __int_as_float(0x7fffffff);
    return f8_pack2(v, 0.f) & 0xffu;
}

// Two floats rounded to bf16 (ties to even, NaN stays NaN), lo in the low half.
__device__ __forceinline__ uint32_t f8_bf16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint16_t f8_bf16(float v) { return (uint16_t)f8_bf16x2(v, 0.f); }

// The two e4m3 values of a 16-bit word as floats (both conversions exact).
__device__ __forceinline__ void f8_unpack2(uint32_t w, float& lo, float& hi) {
    asm("{\n\t.reg .b32 h;\n\t.reg .b16 a, b, c;\n\t"
        "cvt.u16.u32 c, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 h, c;\n\t"
        "mov.b32 {a, b}, h;\n\t"
        "cvt.f32.f16 %0, a;\n\t"
        "cvt.f32.f16 %1, b;\n\t}"
        : "=f"(lo), "=f"(hi)
        : "r"(w));
}
__device__ __forceinline__ void f8_unpack16(uint4 w, float (&f)[16]) {
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < 4; k++) {
        f8_unpack2(a[k] & 0xffffu, f[4 * k], f[4 * k + 1]);
        f8_unpack2(a[k] >> 16, f[4 * k + 2], f[4 * k + 3]);
    }
}

}  // namespace moe
