// 8-bit floats (e4m3) with one float32 scale for each block of 128: the arithmetic of a block, which every kernel that ends in them shares.
//
// A block v becomes q and s with q * s near v: a = max |v|, s = a / 448, q = e4m3(v * (448 / a)), ties to even, so the largest element
// becomes 448 or -448.  A block of zeros has s = 0.  A block that holds an infinity or NaN has s = NaN and q = 0: all that is formed
// from it is NaN, as it would be without the rounding.  The maximum is taken over the bits of |v| as unsigned integers, which order
// like the values and put NaN on top.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

#define FP8_TOP 448.f

// What a block's largest magnitude (its bits) makes of it.
struct Fp8Scale {
    float scale, inverse, before;  // q = e4m3((v * before) * inverse)
    uint32_t keep;                 // 0: the block's values are written as zeros
};
__device__ __forceinline__ Fp8Scale fp8_scale(uint32_t top) {
    Fp8Scale r;
    const float a = __uint_as_float(top);
    const bool finite = top < 0x7f800000u, fine = finite && top > 0;
    r.before = a < 0x1p-100f ? 0x1p64f : 1.f;  // 448 / a stays finite (and the product with `before` is exact)
    r.inverse = fine ? __fdiv_rn(FP8_TOP, a * r.before) : 0.f;
    r.scale = finite ? __fdiv_rn(a, FP8_TOP) : __uint_as_float(0x7fffffffu);
    r.keep = fine ? 0xffffffffu : 0u;
    return r;
}
// One of a block's two quotients, where a warp's lanes share the work of them: what values are multiplied by (0: they are written as
// zeros), or the scale.  The same bits as fp8_scale gives.
struct Fp8Factor {
    float value, before;
};
__device__ __forceinline__ Fp8Factor fp8_factor(uint32_t top, bool inverse) {
    const float a = __uint_as_float(top);
    const bool finite = top < 0x7f800000u;
    Fp8Factor f;
    f.before = a < 0x1p-100f ? 0x1p64f : 1.f;
    const float r = __fdiv_rn(inverse ? FP8_TOP : a, inverse ? a * f.before : FP8_TOP);
    f.value = inverse ? (finite && top > 0 ? r : 0.f) : finite ? r : __uint_as_float(0x7fffffffu);
    return f;
}
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t)lo | (uint32_t)hi << 16;
}
__device__ __forceinline__ uint32_t fp8_quantize4(const float (&v)[4], const Fp8Scale& r) {
    if (r.before == 1.f)
        return fp8_pack4(__fmul_rn(v[0], r.inverse), __fmul_rn(v[1], r.inverse), __fmul_rn(v[2], r.inverse), __fmul_rn(v[3], r.inverse)) & r.keep;
    return fp8_pack4(__fmul_rn(v[0] * r.before, r.inverse), __fmul_rn(v[1] * r.before, r.inverse), __fmul_rn(v[2] * r.before, r.inverse),
                     __fmul_rn(v[3] * r.before, r.inverse)) & r.keep;
}
__device__ __forceinline__ void fp8_values4(uint32_t word, float (&v)[4]) {
    uint32_t lo, hi;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"((uint16_t)word));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"((uint16_t)(word >> 16)));
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}
__device__ __forceinline__ uint32_t fp8_top(uint32_t top, const float (&v)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
    return top;
}
// `left` (up to four) values of a row
__device__ __forceinline__ void fp8_store4(uint8_t* q, int left, uint32_t word) {
    if (left >= 4) {
        *reinterpret_cast<uint32_t*>(q) = word;
        return;
    }
    for (int e = 0; e < left; ++e) q[e] = (uint8_t)(word >> (8 * e));
}
