// 8-bit codes of values relative to a scale: conversions and correctly rounded quotients.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

namespace q8 {

constexpr float MOST_I8 = 127.0f, MOST_E4M3 = 448.0f;            // largest code
constexpr int BLOCK = 32;                                        // tokens of a head that share a scale of the cache

// Four e4m3 codes, nearest, beyond the largest the largest, NaN the code 0x7f; a in the lowest byte.
__device__ __forceinline__ uint32_t e4m3_of(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t)lo | ((uint32_t)hi << 16);
}
// Two f16 from the two codes in the low or high half of w (the lower code in the lower half).
__device__ __forceinline__ uint32_t e4m3_lo(uint32_t w) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(r) : "r"(w));
    return r;
}
__device__ __forceinline__ uint32_t e4m3_hi(uint32_t w) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(w));
    return r;
}
__device__ __forceinline__ void e4m3_values(uint32_t w, float (&f)[4]) {
    const uint32_t a = e4m3_lo(w), b = e4m3_hi(w);
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a)), y = __half22float2(*reinterpret_cast<const __half2*>(&b));
    f[0] = x.x; f[1] = x.y; f[2] = y.x; f[3] = y.y;
}

// f32 value that every later rounding to fewer bits takes for x: x cut off, the last bit set where something was.
__device__ __forceinline__ float round_to_odd(double x) {
    const float f = __double2float_rz(x);
    return (double)f == x ? f : __uint_as_float(__float_as_uint(f) | 1u);
}

// Four codes worked out in 64 bits.
static __device__ __noinline__ uint32_t exact_e4m3(float a, float b, float c, float d, float num, float den) {
    return e4m3_of(round_to_odd((double)a * (double)num / (double)den), round_to_odd((double)b * (double)num / (double)den),
                   round_to_odd((double)c * (double)num / (double)den), round_to_odd((double)d * (double)num / (double)den));
}
static __device__ __noinline__ uint32_t exact_i8(float v, float num, float den) {
    const int q = __double2int_rn((double)v * (double)num / (double)den);
    return (uint32_t)(q > 127 ? 127 : q < -127 ? -127 : q);
}

// Codes of four quotients v[i] * num / den, each the nearest code to the exact quotient (ties to even), given r = num / den rounded.
// v * r is off by at most 2^-23 of itself, so a quotient whose neighbours 2^-21 to either side have one code has that code; the few others are
// worked out in 64 bits.  So the codes follow from the operator's definition alone, not from the order of this kernel's operations.
// wide: r does not stand for the quotient (it overflowed).
template <bool I8>
__device__ __forceinline__ uint32_t codes_of(const float (&v)[4], float r, float num, float den, bool wide) {
    constexpr float DOWN = 1.0f - 4.76837158e-7f, UP = 1.0f + 4.76837158e-7f;
    float t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = v[i] * r;
    if constexpr (I8) {
        constexpr float MAGIC = 12582912.0f;                      // 1.5 * 2^23: the sum's low bits are the nearest whole number
        uint32_t c[4];
        bool near = wide;                                        // (of 127 the error is 2^-16: borders are looked for 2^-13 to either side)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float m = t[i] + MAGIC;
            near |= !(fabsf(t[i] - (m - MAGIC)) < 0.4998f);
            c[i] = __float_as_uint(m);
        }
        if (near) {
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i] = exact_i8(v[i], num, den);
        }
        return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    } else {
        const uint32_t lo = e4m3_of(t[0] * DOWN, t[1] * DOWN, t[2] * DOWN, t[3] * DOWN), hi = e4m3_of(t[0] * UP, t[1] * UP, t[2] * UP, t[3] * UP);
        return lo == hi && !wide ? lo : exact_e4m3(v[0], v[1], v[2], v[3], num, den);
    }
}

}  // namespace q8
