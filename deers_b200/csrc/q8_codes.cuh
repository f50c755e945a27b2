// 8-bit codes of values relative to a scale: conversions and correctly rounded quotients.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "f32_util.cuh"

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
// Four codes of quotients v * num / den worked out in 64 bits: for operands whose products leave f32.
template <bool I8>
static __device__ __noinline__ uint32_t codes_far(float a, float b, float c, float d, float num, float den) {
    const double x[4] = {(double)a * num / den, (double)b * num / den, (double)c * num / den, (double)d * num / den};
    if constexpr (I8) {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) w |= ((uint32_t)__double2int_rn(fmin(fmax(x[i], -127.0), 127.0)) & 0xffu) << (8 * i);
        return w;
    }
    return e4m3_of(round_to_odd(x[0]), round_to_odd(x[1]), round_to_odd(x[2]), round_to_odd(x[3]));
}

// Sign of |v| * num - |mid| * den, exactly: the products' rounding errors are f32 values too.  The products are next to one another, so their
// difference is exact as well.  mid has few bits; num and den are such that nothing overflows or falls among the subnormals.
__device__ __forceinline__ float beyond(float v, float num, float mid, float den) {
    const float a = fabsf(v), m = fabsf(mid), p = a * num, q = m * den;
    return (p - q) + (fmaf(a, num, -p) - fmaf(m, den, -q));
}

// Products of den with a border, or of the quotient's operands, could leave f32.
__device__ __forceinline__ bool den_is_far(float den) { return !(den > 1e-20f && den < 1e20f); }

// The factors that bring values next to their quotients v * num / den: r = num / den is off by 2^-24 of itself, and so is each of the two products that
// follow, so the quotient lies between v * down and v * up.  far: neither says anything, and nothing is between them.
struct Factors { float down, up; };
__device__ __forceinline__ Factors factors(float num, float den, bool far) {
    const float r = num / den;
    return far ? Factors{0.f, __uint_as_float(0x7f800000u)} : Factors{r * (1.0f - 2.38418579e-7f), r * (1.0f + 2.38418579e-7f)};       // 2^-22
}

// Of values whose quotient may lie on either side of a border, the code by an exact comparison with it; ties to even.
static __device__ __noinline__ uint32_t decide_e4m3(uint32_t lo, uint32_t hi, float v0, float v1, float v2, float v3, float num, float den) {
    if (den_is_far(den) || !(num > 1e-20f)) return codes_far<false>(v0, v1, v2, v3, num, den);
    const float v[4] = {v0, v1, v2, v3};
    float a[4], b[4];
    e4m3_values(lo, a);
    e4m3_values(hi, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t mask = 0xffu << (8 * i);
        if ((lo ^ hi) & mask) {                                  // neighbours of one sign, hi the larger
            const float side = beyond(v[i], num, 0.5f * (a[i] + b[i]), den);
            if (side > 0.f || (side == 0.f && (lo >> (8 * i)) & 1u)) lo = (lo & ~mask) | (hi & mask);
        }
    }
    return lo;
}
static __device__ __noinline__ uint32_t decide_i8(float v0, float v1, float v2, float v3, float num, float den) {
    if (den_is_far(den)) return codes_far<true>(v0, v1, v2, v3, num, den);
    const float v[4] = {v0, v1, v2, v3};
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float low = fminf(floorf(fabsf(v[i] * (num / den))), 126.f);           // the two sizes: low, low + 1 (or the quotient is whole)
        const float side = beyond(v[i], num, low + 0.5f, den);
        int size = (int)low + (side > 0.f || (side == 0.f && ((int)low & 1)) ? 1 : 0);
        w |= ((uint32_t)(v[i] < 0.f ? -size : size) & 0xffu) << (8 * i);
    }
    return w;
}

// e4m3 codes of four quotients v[i] * num / den whose numerators are f32 values.  A quotient within its last bit leaves a remainder that is an f32 value too,
// and the remainder's sign says on which side of it the exact one lies: cut off, the last bit set where something was, it rounds as the exact one does.
static __device__ __noinline__ uint32_t quotients_e4m3(float v0, float v1, float v2, float v3, float num, float den) {
    if (den_is_far(den)) return codes_far<false>(v0, v1, v2, v3, num, den);
    const float v[4] = {v0, v1, v2, v3}, r = 1.0f / den;
    float t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float x = v[i] * num, near = x * r, q = fmaf(fmaf(-near, den, x), r, near), rest = fmaf(-q, den, x);
        const uint32_t bits = __float_as_uint(q);
        t[i] = __uint_as_float(rest != 0.f ? (bits - ((bits ^ __float_as_uint(rest)) >> 31)) | 1u : bits);
    }
    return e4m3_of(t[0], t[1], t[2], t[3]);
}

// Codes of both bounds of four quotients: one where they are equal.
__device__ __forceinline__ void bounds_e4m3(const float (&v)[4], const Factors& f, uint32_t& lo, uint32_t& hi) {
    const uint64_t v01 = pack_f32x2(v[0], v[1]), v23 = pack_f32x2(v[2], v[3]), up = pack_f32x2(f.up, f.up), down = pack_f32x2(f.down, f.down);
    float u[4], d[4];
    unpack_f32x2(mul2(v01, up), u[0], u[1]);
    unpack_f32x2(mul2(v23, up), u[2], u[3]);
    unpack_f32x2(mul2(v01, down), d[0], d[1]);
    unpack_f32x2(mul2(v23, down), d[2], d[3]);
    lo = e4m3_of(d[0], d[1], d[2], d[3]);
    hi = e4m3_of(u[0], u[1], u[2], u[3]);
}

// Codes of four quotients v[i] * num / den, each the nearest code to the exact quotient (ties to even).  Where both bounds of a quotient have one
// code, that is it; the few others are decided exactly, so the codes follow from the operator's definition alone, not from the order of this
// kernel's operations.  (f16 values meet borders often: three normal ones in ten thousand, and a warp asks for 128 at once.)  EXACT: v[i] * num are f32 values,
// which makes the decision short (norm of 16384 x 2048 f16 42.0 -> 41.3 us).
template <bool I8, bool EXACT = false>
__device__ __forceinline__ uint32_t codes_of(const float (&v)[4], const Factors& f, float num, float den) {
    if constexpr (I8) {
        float u[4];
        unpack_f32x2(mul2(pack_f32x2(v[0], v[1]), pack_f32x2(f.up, f.up)), u[0], u[1]);
        unpack_f32x2(mul2(pack_f32x2(v[2], v[3]), pack_f32x2(f.up, f.up)), u[2], u[3]);
        constexpr float MAGIC = 12582912.0f;                      // 1.5 * 2^23: the sum's low bits are the nearest whole number
        uint32_t c[4];
        bool near = false;                                       // (of 127, 2^-22 and three roundings are 2^-14.2 at most: borders are looked for 2^-12.7 to either side)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float m = u[i] + MAGIC;
            near |= !(fabsf(u[i] - (m - MAGIC)) < 0.49985f);
            c[i] = __float_as_uint(m);
        }
        if (near) return decide_i8(v[0], v[1], v[2], v[3], num, den);
        return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    } else {
        uint32_t lo, hi;
        bounds_e4m3(v, f, lo, hi);
        if (lo == hi) return lo;
        if constexpr (EXACT) return quotients_e4m3(v[0], v[1], v[2], v[3], num, den);
        else return decide_e4m3(lo, hi, v[0], v[1], v[2], v[3], num, den);
    }
}

// |v| into a running maximum that passes over NaN; the four values as f32.
__device__ __forceinline__ void look_at(float& top, const float (&v)[4]) { top = fmaxf(fmaxf(top, fmaxf(fabsf(v[0]), fabsf(v[1]))), fmaxf(fabsf(v[2]), fabsf(v[3]))); }
__device__ __forceinline__ void four(const float* v, float (&f)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = v[e];
}
__device__ __forceinline__ void four(const __half* v, float (&f)[4]) {
    const float2 a = __half22float2(__halves2half2(v[0], v[1])), b = __half22float2(__halves2half2(v[2], v[3]));
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
}
// |v| of eight values into a running maximum that passes over NaN.
__device__ __forceinline__ void look_at8(float& top, const float* v) {
#pragma unroll
    for (int e = 0; e < 8; e += 4) look_at(top, *reinterpret_cast<const float(*)[4]>(v + e));
}
__device__ __forceinline__ void look_at8(float& top, const __half* v) {
    __half2 m = __habs2(__halves2half2(v[0], v[1]));
#pragma unroll
    for (int e = 2; e < 8; e += 2) m = __hmax2(m, __habs2(__halves2half2(v[e], v[e + 1])));
    const float2 f = __half22float2(m);
    top = fmaxf(top, fmaxf(f.x, f.y));
}

}  // namespace q8
