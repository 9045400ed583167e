// Eight values of a row at a time, and the int8 codes of rows: what the
// kernels that quantize rows share.
#pragma once

#include "devmath.h"

namespace rocm {

// Eight consecutive values at p, of which the first n exist (the rest read as
// 0). Rows may start at any element, so the vectors are read at its alignment.
template <typename H> __device__ __forceinline__ void read8(const H *p, int n, float (&v)[8]) {
    typedef H loose8 __attribute__((ext_vector_type(8), aligned(sizeof(H))));
    if (n >= 8) {
        const loose8 q = *(const loose8 *)p;
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = to_f32(q[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = k < n ? to_f32(p[k]) : 0.0f;
    }
}

template <typename H> __device__ __forceinline__ void write8(H *p, int n, const float (&v)[8]) {
    typedef H loose8 __attribute__((ext_vector_type(8), aligned(sizeof(H))));
    if (n >= 8) {
        loose8 q;
#pragma unroll
        for (int k = 0; k < 8; ++k) q[k] = from_f32<H>(v[k]);
        *(loose8 *)p = q;
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < n) p[k] = from_f32<H>(v[k]);
    }
}

// d as an F32 that rounds to 16 bits as d itself does: cut off, and odd where
// anything was. (Below F32's smallest normal number its own rounding still
// comes first.) 65536 x 1024 F16 rows and their norm take 54.4 us so, 51.0 with
// d rounded to F32, one output in some 15,000 to the wrong side.
__device__ __forceinline__ float odd_f32(double d) {
    constexpr uint32_t REST = 0x1fffffff;   // what F32 has no room for
    const uint64_t u = __builtin_bit_cast(uint64_t, d);
    const uint32_t low = (uint32_t)u, odd = low | ((low & REST) + REST);
    return (float)__builtin_bit_cast(double, (u >> 32 << 32) | (odd & ~REST));
}

// The whole number nearest to 127 c / top (ties to even), |c| <= top, without
// rounding: low, the whole number below it, and a half are compared with it as
// exact sums of two numbers each.
__device__ __forceinline__ int nearest_code(double c, double top, double low) {
#pragma clang fp contract(off)
    const double half = low + 0.5, a = 127.0 * c, b = half * top;
    const double d = (a - b) + (fma(127.0, c, -a) - fma(half, top, -b));
    return (int)(d > 0.0 ? low + 1.0 : d < 0.0 ? low : 2.0 * rint(0.5 * half));
}

// The codes of eight of a row's values, top the largest magnitude of the row
// (finite and not 0, but where `fine` is not set: then they are 0): those of
// nearest_code, by an F32 quotient where no border is nearer than its error.
__device__ __forceinline__ void codes_of8(const float (&v)[8], float top, bool fine, uint32_t (&q)[2]) {
    const double k127 = fine && top > 0.0f ? 127.0 / top : 0.0;
    const float factor = (float)k127;
    // (Rows so large or small that F32 does not hold the steps.)
    const bool far = k127 > 1e30 || (k127 > 0.0 && k127 < 1e-30);
    float near = 0.0f;   // the largest distance from a whole number
    int code[8];
    float t[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        t[k] = v[k] * factor;
        const float whole = rintf(t[k]);
        near = fmaxf(near, fabsf(t[k] - whole));
        code[k] = fine ? (int)whole : 0;
    }
    if (fine && (near > 0.5f - 2.5e-5f || far)) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            code[k] = nearest_code(v[k], top, far ? floor(127.0 * v[k] / top) : (double)floorf(t[k]));
    }
    q[0] = q[1] = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) q[k >> 2] |= (uint32_t)(uint8_t)(int8_t)code[k] << (8 * (k & 3));
}

}  // namespace rocm
