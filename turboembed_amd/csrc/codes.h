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

// The same in F32, where nothing of it over- or underflows: (127 c - half top) is
// decided by the rounded products' difference, which is exact as they lie within
// a factor of 2, and their errors'.
__device__ __forceinline__ float nearest_code_f32(float c, float top, float low) {
#pragma clang fp contract(off)
    const float half = low + 0.5f, a = 127.0f * c, b = half * top;
    const float d = (a - b) + (fmaf(127.0f, c, -a) - fmaf(half, top, -b));
    return d > 0.0f ? low + 1.0f : d < 0.0f ? low : 2.0f * rintf(0.5f * half);
}

// The codes of eight of a row's values, top the largest magnitude of the row
// (finite, but where `fine` is not set: then they are 0): those of nearest_code,
// by an F32 quotient where no border is nearer than its error, 4 2^-24 of 127.
// (Of 16-bit rows a third has a value that is half of its largest: 63.5.)
__device__ __forceinline__ void codes_of8(const float (&v)[8], float top, bool fine, uint32_t (&q)[2]) {
    const float factor = top > 0.0f ? 127.0f * __builtin_amdgcn_rcpf(top) : 0.0f;
    // 1.5 2^23 and a small number: the whole number next to it, its lowest byte the code.
    constexpr float SHIFT = 12582912.0f, NEAR = 0.5f - 3.5e-5f;
    float near = 0.0f, t[8], off[8];   // the distances from a whole number
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        t[k] = fmaf(v[k], factor, SHIFT);
        off[k] = fmaf(v[k], factor, SHIFT - t[k]);
        near = fmaxf(near, fabsf(off[k]));
    }
    // (Rows so large or small that F32 does not hold the steps.)
    if (fine && top > 0.0f && (top > 1e30f || top < 1e-28f)) {
#pragma unroll
        for (int k = 0; k < 8; ++k) t[k] = SHIFT + (float)nearest_code(v[k], top, floor(127.0 * v[k] / top));
    } else if (fine && near > NEAR) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (fabsf(off[k]) > NEAR) t[k] = SHIFT + nearest_code_f32(v[k], top, floorf(v[k] * factor));
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const auto bits = [&](int k) { return __float_as_uint(t[4 * w + k]); };
        const uint32_t lo = __builtin_amdgcn_perm(bits(1), bits(0), 0x0c0c0400u), hi = __builtin_amdgcn_perm(bits(3), bits(2), 0x0c0c0400u);
        q[w] = fine ? lo | hi << 16 : 0;
    }
}

}  // namespace rocm
