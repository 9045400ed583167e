// RMS norm with the residual's addition and int8 codes out, and the codes of
// rows alone.
//
// A row is held in registers by a few lanes, a wave or a workgroup: x (and the
// residual) are read once, everything else is made from the registers, and
// the outputs are written once. The weight is read twice, from the caches.
// Bound by those bytes: 4807 x 1023 F32 rows and their norm take 15.4 us (5.1
// TB/s, a large copy's rate), 65536 x 1024 F16 rows to codes 44.4 (4.5), 65536 x
// 4096 BF16 rows with a residual to codes 443 (4.25, as the norm alone does: a
// workgroup reads its row, exchanges sums and writes in turn). 16-bit rows that
// no vector's alignment divides reach two thirds of that (26214 x 2500 F16, the
// same: 2.8; x 2504: 3.2).
//
// The codes are those of the definition, not of a rounded norm: code_i = the
// whole number nearest to 127 y_i / max|y| = 127 c_i / max|c|, c = v w, as the
// norm's factor is common to the row. c is exact in 64 bits (24 by 24 bits),
// so a code can only go wrong next to the border of two codes: F32 products
// give the quotient to 3 2^-24 of it, 2.3e-5, and where a border is nearer than
// 2.5e-5 (one value in 20,000) it is decided again without rounding
// (nearest_code).
#include <hip/hip_runtime.h>

#include "devmath.h"
#include "launch.h"
#include "operators.h"

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

__device__ __forceinline__ void write8(void *p, Dt t, uint64_t at, int n, const float (&v)[8]) {
    if (t == Dt::F32) write8((float *)p + at, n, v);
    else if (t == Dt::F16) write8((_Float16 *)p + at, n, v);
    else write8((__bf16 *)p + at, n, v);
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

// A row's sum of squares, largest magnitude and sign of what is no number.
struct Stats {
    double ss, top;
    float bad;
};

// Over the LANES lanes that share a row (a power of 2 of a wave's, or whole
// waves); red is the waves' LDS, another for the next row. Every lane of them
// calls it.
template <int LANES> __device__ __forceinline__ Stats row_stats(Stats v, Stats *red) {
    constexpr int WAVES = LANES / 64;
#pragma unroll
    for (int o = LANES < 64 ? LANES / 2 : 32; o > 0; o >>= 1) {
        v.ss += __shfl_xor(v.ss, o, 64);
        v.top = fmax(v.top, __shfl_xor(v.top, o, 64));
        v.bad += __shfl_xor(v.bad, o, 64);
    }
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) {
            const Stats u = red[i];
            v.ss += u.ss, v.top = fmax(v.top, u.top), v.bad += u.bad;
        }
    }
    return v;
}

// X: x's type; R: the residual's (and v's); NORM: rms_norm, else the codes of
// x. LANES lanes hold a row, lane l of them columns 8 (l + LANES g) .. + 7 of
// each group g < G; a workgroup is at least 256.
template <typename X, typename R, bool NORM, int LANES, int G>
__global__ void __launch_bounds__(LANES < 256 ? 256 : LANES) row_codes_kernel(RowArgs a) {
    constexpr int ROWS = LANES < 256 ? 256 / LANES : 1;
    // (Two rows' worth: a wave may be a row ahead of the slowest.)
    __shared__ Stats red[2][LANES < 64 ? 1 : LANES / 64];
    const int lane = threadIdx.x % LANES;
    int turn = 0;
    // (Unsigned: the last step passes 31 bits.)
    for (uint32_t row = blockIdx.x * ROWS + threadIdx.x / LANES; row < (uint32_t)a.rows; row += gridDim.x * ROWS) {
        float v[G][8];
        double ss = 0.0, top = 0.0;
        float top32 = 0.0f, bad = 0.0f;   // bad is not 0: an infinity or a NaN among the values
        // (A weight of either type, 1 without one.)
        auto weight = [&](int c, int n, float(&w)[8]) {
            if constexpr (NORM) {
                if (a.wt == Dt::F32) read8((const float *)a.w + c, n, w);
                else read8((const X *)a.w + c, n, w);
            }
        };
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int c = 8 * (lane + LANES * g), n = a.cols - c;
            if (n > 0) {
                read8((const X *)a.x + row * a.ldx + c, n, v[g]);
                if (NORM && a.res) {
                    float r[8];
                    read8((const R *)a.res + row * a.ldr + c, n, r);
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[g][k] = to_f32(from_f32<R>(v[g][k] + r[k]));
                }
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) v[g][k] = 0.0f;
            }
        }
        if (NORM && a.sum)
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const int c = 8 * (lane + LANES * g), n = a.cols - c;
                if (n > 0) write8((R *)a.sum + row * a.lds + c, n, v[g]);
            }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int c = 8 * (lane + LANES * g), n = a.cols - c;
            if (n <= 0) continue;
            float w[8];
            if (a.scales) weight(c, n, w);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const double d = v[g][k];
                if constexpr (NORM) ss = fma(d, d, ss);
                if (a.scales) {
                    if constexpr (NORM) {
                        top = fmax(top, fabs(d * w[k]));
                        bad = fmaf(v[g][k] * 0.0f, w[k], bad);
                    } else {
                        top32 = fmaxf(top32, fabsf(v[g][k]));
                        bad = fmaf(v[g][k], 0.0f, bad);
                    }
                }
            }
        }
        const Stats all = row_stats<LANES>(Stats{ss, NORM ? top : (double)top32, bad}, red[turn]);
        turn ^= 1;
        double r = 1.0;
        if constexpr (NORM) r = 1.0 / sqrt(all.ss / a.cols + a.eps);
        if (NORM && a.out)
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const int c = 8 * (lane + LANES * g), n = a.cols - c;
                if (n <= 0) continue;
                float w[8], y[8];
                weight(c, n, w);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    y[k] = a.ot == Dt::F32 ? (float)(v[g][k] * r * w[k]) : odd_f32(v[g][k] * r * w[k]);
                write8(a.out, a.ot, row * a.ldo + c, n, y);
            }
        if (!a.scales) continue;
        top = all.top;
        const bool fine = all.bad == 0.0f;
        const double k127 = fine && top > 0.0 ? 127.0 / top : 0.0;
        const float factor = (float)k127;
        // (Rows so large or small that F32 does not hold the steps.)
        const bool far = k127 > 1e30 || (k127 > 0.0 && k127 < 1e-30);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int c = 8 * (lane + LANES * g), n = a.cols - c;
            if (n <= 0) continue;
            float w[8], t[8];
            weight(c, n, w);
            float near = 0.0f;   // the largest distance from a whole number
            int code[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                t[k] = (NORM ? v[g][k] * w[k] : v[g][k]) * factor;
                const float whole = rintf(t[k]);
                near = fmaxf(near, fabsf(t[k] - whole));
                code[k] = fine ? (int)whole : 0;
            }
            if (near > 0.5f - 2.5e-5f || far) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const double e = NORM ? (double)v[g][k] * w[k] : (double)v[g][k];
                    code[k] = nearest_code(e, top, far ? floor(127.0 * e / top) : (double)floorf(t[k]));
                    if (!fine) code[k] = 0;
                }
            }
            uint32_t q[2] = {0, 0};
#pragma unroll
            for (int k = 0; k < 8; ++k) q[k >> 2] |= (uint32_t)(uint8_t)(int8_t)code[k] << (8 * (k & 3));
            int8_t *p = a.codes + row * a.ldc + c;
            if (n >= 8) {
                typedef uint32_t loose2 __attribute__((ext_vector_type(2), aligned(1)));
                *(loose2 *)p = loose2{q[0], q[1]};
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (k < n) p[k] = (int8_t)(q[k >> 2] >> (8 * (k & 3)));
            }
        }
        if (lane == 0) a.scales[row] = !fine ? __builtin_nanf("") : top > 0.0 ? (float)(top * r / 127.0) : 0.0f;
    }
}

template <typename X, typename R, bool NORM> static hipError_t launch_rows(hipStream_t s, const RowArgs &a) {
    // Lanes a row and values a lane as measured, GB/s of norm, residual and
    // codes, F16 or BF16: 4096 columns 256 x 16 4140, 64 x 64 3371, 128 x 32
    // 3751, 512 x 16 2985; 8192: 256 x 32 3740, 512 x 16 3520; 16384: 512 x 32
    // 3784, 256 x 64 2698, 1024 x 32 2153. Narrow rows share a wave, or most of
    // it holds nothing: 2^20 rows of 64 in 8 lanes 4112, in 64 665; 2^18 of 256
    // in 32 lanes 3981, in 64 2319.
    // Workgroups enough for every row, up to a bound past which they take
    // several (a launch holds less than 2^32 threads; and a row a workgroup
    // spends a fortieth of its time on starting one: 65536 x 4096 452 us, 440 in
    // 2^14 of them).
    auto go = [&](auto kernel, int lanes) {
        const int per = lanes < 256 ? 256 / lanes : 1, threads = lanes < 256 ? 256 : lanes;
        const int blocks = (a.rows - 1) / per + 1;
        const int most = lanes < 256 ? 1 << 20 : 1 << 14;
        return enqueue(kernel, dim3(blocks < most ? blocks : most), dim3(threads), 0, s, a);
    };
#define ROWS(L, G) return go(row_codes_kernel<X, R, NORM, L, G>, L)
    if (a.cols <= 64) ROWS(8, 1);
    if (a.cols <= 128) ROWS(16, 1);
    if (a.cols <= 256) ROWS(32, 1);
    if (a.cols <= 512) ROWS(64, 1);
    if (a.cols <= 1024) ROWS(64, 2);
    if (a.cols <= 2048) ROWS(64, 4);
    if (a.cols <= 4096) ROWS(256, 2);
    if (a.cols <= 8192) ROWS(256, 4);
    if (a.cols <= 16384) ROWS(512, 4);
    if (a.cols <= 32768) ROWS(512, 8);
    ROWS(1024, 8);
#undef ROWS
}

hipError_t row_codes(hipStream_t s, const RowArgs &a) {
    if (a.rows <= 0) return hipSuccess;
    if (!a.w) {
        if (a.xt == Dt::F32) return launch_rows<float, float, false>(s, a);
        if (a.xt == Dt::F16) return launch_rows<_Float16, _Float16, false>(s, a);
        return launch_rows<__bf16, __bf16, false>(s, a);
    }
    if (a.xt == Dt::F32) return launch_rows<float, float, true>(s, a);
    if (a.xt == Dt::F16)
        return a.rt == Dt::F32 ? launch_rows<_Float16, float, true>(s, a) : launch_rows<_Float16, _Float16, true>(s, a);
    return a.rt == Dt::F32 ? launch_rows<__bf16, float, true>(s, a) : launch_rows<__bf16, __bf16, true>(s, a);
}

}  // namespace rocm
