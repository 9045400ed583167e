// What the attention kernels over a caller's memory share: a row's two halves
// of a wave, chunks of 16 bytes, and a weight as two numbers.
#pragma once

#include <type_traits>

#include "devmath.h"
#include "gemm_tile.h"

namespace rocm {

// The sum of a lane's value and the lane 32 away's, and the larger of the two.
__device__ __forceinline__ float both_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float both_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

typedef float f32x4 __attribute__((ext_vector_type(4)));

// ...of the four lanes 16 apart.
__device__ __forceinline__ float four_sum(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return both_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}
__device__ __forceinline__ float four_max(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return both_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}

template <typename T> struct Chunk {   // 16 bytes of a row
    static constexpr int N = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
    typedef T loose __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// The N elements at p, of which n exist (the rest 0).
template <typename T> __device__ __forceinline__ typename Chunk<T>::vec read_chunk(const T *p, int n) {
    typename Chunk<T>::vec v;
    if (n >= Chunk<T>::N) return *(const typename Chunk<T>::loose *)p;
#pragma unroll
    for (int i = 0; i < Chunk<T>::N; ++i) v[i] = i < n ? p[i] : (T)0.0f;
    return v;
}

// Of each of two weights (0 or more) a number of T one to two of its steps
// below, so that what is left of it is at least a step: both terms of a weight
// are positive, and an infinite value stays what its product gives.
template <typename T>
__device__ __forceinline__ auto below(float w0, float w1) {
    typedef unsigned short bits2 __attribute__((ext_vector_type(2)));
    typedef T two __attribute__((ext_vector_type(2)));
    bits2 b;
    if constexpr (std::is_same<T, _Float16>::value) b = __builtin_bit_cast(bits2, __builtin_amdgcn_cvt_pkrtz(w0, w1));
    else b = bits2{(unsigned short)(__float_as_uint(w0) >> 16), (unsigned short)(__float_as_uint(w1) >> 16)};
    return __builtin_bit_cast(two, __builtin_elementwise_sub_sat(b, bits2{1, 1}));
}

// LDS reads that transpose, N of them of each of A addresses, the second OFF
// bytes behind the first, all from AT on, waited for here: for the builtins the
// compiler waits for every load to LDS that is on its way too, those of the next
// tile, which these do not read.
typedef uint32_t words2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) const void *lds_ptr;
#define TURBO_READS_8(OP)                                                                                              \
    asm volatile(OP " %0, %8 offset:%12\n\t" OP " %1, %8 offset:%13\n\t" OP " %2, %9 offset:%12\n\t"                  \
                 OP " %3, %9 offset:%13\n\t" OP " %4, %10 offset:%12\n\t" OP " %5, %10 offset:%13\n\t"                 \
                 OP " %6, %11 offset:%12\n\t" OP " %7, %11 offset:%13\n\ts_waitcnt lgkmcnt(0)"                        \
                 : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7]) \
                 : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(AT), "n"(AT + OFF)                               \
                 : "memory")
#define TURBO_READS_4(OP)                                                                                              \
    asm volatile(OP " %0, %4 offset:%8\n\t" OP " %1, %5 offset:%8\n\t" OP " %2, %6 offset:%8\n\t" OP                 \
                    " %3, %7 offset:%8\n\ts_waitcnt lgkmcnt(0)"                                                         \
                 : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])                                                   \
                 : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(AT)                                              \
                 : "memory")
// 16-bit elements: two reads of each address, v[2 i] and v[2 i + 1].
template <int AT, int OFF> __device__ __forceinline__ void read_tr16(words2 (&v)[8], const uint32_t (&at)[4]) {
    TURBO_READS_8("ds_read_b64_tr_b16");
}
// Bytes: one of each.
template <int AT> __device__ __forceinline__ void read_tr8(words2 (&v)[4], const uint32_t (&at)[4]) {
    TURBO_READS_4("ds_read_b64_tr_b8");
}
#undef TURBO_READS_8
#undef TURBO_READS_4

// The product whose result has M rows and columns: lane l has column l % M of
// it, and rows 4 (64 / M) (i / 4) + 4 (l / M) + i % 4 in register i. 16-bit
// operands: row or column l % M, 8 steps of the inner width from 8 (l / M) on.
template <typename T, int M> struct Product : Mma<T> {};
template <> struct Product<_Float16, 16> {
    typedef half8 frag;
    typedef floatx4 acc;
    static __device__ __forceinline__ acc run(frag a, frag b, acc c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};
template <> struct Product<__bf16, 16> {
    typedef bf16x8 frag;
    typedef floatx4 acc;
    static __device__ __forceinline__ acc run(frag a, frag b, acc c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};

// Codes as numbers of T, a word's four at a time.
__device__ __forceinline__ void numbers_of(uint32_t w, float *v) {
    // (Of the word and of its upper three bytes, as the conversions that pick a
    // byte take them: bytes 0 and 2 of each.)
    uint32_t u = w >> 8;
    asm volatile("" : "+v"(u));
    v[0] = (float)(int8_t)w, v[1] = (float)(int8_t)u, v[2] = (float)(int8_t)(w >> 16), v[3] = (float)(int8_t)(u >> 16);
}
template <typename T> __device__ __forceinline__ void numbers_of(uint32_t w, T *v) {
    if constexpr (std::is_same<T, _Float16>::value) {
        // 1024 and a number of 10 bits is 0x6400 and its bits: each code plus
        // 128, less 1152, exactly.
        typedef _Float16 two __attribute__((ext_vector_type(2)));
        const uint32_t u = w ^ 0x80808080u;
        const two a = __builtin_bit_cast(two, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - two{1152, 1152};
        const two b = __builtin_bit_cast(two, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - two{1152, 1152};
        v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1];
    } else {
        float f[4];
        numbers_of(w, f);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = from_f32<T>(f[e]);
    }
}

}  // namespace rocm
