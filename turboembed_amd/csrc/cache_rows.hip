// Rows into the pages of a cache, as they are or as int8 codes, and back.
//
// A few lanes hold a head's row, eight values each, so a wave moves several
// rows of K and of V at once. A wave looks for its first row's sequence 64
// sequences a step, the lanes go on from there.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "cache_find.h"
#include "codes.h"
#include "launch.h"

namespace rocm {

struct RowsArgs {
    CacheArgs c;
    void *k, *v;              // the call's rows
    uint64_t ks[2], vs[2];
};

template <typename T> struct Eight {
    typedef T loose __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};

// Eight elements from one place to another, n of them there.
template <typename T> __device__ __forceinline__ void copy8(T *to, const T *from, int n) {
    typedef typename Eight<T>::loose loose;
    if (n >= 8) {
        *(loose *)to = *(const loose *)from;
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < n) to[k] = from[k];
    }
}

// The codes of eight of a head's values into its slot, and its scale.
template <typename T, int LANES>
__device__ __forceinline__ void write_codes(const T *from, int n, bool there, int8_t *to, float *scale) {
    float v[8], top = 0.0f, bad = 0.0f;   // bad is not 0: an infinity or a NaN among the values
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = 0.0f;
    if (there && n > 0) read8(from, n, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(v[k])), bad = fmaf(v[k], 0.0f, bad);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64)), bad += __shfl_xor(bad, o, 64);
    if (!there) return;
    const bool fine = bad == 0.0f;
    if (n > 0) {
        uint32_t q[2];
        codes_of8(v, top, fine, q);
        if (n >= 8) {
            typedef uint32_t loose2 __attribute__((ext_vector_type(2), aligned(1)));
            *(loose2 *)to = loose2{q[0], q[1]};
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k < n) to[k] = (int8_t)(q[k >> 2] >> (8 * (k & 3)));
        }
    }
    if (threadIdx.x % LANES == 0) *scale = fine ? (float)((double)top / 127.0) : __builtin_nanf("");
}

// Eight codes times their scale, rounded once to T.
template <typename T> __device__ __forceinline__ void read_codes(const int8_t *from, float scale, int n, T *to) {
    uint32_t q[2] = {0, 0};
    if (n >= 8) {
        typedef uint32_t loose2 __attribute__((ext_vector_type(2), aligned(1)));
        const loose2 x = *(const loose2 *)from;
        q[0] = x[0], q[1] = x[1];
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < n) q[k >> 2] |= (uint32_t)(uint8_t)from[k] << (8 * (k & 3));
    }
    float v[8];
    bool tie = false;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        v[k] = (float)(int8_t)(q[k >> 2] >> (8 * (k & 3))) * scale;
        // (A product that F32 has rounded onto the border of two 16-bit numbers
        // would be rounded a second time, from there.)
        const uint32_t u = __float_as_uint(v[k]);
        if (std::is_same<T, __bf16>::value) tie |= (u & 0xffffu) == 0x8000u;
        if (std::is_same<T, _Float16>::value) tie |= (u & 0x1fffu) == 0x1000u || (u & 0x7fffffffu) < 0x38800000u;
    }
    if (!std::is_same<T, float>::value && tie)
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = odd_f32((double)(int8_t)(q[k >> 2] >> (8 * (k & 3))) * scale);
    write8(to, n, v);
}

// LANES lanes a head's row. WRITE: the call's rows into the cache, else back.
template <typename T, bool I8, bool WRITE, int LANES> __global__ void __launch_bounds__(256) cache_rows(RowsArgs a) {
    typedef typename std::conditional<I8, int8_t, T>::type H;   // as the cache holds them
    constexpr int PER = 64 / LANES;
    const CacheArgs &c = a.c;
    const int lane = threadIdx.x & 63, col = 8 * (lane % LANES), n = c.width - col;
    const uint32_t rows = (uint32_t)c.tokens * (uint32_t)c.kv;   // (below 2^31)
    const uint32_t stride = gridDim.x * 4 * PER;
    for (uint32_t r0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * PER; r0 < rows; r0 += stride) {
        int seq = seq_before(c, (int)(r0 / (uint32_t)c.kv));
        const uint32_t r = r0 + lane / LANES;
        const int t = (int)(r / (uint32_t)c.kv);
        const uint64_t head = r - (uint32_t)t * (uint32_t)c.kv;
        // (Rows past the last belong to no sequence: a call's tokens end before them.)
        const int p = r < rows ? position_of(c, t, seq) : -1;
        const bool own = r < rows && seq >= 0 && seq < c.seqs && t >= within(c.starts[seq], 0, c.tokens);
        const int slot = p >= 0 ? slot_of(c, seq, p) : -1;
        T *k = (T *)a.k + t * a.ks[0] + head * a.ks[1] + col, *v = (T *)a.v + t * a.vs[0] + head * a.vs[1] + col;
        const uint64_t at = slot < 0 ? 0 : slot;
        H *hk = (H *)c.k + at * c.ks[0] + head * c.ks[1] + col, *hv = (H *)c.v + at * c.vs[0] + head * c.vs[1] + col;
        float *sk = c.k_scales + at * c.kss + head, *sv = c.v_scales + at * c.vss + head;
        if constexpr (WRITE && I8) {
            write_codes<T, LANES>(k, n, slot >= 0, hk, sk);
            write_codes<T, LANES>(v, n, slot >= 0, hv, sv);
        } else if constexpr (WRITE) {
            if (slot >= 0 && n > 0) copy8(hk, k, n), copy8(hv, v, n);
        } else if (own && n > 0) {
            if (slot < 0) {
                const float zero[8] = {};
                write8(k, n, zero), write8(v, n, zero);
            } else if constexpr (I8) {
                read_codes(hk, *sk, n, k), read_codes(hv, *sv, n, v);
            } else {
                copy8(k, hk, n), copy8(v, hv, n);
            }
        }
    }
}

template <typename T, bool I8, bool WRITE> static hipError_t launch_rows(hipStream_t s, const RowsArgs &a) {
    const auto go = [&](auto kernel, int lanes) {
        const uint64_t rows = (uint64_t)a.c.tokens * a.c.kv, per = 4 * (64 / lanes);
        const uint64_t blocks = std::min<uint64_t>((rows + per - 1) / per, 1 << 20);
        return enqueue(kernel, dim3((uint32_t)blocks), dim3(256), 0, s, a);
    };
    if (a.c.width <= 32) return go(cache_rows<T, I8, WRITE, 4>, 4);
    if (a.c.width <= 64) return go(cache_rows<T, I8, WRITE, 8>, 8);
    return go(cache_rows<T, I8, WRITE, 16>, 16);
}

template <bool WRITE> static hipError_t rows_of(hipStream_t s, const RowsArgs &a, Dt t, bool i8) {
    if (a.c.tokens == 0 || a.c.kv == 0 || a.c.seqs == 0) return hipSuccess;
    const auto go = [&](auto zero) {
        typedef decltype(zero) T;
        return i8 ? launch_rows<T, true, WRITE>(s, a) : launch_rows<T, false, WRITE>(s, a);
    };
    if (t == Dt::F32) return go(0.0f);
    if (t == Dt::F16) return go((_Float16)0.0f);
    return go((__bf16)0.0f);
}

hipError_t cache_write(hipStream_t s, const CacheArgs &a, Dt rows, bool i8, const void *k, const void *v,
                       const uint64_t (&ks)[2], const uint64_t (&vs)[2]) {
    return rows_of<true>(s, RowsArgs{a, const_cast<void *>(k), const_cast<void *>(v), {ks[0], ks[1]}, {vs[0], vs[1]}},
                         rows, i8);
}

hipError_t cache_read(hipStream_t s, const CacheArgs &a, Dt rows, bool i8, void *k, void *v, const uint64_t (&ks)[2],
                      const uint64_t (&vs)[2]) {
    return rows_of<false>(s, RowsArgs{a, k, v, {ks[0], ks[1]}, {vs[0], vs[1]}}, rows, i8);
}

}  // namespace rocm
