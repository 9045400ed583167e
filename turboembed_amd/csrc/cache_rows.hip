// Rows into the pages of a cache, as they are or as int8 codes, and back.
//
// A few lanes hold a head's row, eight values each, so a wave moves several
// rows of K and of V at once: what does not depend on where a row goes is on its
// way before that is known. A wave
// looks for its first row's sequence 64 sequences a step, the lanes go on from
// there. Bytes bound long calls: 8 x 4096 BF16 tokens of 8 heads of 128 into int8
// pages take 60 us (3.4 TB/s), 8 x 2048-4096 of 16 heads of 64 out of them as
// F16 36 us (4.2); short ones a launch and four reads in turn (4 us).
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

// Eight elements, n of them there.
template <typename T> struct Group {
    typename Eight<T>::loose v;
    __device__ __forceinline__ void read(const T *from, int n) {
        if (n >= 8) {
            v = *(const typename Eight<T>::loose *)from;
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = k < n ? from[k] : (T)0;
        }
    }
    template <bool PAST = false> __device__ __forceinline__ void write(T *to, int n) const {
        if (n >= 8) {
            if constexpr (PAST) __builtin_nontemporal_store(v, (typename Eight<T>::loose *)to);
            else *(typename Eight<T>::loose *)to = v;
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k < n) to[k] = v[k];
        }
    }
};

// The largest of LANES lanes' numbers that share a row, as each of them has it.
template <int LANES> __device__ __forceinline__ uint32_t row_max(uint32_t v) {
    const auto with = [&](int other) { v = max(v, (uint32_t)other); };
    if constexpr (LANES == 16) {
        with(__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, true));   // 8 lanes on, of 16
        with(__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, true));   // 4
        with(__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, true));
        with(__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, true));
    } else {
        if constexpr (LANES == 8) with(__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true));   // 7 - lane, of 8
        with(__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, true));    // lane ^ 1
        with(__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, true));    // lane ^ 2
    }
    return v;
}

// The codes of eight of a head's values, and its scale.
template <typename T, int LANES>
__device__ __forceinline__ void write_codes(const Group<T> &x, int n, bool there, int8_t *to, float *scale) {
    // (The bits of numbers of 0 or more are in their order, an infinity's and a
    // NaN's behind them all.)
    float v[8];
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = to_f32(x.v[k]), most = max(most, __float_as_uint(v[k]) & 0x7fffffffu);
    most = row_max<LANES>(most);
    const float top = __uint_as_float(most);
    if (!there) return;
    const bool fine = most < 0x7f800000u;
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
    if (threadIdx.x % LANES == 0) {
        // top / 127 rounded to F32: a quotient corrected by its exact remainder.
        constexpr float INV = 1.0f / 127.0f;
        const float near = top * INV, s = top < 1e-30f ? __fdiv_rn(top, 127.0f) : fmaf(fmaf(-127.0f, near, top), INV, near);
        *scale = fine ? s : __builtin_nanf("");
    }
}

// Eight codes times their scale, rounded once to T.
template <typename T> __device__ __forceinline__ Group<T> values_of(const Group<int8_t> &q, float scale) {
    float v[8];
    // (A product that F32 has rounded onto the border of two 16-bit numbers would
    // be rounded a second time, from there; among F16's smallest the borders are
    // elsewhere.)
    bool tie = std::is_same<T, _Float16>::value && fabsf(scale) < 6.103515625e-5f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        v[k] = (float)q.v[k] * scale;
        const uint32_t u = __float_as_uint(v[k]);
        if (std::is_same<T, __bf16>::value) tie |= (u & 0xffffu) == 0x8000u;
        if (std::is_same<T, _Float16>::value) tie |= (u & 0x1fffu) == 0x1000u;
    }
    if (!std::is_same<T, float>::value && tie)
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = odd_f32((double)q.v[k] * scale);
    Group<T> g;
#pragma unroll
    for (int k = 0; k < 8; ++k) g.v[k] = from_f32<T>(v[k]);
    return g;
}

// LANES lanes a head's row, U rows each. WRITE: the call's rows into the cache,
// else back; PAST: the rows go past the caches, which keep states instead.
template <typename T, bool I8, bool WRITE, int LANES, int U, bool PAST> __global__ void __launch_bounds__(256) cache_rows(RowsArgs a) {
    typedef typename std::conditional<I8, int8_t, T>::type H;   // as the cache holds them
    typedef typename std::conditional<WRITE, T, H>::type From;
    constexpr int PER = 64 / LANES;
    const CacheArgs &c = a.c;
    const int lane = threadIdx.x & 63, col = 8 * (lane % LANES), n = c.width - col;
    const uint32_t rows = (uint32_t)c.tokens * (uint32_t)c.kv;   // (below 2^31)
    const uint32_t stride = gridDim.x * 4 * PER * U;
    for (uint32_t r0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * PER * U; r0 < rows; r0 += stride) {
        int t[U], slot[U];
        uint32_t head[U];
        bool own[U];
        Group<From> k[U], v[U];
        float sk[U], sv[U];
        const auto row = [&](void *p, const uint64_t (&s)[2], int u) { return (T *)p + t[u] * s[0] + head[u] * s[1] + col; };
        const auto state = [&](void *p, const uint64_t (&s)[2], int u) {
            return (H *)p + (uint64_t)max(0, slot[u]) * s[0] + head[u] * s[1] + col;
        };
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // (Rows past the last: the last one, for which nothing is done.)
            const uint32_t r = min(r0 + u * PER + lane / LANES, rows - 1);
            own[u] = r == r0 + u * PER + lane / LANES;
            t[u] = (int)(r / (uint32_t)c.kv), head[u] = r - (uint32_t)t[u] * (uint32_t)c.kv;
            if constexpr (WRITE) k[u].read(row(a.k, a.ks, u), n), v[u].read(row(a.v, a.vs, u), n);
        }
        int seq = seq_before(c, (int)(r0 / (uint32_t)c.kv));
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int p = position_of(c, t[u], seq);
            own[u] = own[u] && seq >= 0 && seq < c.seqs && t[u] >= within(c.starts[seq], 0, c.tokens);
            slot[u] = own[u] && p >= 0 ? slot_of(c, seq, p) : -1;
        }
        if constexpr (!WRITE)
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (slot[u] >= 0) {
                    k[u].read(state(c.k, c.ks, u), n), v[u].read(state(c.v, c.vs, u), n);
                    if constexpr (I8)
                        sk[u] = c.k_scales[(uint64_t)slot[u] * c.kss + head[u]], sv[u] = c.v_scales[(uint64_t)slot[u] * c.vss + head[u]];
                }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if constexpr (WRITE && I8) {
                const uint64_t at = (uint64_t)max(0, slot[u]);
                write_codes<T, LANES>(k[u], n, slot[u] >= 0, state(c.k, c.ks, u), c.k_scales + at * c.kss + head[u]);
                write_codes<T, LANES>(v[u], n, slot[u] >= 0, state(c.v, c.vs, u), c.v_scales + at * c.vss + head[u]);
            } else if constexpr (WRITE) {
                if (slot[u] >= 0) k[u].write(state(c.k, c.ks, u), n), v[u].write(state(c.v, c.vs, u), n);
            } else if (own[u]) {
                if (slot[u] < 0) {
                    const Group<T> zero{};
                    zero.write(row(a.k, a.ks, u), n), zero.write(row(a.v, a.vs, u), n);
                } else if constexpr (I8) {
                    values_of<T>(k[u], sk[u]).template write<PAST>(row(a.k, a.ks, u), n);
                    values_of<T>(v[u], sv[u]).template write<PAST>(row(a.v, a.vs, u), n);
                } else {
                    k[u].template write<PAST>(row(a.k, a.ks, u), n), v[u].template write<PAST>(row(a.v, a.vs, u), n);
                }
            }
        }
    }
}

template <typename T, bool I8, bool WRITE> static hipError_t launch_rows(hipStream_t s, const RowsArgs &a) {
    // Reads, where they leave two workgroups for every compute unit: two rows a
    // lane of codes, and stores past the caches. (8 x 2048-4096 tokens of 16 heads
    // of 64, codes as F16, states that no cache holds: 68 us with four rows a lane
    // and plain stores, 45 with one row, 40 so; 8 x 4096 BF16 tokens of 8 heads of 128, copied,
    // 71, and 61 with one row. Writes of these 64 us with four rows a lane, 59 with
    // one; their stores stay in the caches, where the attention will look.)
    const uint64_t rows = (uint64_t)a.c.tokens * a.c.kv;
    const auto go = [&](auto kernel, int per) {
        const uint64_t blocks = std::min<uint64_t>((rows + per - 1) / per, 1 << 20);
        return enqueue(kernel, dim3((uint32_t)blocks), dim3(256), 0, s, a);
    };
    constexpr int LONG = I8 && !WRITE ? 2 : 1;
#define ROWS(L)                                                                                 \
    if constexpr (!WRITE)                                                                       \
        if (rows >= 256 * 2 * LONG * (256 / L))                                                 \
            return go(cache_rows<T, I8, WRITE, L, LONG, true>, LONG * (256 / L));               \
    return go(cache_rows<T, I8, WRITE, L, 1, false>, 256 / L)
    if (a.c.width <= 32) { ROWS(4); }
    if (a.c.width <= 64) { ROWS(8); }
    ROWS(16);
#undef ROWS
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
