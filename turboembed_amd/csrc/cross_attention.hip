// Attention of queries to an encoder's states of another length.
//
// A workgroup takes an item of the plan: 32 rows a wave (a row is a query
// token's head; those that share a key head are rows of one item, so that its
// keys and values are read once for them) against a run of keys. K and V
// pass through LDS in tiles of KB keys, two of each: the next tile's loads are
// in registers while one is computed. Scores are computed transposed, S^T =
// K Q^T, so that a lane holds one row (lane % 32) and 16 of 32 keys, the other
// 16 in the lane 32 away; O^T += V^T P^T then takes P as the score registers
// hold it, against V's columns for the same keys in that order (16-bit values
// by LDS reads that transpose, F32 values one by one).
//
// The softmax is the running one, in base 2 and F32; its maximum moves only
// when a score passes it by more than 2^8, so most tiles rescale nothing. The
// scale is positive here (the launcher turns q around for a negative one).
#include <hip/hip_runtime.h>

#include <type_traits>

#include "devmath.h"
#include "gemm_tile.h"
#include "launch.h"
#include "operators.h"

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

// a b, rounded, less c.
__device__ __forceinline__ float rounded_less(float a, float b, float c) {
#pragma clang fp contract(off)
    return a * b - c;
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

// Where a part of `rows` rows lies in the workspace.
__device__ __forceinline__ float *part_of(const CrossArgs &a, int part) {
    return a.ws + (uint64_t)part * a.part_rows * (a.width + 2);
}

// DP: the head width rounded up to 32, 64, 96 or 128.
template <typename T, int DP, int WAVES> struct CrossTile {
    static constexpr bool F32 = std::is_same<T, float>::value;
    static constexpr int KB = WAVES == 1 || (F32 && DP > 64) ? 32 : 64;
    static constexpr int PITCH = DP * (int)sizeof(T) + 16;   // 16 bytes more: rows in different banks
    static constexpr int BUF = KB * PITCH;
    static constexpr int LDS = 4 * BUF;                      // K and V, two tiles of each
};

template <typename T, int DP, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) cross_tiles(CrossArgs a) {
    using C = CrossTile<T, DP, WAVES>;
    constexpr bool F32 = C::F32;
    constexpr int KB = C::KB, SUB = KB / 32, PITCH = C::PITCH, BUF = C::BUF, DT = DP / 32;
    constexpr int E = Chunk<T>::N, CPR = DP / E, THREADS = 64 * WAVES, NL = KB * CPR / THREADS;
    static_assert(NL * THREADS == KB * CPR, "whole loads a thread");
    constexpr float LAG = 8.0f;
    typedef typename Chunk<T>::vec vec;
    typedef typename Mma<T>::frag frag;
    extern __shared__ __attribute__((aligned(16))) char smem[];

    const CrossItem it = a.items[blockIdx.x];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, h = lane >> 5, d = a.width;
    const bool work = 32 * wave < it.rows;   // this wave has rows
    const int row = it.row0 + min(32 * wave + r, it.rows - 1);
    const uint64_t token = (uint64_t)it.q0 + row / a.share, head = (uint64_t)it.kv * a.share + row % a.share;

    // This row's q: of each 2 E columns the lane's half's E.
    vec q[CPR / 2];
    {
        const T *p = (const T *)a.q + token * a.qs[0] + head * a.qs[1];
#pragma unroll
        for (int s = 0; s < CPR / 2; ++s) {
            const int c = (2 * s + h) * E;
            q[s] = read_chunk(p + c, d - c);
#pragma unroll
            for (int e = 0; e < E; ++e) q[s][e] = from_f32<T>(to_f32(q[s][e]) * a.turn);
        }
    }

    // This thread's chunks of a tile.
    const T *kp[NL], *vp[NL];
    {
        const T *K = (const T *)a.k + (uint64_t)it.k0 * a.ks[0] + it.kv * a.ks[1];
        const T *V = (const T *)a.v + (uint64_t)it.k0 * a.vs[0] + it.kv * a.vs[1];
#pragma unroll
        for (int j = 0; j < NL; ++j) {
            const int i = tid + j * THREADS, key = i / CPR, c = i % CPR * E;
            kp[j] = K + key * a.ks[0] + c;
            vp[j] = V + key * a.vs[0] + c;
        }
    }
    const int32_t *mask = a.mask ? a.mask + it.k0 : nullptr;
    vec kr[NL], vr[NL];
    int alive = 0;   // of the held tile: key `lane` is live
    auto load = [&](int kb) {
        const bool mine = lane < KB && kb + lane < it.nk;
        alive = mine && mask ? mask[kb + lane] : mine;
#pragma unroll
        for (int j = 0; j < NL; ++j) {
            const int i = tid + j * THREADS, key = i / CPR, n = d - i % CPR * E;
            kr[j] = vr[j] = vec{};
            if (kb + key < it.nk) {
                kr[j] = read_chunk(kp[j] + kb * a.ks[0], n);
                // (A masked value weighs 0, but not if it is no number.)
                if (!mask || mask[kb + key] != 0) vr[j] = read_chunk(vp[j] + kb * a.vs[0], n);
            }
        }
    };
    auto place = [&](int buf) {
        char *K = smem + buf * 2 * BUF, *V = K + BUF;
#pragma unroll
        for (int j = 0; j < NL; ++j) {
            const int i = tid + j * THREADS, at = i / CPR * PITCH + i % CPR * 16;
            *(vec *)(K + at) = kr[j];
            *(vec *)(V + at) = vr[j];
        }
    };

    floatx16 o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] = floatx16{};
    float m = -INFINITY, l = 0.0f;
    bool any = false;   // a live key so far

    auto compute = [&](int buf, uint64_t live) {
        const char *K = smem + buf * 2 * BUF, *V = K + BUF;
        floatx16 s[SUB];
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            s[u] = floatx16{};
#pragma unroll
            for (int c = 0; c < CPR / 2; ++c) {
                const vec k = *(const vec *)(K + (32 * u + r) * PITCH + (2 * c + h) * 16);
                if constexpr (F32) {
#pragma unroll
                    for (int e = 0; e < E; ++e) s[u] = Mma<T>::run(k[e], q[c][e], s[u]);
                } else {
                    s[u] = Mma<T>::run(k, q[c], s[u]);
                }
            }
        }
        // Register i is key 8 (i / 4) + 4 h + i % 4 of its 32.
        if (live != (KB == 64 ? ~0ull : 0xffffffffull))   // uniform
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                const uint32_t word = (uint32_t)(live >> (32 * u)) >> (4 * h);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[u][i] = (word >> (8 * (i >> 2) + (i & 3))) & 1u ? s[u][i] : -INFINITY;
            }
        float mx = s[0][0];
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[u][i]);
        mx = both_max(mx) * a.scale;
        if (__ballot(mx > m + LAG) != 0) {
            const float mn = fmaxf(m, mx);
            // (Equal: both infinite, of one sign.)
            const float f = __builtin_amdgcn_exp2f(m == mn ? 0.0f : m - mn);
#pragma unroll
            for (int t = 0; t < DT; ++t) o[t] *= f;
            l *= f;
            m = mn;
        }
        const float base = m == -INFINITY ? 0.0f : m;
        float sum = 0.0f;
        // A score's distance from the maximum in one rounding; where the
        // maximum is so large that its own rounding shows, from the rounded
        // score, which is no larger.
        if (__ballot(fabsf(base) > 16777216.0f) == 0) {
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    s[u][i] = __builtin_amdgcn_exp2f(fmaf(s[u][i], a.scale, -base));
                    sum += s[u][i];
                }
        } else {
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    s[u][i] = __builtin_amdgcn_exp2f(rounded_less(s[u][i], a.scale, base));
                    sum += s[u][i];
                }
        }
        l += sum;
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            if constexpr (F32) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const char *at = V + (32 * u + 8 * (i >> 2) + 4 * h + (i & 3)) * PITCH + r * 4;
#pragma unroll
                    for (int t = 0; t < DT; ++t) o[t] = Mma<T>::run(*(const float *)(at + t * 128), s[u][i], o[t]);
                }
            } else {
                // 16 keys a product: registers 8 b .. 8 b + 7. A group of 16 lanes
                // reads 4 keys by 16 columns, and a lane gets its column's 4.
                typedef short s4 __attribute__((ext_vector_type(4)));
                const int g = lane >> 4, n = lane & 15;
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    frag p;
#pragma unroll
                    for (int e = 0; e < 8; ++e) p[e] = from_f32<T>(s[u][8 * b + e]);
                    const char *at = V + (32 * u + 16 * b + 4 * (g >> 1) + (n >> 2)) * PITCH + (16 * (g & 1) + 4 * (n & 3)) * 2;
#pragma unroll
                    for (int t = 0; t < DT; ++t) {
                        struct {
                            s4 lo, hi;
                        } v;
                        v.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) s4 *)(at + 64 * t));
                        v.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) s4 *)(at + 64 * t + 8 * PITCH));
                        o[t] = Mma<T>::run(__builtin_bit_cast(frag, v), p, o[t]);
                    }
                }
            }
        }
    };

    if (it.nk > 0) {
        load(0);
        place(0);
    }
    for (int kb = 0, buf = 0; kb < it.nk; kb += KB, buf ^= 1) {
        const uint64_t live = __ballot(alive != 0);
        __syncthreads();   // the tile is in LDS, and the other one read
        if (kb + KB < it.nk) load(kb + KB);
        any |= live != 0;
        if (work && live != 0) compute(buf, live);
        if (kb + KB < it.nk) place(buf ^ 1);
    }
    if (!work) return;

    l = both_sum(l);
    if (32 * wave + r >= it.rows) return;
    if (it.part < 0) {
        const float inv = any ? 1.0f / l : 0.0f;   // (all scores minus infinity: 0 times infinity)
        T *out = (T *)a.out + token * a.os[0] + head * a.os[1];
        typedef T loose4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = 32 * t + 8 * g + 4 * h;
                const loose4 y{from_f32<T>(o[t][4 * g] * inv), from_f32<T>(o[t][4 * g + 1] * inv),
                               from_f32<T>(o[t][4 * g + 2] * inv), from_f32<T>(o[t][4 * g + 3] * inv)};
                if (c + 4 <= d) {
                    *(loose4 *)(out + c) = y;
                } else {
#pragma unroll
                    for (int e = 0; e < 3; ++e)
                        if (c + e < d) out[c + e] = y[e];
                }
            }
        return;
    }
    float *p = part_of(a, it.part), *po = p + (uint64_t)(32 * wave + r) * d;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int c = 32 * t + 8 * (i >> 2) + 4 * h + (i & 3);
            if (c < d) po[c] = o[t][i];
        }
    if (h == 0) {
        float *ml = p + (uint64_t)a.part_rows * d + 2 * (32 * wave + r);
        ml[0] = m;
        ml[1] = any && m == -INFINITY && l == 0.0f ? 1.0f : l;
    }
}

// The parts of rows whose keys were cut: a wave a row, a lane a column of each 64.
template <typename T> __global__ void __launch_bounds__(256) cross_join(CrossArgs a) {
    const CrossJoin j = a.joins[blockIdx.x];
    const int lane = threadIdx.x & 63, d = a.width;
    for (int i = blockIdx.y * 4 + (threadIdx.x >> 6); i < j.rows; i += gridDim.y * 4) {
        float m = -INFINITY;
        for (int p = 0; p < j.parts; ++p) m = fmaxf(m, part_of(a, j.part0 + p)[(uint64_t)a.part_rows * d + 2 * i]);
        float l = 0.0f, o[2] = {0.0f, 0.0f};
        for (int p = 0; p < j.parts; ++p) {
            const float *part = part_of(a, j.part0 + p), *ml = part + (uint64_t)a.part_rows * d + 2 * i;
            const float w = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ml[0] - m);
            l = fmaf(w, ml[1], l);
#pragma unroll
            for (int u = 0; u < 2; ++u)
                if (lane + 64 * u < d) o[u] = fmaf(w, part[(uint64_t)i * d + lane + 64 * u], o[u]);
        }
        // No maximum: no live key (0), or scores of minus infinity alone.
        const float inv = m == -INFINITY ? (l == 0.0f ? 0.0f : __builtin_nanf("")) : 1.0f / l;
        const int row = j.row0 + i;
        T *out = (T *)a.out + ((uint64_t)j.q0 + row / a.share) * a.os[0] +
                 ((uint64_t)j.kv * a.share + row % a.share) * a.os[1];
#pragma unroll
        for (int u = 0; u < 2; ++u)
            if (lane + 64 * u < d) out[lane + 64 * u] = from_f32<T>(o[u] * inv);
    }
}

template <typename T> static hipError_t launch_cross(hipStream_t s, const CrossArgs &a) {
    const dim3 grid(a.n_items);
#define TILES(DP)                                                                                                \
    if (a.part_rows == 32) enqueue(cross_tiles<T, DP, 1>, grid, dim3(64), CrossTile<T, DP, 1>::LDS, s, a);        \
    else enqueue(cross_tiles<T, DP, 4>, grid, dim3(256), CrossTile<T, DP, 4>::LDS, s, a)
    if (a.width <= 32) { TILES(32); }
    else if (a.width <= 64) { TILES(64); }
    else if (a.width <= 96) { TILES(96); }
    else { TILES(128); }
#undef TILES
    if (a.n_joins) enqueue(cross_join<T>, dim3(a.n_joins, a.part_rows == 32 ? 2 : 8), dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t cross_attention(hipStream_t s, const CrossArgs &a) {
    if (a.n_items == 0) return hipSuccess;
    if (a.dt == Dt::F32) return launch_cross<float>(s, a);
    if (a.dt == Dt::F16) return launch_cross<_Float16>(s, a);
    return launch_cross<__bf16>(s, a);
}

}  // namespace rocm
