// Attention of queries to an encoder's states of another length.
//
// A workgroup takes an item of the plan: 32 rows a wave (a row is a query
// token's head; those that share a key head are rows of one item, so that its
// keys and values are read once for them) against a run of keys. K and V
// pass through LDS in tiles of KB keys, two of each: the next tile is on its
// way while one is computed. Scores are computed transposed, S^T = K Q^T, so
// that a lane holds one row (lane % 32) and 16 of 32 keys, the other 16 in the
// lane 32 away; O^T += V^T P^T then takes P as the score registers hold it,
// against V's columns for the same keys in that order (16-bit values by LDS
// reads that transpose, F32 values one by one).
//
// The softmax is the running one, in base 2 and F32, and most tiles rescale
// nothing: what it takes for a row's maximum moves only when a score is 2^8
// above the one that it was set by. The scale is positive here (the launcher
// turns q around for a negative one).
//
// One token a sequence is bound by the keys' and values' bytes: 48 by 200 to
// 4096 states, 16 heads of 64, BF16, take 93 us with the join (4.5 TB/s). Long
// F16 queries are bound by the softmax's vector instructions beside the
// products: 8 x 1024-2048 tokens by 2048-8192 states, 16 heads of 64, take 289
// us (815 TFLOP/s); 4 x 1024 by 4096, 16 heads of 128 in BF16, 137 (1000). F32
// is bound by its matrix instructions, 64 cycles each: a tile of 32 keys by 32
// rows of 64 is 4096 cycles; 24 x 5-77 tokens by 33-500 states, 12 heads, take
// 33 us.
// (Tiles of 32 keys where a wave is alone, so that more of them fit; of 64
// where four share them, which halves the barriers.)
#include <hip/hip_runtime.h>

#include <algorithm>
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

typedef float f32x4 __attribute__((ext_vector_type(4)));

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

// Where a part of `rows` rows lies in the workspace.
__device__ __forceinline__ float *part_of(const CrossArgs &a, int part) {
    return a.ws + (uint64_t)part * cross_part_floats(a.most_rows, a.width);
}

// DP: the head width rounded up to 32, 64, 96 or 128. A tile's rows are DP
// elements in LDS, chunk c of key k at place c ^ swap(k), so that what a
// read's pass reads lies in different banks.
// DIRECT: keys and values in aligned whole chunks, which go to LDS by themselves
// (a kernel of its own: the other's registers cost it a wave a SIMD).
template <typename T, int DP, int WAVES, bool DIRECT> struct CrossTile {
    static constexpr bool F32 = std::is_same<T, float>::value;
    static constexpr int KB = WAVES == 1 || F32 ? 32 : 64;
    static constexpr int PITCH = DP * (int)sizeof(T), CPR = PITCH / 16;
    static constexpr int BUF = KB * PITCH;
    static constexpr int LDS = 4 * BUF;   // K and V, two tiles of each
    // Waves a SIMD, at least.
    static constexpr int OCC = F32 ? (DP <= (DIRECT ? 96 : 64) || WAVES == 4 ? 2 : 1) : DP <= 64 ? 3 : 2;
    // LDS serves 256 bytes a cycle: 16 keys of one chunk of K (a 16-byte
    // read's pass), 4 keys of 4 chunks of V (a transposing read's).
    static constexpr int PERIOD = CPR % 16 == 0 ? 1 : CPR % 8 == 0 ? 2 : 4;   // keys until the banks repeat
    static __device__ __forceinline__ int swap_k(int key) { return key / PERIOD % (16 / PERIOD); }
    static __device__ __forceinline__ int swap_v(int key) {
        if (F32) return CPR % 16 == 0 ? (key >> 2 & 1) * 8 : 0;   // (a read's pass: 8 chunks of keys k and k + 4)
        return PERIOD == 1 ? (key & 3) * 4 : PERIOD == 2 ? (key >> 1 & 1) * 4 : 0;
    }
};

// TWO: 16-bit weights are two numbers of T each for the product with V, not one.
// That is so where no item has more than a wave's rows: the keys' and values'
// bytes bound it, and the second product mostly hides behind them (48 x 1 by
// 200-4096, BF16: heads of 64 93.0 us for 92.4, of 128 165.7 for 162.7; 64 x 4
// by 1024, four heads of 80 a key head, where one wave computes and three
// load, 31.8 for 27.6; the first's error 2.3e-3 with one, 1.7e-3, the output's
// own rounding, with two). Where four waves compute, the vector instructions
// bound it: two numbers would take 407 us for 290 (8 x 1024-2048 by 2048-8192,
// F16; errors 2.1e-4 and 2.9e-4), so a weight is rounded once.
template <typename T, int DP, int WAVES, bool DIRECT, bool TWO>
__global__ void __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(CrossTile<T, DP, WAVES, DIRECT>::OCC)))
cross_tiles(CrossArgs a) {
    using C = CrossTile<T, DP, WAVES, DIRECT>;
    constexpr bool F32 = C::F32;
    constexpr int KB = C::KB, SUB = KB / 32, PITCH = C::PITCH, BUF = C::BUF, CPR = C::CPR, DT = DP / 32;
    constexpr int E = Chunk<T>::N, NL = KB * CPR / 64 / WAVES;
    static_assert(NL * 64 * WAVES == KB * CPR, "whole loads a wave");
    // m is LEAD above the maximum (base 2) that it was set by, and is set again
    // by one that is LAG above that. With a LEAD of LAG weights are 1 at most, so
    // that values of F32's size add up to finite sums. F16's need no such room,
    // and its weights have no range to give away: there they reach 2^LAG.
    constexpr float LAG = 8.0f, LEAD = std::is_same<T, _Float16>::value ? 0.0f : LAG;
    constexpr uint64_t FULL = KB == 64 ? ~0ull : 0xffffffffull;
    typedef typename Chunk<T>::vec vec;
    typedef typename Mma<T>::frag frag;
    extern __shared__ __attribute__((aligned(1024))) char smem[];

    const CrossItem it = a.items[blockIdx.x];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, h = lane >> 5, d = a.width;
    const bool work = 32 * wave < it.rows;   // this wave has rows
    const int row = it.row0 + min(32 * wave + r, it.rows - 1);
    const int of_token = a.share == 1 ? row : row / a.share;
    const uint64_t token = (uint64_t)it.q0 + of_token, head = (uint64_t)it.kv * a.share + (row - of_token * a.share);

    // This lane's places of a tile: load j of the wave fills 64 chunks in order.
    const T *K0 = (const T *)a.k + (uint64_t)it.k0 * a.ks[0] + it.kv * a.ks[1];
    const T *V0 = (const T *)a.v + (uint64_t)it.k0 * a.vs[0] + it.kv * a.vs[1];
    const auto key_of = [&](int j) { return ((wave * NL + j) * 64 + lane) / CPR; };
    const auto col_k = [&](int j) { return (((wave * NL + j) * 64 + lane) % CPR ^ C::swap_k(key_of(j))) * E; };
    const auto col_v = [&](int j) { return (((wave * NL + j) * 64 + lane) % CPR ^ C::swap_v(key_of(j))) * E; };
    // (DIRECT: bytes from a tile's first key, which 31 bits hold; else elements.)
    typedef typename std::conditional<DIRECT, uint32_t, uint64_t>::type place;
    place ko[NL], vo[NL];
#pragma unroll
    for (int j = 0; j < NL; ++j) {
        constexpr place size = DIRECT ? sizeof(T) : 1;
        ko[j] = (key_of(j) * (place)a.ks[0] + col_k(j)) * size, vo[j] = (key_of(j) * (place)a.vs[0] + col_v(j)) * size;
    }
    const int32_t *mask = a.mask ? a.mask + it.k0 : nullptr;
    int alive = 1;   // of the tile on its way: key `lane` is live

    // Starts a tile on its way to LDS: aligned rows of whole chunks go there by
    // themselves, others through registers at once. Keys past the last repeat it.
    const auto load = [&](int kb, int buf) {
        char *K = smem + buf * 2 * BUF, *V = K + BUF;
        const T *kt = K0 + kb * a.ks[0], *vt = V0 + kb * a.vs[0];
        const int last = it.nk - 1 - kb;
        if (mask || last < KB - 1) {   // uniform
            const int key = min(lane, last);
            alive = lane <= last && (!mask || mask[kb + key] != 0);
        }
        if constexpr (DIRECT) {
            // (As buffer loads: those count as vector memory alone, so the reads
            // of LDS below wait for no load.)
            typedef __attribute__((address_space(3))) void *to;
            const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc((void *)kt, (short)0, -1, 0x00020000);
            const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc((void *)vt, (short)0, -1, 0x00020000);
            const auto send = [&](__amdgpu_buffer_rsrc_t tile, uint32_t at, char *dst) {
                __builtin_amdgcn_raw_ptr_buffer_load_lds(tile, (to)dst, 16, (int)at, 0, 0, 0);
            };
            if (last >= KB - 1 && d == DP) {   // uniform
#pragma unroll
                for (int j = 0; j < NL; ++j)
                    send(kr, ko[j], K + (wave * NL + j) * 1024);
#pragma unroll
                for (int j = 0; j < NL; ++j)
                    send(vr, vo[j], V + (wave * NL + j) * 1024);
            } else {
#pragma unroll
                for (int j = 0; j < NL; ++j) {
                    const uint32_t back = max(0, key_of(j) - last) * (uint32_t)sizeof(T);
                    // (Columns past the width keep the zeros they began with.)
                    if (col_k(j) < d) send(kr, ko[j] - back * (uint32_t)a.ks[0], K + (wave * NL + j) * 1024);
                    if (col_v(j) < d) send(vr, vo[j] - back * (uint32_t)a.vs[0], V + (wave * NL + j) * 1024);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < NL; ++j) {
                const int64_t back = min(0, last - key_of(j));
                const int at = ((wave * NL + j) * 64 + lane) * 16, nk = d - col_k(j), nv = d - col_v(j);
                *(vec *)(K + at) = nk > 0 ? read_chunk(kt + ko[j] + back * (int64_t)a.ks[0], nk) : vec{};
                *(vec *)(V + at) = nv > 0 ? read_chunk(vt + vo[j] + back * (int64_t)a.vs[0], nv) : vec{};
            }
        }
    };

    if (DIRECT && d < DP) {   // uniform
        for (int i = tid; i < C::LDS / 16; i += 64 * WAVES) *(vec *)(smem + i * 16) = vec{};
        __syncthreads();
    }
    if (it.nk > 0) load(0, 0);
    // This row's q: of each 2 E columns the lane's half's E.
    vec q[CPR / 2];
    {
        const T *p = (const T *)a.q + token * a.qs[0] + head * a.qs[1];
#pragma unroll
        for (int s = 0; s < CPR / 2; ++s) {
            const int c = (2 * s + h) * E;
            q[s] = read_chunk(p + c, d - c);
        }
        if (a.turn != 1.0f)   // uniform
#pragma unroll
            for (int s = 0; s < CPR / 2; ++s)
#pragma unroll
                for (int e = 0; e < E; ++e) q[s][e] = from_f32<T>(to_f32(q[s][e]) * a.turn);
    }

    floatx16 o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] = floatx16{};
    float m = -INFINITY, l = 0.0f;
    bool any = false, far = false;   // a live key so far; a maximum past 2^24

    // S^T of 32 keys. Register i is key 8 (i / 4) + 4 h + i % 4.
    const int kr = r * PITCH, ks = C::swap_k(r);   // (32 keys on, the swap is the same)
    const auto scores = [&](const char *K, floatx16 (&s)[SUB]) {
#pragma unroll
        for (int u = 0; u < SUB; ++u) s[u] = floatx16{};
        const auto chunk = [&](int c, int u) {
            return *(const vec *)(K + 32 * u * PITCH + kr + ((2 * c + h) ^ ks) * 16);
        };
        if constexpr (F32) {
            // (A chunk read two ahead of its products, which are slow enough to hide it.)
            vec k[3] = {chunk(0, 0), chunk(1, 0)};
#pragma unroll
            for (int c = 0; c < CPR / 2; ++c) {
                if (c + 2 < CPR / 2) k[(c + 2) % 3] = chunk(c + 2, 0);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int e = 0; e < E; ++e) s[0] = Mma<T>::run(k[c % 3][e], q[c][e], s[0]);
            }
        } else {
#pragma unroll
            for (int c = 0; c < CPR / 2; ++c)
#pragma unroll
                for (int u = 0; u < SUB; ++u) s[u] = Mma<T>::run(chunk(c, u), q[c], s[u]);
        }
    };
    // O^T += V^T P^T over 32 keys; weight(i) is register i's, in order.
    const auto add_values = [&](const char *V, auto weight) {
        if constexpr (F32) {
            // (Values and weights two keys ahead of their products.)
            float v[3][DT], p[3];
            const auto ahead = [&](int i) {
                const int key = 8 * (i >> 2) + 4 * h + (i & 3);
#pragma unroll
                for (int t = 0; t < DT; ++t)
                    v[i % 3][t] =
                        *(const float *)(V + key * PITCH + (((r >> 2) + 8 * t) ^ C::swap_v(key)) * 16 + (r & 3) * 4);
                p[i % 3] = weight(i);
            };
            ahead(0), ahead(1);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (i + 2 < 16) ahead(i + 2);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int t = 0; t < DT; ++t) o[t] = Mma<T>::run(v[i % 3][t], p[i % 3], o[t]);
            }
        } else {
            // 16 keys a product: registers 8 j .. 8 j + 7. A group of 16 lanes
            // reads 4 keys by 16 columns, and a lane gets its column's 4.
            typedef short s4 __attribute__((ext_vector_type(4)));
            const int g = lane >> 4, n = lane & 15, key = 4 * (g >> 1) + (n >> 2);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                frag f, rest, vt[DT];
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float w0 = weight(8 * j + e), w1 = weight(8 * j + e + 1);
                    if constexpr (TWO) {
                        const auto hi = below<T>(w0, w1);
                        f[e] = hi[0], f[e + 1] = hi[1];
                        rest[e] = from_f32<T>(w0 - to_f32(hi[0])), rest[e + 1] = from_f32<T>(w1 - to_f32(hi[1]));
                    } else {
                        f[e] = from_f32<T>(w0), f[e + 1] = from_f32<T>(w1);
                    }
                }
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    const int c = 4 * t + 2 * (g & 1) + ((n >> 1) & 1);
                    const auto at = [&](int k) {
                        return (__attribute__((address_space(3))) s4 *)(V + k * PITCH + (c ^ C::swap_v(k)) * 16 + (n & 1) * 8);
                    };
                    struct {
                        s4 lo, hi;
                    } v;
                    v.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at(16 * j + key));
                    v.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at(16 * j + 8 + key));
                    vt[t] = __builtin_bit_cast(frag, v);
                    o[t] = Mma<T>::run(vt[t], f, o[t]);
                }
                if constexpr (TWO)
#pragma unroll
                    for (int t = 0; t < DT; ++t) o[t] = Mma<T>::run(vt[t], rest, o[t]);
            }
        }
    };
    const auto raise = [&](float mx) {   // m, for scores of up to mx
        if (__ballot(mx > m + (LAG - LEAD)) == 0) return;
        const float mn = fmaxf(m, mx + LEAD);
        // (Equal: both infinite, of one sign.)
        const float f = __builtin_amdgcn_exp2f(m == mn ? 0.0f : m - mn);
#pragma unroll
        for (int t = 0; t < DT; ++t) o[t] *= f;
        l *= f;
        m = mn;
        far = __ballot(fabsf(m) > 16777216.0f && m != -INFINITY) != 0;
    };
    const auto tile = [&](const char *K, uint64_t live) {
        floatx16 s[SUB];
        scores(K, s);
        if (live != FULL) {   // uniform
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                const uint32_t word = (uint32_t)(live >> (32 * u)) >> (4 * h);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[u][i] = (word >> (8 * (i >> 2) + (i & 3))) & 1u ? s[u][i] : -INFINITY;
            }
        }
        float mx = s[0][0];
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[u][i]);
        raise(both_max(mx) * a.scale);
        const float base = m == -INFINITY ? 0.0f : m;
        // A score's distance from the maximum in one rounding; where the
        // maximum is so large that its own rounding shows, from the rounded
        // score, which is no larger.
        float scale = a.scale;
        if (far) {   // uniform
#pragma unroll
            for (int u = 0; u < SUB; ++u) s[u] *= scale;
            scale = 1.0f;
        }
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            float sum = 0.0f;
            add_values(K + BUF + 32 * u * PITCH, [&](int i) {
                const float w = __builtin_amdgcn_exp2f(fmaf(s[u][i], scale, -base));
                sum += w;
                return w;
            });
            l += sum;
        }
    };

    for (int kb = 0, buf = 0; kb < it.nk; kb += KB, buf ^= 1) {
        __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): this wave's loads are in LDS
        const uint64_t live = __ballot(lane < KB && alive);
        if (live != FULL) {   // uniform
            // A masked value weighs 0, but not if it is no number.
#pragma unroll
            for (int j = 0; j < NL; ++j)
                if (!((live >> key_of(j)) & 1))
                    *(vec *)(smem + buf * 2 * BUF + BUF + ((wave * NL + j) * 64 + lane) * 16) = vec{};
        }
        __syncthreads();   // the tile is there, and the other one read
        if (kb + KB < it.nk) load(kb + KB, buf ^ 1);
        any |= live != 0;
        if (work && live != 0) tile(smem + buf * 2 * BUF, live);
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
    // Four columns of every row, then the next four; then the maxima and sums.
    f32x4 *p = (f32x4 *)part_of(a, it.part);
    const int at = 32 * wave + r, groups = (d + 3) / 4;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = 8 * t + 2 * g + h;
            if (c < groups) p[c * it.rows + at] = f32x4{o[t][4 * g], o[t][4 * g + 1], o[t][4 * g + 2], o[t][4 * g + 3]};
        }
    if (h == 0) {
        float2 *ml = (float2 *)(p + groups * it.rows);
        ml[at] = float2{m, any && m == -INFINITY && l == 0.0f ? 1.0f : l};
    }
}

// The parts of rows whose keys were cut: a wave a row, a lane a column of each 64.
template <typename T> __global__ void __launch_bounds__(256) cross_join(CrossArgs a) {
    const CrossJoin j = a.joins[blockIdx.x];
    const int lane = threadIdx.x & 63, waves = blockDim.x >> 6, d = a.width, groups = (d + 3) / 4;
    const uint64_t pitch = cross_part_floats(a.most_rows, d);
    const float *first = part_of(a, j.part0);
    for (int i = blockIdx.y * waves + (threadIdx.x >> 6); i < j.rows; i += gridDim.y * waves) {
        // A lane a part: its maximum and sum.
        const float *ml = first + 4 * groups * j.rows + 2 * i;
        float m = -INFINITY;
        for (int p = lane; p < j.parts; p += 64) m = fmaxf(m, ml[p * pitch]);
#pragma unroll
        for (int w = 32; w > 0; w >>= 1) m = fmaxf(m, __shfl_xor(m, w, 64));
        float l = 0.0f, o[2] = {0.0f, 0.0f};
        for (int p0 = 0; p0 < j.parts; p0 += 64) {
            const int n = min(64, j.parts - p0);
            float w = 0.0f;
            if (lane < n) {
                const float *q = ml + (p0 + lane) * pitch;
                w = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(q[0] - m);
                l = fmaf(w, q[1], l);
            }
            const float *part = first + p0 * pitch + 4 * i + (lane & 3);
#pragma unroll 4
            for (int p = 0; p < n; ++p, part += pitch) {
                const float wp = __shfl(w, p, 64);
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    if (lane + 64 * u < d) o[u] = fmaf(wp, part[((lane >> 2) + 16 * u) * 4 * j.rows], o[u]);
            }
        }
        l = wave_sum(l);
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

template <typename T, bool DIRECT> static hipError_t launch_cross(hipStream_t s, const CrossArgs &a) {
    const dim3 grid(a.n_items);
    constexpr bool F32 = std::is_same<T, float>::value;
    hipError_t e;
#define WAVES(DP, W, TWO) \
    e = enqueue(cross_tiles<T, DP, W, DIRECT, TWO>, grid, dim3(64 * W), CrossTile<T, DP, W, DIRECT>::LDS, s, a)
#define TILES(DP)                                   \
    if (a.part_rows == 32) WAVES(DP, 1, !F32);      \
    else if (a.one_wave) WAVES(DP, 4, !F32);        \
    else WAVES(DP, 4, false)
    if (a.width <= 32) { TILES(32); }
    else if (a.width <= 64) { TILES(64); }
    else if (a.width <= 96) { TILES(96); }
    else { TILES(128); }
#undef TILES
#undef WAVES
    if (e != hipSuccess || a.n_joins == 0) return e;
    const int waves = a.most_rows < 4 ? a.most_rows : 4;
    return enqueue(cross_join<T>, dim3(a.n_joins, (a.most_rows + 2 * waves - 1) / (2 * waves)), dim3(64 * waves), 0, s, a);
}

hipError_t cross_attention(hipStream_t s, const CrossArgs &a) {
    if (a.n_items == 0) return hipSuccess;
    const auto whole = [&](const void *p, const uint64_t (&stride)[2]) {
        const uint64_t size = dt_bytes(a.dt);
        return (reinterpret_cast<uintptr_t>(p) | stride[0] * size | stride[1] * size) % 16 == 0;
    };
    // (Keys and values in aligned whole chunks, a tile of them within 31 bits.)
    const bool direct = a.width * dt_bytes(a.dt) % 16 == 0 && whole(a.k, a.ks) && whole(a.v, a.vs) &&
                        std::max(a.ks[0], a.vs[0]) < (1u << 31) / 64 / 4;
    const auto go = [&](auto zero) {
        typedef decltype(zero) T;
        return direct ? launch_cross<T, true>(s, a) : launch_cross<T, false>(s, a);
    };
    if (a.dt == Dt::F32) return go(0.0f);
    if (a.dt == Dt::F16) return go((_Float16)0.0f);
    return go((__bf16)0.0f);
}

}  // namespace rocm
