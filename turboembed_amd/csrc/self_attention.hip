// Attention of a call's own tokens: each to the states of its sequence up to
// its own, over the rows of the call (a whole prompt) or over the pages of a
// cache.
//
// A wave takes a row (a token's head): a lane a key of each 64, then a lane a
// column of the values, with the running softmax in base 2 and F32.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "cache_find.h"
#include "devmath.h"
#include "launch.h"

namespace rocm {

template <typename T, bool I8> __global__ void __launch_bounds__(256) self_rows(SelfArgs a) {
    typedef typename std::conditional<I8, int8_t, T>::type H;
    const CacheArgs &c = a.c;
    const int lane = threadIdx.x & 63, d = c.width, heads = c.kv * a.share;
    const uint32_t rows = (uint32_t)c.tokens * (uint32_t)heads;
    for (uint32_t r = blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += gridDim.x * 4) {
        const int t = (int)(r / (uint32_t)heads), head = (int)(r - (uint32_t)t * (uint32_t)heads), g = head / a.share;
        int seq = seq_before(c, t);
        const int pos = position_of(c, t, seq);
        if (seq < 0 || seq >= c.seqs || t < within(c.starts[seq], 0, c.tokens)) continue;
        const T *q = (const T *)a.q + t * a.qs[0] + head * a.qs[1];
        float m = -INFINITY, l = 0.0f, o[2] = {0.0f, 0.0f};
        bool any = false;
        const int last = c.paged ? min(pos, room(c) - 1) : pos;
        for (int k0 = a.window > pos ? 0 : pos - a.window + 1; k0 <= last; k0 += 64) {
            const int p = k0 + lane;
            const int slot = p > last ? -1 : c.paged ? slot_of(c, seq, p) : within(c.starts[seq], 0, c.tokens) + p;
            float s = -INFINITY;
            if (slot >= 0) {
                const H *k = (const H *)c.k + (uint64_t)slot * c.ks[0] + g * c.ks[1];
                s = 0.0f;
                for (int e = 0; e < d; ++e) s = fmaf((float)q[e] * a.turn, (float)k[e], s);
                if constexpr (I8) s *= c.k_scales[(uint64_t)slot * c.kss + g];
                s *= a.scale;
            }
            const uint64_t live = __ballot(slot >= 0);
            any |= live != 0;
            float top = s;
#pragma unroll
            for (int w = 32; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor(top, w, 64));
            top = fmaxf(m, top);
            const float f = m == top ? 1.0f : exp2f(m - top), base = top == -INFINITY ? 0.0f : top;
            m = top;
            const float w = slot >= 0 ? exp2f(s - base) : 0.0f;
            l = l * f + wave_sum(w);
#pragma unroll
            for (int u = 0; u < 2; ++u) o[u] *= f;
            for (uint64_t rest = live; rest; rest &= rest - 1) {
                const int j = __ffsll((unsigned long long)rest) - 1;
                const uint64_t at = (uint64_t)__shfl(slot, j, 64);
                float wj = __shfl(w, j, 64);
                if constexpr (I8) wj *= c.v_scales[at * c.vss + g];
                const H *v = (const H *)c.v + at * c.vs[0] + g * c.vs[1];
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    if (lane + 64 * u < d) o[u] = fmaf(wj, (float)v[lane + 64 * u], o[u]);
            }
        }
        const float inv = any ? 1.0f / l : 0.0f;
        T *out = (T *)a.out + t * a.os[0] + head * a.os[1];
#pragma unroll
        for (int u = 0; u < 2; ++u)
            if (lane + 64 * u < d) out[lane + 64 * u] = from_f32<T>(o[u] * inv);
    }
}

hipError_t self_attention(hipStream_t s, const SelfArgs &a) {
    if (a.c.tokens == 0 || a.c.seqs == 0) return hipSuccess;
    const uint64_t rows = (uint64_t)a.c.tokens * a.c.kv * a.share;
    const dim3 grid((uint32_t)std::min<uint64_t>((rows + 3) / 4, 1 << 22));
    const auto go = [&](auto zero) {
        typedef decltype(zero) T;
        return a.i8 ? enqueue(self_rows<T, true>, grid, dim3(256), 0, s, a)
                    : enqueue(self_rows<T, false>, grid, dim3(256), 0, s, a);
    };
    if (a.dt == Dt::F32) return go(0.0f);
    if (a.dt == Dt::F16) return go((_Float16)0.0f);
    return go((__bf16)0.0f);
}

uint64_t self_workspace(uint64_t, uint64_t, int, int, int, Dt) { return 0; }

}  // namespace rocm
