// Attention of queries to an encoder's states of another length.
#include <hip/hip_runtime.h>

#include "devmath.h"
#include "launch.h"
#include "operators.h"

namespace rocm {

// A wave a row; a lane a key of each 64, then a lane two columns of V.
template <typename T> __global__ void __launch_bounds__(256) cross_plain(CrossArgs a) {
    const CrossItem it = a.items[blockIdx.x];
    const int lane = threadIdx.x & 63, d = a.width;
    for (int r = it.row0 + (threadIdx.x >> 6); r < it.row0 + it.rows; r += 4) {
        const uint64_t token = it.q0 + r / a.share, head = it.kv * a.share + r % a.share;
        const T *q = (const T *)a.q + token * a.qs[0] + head * a.qs[1];
        const T *K = (const T *)a.k + it.kv * a.ks[1], *V = (const T *)a.v + it.kv * a.vs[1];
        float m = -INFINITY, l = 0.0f, o[2] = {0.0f, 0.0f};
        bool any = false;
        for (int kb = 0; kb < it.nk; kb += 64) {
            const uint64_t key = (uint64_t)it.k0 + kb + lane;
            const bool live = kb + lane < it.nk && (!a.mask || a.mask[key] != 0);
            float s = 0.0f;
            if (live) {
                const T *k = K + key * a.ks[0];
                for (int c = 0; c < d; ++c) s = fmaf(to_f32(q[c]), to_f32(k[c]), s);
                s *= a.scale;
            }
            const uint64_t alive = __ballot(live);
            any |= alive != 0;
            float top = live ? s : -INFINITY;
#pragma unroll
            for (int w = 32; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor(top, w, 64));
            const float mn = fmaxf(m, top), safe = mn == -INFINITY ? 0.0f : mn;
            const float f = __builtin_amdgcn_exp2f(m == mn ? 0.0f : m - safe);
            const float p = live ? __builtin_amdgcn_exp2f(s - safe) : 0.0f;
            l = l * f + wave_sum(p);
            o[0] *= f, o[1] *= f;
            m = mn;
            for (int j = 0; j < 64 && kb + j < it.nk; ++j) {
                if (!((alive >> j) & 1)) continue;
                const float pj = __shfl(p, j, 64);
                const T *v = V + ((uint64_t)it.k0 + kb + j) * a.vs[0];
                for (int u = 0; u < 2; ++u)
                    if (lane + 64 * u < d) o[u] = fmaf(pj, to_f32(v[lane + 64 * u]), o[u]);
            }
        }
        T *out = (T *)a.out + token * a.os[0] + head * a.os[1];
        for (int u = 0; u < 2; ++u)
            if (lane + 64 * u < d) out[lane + 64 * u] = from_f32<T>(any ? o[u] / l : 0.0f);
    }
}

hipError_t cross_attention(hipStream_t s, const CrossArgs &a) {
    if (a.n_items == 0) return hipSuccess;
    const dim3 grid(a.n_items), block(256);
    if (a.dt == Dt::F32) enqueue(cross_plain<float>, grid, block, 0, s, a);
    else if (a.dt == Dt::F16) enqueue(cross_plain<_Float16>, grid, block, 0, s, a);
    else enqueue(cross_plain<__bf16>, grid, block, 0, s, a);
    return hipGetLastError();
}

}  // namespace rocm
