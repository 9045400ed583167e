// The int8 product on the caller's codes and scales.
#include <hip/hip_runtime.h>

#include "devmath.h"
#include "launch.h"
#include "operators.h"

namespace rocm {

// An output from its exact sum: both scales, then the bias, each rounded.
__device__ __forceinline__ float scaled(int sum, float as, float ws, float bias) {
#pragma clang fp contract(off)
    return (float)sum * as * ws + bias;
}

__device__ __forceinline__ void put(void *out, Dt t, uint64_t at, float v) {
    if (t == Dt::F32) ((float *)out)[at] = v;
    else if (t == Dt::F16) ((_Float16 *)out)[at] = (_Float16)v;
    else ((__bf16 *)out)[at] = (__bf16)v;
}

// An output a lane, its products one by one.
__global__ void __launch_bounds__(256) linear_i8_plain(LinearArgs a) {
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < (uint64_t)a.m * a.n; i += (uint64_t)gridDim.x * 256) {
        const uint64_t m = i / a.n, n = i % a.n;
        int sum = 0;
        for (int k = 0; k < a.k; ++k) sum += (int)a.a[m * a.lda + k] * a.w[n * a.ldw + k];
        put(a.out, a.ot, m * a.ldo + n, scaled(sum, a.as[m], a.ws[n], a.bias ? a.bias[n] : 0.0f));
    }
}

hipError_t linear_i8(hipStream_t s, const LinearArgs &a) {
    if (a.m <= 0 || a.n <= 0) return hipSuccess;
    const uint64_t blocks = ((uint64_t)a.m * a.n + 255) / 256;
    enqueue(linear_i8_plain, dim3((uint32_t)(blocks < (1 << 20) ? blocks : 1 << 20)), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace rocm
