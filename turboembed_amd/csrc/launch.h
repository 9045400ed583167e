// The one way the kernel sources enqueue a kernel: through the launch hook
// (LaunchTiming), so a timed run's events are bound to the kernels' own
// dispatch packets. The status is the launch's own; hipGetLastError's may be
// of any call that this thread's program has made before.
#pragma once

#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>

#include <tuple>

#include "kernels.h"

namespace rocm {

template <typename... Formals, typename... Actuals>
inline hipError_t enqueue(void (*k)(Formals...), dim3 grid, dim3 block, uint32_t lds, hipStream_t s, Actuals... a) {
    LaunchTiming &t = launch_timing();
    std::tuple<Formals...> args{static_cast<Formals>(a)...};
    const hipError_t e = std::apply(
        [&](auto &...arg) {
            void *at[] = {(void *)&arg...};
            return hipExtLaunchKernel((const void *)k, grid, block, at, lds, s, t.start, t.stop, 0);
        },
        args);
    if (t.stop) {
        t.start = nullptr;
        t.bound = true;
    }
    return e;
}

}  // namespace rocm
