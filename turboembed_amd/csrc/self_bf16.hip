// The kernels of self_tiles.h for BF16 rows.
#include "self_tiles.h"

namespace rocm {

hipError_t self_bf16(hipStream_t s, const SelfArgs &a, const SelfLaunch &f) { return launch_self<__bf16>(s, a, f); }

}  // namespace rocm
