// The kernels of self_tiles.h for F32 rows.
#include "self_tiles.h"

namespace rocm {

hipError_t self_f32(hipStream_t s, const SelfArgs &a, const SelfLaunch &f) { return launch_self<float>(s, a, f); }

}  // namespace rocm
