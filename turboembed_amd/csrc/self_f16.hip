// The kernels of self_tiles.h for F16 rows.
#include "self_tiles.h"

namespace rocm {

hipError_t self_f16(hipStream_t s, const SelfArgs &a, const SelfLaunch &f) { return launch_self<_Float16>(s, a, f); }

}  // namespace rocm
