// Head norm + rotation kernels for f32 elements.
#include "fln_rotary.cuh"

namespace fln {
FLN_ROTARY_INSTANTIATE(float)
}  // namespace fln
