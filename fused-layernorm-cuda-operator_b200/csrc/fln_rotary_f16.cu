// Head norm + rotation kernels for f16 elements.
#include "fln_rotary.cuh"

namespace fln {
FLN_ROTARY_INSTANTIATE(__half)
}  // namespace fln
