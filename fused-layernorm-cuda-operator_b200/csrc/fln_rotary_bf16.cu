// Head norm + rotation kernels for bf16 elements.
#include "fln_rotary.cuh"

namespace fln {
FLN_ROTARY_INSTANTIATE(__nv_bfloat16)
}  // namespace fln
