// Row-in-registers kernels of norm - gate - add - norm for bf16 elements.
#include "fln_nga_rows.cuh"

namespace fln {
FLN_NGA_INSTANTIATE(__nv_bfloat16)
}  // namespace fln
