// Row-in-registers kernels of norm - gate - add - norm for f32 elements.
#include "fln_nga_rows.cuh"

namespace fln {
FLN_NGA_INSTANTIATE(float)
}  // namespace fln
