// Row-in-registers kernels of norm - gate - add - norm for f16 elements.
#include "fln_nga_rows.cuh"

namespace fln {
FLN_NGA_INSTANTIATE(__half)
}  // namespace fln
