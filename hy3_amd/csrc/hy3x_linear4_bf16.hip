// hy3x_linear4_bf16.hip -- the products of 4-bit weights for bf16 x.
#include "hy3x_linear4_kernels.h"

namespace hy3x {
template void launch_linear4<__hip_bfloat16>(const Linear4Call &c, hipStream_t st);
}
