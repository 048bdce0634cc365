// hy3x_linear4_f32.hip -- the products of 4-bit weights for f32 x.
#include "hy3x_linear4_kernels.h"

namespace hy3x {
template void launch_linear4<float>(const Linear4Call &c, hipStream_t st);
}
