// hy3x_linear4_f16.hip -- the products of 4-bit weights for f16 x.
#include "hy3x_linear4_kernels.h"

namespace hy3x {
template void launch_linear4<__half>(const Linear4Call &c, hipStream_t st);
}
