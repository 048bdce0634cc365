// hy3x_mfma_raw.hip -- the narrow shape's gate/up GEMM for a shared expert with
// adapters: the same source, compiled with HY3X_MFMA_RAW into namespace
// hy3x::mfma_raw. The shared expert's gate and up products are stored too, in
// fp32 (out[token][gate | up]), for the adapters to add to.
#define HY3X_MFMA_RAW
#include "hy3x_mfma.hip"
