// hy3x_mfma_raw_wide.hip -- hy3x_mfma_raw.hip in the wide shape, namespace
// hy3x::mfma_raw_wide.
#define HY3X_MFMA_RAW
#define HY3X_MFMA_WIDE
#include "hy3x_mfma.hip"
