// hy3x_ops.h -- the operators' launches, arguments already checked, for the
// entry points of other translation units (the layer's forward).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/hy3x_moe.h"

namespace hy3x {

// HY3X_OK, or the error of hy3x_route_experts for this rule.
int check_route_spec(const hy3x_route_spec *spec);
void launch_route(const hy3x_route_spec &spec, const void *logits, int type, int64_t row_stride,
                  const float *bias, int T, int32_t *ids, float *w, hipStream_t st);

struct AdaptersShape {
  int d_in, d_out, device;
};
AdaptersShape adapters_shape(const hy3x_adapters *h);
void launch_adapters(const hy3x_adapters *h, const int32_t *ids, const void *x, int x_type,
                     int64_t x_stride, const void *base, int64_t base_stride, void *y, int y_type,
                     int64_t y_stride, int T, hipStream_t st);

}  // namespace hy3x
