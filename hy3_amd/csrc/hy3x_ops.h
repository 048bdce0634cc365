// hy3x_ops.h -- the operators' launches, arguments already checked, for the
// entry points of other translation units (the layer's forward), and a check that
// several of them make.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/hy3x_moe.h"

namespace hy3x {

// HY3X_OK, or the error of hy3x_route_experts for this rule.
int check_route_spec(const hy3x_route_spec *spec);
void launch_route(const hy3x_route_spec &spec, const void *logits, int type, int64_t row_stride,
                  const float *bias, int T, int32_t *ids, float *w, hipStream_t st);

// Whether T rows of a_row bytes, a_step apart from a, and T rows of b share a
// byte. Rows of one wider buffer (equal steps) may lie between each other.
inline bool rows_overlap(const void *a, int64_t a_step, int64_t a_row, const void *b,
                         int64_t b_step, int64_t b_row, int T) {
  const uintptr_t a0 = (uintptr_t)a, b0 = (uintptr_t)b;
  const uintptr_t a1 = a0 + (uintptr_t)((T - 1) * a_step + a_row);
  const uintptr_t b1 = b0 + (uintptr_t)((T - 1) * b_step + b_row);
  if (a1 <= b0 || b1 <= a0) return false;
  if (a_step != b_step || T == 1) return true;
  const int64_t off = (int64_t)((b0 >= a0 ? b0 - a0 : a0 - b0) % (uintptr_t)a_step);
  const int64_t ab = b0 >= a0 ? off : (a_step - off) % a_step;  // b's place in a's rows
  return ab < a_row || ab + b_row > a_step;
}

struct AdaptersShape {
  int d_in, d_out, device;
};
AdaptersShape adapters_shape(const hy3x_adapters *h);
void launch_adapters(const hy3x_adapters *h, const int32_t *ids, const void *x, int x_type,
                     int64_t x_stride, const void *base, int64_t base_stride, void *y, int y_type,
                     int64_t y_stride, int T, hipStream_t st);

}  // namespace hy3x
