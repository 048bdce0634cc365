// hy3x_error.h -- the error channel of the library's entry points, for the
// translation units beside hy3x_layer.hip (which holds the message).
#pragma once
#include <stdarg.h>
#include <stdio.h>

namespace hy3x {

int set_error(int code, const char *msg);  // the message hy3x_last_error() returns

static int op_fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
static int op_fail(int code, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return set_error(code, buf);
}

}  // namespace hy3x

#define OP_HIP_TRY(call)                                                              \
  do {                                                                                \
    hipError_t e_ = (call);                                                           \
    if (e_ != hipSuccess)                                                             \
      return hy3x::op_fail(HY3X_E_HIP, "%s failed: %s (%s:%d)", #call,                \
                           hipGetErrorString(e_), __FILE__, __LINE__);                \
  } while (0)
