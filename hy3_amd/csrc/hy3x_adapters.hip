// hy3x_adapters.hip -- low-rank adapters of many requests at once beside a
// shared projection (hy3x_adapters_*):
//
//   u = A_a x_t            (fp32 sums over d_in)
//   y_t = base_t + scale_a (B_a u)   (fp32 sums over the rank, y rounded once)
//
// The handle keeps every adapter's A and B padded with zeros to whole tiles.
// A block takes one token and a slice of its outputs and forms u for itself:
// nothing passes between blocks, so there is no scratch memory and no second
// launch.
#include <hip/hip_bf16.h>
#include <string.h>

#include <new>

#include "../../include/hy3x_moe.h"
#include "hy3x_common.h"
#include "hy3x_error.h"

struct hy3x_adapters {
  int device = 0, count = 0, rank = 0, d_in = 0, d_out = 0, type = 0;
  int rp = 0, kp = 0, np = 0;  // rank, d_in and d_out padded to whole tiles
  uint16_t *a = nullptr;       // [count][rp][kp]
  uint16_t *b = nullptr;       // [count][np][rp]
  float *scale = nullptr;      // [count]
};

namespace hy3x {
namespace {

__device__ __forceinline__ float elem(float v) { return v; }
__device__ __forceinline__ float elem(__half v) { return __half2float(v); }
__device__ __forceinline__ float elem(__hip_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float *p, float v) { *p = v; }
__device__ __forceinline__ void put(__half *p, float v) { *p = __float2half(v); }
__device__ __forceinline__ void put(__hip_bfloat16 *p, float v) { *p = __float2bfloat16(v); }

constexpr int SLICE = 256;  // outputs per block

template <class W, class X, class Y>
__global__ __launch_bounds__(256) void k_adapters(
    const W *__restrict__ a, const W *__restrict__ b, const float *__restrict__ scale, int count,
    int rp, int kp, int np, int d_in, int d_out, const int32_t *__restrict__ ids,
    const X *__restrict__ x, int64_t x_stride, const Y *base, int64_t base_stride, Y *y,
    int64_t y_stride) {
  __shared__ float u[HY3X_ADAPTERS_MAX_RANK];
  const int t = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int id = ids[t];
  const bool has = id >= 0 && id < count;
  if (has) {
    for (int r = wave; r < rp; r += 4) {
      const W *ar = a + ((int64_t)id * rp + r) * kp;
      float sum = 0.0f;
      for (int k = lane; k < d_in; k += 64) sum += elem(ar[k]) * elem(x[t * x_stride + k]);
      sum = wave_sum(sum);
      if (lane == 0) u[r] = sum;
    }
  }
  __syncthreads();
  const int c = blockIdx.y * SLICE + threadIdx.x;
  if (c >= d_out) return;
  float v = base ? elem(base[t * base_stride + c]) : 0.0f;
  if (has) {
    const W *br = b + ((int64_t)id * np + c) * rp;
    float sum = 0.0f;
    for (int r = 0; r < rp; r++) sum += elem(br[r]) * u[r];
    v += scale[id] * sum;
  }
  put(y + t * y_stride + c, v);
}

template <class W, class X, class Y>
void launch(const hy3x_adapters *h, const int32_t *ids, const void *x, int64_t x_stride,
            const void *base, int64_t base_stride, void *y, int64_t y_stride, int T,
            hipStream_t st) {
  k_adapters<W, X, Y><<<dim3(T, (h->d_out + SLICE - 1) / SLICE), 256, 0, st>>>(
      (const W *)h->a, (const W *)h->b, h->scale, h->count, h->rp, h->kp, h->np, h->d_in,
      h->d_out, ids, (const X *)x, x_stride, (const Y *)base, base_stride, (Y *)y, y_stride);
}

template <class W>
void launch_types(const hy3x_adapters *h, const int32_t *ids, const void *x, bool x32,
                  int64_t x_stride, const void *base, int64_t base_stride, void *y, bool y32,
                  int64_t y_stride, int T, hipStream_t st) {
  if (x32 && y32)
    launch<W, float, float>(h, ids, x, x_stride, base, base_stride, y, y_stride, T, st);
  else if (x32)
    launch<W, float, W>(h, ids, x, x_stride, base, base_stride, y, y_stride, T, st);
  else if (y32)
    launch<W, W, float>(h, ids, x, x_stride, base, base_stride, y, y_stride, T, st);
  else
    launch<W, W, W>(h, ids, x, x_stride, base, base_stride, y, y_stride, T, st);
}

// Rows of a dense matrix into rows of a padded one (the padding is zero since
// the handle was made).
int copy_rows(uint16_t *dst, int dst_row, const void *src, int rows, int row, hipMemcpyKind kind) {
  OP_HIP_TRY(hipMemcpy2D(dst, (size_t)dst_row * 2, src, (size_t)row * 2, (size_t)row * 2, rows,
                         kind));
  return HY3X_OK;
}

// Whether T rows of a_row bytes, a_step apart from a, and T rows of b share a
// byte. Rows of one wider buffer (equal steps) may lie between each other.
bool overlap(const void *a, int64_t a_step, int64_t a_row, const void *b, int64_t b_step,
             int64_t b_row, int T) {
  const uintptr_t a0 = (uintptr_t)a, b0 = (uintptr_t)b;
  const uintptr_t a1 = a0 + (uintptr_t)((T - 1) * a_step + a_row);
  const uintptr_t b1 = b0 + (uintptr_t)((T - 1) * b_step + b_row);
  if (a1 <= b0 || b1 <= a0) return false;
  if (a_step != b_step || T == 1) return true;
  const int64_t off = (int64_t)((b0 >= a0 ? b0 - a0 : a0 - b0) % (uintptr_t)a_step);
  const int64_t ab = b0 >= a0 ? off : (a_step - off) % a_step;  // b's place in a's rows
  return ab < a_row || ab + b_row > a_step;
}

}  // namespace


}  // namespace hy3x

using namespace hy3x;

extern "C" {

int hy3x_adapters_destroy(hy3x_adapters *h) {
  if (!h) return HY3X_OK;
  void *ptrs[] = {h->a, h->b, h->scale};
  for (void *p : ptrs)
    if (p) (void)hipFree(p);
  delete h;
  return HY3X_OK;
}

int hy3x_adapters_create(hy3x_adapters **out, int count, int rank, int d_in, int d_out, int type) {
  if (!out) return op_fail(HY3X_E_ARG, "out is NULL");
  *out = nullptr;
  if (count < 1 || count > HY3X_ADAPTERS_MAX_COUNT)
    return op_fail(HY3X_E_ARG, "count %d outside [1,%d]", count, HY3X_ADAPTERS_MAX_COUNT);
  if (rank < 1 || rank > HY3X_ADAPTERS_MAX_RANK)
    return op_fail(HY3X_E_ARG, "rank %d outside [1,%d]", rank, HY3X_ADAPTERS_MAX_RANK);
  if (d_in < 1 || d_in > HY3X_ADAPTERS_MAX_DIM || d_out < 1 || d_out > HY3X_ADAPTERS_MAX_DIM)
    return op_fail(HY3X_E_ARG, "d_in %d or d_out %d outside [1,%d]", d_in, d_out,
                   HY3X_ADAPTERS_MAX_DIM);
  if (type != HY3X_F16 && type != HY3X_BF16)
    return op_fail(HY3X_E_ARG, "adapter type %d is neither HY3X_F16 nor HY3X_BF16", type);
  hy3x_adapters *h = new (std::nothrow) hy3x_adapters();
  if (!h) return op_fail(HY3X_E_NOMEM, "out of host memory");
  h->count = count;
  h->rank = rank;
  h->d_in = d_in;
  h->d_out = d_out;
  h->type = type;
  h->rp = rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : 128;
  h->kp = (d_in + 31) & ~31;
  h->np = (d_out + 63) & ~63;
  const hipError_t e = hipGetDevice(&h->device);
  if (e != hipSuccess) {
    delete h;
    return op_fail(HY3X_E_HIP, "hipGetDevice failed: %s", hipGetErrorString(e));
  }
  const size_t na = (size_t)count * h->rp * h->kp * 2, nb = (size_t)count * h->rp * h->np * 2;
  if (hipMalloc(&h->a, na) != hipSuccess || hipMalloc(&h->b, nb) != hipSuccess ||
      hipMalloc(&h->scale, (size_t)count * sizeof(float)) != hipSuccess) {
    (void)hipGetLastError();
    hy3x_adapters_destroy(h);
    return op_fail(HY3X_E_NOMEM, "hipMalloc of %d adapters (%zu bytes) failed", count, na + nb);
  }
  if (hipMemset(h->a, 0, na) != hipSuccess || hipMemset(h->b, 0, nb) != hipSuccess ||
      hipMemset(h->scale, 0, (size_t)count * sizeof(float)) != hipSuccess ||
      hipDeviceSynchronize() != hipSuccess) {
    hy3x_adapters_destroy(h);
    return op_fail(HY3X_E_HIP, "clearing the adapters failed");
  }
  *out = h;
  return HY3X_OK;
}

static int check_device(const hy3x_adapters *h) {
  int dev = -1;
  OP_HIP_TRY(hipGetDevice(&dev));
  if (dev != h->device)
    return op_fail(HY3X_E_ARG, "the adapters live on device %d, the current device is %d",
                   h->device, dev);
  return HY3X_OK;
}

int hy3x_adapters_set(hy3x_adapters *h, int index, const void *a, const void *b, float scale,
                      int src_on_device) {
  if (!h || !a || !b) return op_fail(HY3X_E_ARG, "NULL argument");
  if (index < 0 || index >= h->count)
    return op_fail(HY3X_E_ARG, "adapter %d outside [0,%d)", index, h->count);
  int rc = check_device(h);
  if (rc) return rc;
  OP_HIP_TRY(hipDeviceSynchronize());
  const hipMemcpyKind kind = src_on_device ? hipMemcpyDeviceToDevice : hipMemcpyHostToDevice;
  if ((rc = copy_rows(h->a + (size_t)index * h->rp * h->kp, h->kp, a, h->rank, h->d_in, kind)) ||
      (rc = copy_rows(h->b + (size_t)index * h->rp * h->np, h->rp, b, h->d_out, h->rank, kind)))
    return rc;
  OP_HIP_TRY(hipMemcpy(h->scale + index, &scale, sizeof(float), hipMemcpyHostToDevice));
  OP_HIP_TRY(hipDeviceSynchronize());
  return HY3X_OK;
}

int hy3x_adapters_apply(const hy3x_adapters *h, const int32_t *ids, const void *x, int x_type,
                        int64_t x_stride, const void *base, int64_t base_stride, void *y,
                        int y_type, int64_t y_stride, int T, void *stream) {
  if (!h) return op_fail(HY3X_E_ARG, "NULL adapters");
  if ((x_type != HY3X_F32 && x_type != h->type) || (y_type != HY3X_F32 && y_type != h->type))
    return op_fail(HY3X_E_ARG, "x type %d and y type %d: each is HY3X_F32 or the adapters' %d",
                   x_type, y_type, h->type);
  if (T < 0 || T > HY3X_ADAPTERS_MAX_TOKENS)
    return op_fail(HY3X_E_ARG, "T=%d outside [0,%d]", T, HY3X_ADAPTERS_MAX_TOKENS);
  const int64_t most = (int64_t)1 << 32;  // T rows of it stay inside 64-bit byte offsets
  if (x_stride < h->d_in || y_stride < h->d_out || (base && base_stride < h->d_out) ||
      x_stride > most || y_stride > most || (base && base_stride > most))
    return op_fail(HY3X_E_ARG, "a row stride lies below its row's length, or above %lld",
                   (long long)most);
  if (T == 0) return HY3X_OK;
  if (!ids || !x || !y) return op_fail(HY3X_E_ARG, "NULL ids, x or y");
  const int64_t xs = x_type == HY3X_F32 ? 4 : 2, ys = y_type == HY3X_F32 ? 4 : 2;
  if ((uintptr_t)ids % 4 || (uintptr_t)x % xs || (uintptr_t)y % ys || (uintptr_t)base % ys)
    return op_fail(HY3X_E_ARG, "a pointer is not aligned to its elements");
  if (overlap(x, x_stride * xs, h->d_in * xs, y, y_stride * ys, h->d_out * ys, T))
    return op_fail(HY3X_E_ARG, "y overlaps x");
  if (base && !(base == y && (base_stride == y_stride || T == 1)) &&
      overlap(base, base_stride * ys, h->d_out * ys, y, y_stride * ys, h->d_out * ys, T))
    return op_fail(HY3X_E_ARG, "y overlaps base without being base");
  const int rc = check_device(h);
  if (rc) return rc;
  hipStream_t st = (hipStream_t)stream;
  if (h->type == HY3X_F16)
    launch_types<__half>(h, ids, x, x_type == HY3X_F32, x_stride, base, base_stride, y,
                         y_type == HY3X_F32, y_stride, T, st);
  else
    launch_types<__hip_bfloat16>(h, ids, x, x_type == HY3X_F32, x_stride, base, base_stride, y,
                                 y_type == HY3X_F32, y_stride, T, st);
  OP_HIP_TRY(hipGetLastError());
  return HY3X_OK;
}

}  // extern "C"
