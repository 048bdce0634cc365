// hy3x_linear4.hip -- products of 4-bit weights with group scales (hy3x_linear4_*):
// the handle, its weights' layout and the entry points. The kernels are in hy3x_linear4_kernels.h.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>
#include <atomic>
#include <new>

#include "hy3x_error.h"
#include "hy3x_linear4.h"
#include "hy3x_ops.h"

struct hy3x_linear4 {
  int device = 0, d_out = 0, d_in = 0, group = 0, type = 0;
  int tiles = 0, chunks = 0, quads = 0;  // row tiles of 16, chunks of 128 k, quads of chunks
  bool set = false, zeros = false;
  mutable std::atomic<bool> kept{false};  // a captured call knows of no zero points
  uint32_t *q = nullptr;
  uint16_t *s = nullptr;
  uint8_t *z = nullptr;
};

namespace hy3x {
namespace {

// q [d_out x ceil(d_in / 2)] bytes (element k in byte k / 2, even k low), scales and
// zeros [d_out x groups] to the kernels' layout.
__global__ __launch_bounds__(256) void k_pack_q(const uint8_t *q, int d_out, int d_in, int chunks,
                                                int64_t n, uint32_t *out) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n;  // a dword
       i += (int64_t)gridDim.x * 256) {
    const int j = (int)(i & 3), lane = (int)(i >> 2 & 63);
    const int64_t tile = i >> 8;
    const int64_t row = linear4_row(tile / chunks, lane & 15);
    const int k0 = (int)(tile % chunks) * 128 + 32 * j + 8 * (lane >> 4);
    uint32_t w = 0;
    if (row < d_out)
      for (int e = 0; e < 8; e++) {
        const int k = k0 + e;
        if (k >= d_in) break;
        w |= linear4_code(q[row * ((d_in + 1) / 2) + k / 2] >> (4 * (k & 1)) & 15, e);
      }
    out[i] = w;
  }
}
__global__ __launch_bounds__(256) void k_pack_s(const uint16_t *s, const uint8_t *z, int d_out,
                                                int groups, int quads, int gp, int64_t n,
                                                uint16_t *so, uint8_t *zo) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n;  // a group
       i += (int64_t)gridDim.x * 256) {
    const int64_t tile = i / (64 * gp);
    const int64_t row = linear4_row(tile / quads, (int)(i / (4 * gp) % 16));
    const int64_t g = tile % quads * (4 * gp) + i % (4 * gp);
    const bool in = row < d_out && g < groups;
    so[i] = in ? s[row * groups + g] : 0;
    zo[i] = 2 * (!z ? 8 : in ? z[row * groups + g] : 0) - 15;
  }
}
__global__ __launch_bounds__(256) void k_check_zeros(const uint8_t *z, int64_t n, int *bad) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    if (z[i] > 16) *bad = 1;
}

}  // namespace
}  // namespace hy3x

using namespace hy3x;

extern "C" {

int hy3x_linear4_destroy(hy3x_linear4 *h) {
  if (!h) return HY3X_OK;
  void *ptrs[] = {h->q, h->s, h->z};
  for (void *p : ptrs)
    if (p) (void)hipFree(p);
  delete h;
  return HY3X_OK;
}

int hy3x_linear4_create(hy3x_linear4 **out, int d_out, int d_in, int group, int type) {
  if (!out) return op_fail(HY3X_E_ARG, "out is NULL");
  *out = nullptr;
  if (d_out < 1 || d_out > HY3X_LINEAR4_MAX_OUT)
    return op_fail(HY3X_E_ARG, "d_out %d outside [1,%d]", d_out, HY3X_LINEAR4_MAX_OUT);
  if (d_in < HY3X_LINEAR4_MIN_IN || d_in > HY3X_LINEAR4_MAX_IN)
    return op_fail(HY3X_E_ARG, "d_in %d outside [%d,%d]", d_in, HY3X_LINEAR4_MIN_IN,
                   HY3X_LINEAR4_MAX_IN);
  if (group != 32 && group != 64 && group != 128)
    return op_fail(HY3X_E_ARG, "group %d is none of 32, 64, 128", group);
  if (type != HY3X_F16 && type != HY3X_BF16)
    return op_fail(HY3X_E_ARG, "scale type %d is neither HY3X_F16 nor HY3X_BF16", type);
  hy3x_linear4 *h = new (std::nothrow) hy3x_linear4();
  if (!h) return op_fail(HY3X_E_NOMEM, "out of host memory");
  h->d_out = d_out;
  h->d_in = d_in;
  h->group = group;
  h->type = type;
  h->tiles = (d_out + 63) / 64 * 4;
  h->chunks = (d_in + 127) / 128;
  h->quads = (h->chunks + 3) / 4;
  const hipError_t e = hipGetDevice(&h->device);
  if (e != hipSuccess) {
    delete h;
    return op_fail(HY3X_E_HIP, "hipGetDevice failed: %s", hipGetErrorString(e));
  }
  const size_t nq = (size_t)h->tiles * h->chunks * 1024;
  const size_t ns = (size_t)h->tiles * h->quads * 64 * (128 / group);
  if (hipMalloc(&h->q, nq) != hipSuccess || hipMalloc(&h->s, 2 * ns) != hipSuccess ||
      hipMalloc(&h->z, ns) != hipSuccess) {
    (void)hipGetLastError();
    hy3x_linear4_destroy(h);
    return op_fail(HY3X_E_NOMEM, "hipMalloc of a %d x %d matrix (%zu bytes) failed", d_out, d_in,
                   nq + 3 * ns);
  }
  *out = h;
  return HY3X_OK;
}

static int check_device(const hy3x_linear4 *h) {
  int dev = -1;
  OP_HIP_TRY(hipGetDevice(&dev));
  if (dev != h->device)
    return op_fail(HY3X_E_ARG, "the weights live on device %d, the current device is %d",
                   h->device, dev);
  return HY3X_OK;
}

int hy3x_linear4_set(hy3x_linear4 *h, const void *q, const void *scales, const void *zeros,
                     int src_on_device) {
  if (!h || !q || !scales) return op_fail(HY3X_E_ARG, "NULL argument");
  if ((uintptr_t)scales % 2) return op_fail(HY3X_E_ARG, "scales is not aligned to its elements");
  if (zeros && h->kept)
    return op_fail(HY3X_E_STATE, "zero points for weights that a captured call has without them");
  const int rc = check_device(h);
  if (rc) return rc;
  OP_HIP_TRY(hipDeviceSynchronize());
  const int groups = (h->d_in + h->group - 1) / h->group;
  const size_t nq = (size_t)h->d_out * ((h->d_in + 1) / 2), ng = (size_t)h->d_out * groups;
  struct Stage {
    uint8_t *p = nullptr;
    ~Stage() {
      if (p) (void)hipFree(p);
    }
  } stage;
  // the flag of a bad zero point, then the scales (2-byte elements), zeros and q
  const size_t held = src_on_device ? 0 : 3 * ng + nq;
  if (hipMalloc(&stage.p, 16 + held) != hipSuccess) {
    (void)hipGetLastError();
    return op_fail(HY3X_E_NOMEM, "hipMalloc of the weights' staging buffer failed");
  }
  if (!src_on_device) {
    uint8_t *p = stage.p + 16;
    OP_HIP_TRY(hipMemcpy(p, scales, 2 * ng, hipMemcpyHostToDevice));
    if (zeros) OP_HIP_TRY(hipMemcpy(p + 2 * ng, zeros, ng, hipMemcpyHostToDevice));
    OP_HIP_TRY(hipMemcpy(p + 3 * ng, q, nq, hipMemcpyHostToDevice));
    scales = p;
    if (zeros) zeros = p + 2 * ng;
    q = p + 3 * ng;
  }
  if (zeros) {
    int bad = 0;
    OP_HIP_TRY(hipMemset(stage.p, 0, sizeof(int)));
    k_check_zeros<<<(uint32_t)std::min<size_t>((ng + 255) / 256, 2048), 256>>>(
        (const uint8_t *)zeros, (int64_t)ng, (int *)stage.p);
    OP_HIP_TRY(hipGetLastError());
    OP_HIP_TRY(hipMemcpy(&bad, stage.p, sizeof(int), hipMemcpyDeviceToHost));
    if (bad) return op_fail(HY3X_E_ARG, "a zero point is above 16");
  }
  const int gp = 128 / h->group;
  const int64_t dwords = (int64_t)h->tiles * h->chunks * 256;
  const int64_t spots = (int64_t)h->tiles * h->quads * 64 * gp;
  const auto blocks = [](int64_t n) {
    return (uint32_t)std::min<int64_t>((n + 255) / 256, 1 << 20);
  };
  k_pack_q<<<blocks(dwords), 256>>>((const uint8_t *)q, h->d_out, h->d_in, h->chunks, dwords,
                                    h->q);
  OP_HIP_TRY(hipGetLastError());
  k_pack_s<<<blocks(spots), 256>>>((const uint16_t *)scales, (const uint8_t *)zeros, h->d_out,
                                   groups, h->quads, gp, spots, h->s, h->z);
  OP_HIP_TRY(hipGetLastError());
  OP_HIP_TRY(hipDeviceSynchronize());
  h->zeros = zeros != nullptr;
  h->set = true;
  return HY3X_OK;
}

int hy3x_linear4_apply(const hy3x_linear4 *h, const void *x, int x_type, int64_t x_stride,
                       const void *base, int64_t base_stride, void *y, int y_type,
                       int64_t y_stride, int T, void *stream) {
  if (!h) return op_fail(HY3X_E_ARG, "NULL weights");
  if (!h->set) return op_fail(HY3X_E_STATE, "the weights are not set");
  if (x_type < HY3X_F32 || x_type > HY3X_BF16 || y_type < HY3X_F32 || y_type > HY3X_BF16)
    return op_fail(HY3X_E_ARG, "x type %d or y type %d is none of HY3X_F32, _F16, _BF16", x_type,
                   y_type);
  if (T < 0 || T > HY3X_LINEAR4_MAX_TOKENS)
    return op_fail(HY3X_E_ARG, "T=%d outside [0,%d]", T, HY3X_LINEAR4_MAX_TOKENS);
  const int64_t most = (int64_t)1 << 32;  // T rows of it stay inside 64-bit byte offsets
  if (x_stride < h->d_in || y_stride < h->d_out || (base && base_stride < h->d_out) ||
      x_stride > most || y_stride > most || (base && base_stride > most))
    return op_fail(HY3X_E_ARG, "a row stride lies below its row's length, or above %lld",
                   (long long)most);
  if (T == 0) return HY3X_OK;
  if (!x || !y) return op_fail(HY3X_E_ARG, "NULL x or y");
  const int64_t xs = x_type == HY3X_F32 ? 4 : 2, ys = y_type == HY3X_F32 ? 4 : 2;
  if ((uintptr_t)x % xs || (uintptr_t)y % ys || (uintptr_t)base % ys)
    return op_fail(HY3X_E_ARG, "a pointer is not aligned to its elements");
  if (rows_overlap(x, x_stride * xs, h->d_in * xs, y, y_stride * ys, h->d_out * ys, T))
    return op_fail(HY3X_E_ARG, "y overlaps x");
  if (base && !(base == y && (base_stride == y_stride || T == 1)) &&
      rows_overlap(base, base_stride * ys, h->d_out * ys, y, y_stride * ys, h->d_out * ys, T))
    return op_fail(HY3X_E_ARG, "y overlaps base without being base");
  const int rc = check_device(h);
  if (rc) return rc;
  Linear4Call c;
  c.q = (const u4v *)h->q;
  c.s = h->s;
  c.z = h->z;
  c.z_quad = h->zeros ? 64 * (128 / h->group) : 0;
  c.z_tile = c.z_quad * h->quads;
  c.d_out = h->d_out;
  c.d_in = h->d_in;
  c.tiles = h->tiles;
  c.chunks = h->chunks;
  c.quads = h->quads;
  c.group = h->group;
  c.s16 = h->type == HY3X_F16;
  c.x_stride = x_stride;
  c.base_stride = base_stride;
  c.y_stride = y_stride;
  c.y_type = y_type;
  const hipStream_t st = (hipStream_t)stream;
  if (!h->zeros && st && !h->kept) {  // its replays will read one quad's zero points for all
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    OP_HIP_TRY(hipStreamIsCapturing(st, &status));
    if (status == hipStreamCaptureStatusActive) h->kept = true;
  }
  // A launch has less than 2^32 threads; the smallest tiles of that many outputs, 32 tokens
  // and 8 row tiles, have 256.
  const int most_tokens = 32 * (((1 << 24) - 1) / ((h->tiles + 7) / 8));
  for (int t = 0; t < T; t += c.T) {
    c.x = (const uint8_t *)x + t * x_stride * xs;
    c.base = base ? (const uint8_t *)base + t * base_stride * ys : nullptr;
    c.y = (uint8_t *)y + t * y_stride * ys;
    c.T = std::min(T - t, most_tokens);
    if (x_type == HY3X_F32) launch_linear4<float>(c, st);
    else if (x_type == HY3X_F16) launch_linear4<__half>(c, st);
    else launch_linear4<__hip_bfloat16>(c, st);
    OP_HIP_TRY(hipGetLastError());
  }
  return HY3X_OK;
}

}  // extern "C"
