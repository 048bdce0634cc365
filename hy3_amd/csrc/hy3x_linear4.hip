// hy3x_linear4.hip -- products of 4-bit weights with a scale, and perhaps a
// zero point, for each group of a row's weights (hy3x_linear4_*):
//
//   W[n][k] = s[n][k / group] (q[n][k] - z[n][k / group])
//   y[t][n] = base[t][n] + sum_k W[n][k] x[t][k]        (fp32 sums, y rounded once)
//
// Products: v_mfma_f32_16x16x32_{bf16,f16}, rows = tokens, columns = 16 rows of
// W. The integers q and -z are exact in both types, so a group's sum
// sum_k x (q - z) is the fp32 accumulator of its MFMAs, and its scale is one FMA.
// fp32 x meets them as three bf16 parts (hi + mid + lo, 24 bits), each a row of
// the MFMA.
//
// Weights as the MFMAs read them:
//   q  [row tile][chunk of 128 k][lane][4 dwords]: dword j of lane l holds k =
//      128 c + 32 j + 8 (l / 16) + i of row 16 rt + l % 16, element i < 4 in the
//      low half of byte i, i >= 4 in the high half of byte i - 4: both halves are
//      bytes q, which v_cvt_scalef32_pk_{bf16,f16}_fp8 turns into the numbers q,
//      as e4m3 bytes below 16 stand for q 2^-9;
//   s  [row tile][quad of chunks][row][4 GP] (GP groups in a chunk), 0 beyond d_in
//      and d_out; z the same, in bytes.
#include <hip/hip_bf16.h>
#include <string.h>

#include <algorithm>
#include <new>

#include "../../include/hy3x_moe.h"
#include "hy3x_common.h"
#include "hy3x_error.h"
#include "hy3x_ops.h"

struct hy3x_linear4 {
  int device = 0, d_out = 0, d_in = 0, group = 0, type = 0;
  int tiles = 0, chunks = 0, quads = 0;  // row tiles of 16, chunks of 128 k, quads of chunks
  bool set = false, zeros = false;
  uint32_t *q = nullptr;
  uint16_t *s = nullptr;
  uint8_t *z = nullptr;
};

namespace hy3x {
namespace {

typedef float f4v __attribute__((ext_vector_type(4)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));
typedef __bf16 bf2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf8v __attribute__((ext_vector_type(8)));
typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));

// The MFMAs' operand type for x: its own two-byte type, bf16 parts of fp32.
template <class X>
struct Op;
template <>
struct Op<__half> {
  static constexpr int PARTS = 1;
  static __device__ __forceinline__ f4v mma(u4v a, u4v b, f4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8v, a),
                                                  __builtin_bit_cast(h8v, b), c, 0, 0, 0);
  }
  template <bool HI>
  static __device__ __forceinline__ uint32_t ints(uint32_t bytes) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(bytes, 512.0f, HI));
  }
  static __device__ __forceinline__ uint32_t both(float v) {  // v in both halves
    return 0x10001u * __builtin_bit_cast(uint16_t, (_Float16)v);
  }
};
template <>
struct Op<__hip_bfloat16> {
  static constexpr int PARTS = 1;
  static __device__ __forceinline__ f4v mma(u4v a, u4v b, f4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, a),
                                                   __builtin_bit_cast(bf8v, b), c, 0, 0, 0);
  }
  template <bool HI>
  static __device__ __forceinline__ uint32_t ints(uint32_t bytes) {
    return __builtin_bit_cast(uint32_t,
                              __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(bytes, 512.0f, HI));
  }
  static __device__ __forceinline__ uint32_t both(float v) {  // exact: at most 8 bits
    return (__float_as_uint(v) >> 16) * 0x10001u;
  }
};
template <>
struct Op<float> : Op<__hip_bfloat16> {
  static constexpr int PARTS = 3;
};

// 8 weights of a lane as an operand.
template <class X>
__device__ __forceinline__ u4v weights(uint32_t w) {
  const uint32_t lo = w & 0x0f0f0f0fu, hi = w >> 4 & 0x0f0f0f0fu;
  return (u4v){Op<X>::template ints<false>(lo), Op<X>::template ints<true>(lo),
               Op<X>::template ints<false>(hi), Op<X>::template ints<true>(hi)};
}

// Part p of v in bf16: v = p0 + p1 + p2. An infinity is its first part, the
// others 0.
__device__ __forceinline__ float trunc16(float v) {
  return __uint_as_float(__float_as_uint(v) & 0xffff0000u);
}
__device__ __forceinline__ uint32_t part_of(float v, int p) {
  const float a = trunc16(v), r = fabsf(v) == INFINITY ? 0.0f : v - a, b = trunc16(r);
  return __float_as_uint(p == 0 ? a : p == 1 ? b : p == 2 ? r - b : 0.0f) >> 16;
}

// Elements k .. k + 7 of a row of n as an operand, zeros beyond it.
template <class X>
__device__ __forceinline__ u4v operand(const X *row, int k, int n, int part) {
  u4v out;
  if constexpr (sizeof(X) == 2) {
    if (k + 8 <= n) {
      __builtin_memcpy(&out, row + k, 16);
    } else {
      uint16_t e[8];
#pragma unroll
      for (int j = 0; j < 8; j++) {
        __builtin_memcpy(&e[j], row + min(k + j, n - 1), 2);
        if (k + j >= n) e[j] = 0;
      }
#pragma unroll
      for (int j = 0; j < 4; j++) out[j] = e[2 * j] | (uint32_t)e[2 * j + 1] << 16;
    }
  } else {
    float e[8];
    if (k + 8 <= n) {
      __builtin_memcpy(e, row + k, 32);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) {
        e[j] = row[min(k + j, n - 1)];
        if (k + j >= n) e[j] = 0.0f;
      }
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
      out[j] = part_of(e[2 * j], part) | part_of(e[2 * j + 1], part) << 16;
  }
  return out;
}

struct Call {
  const u4v *q;
  const uint16_t *s;
  const uint8_t *z;  // NULL: 8 everywhere
  int d_out, d_in, tiles, chunks, quads;
  bool s16;  // scales are fp16
  const void *x, *base;
  void *y;
  int64_t x_stride, base_stride, y_stride;
  int T, y_type;
};

__device__ __forceinline__ float scale_of(uint32_t bits, bool s16) {
  return s16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)bits) : __uint_as_float(bits << 16);
}

__device__ __forceinline__ float load_y(const void *p, int64_t at, int type) {
  if (type == HY3X_F32) return ((const float *)p)[at];
  if (type == HY3X_F16) return __half2float(((const __half *)p)[at]);
  return __bfloat162float(((const __hip_bfloat16 *)p)[at]);
}
__device__ __forceinline__ void store_y(void *p, int64_t at, int type, float v) {
  if (type == HY3X_F32) ((float *)p)[at] = v;
  else if (type == HY3X_F16) ((__half *)p)[at] = __float2half(v);
  else ((__hip_bfloat16 *)p)[at] = __float2bfloat16(v);
}

constexpr int WAVES = 4;

// One row tile and one token tile at a time; the waves split the quads.
template <class X, int GP>
__global__ __launch_bounds__(64 * WAVES) void k_linear4(Call c) {
  constexpr int TT = Op<X>::PARTS == 1 ? 16 : 4;  // tokens of a tile
  __shared__ float red[WAVES][4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, h = lane >> 4;
  const int token_tiles = (c.T + TT - 1) / TT;
  const int64_t all = (int64_t)token_tiles * c.tiles;
  for (int64_t item = blockIdx.x; item < all; item += gridDim.x) {
    const int rt = (int)(item % c.tiles);
    const int64_t t0 = item / c.tiles * TT;
    const int part = TT == 4 ? col & 3 : 0;
    const int64_t t = min(t0 + (TT == 4 ? col >> 2 : col), (int64_t)c.T - 1);
    const X *row = (const X *)c.x + t * c.x_stride;
    f4v acc = {0, 0, 0, 0};
    for (int qd = wave; qd < c.quads; qd += WAVES) {
      const size_t at = (((size_t)rt * c.quads + qd) * 16 + col) * (4 * GP);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int ch = 4 * qd + i;
        if (ch >= c.chunks) break;
        const u4v w = c.q[((size_t)rt * c.chunks + ch) * 64 + lane];
#pragma unroll
        for (int g = 0; g < GP; g++) {
          const float s = scale_of(c.s[at + i * GP + g], c.s16);
          const uint32_t zz = Op<X>::both(c.z ? -(float)c.z[at + i * GP + g] : -8.0f);
          const u4v z = {zz, zz, zz, zz};
          f4v d = {0, 0, 0, 0};
#pragma unroll
          for (int j = g * 4 / GP; j < (g + 1) * 4 / GP; j++) {
            const u4v a = operand(row, 128 * ch + 32 * j + 8 * h, c.d_in, part);
            d = Op<X>::mma(a, weights<X>(w[j]), d);
            d = Op<X>::mma(a, z, d);
          }
#pragma unroll
          for (int r = 0; r < 4; r++) acc[r] = fmaf(s, d[r], acc[r]);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < 4; r++) red[wave][r][lane] = acc[r];
    __syncthreads();
    // thread: register r of a lane
    const int r = wave;
    float v = 0.0f;
    if (TT == 16) {
      for (int w = 0; w < WAVES; w++) v += red[w][r][lane];
    } else if (r == 0) {
      for (int w = 0; w < WAVES; w++) v += red[w][0][lane] + (red[w][1][lane] + red[w][2][lane]);
    }
    const int64_t token = t0 + (TT == 16 ? 4 * h + r : h);
    const int n = 16 * rt + col;
    if ((TT == 16 || r == 0) && token < c.T && n < c.d_out) {
      if (c.base) v += load_y(c.base, token * c.base_stride + n, c.y_type);
      store_y(c.y, token * c.y_stride + n, c.y_type, v);
    }
    __syncthreads();
  }
}

// q [d_out x ceil(d_in / 2)] bytes (element k in byte k / 2, even k low), scales and
// zeros [d_out x groups] to the kernels' layout.
__global__ __launch_bounds__(256) void k_pack_q(const uint8_t *q, int d_out, int d_in, int chunks,
                                                int64_t n, uint32_t *out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;  // a dword
  if (i >= n) return;
  const int j = (int)(i & 3), lane = (int)(i >> 2 & 63);
  const int64_t tile = i >> 8;
  const int64_t row = tile / chunks * 16 + (lane & 15);
  const int k0 = (int)(tile % chunks) * 128 + 32 * j + 8 * (lane >> 4);
  uint32_t w = 0;
  if (row < d_out)
    for (int e = 0; e < 8; e++) {
      const int k = k0 + e;
      if (k >= d_in) break;
      const uint32_t v = q[row * ((d_in + 1) / 2) + k / 2] >> (4 * (k & 1)) & 15;
      w |= v << (8 * (e & 3) + 4 * (e >> 2));
    }
  out[i] = w;
}
__global__ __launch_bounds__(256) void k_pack_s(const uint16_t *s, const uint8_t *z, int d_out,
                                                int groups, int quads, int gp, int64_t n,
                                                uint16_t *so, uint8_t *zo) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;  // a group
  if (i >= n) return;
  const int64_t tile = i / (64 * gp);
  const int64_t row = tile / quads * 16 + i / (4 * gp) % 16;
  const int64_t g = tile % quads * (4 * gp) + i % (4 * gp);
  const bool in = row < d_out && g < groups;
  so[i] = in ? s[row * groups + g] : 0;
  if (z) zo[i] = in ? z[row * groups + g] : 0;
}
__global__ __launch_bounds__(256) void k_check_zeros(const uint8_t *z, int64_t n, int *bad) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    if (z[i] > 16) *bad = 1;
}

template <class X>
void launch(const Call &c, int group, hipStream_t st) {
  constexpr int TT = Op<X>::PARTS == 1 ? 16 : 4;
  const int64_t all = (int64_t)((c.T + TT - 1) / TT) * c.tiles;
  const dim3 grid((uint32_t)std::min<int64_t>(all, 1 << 20)), block(64 * WAVES);
  if (group == 128) k_linear4<X, 1><<<grid, block, 0, st>>>(c);
  else if (group == 64) k_linear4<X, 2><<<grid, block, 0, st>>>(c);
  else k_linear4<X, 4><<<grid, block, 0, st>>>(c);
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
  if (d_in < 1 || d_in > HY3X_LINEAR4_MAX_IN)
    return op_fail(HY3X_E_ARG, "d_in %d outside [1,%d]", d_in, HY3X_LINEAR4_MAX_IN);
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
  h->tiles = (d_out + 15) / 16;
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
  k_pack_q<<<(uint32_t)((dwords + 255) / 256), 256>>>((const uint8_t *)q, h->d_out, h->d_in,
                                                       h->chunks, dwords, h->q);
  OP_HIP_TRY(hipGetLastError());
  k_pack_s<<<(uint32_t)((spots + 255) / 256), 256>>>((const uint16_t *)scales,
                                                      (const uint8_t *)zeros, h->d_out, groups,
                                                      h->quads, gp, spots, h->s, h->z);
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
  Call c;
  c.q = (const u4v *)h->q;
  c.s = h->s;
  c.z = h->zeros ? h->z : nullptr;
  c.d_out = h->d_out;
  c.d_in = h->d_in;
  c.tiles = h->tiles;
  c.chunks = h->chunks;
  c.quads = h->quads;
  c.s16 = h->type == HY3X_F16;
  c.x = x;
  c.base = base;
  c.y = y;
  c.x_stride = x_stride;
  c.base_stride = base_stride;
  c.y_stride = y_stride;
  c.T = T;
  c.y_type = y_type;
  const hipStream_t st = (hipStream_t)stream;
  if (x_type == HY3X_F32) launch<float>(c, h->group, st);
  else if (x_type == HY3X_F16) launch<__half>(c, h->group, st);
  else launch<__hip_bfloat16>(c, h->group, st);
  OP_HIP_TRY(hipGetLastError());
  return HY3X_OK;
}

}  // extern "C"
