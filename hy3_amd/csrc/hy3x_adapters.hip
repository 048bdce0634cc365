// hy3x_adapters.hip -- low-rank adapters of many requests at once beside a
// shared projection (hy3x_adapters_*):
//
//   u = A_a x_t                      (fp32 sums over d_in)
//   y_t = base_t + scale_a (B_a u)   (fp32 sums over the rank, y rounded once)
//
// One launch: a block takes TOK tokens and a slice of their outputs, and forms
// u for itself, so nothing passes between blocks: no scratch memory, no second
// launch, no order of blocks in the results. Its waves split d_in, join their
// parts of u in LDS, then split the outputs.
//
// TOK = 16: 16 consecutive tokens, the columns of every MFMA. The adapters that
// occur among them are taken one after another: each forms its products for all
// 16 columns, and the columns of its own tokens are selected, so a token never
// meets another adapter's values (not even their infinities). TOK = 1: one
// token in every column.
//
// Products. u: v_mfma_f32_16x16x32_{f16,bf16} (rows = 16 ranks, columns =
// tokens) where x has the weights' type, v_mfma_f32_16x16x4_f32 where x is
// fp32. B u: v_mfma_f32_16x16x4_f32, as u has fp32's range and precision.
//
// Weights as the MFMAs read them, one coalesced 16-byte load per lane:
//   A  [count][kp / 32][rank tile][lane][8]: rank 16 rt + lane % 16, k = 32 kt
//      + 8 (lane / 16) + j, zero beyond rank and d_in;
//   B  [count][np / 64][chunk][lane][8]: element f = 8 chunk + j of the lane's
//      rp (f = q rp / 4 + s): output 64 cb + 16 (m / 4) + 4 q + m % 4 with m =
//      lane % 16, rank (lane / 16) rp / 4 + s, zero beyond rank and d_out. With
//      this order of outputs over four MFMAs (q) a lane ends with 16
//      consecutive outputs of one token.
#include <hip/hip_bf16.h>
#include <string.h>

#include <algorithm>
#include <new>

#include "../../include/hy3x_moe.h"
#include "hy3x_common.h"
#include "hy3x_error.h"

struct hy3x_adapters {
  int device = 0, count = 0, rank = 0, d_in = 0, d_out = 0, type = 0;
  int rp = 0, kp = 0, np = 0;  // rank, d_in and d_out padded to whole tiles
  uint16_t *a = nullptr, *b = nullptr;
  float *scale = nullptr;  // [count]
};

namespace hy3x {
namespace {

typedef float f4v __attribute__((ext_vector_type(4)));
typedef __bf16 bf8v __attribute__((ext_vector_type(8)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));

constexpr int WAVES = 8;
constexpr int SINGLE_MAX_T = 256;   // up to this many tokens a block takes one token
constexpr int TARGET_BLOCKS = 512;  // blocks that the slices are made for

__device__ __forceinline__ float elem(float v) { return v; }
__device__ __forceinline__ float elem(__half v) { return __half2float(v); }
__device__ __forceinline__ float elem(__hip_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float *p, float v) { *p = v; }
__device__ __forceinline__ void put(__half *p, float v) { *p = __float2half(v); }
__device__ __forceinline__ void put(__hip_bfloat16 *p, float v) { *p = __float2bfloat16(v); }

// Eight elements as loaded, and element j of them in fp32.
template <class T>
struct Eight {
  uint4 v;
  __device__ float at(int j) const {
    const uint32_t w = j < 4 ? (j < 2 ? v.x : v.y) : (j < 6 ? v.z : v.w);
    const uint16_t h = (uint16_t)(w >> (16 * (j & 1)));
    return elem(__builtin_bit_cast(T, h));
  }
};
template <>
struct Eight<float> {
  float4 lo, hi;
  __device__ float at(int j) const {
    const float4 f = j < 4 ? lo : hi;
    return (j & 3) == 0 ? f.x : (j & 3) == 1 ? f.y : (j & 3) == 2 ? f.z : f.w;
  }
};

// Elements k .. k + 7 of a row of n, zeros beyond its end. vec: n % 8 == 0 and
// the row is 16-byte aligned.
template <class T>
__device__ __forceinline__ Eight<T> load8(const T *row, int k, int n, bool vec) {
  Eight<T> r;
  T e[8];
  if (vec && k < n) {
    __builtin_memcpy(&r, __builtin_assume_aligned(row + k, 16), sizeof(r));
    return r;
  }
#pragma unroll
  for (int j = 0; j < 8; j++) {
    e[j] = T(0.0f);
    if (!vec && k + j < n) e[j] = row[k + j];
  }
  __builtin_memcpy(&r, e, sizeof(r));
  return r;
}

__device__ __forceinline__ f4v mma(const Eight<__half> &a, const Eight<__half> &b, f4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8v, a.v),
                                                __builtin_bit_cast(h8v, b.v), c, 0, 0, 0);
}
__device__ __forceinline__ f4v mma(const Eight<__hip_bfloat16> &a, const Eight<__hip_bfloat16> &b,
                                   f4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, a.v),
                                                 __builtin_bit_cast(bf8v, b.v), c, 0, 0, 0);
}
template <class W>
__device__ __forceinline__ f4v mma(const Eight<W> &a, const Eight<float> &b, f4v c) {
#pragma unroll
  for (int j = 0; j < 8; j++)
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.at(j), b.at(j), c, 0, 0, 0);
  return c;
}

template <class X, class Y>
struct Call {
  const uint16_t *a, *b;
  const float *scale;
  int count, kt, nb, d_in, d_out;  // kt = kp / 32, nb = np / 64
  const int32_t *ids;
  const X *x;
  const Y *base;
  Y *y;
  int64_t x_stride, base_stride, y_stride;
  int T, per;   // per: 64-output blocks of a slice
  bool vx, vy;  // rows of x / of base and y in whole aligned 16-byte pieces
};

template <class W, class X, class Y, int RT, int TOK>
__global__ __launch_bounds__(64 * WAVES) void k_adapters(const Call<X, Y> c) {
  constexpr int RP = 16 * RT, PITCH = RP + 4;  // floats per token in LDS
  __shared__ __align__(16) float part[WAVES][TOK][PITCH];
  __shared__ __align__(16) float u[TOK][PITCH];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, g = lane >> 4;
  const int64_t tok = (int64_t)blockIdx.x * TOK + (TOK == 1 ? 0 : col);
  const bool in = tok < c.T;
  int id = in ? c.ids[tok] : -1;
  if (id >= c.count) id = -1;
  const X *xr = c.x + (in ? tok : 0) * c.x_stride;

  // u of every token with an adapter, one adapter after another
  for (uint64_t todo = __ballot(id >= 0 && g == 0); todo;) {
    const int a = __builtin_amdgcn_readlane(id, __ffsll((long long)todo) - 1);
    todo &= ~__ballot(id == a);
    f4v acc[RT];
#pragma unroll
    for (int r = 0; r < RT; r++) acc[r] = f4v{0.f, 0.f, 0.f, 0.f};
    const uint16_t *aw = c.a + ((int64_t)a * c.kt * RT * 64 + lane) * 8;
    auto load_a = [&](int kt, int r) {
      Eight<W> v;
      v.v = *reinterpret_cast<const uint4 *>(aw + ((int64_t)kt * RT + r) * 512);
      return v;
    };
    // pairs of 32: 128 bytes of a two-byte x row at a time, U of them in flight
    constexpr int U = RT >= 4 ? 2 : 4;
    int k0 = 2 * wave;
    for (; k0 + 2 * WAVES * (U / 2 - 1) + 1 < c.kt; k0 += WAVES * U) {
      Eight<X> xv[U];
      Eight<W> av[U][RT];
#pragma unroll
      for (int i = 0; i < U; i++) {
        const int kt = k0 + 2 * WAVES * (i / 2) + (i & 1);
        xv[i] = load8(xr, 32 * kt + 8 * g, c.d_in, c.vx);
#pragma unroll
        for (int r = 0; r < RT; r++) av[i][r] = load_a(kt, r);
      }
#pragma unroll
      for (int i = 0; i < U; i++)
#pragma unroll
        for (int r = 0; r < RT; r++) acc[r] = mma(av[i][r], xv[i], acc[r]);
    }
    for (; k0 < c.kt; k0 += 2 * WAVES)
      for (int kt = k0; kt < min(k0 + 2, c.kt); kt++) {
        const Eight<X> xv = load8(xr, 32 * kt + 8 * g, c.d_in, c.vx);
#pragma unroll
        for (int r = 0; r < RT; r++) acc[r] = mma(load_a(kt, r), xv, acc[r]);
      }
    if (TOK == 16 || col == 0)
#pragma unroll
      for (int r = 0; r < RT; r++)
        *reinterpret_cast<f4v *>(&part[wave][TOK == 1 ? 0 : col][16 * r + 4 * g]) = acc[r];
    __syncthreads();
    for (int i = tid; i < TOK * RP; i += 64 * WAVES) {
      const int t = i / RP, r = i % RP;
      if (TOK == 1 || __shfl(id, t, 64) == a) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) sum += part[w][t][r];
        u[t][r] = sum;
      }
    }
    __syncthreads();
  }

  float ur[4 * RT];  // u of this lane's token, ranks 4 RT g ..
  if (id >= 0)
#pragma unroll
    for (int r = 0; r < RT; r++)
      *reinterpret_cast<f4v *>(&ur[4 * r]) =
          *reinterpret_cast<const f4v *>(&u[TOK == 1 ? 0 : col][4 * RT * g + 4 * r]);
  else
#pragma unroll
    for (int r = 0; r < 4 * RT; r++) ur[r] = 0.0f;

  const int last = min(c.nb, (int)(blockIdx.y + 1) * c.per);
  for (int cb = blockIdx.y * c.per + wave; cb < last; cb += WAVES) {
    float out[16];
#pragma unroll
    for (int i = 0; i < 16; i++) out[i] = 0.0f;
    for (uint64_t todo = __ballot(id >= 0 && g == 0); todo;) {
      const int a = __builtin_amdgcn_readlane(id, __ffsll((long long)todo) - 1);
      todo &= ~__ballot(id == a);
      const uint16_t *bw = c.b + (((int64_t)a * c.nb + cb) * 2 * RT * 64 + lane) * 8;
      Eight<W> bv[2 * RT];
#pragma unroll
      for (int j = 0; j < 2 * RT; j++) bv[j].v = *reinterpret_cast<const uint4 *>(bw + j * 512);
      const float sc = c.scale[a];
#pragma unroll
      for (int q = 0; q < 4; q++) {
        f4v acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < 4 * RT; s++) {
          const int f = q * 4 * RT + s;
          acc = __builtin_amdgcn_mfma_f32_16x16x4f32(bv[f / 8].at(f % 8), ur[s], acc, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) out[4 * q + i] = id == a ? sc * acc[i] : out[4 * q + i];
      }
    }
    if (!in || (TOK == 1 && col)) continue;
    const int c0 = 64 * cb + 16 * g;
    const Y *br = c.base ? c.base + tok * c.base_stride : nullptr;
    Y *yr = c.y + tok * c.y_stride;
    constexpr int P = 16 / sizeof(Y);  // elements per 16-byte piece
    if (c.vy) {
#pragma unroll
      for (int p = 0; p < 16; p += P)
        if (c0 + p < c.d_out) {
          __align__(16) Y v[P];
          if (br) __builtin_memcpy(v, __builtin_assume_aligned(br + c0 + p, 16), 16);
#pragma unroll
          for (int i = 0; i < P; i++) put(&v[i], (br ? elem(v[i]) : 0.0f) + out[p + i]);
          __builtin_memcpy(__builtin_assume_aligned(yr + c0 + p, 16), v, 16);
        }
    } else {
#pragma unroll
      for (int i = 0; i < 16; i++)
        if (c0 + i < c.d_out) put(yr + c0 + i, (br ? elem(br[c0 + i]) : 0.0f) + out[i]);
    }
  }
}

// A and B of one adapter into the layouts above, a thread per 16 bytes.
__global__ __launch_bounds__(256) void k_pack_adapter(const uint16_t *__restrict__ a,
                                                      const uint16_t *__restrict__ b, int rank,
                                                      int d_in, int d_out, int rp, int kt, int nb,
                                                      uint16_t *__restrict__ pa,
                                                      uint16_t *__restrict__ pb) {
  const int rt = rp / 16, na = kt * rt * 64, nbl = nb * 2 * rt * 64;
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= na + nbl) return;
  uint16_t v[8];
  if (i < na) {
    const int lane = i & 63, r = 16 * ((i >> 6) % rt) + lane % 16;
    const int k = 32 * ((i >> 6) / rt) + 8 * (lane / 16);
#pragma unroll
    for (int j = 0; j < 8; j++)
      v[j] = r < rank && k + j < d_in ? a[(int64_t)r * d_in + k + j] : (uint16_t)0;
    __builtin_memcpy(pa + (int64_t)i * 8, v, 16);
  } else {
    const int o = i - na, lane = o & 63, chunk = (o >> 6) % (2 * rt), cb = (o >> 6) / (2 * rt);
    const int m = lane % 16, g = lane / 16;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int f = 8 * chunk + j, q = f / (rp / 4), s = f % (rp / 4);
      const int c = 64 * cb + 16 * (m / 4) + 4 * q + m % 4, r = g * (rp / 4) + s;
      v[j] = r < rank && c < d_out ? b[(int64_t)c * rank + r] : (uint16_t)0;
    }
    __builtin_memcpy(pb + (int64_t)o * 8, v, 16);
  }
}

template <class W, class X, class Y>
void launch(const hy3x_adapters *h, const int32_t *ids, const void *x, int64_t x_stride,
            const void *base, int64_t base_stride, void *y, int64_t y_stride, int T,
            hipStream_t st) {
  Call<X, Y> c;
  c.a = h->a;
  c.b = h->b;
  c.scale = h->scale;
  c.count = h->count;
  c.kt = h->kp / 32;
  c.nb = h->np / 64;
  c.d_in = h->d_in;
  c.d_out = h->d_out;
  c.ids = ids;
  c.x = (const X *)x;
  c.base = (const Y *)base;
  c.y = (Y *)y;
  c.x_stride = x_stride;
  c.base_stride = base_stride;
  c.y_stride = y_stride;
  c.T = T;
  c.vx = (uintptr_t)x % 16 == 0 && h->d_in % 8 == 0 &&
         (T == 1 || x_stride * (int64_t)sizeof(X) % 16 == 0);
  c.vy = (uintptr_t)y % 16 == 0 && (uintptr_t)base % 16 == 0 &&
         h->d_out % (16 / (int)sizeof(Y)) == 0 &&
         (T == 1 || (y_stride * (int64_t)sizeof(Y) % 16 == 0 &&
                     (!base || base_stride * (int64_t)sizeof(Y) % 16 == 0)));
  const bool single = T <= SINGLE_MAX_T;
  const int tiles = single ? T : (T + 15) / 16;
  const int slices = std::max(1, std::min(c.nb, TARGET_BLOCKS / tiles));
  c.per = (c.nb + slices - 1) / slices;
  const dim3 grid(tiles, (c.nb + c.per - 1) / c.per), block(64 * WAVES);
#define HY3X_ADAPTERS(RT)                                    \
  if (h->rp == 16 * RT) {                                    \
    if (single)                                              \
      k_adapters<W, X, Y, RT, 1><<<grid, block, 0, st>>>(c); \
    else                                                     \
      k_adapters<W, X, Y, RT, 16><<<grid, block, 0, st>>>(c); \
    return;                                                  \
  }
  HY3X_ADAPTERS(1)
  HY3X_ADAPTERS(2)
  HY3X_ADAPTERS(4)
  HY3X_ADAPTERS(8)
#undef HY3X_ADAPTERS
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
  if ((uintptr_t)a % 2 || (uintptr_t)b % 2)
    return op_fail(HY3X_E_ARG, "a pointer is not aligned to its elements");
  const int rc = check_device(h);
  if (rc) return rc;
  OP_HIP_TRY(hipDeviceSynchronize());
  const size_t na = (size_t)h->rank * h->d_in * 2, nb = (size_t)h->rank * h->d_out * 2;
  struct Stage {
    uint8_t *p = nullptr;
    ~Stage() {
      if (p) (void)hipFree(p);
    }
  } stage;
  if (!src_on_device) {
    if (hipMalloc(&stage.p, na + nb) != hipSuccess) {
      (void)hipGetLastError();
      return op_fail(HY3X_E_NOMEM, "hipMalloc of the adapter's staging buffer failed");
    }
    OP_HIP_TRY(hipMemcpy(stage.p, a, na, hipMemcpyHostToDevice));
    OP_HIP_TRY(hipMemcpy(stage.p + na, b, nb, hipMemcpyHostToDevice));
    a = stage.p;
    b = stage.p + na;
  }
  const int kt = h->kp / 32, ob = h->np / 64;
  const int n = (kt + 2 * ob) * (h->rp / 16) * 64;
  k_pack_adapter<<<(n + 255) / 256, 256>>>(
      (const uint16_t *)a, (const uint16_t *)b, h->rank, h->d_in, h->d_out, h->rp, kt, ob,
      h->a + (size_t)index * h->rp * h->kp, h->b + (size_t)index * h->rp * h->np);
  OP_HIP_TRY(hipGetLastError());
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
