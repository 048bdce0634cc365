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
#include "hy3x_ops.h"

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
typedef _Float16 h4v __attribute__((ext_vector_type(4)));
typedef short s4v __attribute__((ext_vector_type(4)));

// Waves of a block, and blocks that the slices are made for.
#ifndef NW1
#define NW1 16
#endif
#ifndef NW16
#define NW16 8
#endif
#ifndef TB
#define TB 256
#endif
#ifndef R4
#define R4 2
#endif
#ifndef SMT
#define SMT 256
#endif
constexpr int waves_for(int TOK, int RT) { return TOK == 1 && RT <= 2 ? NW1 : NW16; }
constexpr int SINGLE_MAX_T = SMT;   // up to this many tokens a block takes one token
constexpr int TARGET_BLOCKS = TB;

__device__ __forceinline__ float elem(float v) { return v; }
__device__ __forceinline__ float elem(__half v) { return __half2float(v); }
__device__ __forceinline__ float elem(__hip_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T rounded(float v);
template <>
__device__ __forceinline__ float rounded<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half rounded<__half>(float v) {
  return __float2half(v);
}
template <>
__device__ __forceinline__ __hip_bfloat16 rounded<__hip_bfloat16>(float v) {
  return __float2bfloat16(v);
}

// N elements as loaded, and element j of them in fp32. Loads are 16 bytes at
// the elements' own alignment.
template <class T, int N>
struct Run {
  uint32_t w[N * sizeof(T) / 4];
  __device__ __forceinline__ float at(int j) const {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, w[j]);
    else return elem(__builtin_bit_cast(T, (uint16_t)(w[j / 2] >> (16 * (j & 1)))));
  }
  // in the order of j: an even element clears the odd one behind it
  __device__ __forceinline__ void set(int j, float v) {
    if constexpr (sizeof(T) == 4) w[j] = __builtin_bit_cast(uint32_t, v);
    else {
      const uint32_t h = __builtin_bit_cast(uint16_t, rounded<T>(v));
      w[j / 2] = j & 1 ? w[j / 2] | h << 16 : h;
    }
  }
  __device__ __forceinline__ void load(const T *p) { __builtin_memcpy(w, p, sizeof(w)); }
  __device__ __forceinline__ void store(T *p) const { __builtin_memcpy(p, w, sizeof(w)); }
  // elements c .. of a row of n (n >= 1), zeros beyond it: every load in bounds
  // and none waiting for another
  __device__ __forceinline__ void load_part(const T *row, int c, int n) {
    T e[N];
#pragma unroll
    for (int j = 0; j < N; j++) e[j] = row[min(c + j, n - 1)];
#pragma unroll
    for (int j = 0; j < N; j++) set(j, c + j < n ? elem(e[j]) : 0.0f);
  }
  __device__ __forceinline__ void store_part(T *p, int n) const {
#pragma unroll
    for (int j = 0; j < N; j++)
      if (j < n) {
        if constexpr (sizeof(T) == 4) p[j] = __builtin_bit_cast(T, w[j]);
        else p[j] = __builtin_bit_cast(T, (uint16_t)(w[j / 2] >> (16 * (j & 1))));
      }
  }
};

__device__ __forceinline__ f4v mma(const Run<__half, 8> &a, const Run<__half, 8> &b, f4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8v, a),
                                                __builtin_bit_cast(h8v, b), c, 0, 0, 0);
}
__device__ __forceinline__ f4v mma(const Run<__hip_bfloat16, 8> &a,
                                   const Run<__hip_bfloat16, 8> &b, f4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, a),
                                                 __builtin_bit_cast(bf8v, b), c, 0, 0, 0);
}
__device__ __forceinline__ f4v mma(const Run<__half, 4> &a, const Run<__half, 4> &b, f4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(h4v, a),
                                               __builtin_bit_cast(h4v, b), c, 0, 0, 0);
}
__device__ __forceinline__ f4v mma(const Run<__hip_bfloat16, 4> &a,
                                   const Run<__hip_bfloat16, 4> &b, f4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s4v, a),
                                                   __builtin_bit_cast(s4v, b), c, 0, 0, 0);
}
template <class W>
__device__ __forceinline__ f4v mma(const Run<W, 8> &a, const Run<float, 8> &b, f4v c) {
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
  int T, slices, per;  // per: 64-output blocks of a slice
};

// v in PARTS parts of W's precision, largest first: v = 2^e (p0 + p1 + ..).
// fp16 parts are of v 2^-e with e chosen so that the row's largest |v| lies in
// [2^14, 2^15): the parts keep 11 bits each, down to 2^-24 2^-14 of the
// largest. bf16 has fp32's range, and e = 0. An infinity or NaN is its first
// part, the others 0.
__device__ __forceinline__ float part_of(float v, __half *) {
  return (float)__builtin_amdgcn_cvt_pkrtz(v, 0.0f)[0];
}
__device__ __forceinline__ float part_of(float v, __hip_bfloat16 *) {
  return __uint_as_float(__float_as_uint(v) & 0xffff0000u);
}

// Three parts hold all 24 bits of an fp32 u. Two fp16 parts hold 20 bits of
// each value, an error that an fp16 y's rounding (11 bits) covers also where
// the base cancels most of the product; two bf16 parts would hold 14.
template <class W, class Y>
constexpr int parts_for() {
  return __is_same(W, __half) && sizeof(Y) == 2 ? 2 : 3;
}

constexpr int steps_for(int TOK, int RT, int x_size) {
  return RT == 8 ? 1 : x_size == 2 ? (RT == 1 ? 4 : RT == 2 && TOK == 1 ? 2 : RT == 2 ? 4 : R4) : 2;
}

template <class W, class X, class Y, int RT, int TOK>
__global__ __launch_bounds__(64 * waves_for(TOK, RT)) void k_adapters(const Call<X, Y> c) {
  constexpr int WAVES = waves_for(TOK, RT);
  constexpr int RP = 16 * RT, PITCH = RP + 4;  // floats per token in LDS
  constexpr int PARTS = parts_for<W, Y>();
  // 32-element steps of d_in per group; two groups are in flight
  constexpr int U = steps_for(TOK, RT, sizeof(X));
  __shared__ __align__(16) float part[WAVES][TOK][PITCH];
  __shared__ __align__(16) float u[TOK][PITCH];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, g = lane >> 4;
  // each XCD on a contiguous run of (tokens, slice) items: the slices of one
  // tile share x and A in its L2, neighbouring tiles their adapters
  const uint32_t n = gridDim.x, xcd = blockIdx.x % 8;
  const uint32_t item = xcd * (n / 8) + min(xcd, n % 8) + blockIdx.x / 8;
  const uint32_t tile = item / c.slices, slice = item % c.slices;
  const int64_t tok = (int64_t)tile * TOK + (TOK == 1 ? 0 : col);
  const bool in = tok < c.T;
  const int64_t row = in ? tok : 0;  // columns past the last token read row 0, for nothing
  int id = c.ids[row];

  // step n of this wave: pairs of 32 (128 bytes of a two-byte row) in turn over the waves
  const int full = c.d_in / 32;
  auto step = [&](int n) { return 2 * WAVES * (n >> 1) + 2 * wave + (n & 1); };
  const X *xr = c.x + row * c.x_stride;
  Run<X, 8> xv[U], xn[U];
  auto load_x = [&](Run<X, 8>(&v)[U], int n0) {
#pragma unroll
    for (int i = 0; i < U; i++) v[i].load(xr + 32 * min(step(n0 + i), full - 1) + 8 * g);
  };
  // what does not need the token's adapter is asked for first: x, and the base
  // of the first 64 outputs
  if (full) load_x(xv, 0);
  const int last = min(c.nb, (int)(slice + 1) * c.per), cb0 = slice * c.per + wave;
  const Y *br = c.base ? c.base + row * c.base_stride : nullptr;
  auto load_base = [&](Run<Y, 16> &v, int cb) {
    if (br && 64 * cb + 64 <= c.d_out) v.load(br + 64 * cb + 16 * g);
    else if (br) v.load_part(br, 64 * cb + 16 * g, c.d_out);
    else
#pragma unroll
      for (int i = 0; i < 16; i++) v.set(i, 0.0f);
  };
  Run<Y, 16> bv, bn;
  if (cb0 < last) load_base(bv, cb0);

  if (!in || id >= c.count) id = -1;
  const uint64_t mine = __ballot(id >= 0 && g == 0);  // tokens with an adapter
  auto pick = [&](uint64_t &todo) {  // the next adapter of those tokens
    const int a = __builtin_amdgcn_readlane(id, __ffsll((long long)todo) - 1);
    todo &= ~__ballot(id == a);
    return a;
  };
  uint64_t rest = mine;
  const int a0 = mine ? pick(rest) : 0;
  Run<W, 8> wv[2 * RT], wn[2 * RT];
  auto load_b = [&](Run<W, 8>(&v)[2 * RT], int a, int cb) {
    const W *bw = (const W *)c.b + (((int64_t)a * c.nb + cb) * 2 * RT * 64 + lane) * 8;
#pragma unroll
    for (int j = 0; j < 2 * RT; j++) v[j].load(bw + j * 512);
  };

  // u, rank 16 r + 4 g + i of token col in acc[r][i]: groups of U steps, and in
  // each the adapters of these tokens one after another
  // (DOT: this lane's eight elements of rank 16 r + col, in acc[r][0])
  constexpr bool DOT = TOK == 1 && sizeof(X) == 4;
  f4v acc[RT];
#pragma unroll
  for (int r = 0; r < RT; r++) acc[r] = f4v{0.f, 0.f, 0.f, 0.f};
  auto product = [](const Run<W, 8> &a, const Run<X, 8> &b, f4v v) {
    if constexpr (DOT) {
#pragma unroll
      for (int j = 0; j < 8; j++) v[0] = __builtin_fmaf(a.at(j), b.at(j), v[0]);
      return v;
    } else {
      return mma(a, b, v);
    }
  };
  auto load_a = [&](Run<W, 8>(&v)[RT], int a, int kt) {
    const W *aw = (const W *)c.a + (((int64_t)a * c.kt + kt) * RT * 64 + lane) * 8;
#pragma unroll
    for (int r = 0; r < RT; r++) v[r].load(aw + 512 * r);
  };
  if (mine && step(0) < full) {
    Run<W, 8> av[U][RT], an[U][RT];
    auto load_group = [&](Run<W, 8>(&v)[U][RT], int a, int n0) {
#pragma unroll
      for (int i = 0; i < U; i++) load_a(v[i], a, min(step(n0 + i), full - 1));
    };
    int n0 = 0, a = a0;
    uint64_t todo = rest;
    load_group(av, a, 0);
    for (;;) {
      // the next adapter of this group, or the first of the next group: in
      // flight through this one's products
      const int n1 = todo ? n0 : n0 + U;
      const bool more = step(n1) < full;
      int a1 = a0;
      if (todo) a1 = pick(todo);
      else todo = rest;
      if (more) {
        load_group(an, a1, n1);
        if (n1 != n0) load_x(xn, n1);
      }
      __builtin_amdgcn_sched_barrier(0);
      f4v sum[RT];
#pragma unroll
      for (int r = 0; r < RT; r++) sum[r] = acc[r];
#pragma unroll
      for (int i = 0; i < U; i++)
        if (step(n0 + i) < full) {
#pragma unroll
          for (int r = 0; r < RT; r++) sum[r] = product(av[i][r], xv[i], sum[r]);
        }
#pragma unroll
      for (int r = 0; r < RT; r++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[r][i] = id == a ? sum[r][i] : acc[r][i];
      if (!more) break;
#pragma unroll
      for (int i = 0; i < U; i++) {
#pragma unroll
        for (int r = 0; r < RT; r++) av[i][r] = an[i][r];
        if (n1 != n0) xv[i] = xn[i];
      }
      n0 = n1;
      a = a1;
    }
  }
  if (full < c.kt && wave == WAVES - 1) {  // the last, part step of an odd d_in
    Run<X, 8> xt;
    xt.load_part(xr, 32 * full + 8 * g, c.d_in);
    for (uint64_t todo = mine; todo;) {
      const int a = pick(todo);
      Run<W, 8> av[RT];
      load_a(av, a, full);
#pragma unroll
      for (int r = 0; r < RT; r++) {
        const f4v sum = product(av[r], xt, acc[r]);
#pragma unroll
        for (int i = 0; i < 4; i++) acc[r][i] = id == a ? sum[i] : acc[r][i];
      }
    }
  }
  if (mine && cb0 < last) load_b(wv, a0, cb0);
  if (mine) {  // of the block: every wave has the same tokens
    if constexpr (DOT) {
#pragma unroll
      for (int r = 0; r < RT; r++) {
        float v = acc[r][0] + __shfl_xor(acc[r][0], 16, 64);
        v += __shfl_xor(v, 32, 64);
        if (g == 0) part[wave][0][16 * r + col] = v;
      }
    } else if (TOK == 16 || col == 0)
#pragma unroll
      for (int r = 0; r < RT; r++)
        *reinterpret_cast<f4v *>(&part[wave][TOK == 1 ? 0 : col][16 * r + 4 * g]) = acc[r];
    __syncthreads();
    for (int i = tid; i < TOK * RP; i += 64 * WAVES) {
      const int t = i / RP, r = i % RP;
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES; w++) sum += part[w][t][r];
      u[t][r] = sum;
    }
    __syncthreads();
  }

  // this lane's token: ranks 4 RT g .. of its u, in parts
  constexpr int NS = RT == 1 ? 4 : 8, NV = 4 * RT / NS;  // elements and count of MFMA operands
  Run<W, NS> ur[PARTS][NV];
  float back = 1.0f;  // 2^e
  {
    __align__(16) float v[4 * RT];
    float top = 0.0f;
    if (mine)
#pragma unroll
      for (int r = 0; r < RT; r++)
        *reinterpret_cast<f4v *>(&v[4 * r]) =
            *reinterpret_cast<const f4v *>(&u[TOK == 1 ? 0 : col][4 * RT * g + 4 * r]);
    else
#pragma unroll
      for (int r = 0; r < 4 * RT; r++) v[r] = 0.0f;
#pragma unroll
    for (int r = 0; r < 4 * RT; r++) top = fmaxf(top, fabsf(v[r]));
    if (__is_same(W, __half)) {
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const int e = top < INFINITY ? max((int)(__float_as_uint(top) >> 23) - 127 - 14, -126) : 0;
      back = __uint_as_float((uint32_t)(e + 127) << 23);
#pragma unroll
      for (int r = 0; r < 4 * RT; r++) v[r] = __builtin_amdgcn_ldexpf(v[r], -e);
    }
#pragma unroll
    for (int r = 0; r < 4 * RT; r++) {
      const bool finite = fabsf(v[r]) < INFINITY;
#pragma unroll
      for (int p = 0; p < PARTS; p++) {
        const float h = finite ? part_of(v[r], (W *)nullptr) : p ? 0.0f : v[r];
        ur[p][r / NS].set(r % NS, h);
        v[r] -= finite ? h : 0.0f;
      }
    }
  }

  // 64 outputs of each token after another, and for each the adapters of these
  // tokens; the next step's operands in flight through this one's products
  if (cb0 >= last) return;
  float out[16];
#pragma unroll
  for (int i = 0; i < 16; i++) out[i] = 0.0f;
  int cb = cb0, a = a0;
  uint64_t todo = rest;
  float sc = c.scale[a0];
  for (;;) {
    const int cb1 = todo ? cb : cb + WAVES;
    const bool more = cb1 < last, done = !todo;
    int a1 = a0;
    if (todo) a1 = pick(todo);
    else todo = rest;
    float sc1 = sc;
    if (more) {
      if (mine) load_b(wn, a1, cb1);
      if (rest) sc1 = c.scale[a1];
      if (done) load_base(bn, cb1);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (mine)
#pragma unroll
      for (int q = 0; q < 4; q++) {
        f4v acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int p = PARTS - 1; p >= 0; p--)
#pragma unroll
          for (int n = 0; n < NV; n++) {
            Run<W, NS> o;  // elements q 4 RT + NS n .. of the lane's 16 RT
#pragma unroll
            for (int d = 0; d < NS / 2; d++) {
              const int f = (q * 4 * RT + NS * n) / 2 + d;
              o.w[d] = wv[f / 4].w[f % 4];
            }
            acc = mma(o, ur[p][n], acc);
          }
#pragma unroll
        for (int i = 0; i < 4; i++) out[4 * q + i] = id == a ? sc * (back * acc[i]) : out[4 * q + i];
      }
    if (done) {
      if (in && (TOK == 16 || col == 0)) {
#pragma unroll
        for (int i = 0; i < 16; i++) out[i] += bv.at(i);
#pragma unroll
        for (int i = 0; i < 16; i++) bv.set(i, out[i]);
        Y *yr = c.y + row * c.y_stride + 64 * cb + 16 * g;
        if (64 * cb + 64 <= c.d_out) bv.store(yr);
        else bv.store_part(yr, c.d_out - 64 * cb - 16 * g);
      }
      if (!more) break;
#pragma unroll
      for (int i = 0; i < 16; i++) out[i] = 0.0f;
      bv = bn;
    }
#pragma unroll
    for (int j = 0; j < 2 * RT; j++) wv[j] = wn[j];
    cb = cb1;
    a = a1;
    sc = sc1;
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
  const bool single = T <= SINGLE_MAX_T;
  const int tiles = single ? T : (T + 15) / 16;
  const int slices = std::max(1, std::min(c.nb, TARGET_BLOCKS / tiles));
  c.per = (c.nb + slices - 1) / slices;
  c.slices = (c.nb + c.per - 1) / c.per;
  const dim3 grid((uint32_t)tiles * c.slices), block(64 * waves_for(single ? 1 : 16, h->rp / 16));
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

AdaptersShape adapters_shape(const hy3x_adapters *h) { return {h->d_in, h->d_out, h->device}; }

void launch_adapters(const hy3x_adapters *h, const int32_t *ids, const void *x, int x_type,
                     int64_t x_stride, const void *base, int64_t base_stride, void *y, int y_type,
                     int64_t y_stride, int T, hipStream_t st) {
  if (h->type == HY3X_F16)
    launch_types<__half>(h, ids, x, x_type == HY3X_F32, x_stride, base, base_stride, y,
                         y_type == HY3X_F32, y_stride, T, st);
  else
    launch_types<__hip_bfloat16>(h, ids, x, x_type == HY3X_F32, x_stride, base, base_stride, y,
                                 y_type == HY3X_F32, y_stride, T, st);
}

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
  launch_adapters(h, ids, x, x_type, x_stride, base, base_stride, y, y_type, y_stride, T,
                  (hipStream_t)stream);
  OP_HIP_TRY(hipGetLastError());
  return HY3X_OK;
}

}  // extern "C"
