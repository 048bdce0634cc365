// hy3x_adapters.hip -- low-rank adapters of many requests at once beside a
// shared projection (hy3x_adapters_*):
//
//   u = A_a x_t                      (fp32 sums over d_in)
//   y_t = base_t + scale_a (B_a u)   (fp32 sums over the rank, y rounded once)
//
// One launch: a block takes TOK tokens and a slice of their outputs, and forms
// u for itself, so nothing passes between blocks: no scratch memory, no second
// launch, no order of blocks in the results. Its waves split d_in, join their
// parts of u in LDS, then split the outputs. (Two launches over scratch, the
// parts of u by blocks of their own and A and B read for 32 tokens at a time,
// measured 39.0 us against 36.1 at 4096 x 4096 outputs of rank 64.)
//
// Figures in pairs or in braces compare two forms of one step, measured together
// when it was chosen; what the kernel takes as it stands is under "What bounds it".
//
// TOK = 16: 16 consecutive tokens, the columns of every MFMA. The adapters that
// occur among them are taken one after another: each forms its products for all
// 16 columns, and the columns of its own tokens are selected, so a token never
// meets another adapter's values (not even their infinities). Where several blocks
// share a tile's outputs its adapters can be dealt to them (deal_for). TOK = 1: one
// token in every column.
//
// Products: v_mfma_f32_16x16x32_{f16,bf16} (rows = 16 ranks, columns = tokens).
// fp32 x meets A in three two-byte parts (Split), or in fp32 FMAs for one token;
// u meets B in three too (Parts). The parts keep fp32's range and precision.
// (v_mfma_f32_16x16x4_f32 on fp32 x: 512 tokens of 4096 inputs 52.6 us at rank 64,
// 24.3 in parts, 19.2 and 15.3 at rank 16; before tiles dealt their adapters.)
//
// What bounds it (us of the kernel, inputs and weights from HBM, MI355X; a copy
// reaches 5.2 TB/s): many tokens the bytes of x, base and y only in part, 13.0 us for
// 4096 x 4096 fp16 outputs of 4096 inputs without an adapter; with them each tile's
// chain of x, A, LDS, B and y, and the tiles with several adapters, which end last
// (rank 64: 36.2 us for 111 MB, 3.1 TB/s, 58 with two in every tile; rank 16, 2000
// tokens: 16.3 us for 53 MB, 3.2 TB/s, 14.0 where no tile has two); up to 256
// decoded tokens the adapters' weights (256 tokens, 128 adapters: 14.0 us for 40 MB,
// 2.9 TB/s); a few tokens four loads that wait for each other, ids, A, B, the store
// (32 tokens: 6.1 us; one token beside the router: 6.2 us), and the same in few
// tiles (512 tokens, 1536 fp32 inputs, 4096 fp32 outputs, rank 32: 13.3 us for 20
// MB, 2 of it the tiles with two adapters).
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
#include <type_traits>

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

// Waves of a block: 16 where 128 registers a lane hold the operands in flight
// (512 tokens, fp32, rank 32: 12.6 us with 8 waves, 12.1 with 16; one token beside
// the router 9.0 and 7.8), 8 above.
constexpr int waves_for(int TOK, int RT) { return RT == 1 || (RT == 2 && TOK == 16) ? 16 : 8; }
// Up to this many tokens, one per CU, a block takes one token and the order of the
// adapters does not matter; above, tiles of 16. The ids are on the device, so T alone
// decides. us, one token per block | tiles, 4096 -> 4096 of rank 16 in bf16, every
// token another of 128 adapters, and runs of 100 tokens with one:
//   256 tokens         14.3 | 39.5 (not dealt)   10.2 | 9.8
//   320 (a second round of blocks) 21.0 | 20.9   18.4 | 10.9
//   1024               45.1 | 35.0               36.6 | 13.7
// What neither serves are single tokens beside long runs: their tiles of up to 16
// adapters end long after the others (2000 tokens, 64 of them single: 45.0 us, in
// two calls 22.6; 4096 of rank 64, 256 single: 210 and 81).
constexpr int SINGLE_MAX_T = 256;
// Blocks that the outputs are sliced for: one per CU. More slices form u again
// (512 blocks: 32 decoded tokens 9.8 us against 6.1, 512 in fp32 19.1 against
// 13.1, 2000 22.4 against 16.4, 4096 of rank 64 45.0 against 36.2).
constexpr int TARGET_BLOCKS = 256;

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
  // Stores past the caches (non-temporal). Plain ones fill the L2s with y, whose
  // write-back then ends the kernel: 4096 x 4096 outputs at rank 64 49.8 us with
  // plain stores, 36.1 with these; a kernel that reads y next is not slower for it
  // (32 x 1536 to 4096 x 4096).
  __device__ __forceinline__ void store(T *p) const {
    typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(2)));
#pragma unroll
    for (int k = 0; k < N * (int)sizeof(T) / 16; k++)
      __builtin_nontemporal_store((u4){w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]},
                                  (u4 *)p + k);
  }
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
struct Call {
  const uint16_t *a, *b;
  const float *scale;
  int count, rank, kt, nb, d_in, d_out;  // kt = kp / 32, nb = np / 64
  const int32_t *ids;
  const void *x, *base;  // rows in the kernel's X and Y
  void *y;
  int64_t x_stride, base_stride, y_stride;
  int T, slices, per;  // per: 64-output blocks of a slice
  uint64_t deal;       // deal_for
};

// v in parts of W's precision, largest first: v = 2^e (p0 + p1 + p2).
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

// Parts of u: three, which hold all 24 bits of an fp32 value. Two fp16 parts hold 22
// and cut the rest off, which an fp16 y shows where the base cancels the product.
constexpr int PARTS = 3;

// N steps of a token's fp32 x as three two-byte operands each, which hold its 24
// bits: x = 2^e (p0 + p1 + p2). bf16 has fp32's range, and e = 0. fp16: e grows
// with the largest |x| so far, which lies below 2^(e + 15), and what was summed
// before is scaled along; parts reach down to 2^-24, at most 2^-38 of the largest.
template <class W>
struct Wide {
  Run<W, 8> p[3];
};
template <class W>
struct Split {
  int e = -126;
  template <int N, int RT>
  __device__ __forceinline__ void operator()(const Run<float, 8> (&x)[N], Wide<W> (&out)[N],
                                             f4v (&acc)[RT]) {
    float v[N][8], top = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        v[i][j] = x[i].at(j);
        top = fmaxf(top, fabsf(v[i][j]));
      }
    const bool odd = __ballot(top == INFINITY);
    if (odd) {
      top = 0.0f;
#pragma unroll
      for (int i = 0; i < N; i++)
#pragma unroll
        for (int j = 0; j < 8; j++)
          top = fabsf(v[i][j]) < INFINITY ? fmaxf(top, fabsf(v[i][j])) : top;
    }
    if constexpr (__is_same(W, __half)) {
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const int at = max((int)(__float_as_uint(top) >> 23) - 127 - 14, e);
      if (__ballot(at != e)) {
#pragma unroll
        for (int r = 0; r < RT; r++)
#pragma unroll
          for (int i = 0; i < 4; i++) acc[r][i] = __builtin_amdgcn_ldexpf(acc[r][i], e - at);
        e = at;
      }
      const float by = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
      for (int i = 0; i < N; i++)
#pragma unroll
        for (int j = 0; j < 8; j++) v[i][j] *= by;
    }
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
      for (int q = 0; q < 3; q++) {
        float h[8];
#pragma unroll
        for (int d = 0; d < 4; d++) {
          if constexpr (__is_same(W, __half)) {
            const auto two = __builtin_amdgcn_cvt_pkrtz(v[i][2 * d], v[i][2 * d + 1]);
            out[i].p[q].w[d] = __builtin_bit_cast(uint32_t, two);
            h[2 * d] = (float)two[0];
            h[2 * d + 1] = (float)two[1];
          } else {
            const uint32_t lo = __float_as_uint(v[i][2 * d]), hi = __float_as_uint(v[i][2 * d + 1]);
            out[i].p[q].w[d] = __builtin_amdgcn_perm(hi, lo, 0x07060302);
            h[2 * d] = __uint_as_float(lo & 0xffff0000u);
            h[2 * d + 1] = __uint_as_float(hi & 0xffff0000u);
          }
        }
        if (q == 2) break;
        if (odd)  // an infinity is its first part, the others 0
#pragma unroll
          for (int j = 0; j < 8; j++)
            if (fabsf(v[i][j]) == INFINITY) v[i][j] = h[j] = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) v[i][j] -= h[j];
      }
  }
  template <int RT>
  __device__ __forceinline__ void end(f4v (&acc)[RT]) const {
    if constexpr (__is_same(W, __half))
#pragma unroll
      for (int r = 0; r < RT; r++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[r][i] = __builtin_amdgcn_ldexpf(acc[r][i], e);
  }
};

// The tokens of a wave's columns: 16 consecutive ones, or one in all of them.
// Columns past the last token read row 0, for nothing.
struct Tokens {
  int64_t row;
  bool in;
  int id;         // this column's adapter, -1: none
  uint64_t mine;  // lanes below 16 whose column has one

  __device__ __forceinline__ void find(int64_t token, int T, const int32_t *ids) {
    in = token < T;
    row = in ? token : 0;
    id = ids[row];
  }
  __device__ __forceinline__ void settle(int count) {
    if (!in || id >= count) id = -1;
    mine = __ballot(id >= 0) & 0xffffu;
  }
  // the next adapter of the tokens in todo
  __device__ __forceinline__ int pick(uint64_t &todo) const {
    const int a = __builtin_amdgcn_readlane(id, __ffsll((long long)todo) - 1);
    todo &= ~__ballot(id == a);
    return a;
  }
  // Several adapters in a tile whose outputs `slices` blocks share: dealt to parts
  // (deal_for), each with its share of the slices. This block then has the tokens
  // of one part. Returns the number of parts.
  __device__ __forceinline__ int deal(uint64_t table, int slices, int slice) {
    uint64_t todo = mine;
    int n = 0, at = 0;  // adapters, this column's
    while (todo) {
      const int next = pick(todo);
      at = id == next ? n : at;
      n++;
    }
    const int parts = n ? (int)(table >> (4 * n - 4) & 15) + 1 : 1;
    if (parts == 1) return 1;
    if (at % parts != slice % parts) {  // without an adapter: of part 0
      in = false;
      id = -1;
    }
    mine = __ballot(id >= 0) & 0xffffu;
    return parts;
  }
};

// This wave's part of u of its tokens, rank 16 r + 4 g + i of its column in
// acc[r][i]: d_in in steps of 32, pairs of them (128 bytes of a two-byte row) in
// turn over WAVES waves, U steps to a group, two groups in flight; in each group
// the adapters of these tokens one after another.
// DOT: by fp32 products instead of MFMAs (one token), this lane's eight elements
// of a step for rank 16 r + col in acc[r][0].
// SPLIT: fp32 x as three two-byte parts (Split).
template <class W, class X, int RT, int WAVES, int U, bool DOT>
struct Shrink {
  static constexpr bool SPLIT = sizeof(X) == 4 && !DOT;
  using XO = std::conditional_t<SPLIT, Wide<W>, Run<X, 8>>;  // x as the products read it
  Run<X, 8> xv[U];
  Split<W> parts;
  const X *xr;
  f4v acc[RT];
  int full, kt, d_in, lane, wave;  // full: whole steps, kt: all steps

  __device__ __forceinline__ int step(int n) const {
    return 2 * WAVES * (n >> 1) + 2 * wave + (n & 1);
  }
  __device__ __forceinline__ void load_x(Run<X, 8> (&v)[U], int n0) const {
#pragma unroll
    for (int i = 0; i < U; i++)
      v[i].load(xr + 32 * min(step(n0 + i), full - 1) + 8 * (lane >> 4));
  }
  // x of the first group, which needs no adapter yet
  __device__ __forceinline__ void begin(const Call &c, const Tokens &tk, int w) {
    lane = threadIdx.x & 63;
    wave = w;
    d_in = c.d_in;
    full = d_in / 32;
    kt = c.kt;
    xr = (const X *)c.x + tk.row * c.x_stride;
#pragma unroll
    for (int r = 0; r < RT; r++) acc[r] = f4v{0.f, 0.f, 0.f, 0.f};
    if (full) load_x(xv, 0);
  }
  __device__ __forceinline__ void load_a(Run<W, 8> (&v)[RT], const W *a, int step) const {
    const W *aw = a + ((int64_t)step * RT * 64 + lane) * 8;
#pragma unroll
    for (int r = 0; r < RT; r++) v[r].load(aw + 512 * r);
  }
  // x of a group, loaded, as operands
  template <int N>
  __device__ __forceinline__ void take(const Run<X, 8> (&x)[N], XO (&o)[N]) {
    if constexpr (SPLIT) parts(x, o, acc);
    else
#pragma unroll
      for (int i = 0; i < N; i++) o[i] = x[i];
  }
  static __device__ __forceinline__ f4v product(const Run<W, 8> &a, const XO &b, f4v v) {
    if constexpr (SPLIT) {
#pragma unroll
      for (int k = 2; k >= 0; k--) v = mma(a, b.p[k], v);
      return v;
    } else if constexpr (DOT) {
#pragma unroll
      for (int j = 0; j < 8; j++) v[0] = __builtin_fmaf(a.at(j), b.at(j), v[0]);
      return v;
    } else {
      return mma(a, b, v);
    }
  }
  // N steps of adapter a's weights for the columns that use it
  template <int N, class Live>
  __device__ __forceinline__ void add(const Run<W, 8> (&av)[N][RT], const XO (&x)[N],
                                      const Tokens &tk, int a, Live live) {
    f4v sum[RT];
#pragma unroll
    for (int r = 0; r < RT; r++) sum[r] = acc[r];
#pragma unroll
    for (int i = 0; i < N; i++)
      if (live(i)) {
#pragma unroll
        for (int r = 0; r < RT; r++) sum[r] = product(av[i][r], x[i], sum[r]);
      }
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
      for (int i = 0; i < 4; i++) acc[r][i] = tk.id == a ? sum[r][i] : acc[r][i];
  }
  __device__ __forceinline__ void run(const Call &c, const Tokens &tk) {
    uint64_t rest = tk.mine;
    if (!rest) return;
    const int64_t size = (int64_t)kt * RT * 512;  // elements of one adapter's A
    const W *base = (const W *)c.a;
    const int a0 = tk.pick(rest);
    if (step(0) < full) {
      Run<X, 8> xn[U];
      XO xo[U];
      Run<W, 8> av[U][RT], an[U][RT];
      auto load_group = [&](Run<W, 8>(&v)[U][RT], int a, int n0) {
#pragma unroll
        for (int i = 0; i < U; i++) load_a(v[i], base + a * size, min(step(n0 + i), full - 1));
      };
      int n0 = 0, a = a0;
      uint64_t todo = rest;
      load_group(av, a, 0);
      take(xv, xo);
      for (;;) {
        // the next adapter of this group, or the first of the next group
        const int n1 = todo ? n0 : n0 + U;
        const bool more = step(n1) < full;
        int a1 = a0;
        if (todo) a1 = tk.pick(todo);
        else todo = rest;
        if (more) {
          load_group(an, a1, n1);
          if (n1 != n0) load_x(xn, n1);
        }
        __builtin_amdgcn_sched_barrier(0);  // these loads before the products
        add<U>(av, xo, tk, a, [&](int i) { return step(n0 + i) < full; });
        if (!more) break;
#pragma unroll
        for (int i = 0; i < U; i++)
#pragma unroll
          for (int r = 0; r < RT; r++) av[i][r] = an[i][r];
        if (n1 != n0) take(xn, xo);
        n0 = n1;
        a = a1;
      }
    }
    if (full < kt && wave == WAVES - 1) {  // the last, part step of an odd d_in
      Run<X, 8> xt[1];
      XO xo[1];
      xt[0].load_part(xr, 32 * full + 8 * (lane >> 4), d_in);
      take(xt, xo);
      for (uint64_t todo = tk.mine; todo;) {
        const int a = tk.pick(todo);
        Run<W, 8> av[1][RT];
        load_a(av[0], base + a * size, full);
        add<1>(av, xo, tk, a, [](int) { return true; });
      }
    }
    if constexpr (SPLIT) parts.end(acc);
  }
};

// u of a lane's token, ranks 4 RT g + s, as MFMA operands in parts.
template <class W, int RT>
struct Parts {
  static constexpr int NS = RT == 1 ? 4 : 8, NV = 4 * RT / NS;  // elements, operands
  Run<W, NS> p[PARTS][NV];
  float back;  // 2^e

  __device__ __forceinline__ void split(float (&v)[4 * RT]) {
    back = 1.0f;
    if (__is_same(W, __half)) {
      float top = 0.0f;
#pragma unroll
      for (int r = 0; r < 4 * RT; r++) top = fmaxf(top, fabsf(v[r]));
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
      for (int q = 0; q < PARTS; q++) {
        const float h = finite ? part_of(v[r], (W *)nullptr) : q ? 0.0f : v[r];
        p[q][r / NS].set(r % NS, h);
        v[r] -= finite ? h : 0.0f;
      }
    }
  }
  // outputs 16 g + 4 q + i of a block of 64 in acc[i]
  __device__ __forceinline__ f4v product(const Run<W, 8> (&b)[2 * RT], int q) const {
    f4v acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = PARTS - 1; k >= 0; k--)
#pragma unroll
      for (int n = 0; n < NV; n++) {
        Run<W, NS> o;  // elements q 4 RT + NS n .. of the lane's 16 RT
#pragma unroll
        for (int d = 0; d < NS / 2; d++) {
          const int f = (q * 4 * RT + NS * n) / 2 + d;
          o.w[d] = b[f / 4].w[f % 4];
        }
        acc = mma(o, p[k][n], acc);
      }
    return acc;
  }
};

// Where a lane's 16 outputs of a block of 64 lie: two-byte ones in one run of 16
// (32 bytes), fp32 ones in four runs of 4, 16 apart, so that the four lanes of a
// token write 64 bytes at a time (4096 x 4096 fp32 outputs, rank 64: 67.0 us, in one
// run of 64 bytes per lane 76.0; the same without adapters 33.1 and 63.7). Half a line
// at a time past the caches is still more than y: 512 x 4096 outputs, 8.4 MB, write
// 11.9 MB by the counters, two-byte ones 1.07 to 1.1 times y.
template <class Y>
struct Place {
  static constexpr int RUN = sizeof(Y) == 4 ? 4 : 16, N = 16 / RUN;
  static __device__ __forceinline__ int col(int g, int k) {  // of run k
    return sizeof(Y) == 4 ? 16 * k + 4 * g : 16 * g;
  }
};

// The outputs cb0, cb0 + WAVES, .. (blocks of 64) below `last` of the wave's
// tokens, and for each the adapters of these tokens one after another; the next
// step's operands in flight through this one's products.
template <class W, class Y, int RT, int WAVES>
struct Expand {
  using P = Place<Y>;
  using Piece = Run<Y, P::RUN>;
  Piece bv[P::N], bn[P::N];
  Run<W, 8> wv[2 * RT], wn[2 * RT];
  const Y *br;

  __device__ __forceinline__ void load_base(const Call &c, Piece (&v)[P::N], int cb) const {
    const int g = (threadIdx.x & 63) >> 4;
    const bool whole = 64 * cb + 64 <= c.d_out;
#pragma unroll
    for (int k = 0; k < P::N; k++) {
      const int c0 = 64 * cb + P::col(g, k);
      if (br && whole) v[k].load(br + c0);
      else if (br) v[k].load_part(br, c0, c.d_out);
      else
#pragma unroll
        for (int i = 0; i < P::RUN; i++) v[k].set(i, 0.0f);
    }
  }
  // B's rows as the MFMAs of these places read them: row m of MFMA q is output
  // 16 (m / 4) + 4 q + m % 4, as B is laid out, or output 16 q + m, which lies with
  // lane 4 q + m % 4 as its part m / 4
  __device__ __forceinline__ void load_b(const Call &c, Run<W, 8> (&v)[2 * RT], int a,
                                         int cb) const {
    const int lane = threadIdx.x & 63;
    const W *bw = (const W *)c.b + ((int64_t)a * c.nb + cb) * 2 * RT * 512;
    if constexpr (sizeof(Y) == 2) {
#pragma unroll
      for (int j = 0; j < 2 * RT; j++) v[j].load(bw + j * 512 + lane * 8);
    } else {
      const int part = (lane & 15) >> 2;
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const int from = (lane & 48) + 4 * q + (lane & 3);
        if constexpr (RT == 1) {
          Run<W, 4> h;
          h.load(bw + (part >> 1) * 512 + from * 8 + (part & 1) * 4);
          v[q / 2].w[q % 2 * 2] = h.w[0];
          v[q / 2].w[q % 2 * 2 + 1] = h.w[1];
        } else {
#pragma unroll
          for (int j = 0; j < RT / 2; j++)
            v[q * (RT / 2) + j].load(bw + (part * (RT / 2) + j) * 512 + from * 8);
        }
      }
    }
  }
  // the base of the first outputs, which needs no adapter yet
  __device__ __forceinline__ void begin(const Call &c, const Tokens &tk, int cb0, int last) {
    br = c.base && tk.in ? (const Y *)c.base + tk.row * c.base_stride : nullptr;
    if (cb0 < last) load_base(c, bv, cb0);
  }
  // B of the first outputs and adapter
  __device__ __forceinline__ void ahead(const Call &c, const Tokens &tk, int cb0, int last) {
    uint64_t rest = tk.mine;
    if (rest && cb0 < last) load_b(c, wv, tk.pick(rest), cb0);
  }
  template <class U>
  __device__ __forceinline__ void run(const Call &c, const Tokens &tk, const U &u, int cb0,
                                      int last, bool stores) {
    if (cb0 >= last) return;
    uint64_t rest = tk.mine;
    const int a0 = rest ? tk.pick(rest) : 0;
    // -0: what a token without an adapter adds to its base, a base of -0 included
    float out[16];
#pragma unroll
    for (int i = 0; i < 16; i++) out[i] = -0.0f;
    int cb = cb0, a = a0;
    uint64_t todo = rest;
    float sc = c.scale[a0];
    for (;;) {
      const int cb1 = todo ? cb : cb + WAVES;
      const bool more = cb1 < last, done = !todo;
      int a1 = a0;
      if (todo) a1 = tk.pick(todo);
      else todo = rest;
      float sc1 = sc;
      if (more) {
        if (tk.mine) load_b(c, wn, a1, cb1);
        if (rest) sc1 = c.scale[a1];
        if (done) load_base(c, bn, cb1);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (tk.mine)
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const f4v acc = u.product(wv, q);
#pragma unroll
          for (int i = 0; i < 4; i++)
            out[4 * q + i] = tk.id == a ? sc * (u.back * acc[i]) : out[4 * q + i];
        }
      if (done) {
        const int g = (threadIdx.x & 63) >> 4;
        Y *yr = (Y *)c.y + tk.row * c.y_stride;
#pragma unroll
        for (int k = 0; k < P::N; k++) {
          float sum[P::RUN];
#pragma unroll
          for (int i = 0; i < P::RUN; i++) sum[i] = out[P::RUN * k + i] + bv[k].at(i);
#pragma unroll
          for (int i = 0; i < P::RUN; i++) bv[k].set(i, sum[i]);
          const int c0 = 64 * cb + P::col(g, k);
          if (!tk.in || !stores) continue;
          if (64 * cb + 64 > c.d_out) bv[k].store_part(yr + c0, c.d_out - c0);
          else bv[k].store(yr + c0);
        }
        if (!more) break;
#pragma unroll
        for (int i = 0; i < 16; i++) out[i] = -0.0f;
#pragma unroll
        for (int k = 0; k < P::N; k++) bv[k] = bn[k];
      }
#pragma unroll
      for (int j = 0; j < 2 * RT; j++) wv[j] = wn[j];
      cb = cb1;
      a = a1;
      sc = sc1;
    }
  }
};

// Launch order -> item: each XCD on a contiguous run of (tokens, slice) items,
// so that the slices of some tokens share x and A in its L2, and neighbouring
// tokens their adapters.
__device__ __forceinline__ uint32_t item_of(uint32_t block, uint32_t n) {
  const uint32_t xcd = block % 8;
  return xcd * (n / 8) + min(xcd, n % 8) + block / 8;
}

// Steps of a group by register budget: 128 registers a lane with 16 waves, 256
// with 8; split: fp32 x in three parts.
constexpr int steps_for(int waves, int RT, int x_size, bool split) {
  if (RT == 8 || (RT == 2 && split)) return 1;
  return x_size == 4 || RT == 4 || (RT == 2 && waves == 16) ? 2 : 4;
}

template <class W, class X, class Y, int RT, int TOK>
__global__ __launch_bounds__(64 * waves_for(TOK, RT)) void k_adapters(const Call c) {
  constexpr int WAVES = waves_for(TOK, RT);
  constexpr int RP = 16 * RT, PITCH = RP + 4;  // floats per token in LDS
  constexpr bool DOT = TOK == 1 && sizeof(X) == 4;
  __shared__ __align__(16) float part[WAVES][TOK][PITCH];
  __shared__ __align__(16) float u[TOK][PITCH];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4;
  const int col = lane & 15, at = TOK == 1 ? 0 : col;  // at: the column's token of the block
  const uint32_t item = item_of(blockIdx.x, gridDim.x), tile = item / c.slices;
  const int slice = item % c.slices;
  int last = min(c.nb, (slice + 1) * c.per), cb0 = slice * c.per + wave;
  Tokens tk;
  tk.find((int64_t)tile * TOK + at, c.T, c.ids);
  Shrink<W, X, RT, WAVES, steps_for(WAVES, RT, sizeof(X), sizeof(X) == 4 && !DOT), DOT> sh;
  sh.begin(c, tk, wave);
  Expand<W, Y, RT, WAVES> ex;
  ex.begin(c, tk, cb0, last);
  tk.settle(c.count);
  if (TOK > 1 && c.slices > 1) {
    const int parts = tk.deal(c.deal, c.slices, slice);
    if (parts > 1) {
      const int blocks = (c.slices - 1 - slice % parts) / parts + 1;
      const int per = (c.nb + blocks - 1) / blocks;
      last = min(c.nb, (slice / parts + 1) * per);
      cb0 = slice / parts * per + wave;
      ex.begin(c, tk, cb0, last);
    }
  }
  sh.run(c, tk);
  ex.ahead(c, tk, cb0, last);
  Parts<W, RT> pu;
  if (tk.mine) {  // of the block: every wave has the same tokens
    if constexpr (DOT) {
#pragma unroll
      for (int r = 0; r < RT; r++) {
        float s = sh.acc[r][0] + __shfl_xor(sh.acc[r][0], 16, 64);
        s += __shfl_xor(s, 32, 64);
        if (g == 0) part[wave][0][16 * r + col] = s;
      }
    } else if (TOK == 16 || col == 0)
#pragma unroll
      for (int r = 0; r < RT; r++)
        *reinterpret_cast<f4v *>(&part[wave][at][16 * r + 4 * g]) = sh.acc[r];
    __syncthreads();
    for (int i = tid; i < TOK * RP; i += 64 * WAVES) {
      const int t = i / RP, r = i % RP;
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES; w++) s += part[w][t][r];
      u[t][r] = r < c.rank ? s : 0.0f;  // an infinite x makes NaNs of the padding's zeros
    }
    __syncthreads();
    __align__(16) float v[4 * RT];
#pragma unroll
    for (int r = 0; r < RT; r++)
      *reinterpret_cast<f4v *>(&v[4 * r]) =
          *reinterpret_cast<const f4v *>(&u[at][4 * RT * g + 4 * r]);
    pu.split(v);
  }
  ex.run(c, tk, pu, cb0, last, TOK == 16 || col == 0);
}

// A, B and scale of one adapter into the handle, a thread per 16 bytes.
__global__ __launch_bounds__(256) void k_pack_adapter(const uint16_t *__restrict__ a,
                                                      const uint16_t *__restrict__ b, int rank,
                                                      int d_in, int d_out, int rp, int kt, int nb,
                                                      uint16_t *__restrict__ pa,
                                                      uint16_t *__restrict__ pb,
                                                      float scale, float *__restrict__ pscale) {
  const int rt = rp / 16, na = kt * rt * 64, nbl = nb * 2 * rt * 64;
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= na + nbl) return;
  if (i == 0) *pscale = scale;
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

// Into how many parts the n = 1 .. 16 adapters of a tile are dealt (less one, in 4
// bits each), so that a block forms u of fewer adapters, for more outputs: the
// number with the fewest bytes for the block that has the most. a: of one A, b: of
// one B, io: of a tile's base and y, whose tokens may be uneven by 6; 32 KB an
// adapter and 200 KB for the base's first loads again stand for their latencies (a
// CU takes about 100 KB a us). us, not dealt and dealt: 512 tokens of 4096 fp32
// inputs, 1536 outputs, rank 64, two adapters in some tiles 24.0 and 18.7, eight in
// every tile 75.2 and 22.9; 2000 tokens, 4096 x 4096, rank 64 27.0 and 23.9; rank
// 16, which stays at one part, 15.9 and 17.0.
uint64_t deal_for(int slices, float a, float b, float io) {
  uint64_t table = 0;
  for (int n = 2; n <= 16; n++) {
    int parts = 1;
    float least = n * (a + b / slices + 32e3f) + io / slices;
    for (int p = 2; p <= std::min(n, slices); p++) {
      const int m = (n + p - 1) / p;  // adapters of a part
      const float q = slices / p, tokens = std::min(16, 16 * m / n + 6);
      const float bytes = m * (a + b / q + 32e3f) + io / q * tokens / 16 + 200e3f;
      if (bytes < least) {
        parts = p;
        least = bytes;
      }
    }
    table |= (uint64_t)(parts - 1) << (4 * n - 4);
  }
  return table;
}

template <class W, class X, class Y>
void launch(const hy3x_adapters *h, const int32_t *ids, const void *x, int64_t x_stride,
            const void *base, int64_t base_stride, void *y, int64_t y_stride, int T,
            hipStream_t st) {
  Call c;
  c.a = h->a;
  c.b = h->b;
  c.scale = h->scale;
  c.count = h->count;
  c.rank = h->rank;
  c.kt = h->kp / 32;
  c.nb = h->np / 64;
  c.d_in = h->d_in;
  c.d_out = h->d_out;
  c.ids = ids;
  c.x = x;
  c.base = base;
  c.y = y;
  c.x_stride = x_stride;
  c.base_stride = base_stride;
  c.y_stride = y_stride;
  c.T = T;
  auto slice = [&](int tiles) {
    const int slices = std::max(1, std::min(c.nb, TARGET_BLOCKS / tiles));
    c.per = (c.nb + slices - 1) / slices;
    c.slices = (c.nb + c.per - 1) / c.per;
    c.deal = c.slices == 1 ? 0
                           : deal_for(c.slices, 2.0f * h->kp * h->rp, 2.0f * h->np * h->rp,
                                      32.0f * c.d_out * sizeof(Y));
    return dim3((uint32_t)tiles * c.slices);
  };
  const bool single = T <= SINGLE_MAX_T;
#define HY3X_ADAPTERS(RT)                                                                       \
  if (h->rp == 16 * RT) {                                                                       \
    if (single)                                                                                 \
      k_adapters<W, X, Y, RT, 1><<<slice(T), 64 * waves_for(1, RT), 0, st>>>(c);                \
    else                                                                                        \
      k_adapters<W, X, Y, RT, 16><<<slice((T + 15) / 16), 64 * waves_for(16, RT), 0, st>>>(c);  \
    return;                                                                                     \
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
      h->a + (size_t)index * h->rp * h->kp, h->b + (size_t)index * h->rp * h->np, scale,
      h->scale + index);
  OP_HIP_TRY(hipGetLastError());
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
  const uintptr_t i0 = (uintptr_t)ids, y0 = (uintptr_t)y;
  if (i0 < y0 + (uintptr_t)(((T - 1) * y_stride + h->d_out) * ys) && y0 < i0 + (uintptr_t)T * 4)
    return op_fail(HY3X_E_ARG, "y overlaps ids");
  if (rows_overlap(x, x_stride * xs, h->d_in * xs, y, y_stride * ys, h->d_out * ys, T))
    return op_fail(HY3X_E_ARG, "y overlaps x");
  if (base && !(base == y && (base_stride == y_stride || T == 1)) &&
      rows_overlap(base, base_stride * ys, h->d_out * ys, y, y_stride * ys, h->d_out * ys, T))
    return op_fail(HY3X_E_ARG, "y overlaps base without being base");
  const int rc = check_device(h);
  if (rc) return rc;
  launch_adapters(h, ids, x, x_type, x_stride, base, base_stride, y, y_type, y_stride, T,
                  (hipStream_t)stream);
  OP_HIP_TRY(hipGetLastError());
  return HY3X_OK;
}

}  // extern "C"
