// hy3x_linear4_kernels.h -- kernels of the products of 4-bit weights (the
// mathematics and the weights' layout: hy3x_linear4.h).
//
// Products: v_mfma_f32_16x16x32_{bf16,f16}, rows = tokens, columns = 16 rows of W.
// Operands are q - 7.5, exact in both types, so a group's sum is the fp32 accumulator of
// its MFMAs, and its scale is one FMA. fp32 x meets them as three bf16 parts, which hold
// all of its 24 bits (two would leave 2^-16 of it). q itself would take 7 instructions a lane's
// 8 weights in place of 9, and 2048 tokens, 8192 rows of 4096 154 us in place of 159, but
// sums over x of one sign then come to many times the output before the zero points take
// that off again: relative errors of fp32 outputs, 64 tokens of |N(0, 1)|, 4096 rows of 4096,
// 9e-7 (bf16 x) and 4.1e-6 (fp32 x), centred 1.0e-7 and 3.0e-7 (a plain fp32 product 2.1e-7
// and 5.2e-7).
//
// A lane's 8 weights become an operand by 2 shifts, 3 bit selections and 4 conversions, 15 ns a
// wave and SIMD, more than the time of one MFMA (9 ns): weights that only one tile of tokens meets
// cost more to unpack than to multiply, and bytes bound them (few tokens); unpacked once
// for 4 tiles of tokens they are a quarter of that, and the MFMAs bound them (many).
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>

#include "hy3x_dma.h"
#include "hy3x_linear4.h"

namespace hy3x {
namespace linear4 {

typedef __bf16 bf8v __attribute__((ext_vector_type(8)));
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
  // two bytes (the low or the high ones), sign and magnitude below 16, as half of these
  // numbers: as e4m3 they stand for 2^-9 of them
  template <bool HI>
  static __device__ __forceinline__ uint32_t ints(uint32_t bytes) {
    return __builtin_bit_cast(uint32_t,
                              __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(bytes, 256.0f, HI));
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
                              __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(bytes, 256.0f, HI));
  }
  static __device__ __forceinline__ uint32_t both(float v) {  // exact: at most 8 bits
    return (__float_as_uint(v) >> 16) * 0x10001u;
  }
};
template <>
struct Op<float> : Op<__hip_bfloat16> {
  static constexpr int PARTS = 3;
};

// 8 weights of a lane as an operand, q - 7.5 in the order of k.
template <class X>
__device__ __forceinline__ u4v weights(uint32_t w) {
  // a & b | c, then twice a & b | c & ~b: one instruction each
  const uint32_t lo = __builtin_amdgcn_bitop3_b32(w, 0x8e8e8e8eu, 0x01010101u, 0xea);
  const uint32_t m = __builtin_amdgcn_bitop3_b32(w >> 3, 0x0e0e0e0eu, lo, 0xe2);
  const uint32_t hi = __builtin_amdgcn_bitop3_b32(w << 7, 0x80808080u, m, 0xe2);
  return (u4v){Op<X>::template ints<false>(lo), Op<X>::template ints<true>(lo),
               Op<X>::template ints<false>(hi), Op<X>::template ints<true>(hi)};
}

// Part p of v in bf16: v = p0 + p1 + p2 (of an infinity the others are NaN).
__device__ __forceinline__ float trunc16(float v) {
  return __uint_as_float(__float_as_uint(v) & 0xffff0000u);
}
__device__ __forceinline__ float part_of(float v, int p) {
  const float a = trunc16(v), r = v - a, b = trunc16(r);
  return p == 0 ? a : p == 1 ? b : p == 2 ? r - b : 0.0f;
}
__device__ __forceinline__ uint32_t pair16(float lo, float hi) {  // their upper halves
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302);
}

// Elements k .. k + 7 of a row. Loads are 16 bytes at the elements' own alignment.
template <class X>
struct Eight {
  uint32_t w[2 * sizeof(X)];
  __device__ __forceinline__ void load(const X *row, int k) {
    __builtin_memcpy(w, row + k, sizeof(w));
  }
  // of a row of n (n >= 8), zeros beyond it: its last 8, moved down
  __device__ __forceinline__ void load_within(const X *row, int k, int n) {
    load(row, min(k, n - 8));
    const int by = min(max(k + 8 - n, 0), 8);
    if constexpr (sizeof(X) == 4) {
#pragma unroll
      for (int s = 1; s <= 8; s *= 2)
#pragma unroll
        for (int j = 0; j < 8; j++) w[j] = by & s ? (j + s < 8 ? w[j + s] : 0) : w[j];
    } else {
      uint64_t lo = w[0] | (uint64_t)w[1] << 32, hi = w[2] | (uint64_t)w[3] << 32;
      const int bits = 16 * (by & 3);
      if (by & 8) lo = hi = 0;
      lo = by & 4 ? hi : lo;
      hi = by & 4 ? 0 : hi;
      lo = lo >> bits | (hi << 1) << (63 - bits);
      hi >>= bits;
      w[0] = (uint32_t)lo;
      w[1] = (uint32_t)(lo >> 32);
      w[2] = (uint32_t)hi;
      w[3] = (uint32_t)(hi >> 32);
    }
  }
  // as an operand (part `part` of fp32), in the order of k
  __device__ __forceinline__ u4v operand(int part) const {
    u4v out;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if constexpr (sizeof(X) == 4)
        out[j] = pair16(part_of(__uint_as_float(w[2 * j]), part),
                        part_of(__uint_as_float(w[2 * j + 1]), part));
      else out[j] = w[j];
    }
    return out;
  }
};

__device__ __forceinline__ float scale_of(uint32_t bits, bool s16) {
  return s16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)bits) : __uint_as_float(bits << 16);
}

template <class Y>
constexpr int type_of() {
  return __is_same(Y, float) ? HY3X_F32 : __is_same(Y, __half) ? HY3X_F16 : HY3X_BF16;
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
__device__ __forceinline__ void put(const Linear4Call &c, int64_t token, int n, float v) {
  if (c.base) v += load_y(c.base, token * c.base_stride + n, c.y_type);
  store_y(c.y, token * c.y_stride + n, c.y_type, v);
}
// N outputs that follow each other, in one store
template <class Y, int N>
__device__ __forceinline__ void put_run(const Linear4Call &c, int64_t token, int n,
                                        const float (&v)[N]) {
  Y e[N];
  float b[N];
#pragma unroll
  for (int i = 0; i < N; i++) b[i] = 0.0f;
  if (c.base) {
    __builtin_memcpy(e, (const Y *)c.base + token * c.base_stride + n, sizeof(e));
#pragma unroll
    for (int i = 0; i < N; i++) b[i] = load_y(&e[i], 0, type_of<Y>());
  }
#pragma unroll
  for (int i = 0; i < N; i++) store_y(&e[i], 0, type_of<Y>(), v[i] + b[i]);
  __builtin_memcpy((Y *)c.y + token * c.y_stride + n, e, sizeof(e));
}

// A quad's scales and zero points (as 2 z - 15) of one row: 4 GP of each.
template <int GP>
struct Groups {
  uint32_t s[2 * GP], z[GP];
  __device__ __forceinline__ void load(const Linear4Call &c, int rt, int qd, int row) {
    __builtin_memcpy(s, __builtin_assume_aligned(
        c.s + (((size_t)rt * c.quads + qd) * 16 + row) * (4 * GP), 8 * GP), sizeof(s));
    __builtin_memcpy(z, __builtin_assume_aligned(
        c.z + ((size_t)rt * c.z_tile + (size_t)qd * c.z_quad + row * (4 * GP)), 4 * GP), sizeof(z));
  }
  __device__ __forceinline__ float scale(int g, bool s16) const {
    return scale_of(s[g / 2] >> (16 * (g & 1)) & 0xffffu, s16);
  }
  __device__ __forceinline__ float zero(int g) const {  // 2 z - 15
    return (float)(int8_t)(z[g / 4] >> (8 * (g & 3)));
  }
};

// ---- few tokens ---------------------------------------------------------------
// A block's waves split the quads of every row of W; each holds its part of x as
// operands for as long as the block lasts, and the weights stream past, a row tile at
// a time, RING of them in flight. The waves' sums meet in LDS.
//
// What the zero points take off, (z - 7.5) sum x, is formed from sums of x / 2 over the groups,
// which the MFMAs find (times a matrix of halves) while the first weights are on their way.
//
// Tokens: one tile of 16 (fp32: of 4, whose three parts are rows 4 t + p). Token t is row
// 4 (t % 4) + t / 4, so that up to 4 tokens end in one register of the accumulator: NR of
// its 4 are used.
//
// Bytes bound it where W is large: one token of bf16, 120832 rows of 4096, groups of 128: 46
// us, 5.5 TB/s of weights; fp32 51 us. Small ones are a chain of waits (x, operands, their
// sums, the tile, the join): 4096 rows of 4096 4.7 us.

// Waves of a block, at most: the registers of a SIMD are enough for 4, or for 2 with a
// ring or with fp32 on its way to parts.
template <class X, int RING>
constexpr int few_waves() {
  return RING == 1 && Op<X>::PARTS == 1 ? 16 : 8;
}

template <int HQ, int GP>
struct FewWeights {
  u4v q[HQ][4];
  Groups<GP> g[HQ];
  __device__ __forceinline__ void load(const Linear4Call &c, int rt, int wave, int waves,
                                       int lane) {
#pragma unroll
    for (int i = 0; i < HQ; i++) {
      const int qd = min(wave + i * waves, c.quads - 1);
#pragma unroll
      for (int j = 0; j < 4; j++)
        q[i][j] = __builtin_nontemporal_load(
            &c.q[((size_t)rt * c.chunks + min(4 * qd + j, c.chunks - 1)) * 64 + lane]);
      g[i].load(c, rt, qd, lane & 15);
    }
  }
};

template <class X, int GP, int HQ, int NR, int RING>
__global__ __launch_bounds__((64 * few_waves<X, RING>()),
                             (few_waves<X, RING>() / 4)) void k_linear4_few(Linear4Call c) {
  constexpr bool SPLIT = Op<X>::PARTS == 3;
  constexpr int OUT = SPLIT ? 1 : NR, WAVES = few_waves<X, RING>();  // OUT: sums of a lane
  __shared__ float red[RING == 1 ? 1 : 2][WAVES][OUT][64];
  __shared__ alignas(16) float sums[WAVES][HQ * 4 * GP][4][SPLIT ? 1 : 4];  // of x / 2
  const int lane = threadIdx.x & 63, col = lane & 15, h = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;

  // this lane's row of A: token and part
  const int part = SPLIT ? col & 3 : 0, token = SPLIT ? col >> 2 : 4 * (col & 3) + (col >> 2);
  u4v a[HQ][4][4];
  FewWeights<HQ, GP> ring[RING];
  {
    const X *row = (const X *)c.x + (int64_t)min(token, c.T - 1) * c.x_stride;
#pragma unroll
    for (int i = 0; i < HQ; i++) {
      const int k0 = 512 * (wave + i * waves);
      const bool whole = k0 + 512 <= c.d_in;
#pragma unroll
      for (int ch = 0; ch < 4; ch++) {
        Eight<X> e[4];
        if (whole) {
#pragma unroll
          for (int j = 0; j < 4; j++) e[j].load(row, k0 + 128 * ch + 32 * j + 8 * h);
        } else {
#pragma unroll
          for (int j = 0; j < 4; j++)
            e[j].load_within(row, k0 + 128 * ch + 32 * j + 8 * h, c.d_in);
        }
        if (i == 0 && ch == (SPLIT ? 0 : 3)) ring[0].load(c, blockIdx.x, wave, waves, lane);
#pragma unroll
        for (int j = 0; j < 4; j++) a[i][ch][j] = e[j].operand(part);
        if (SPLIT) __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
#pragma unroll
  for (int p = 1; p < RING; p++)
    if (blockIdx.x + p * gridDim.x < (uint32_t)c.tiles)
      ring[p].load(c, blockIdx.x + p * gridDim.x, wave, waves, lane);
  const uint32_t half = Op<X>::both(0.5f);
#pragma unroll
  for (int i = 0; i < HQ; i++)
#pragma unroll
    for (int g = 0; g < 4 * GP; g++) {
      f4v d = {0, 0, 0, 0};
#pragma unroll
      for (int j = g * 4 / GP; j < (g + 1) * 4 / GP; j++)
        d = Op<X>::mma(a[i][j / 4][j % 4], (u4v){half, half, half, half}, d);
      if (col == 0) {
        if constexpr (SPLIT) sums[wave][i * 4 * GP + g][h][0] = d[0] + (d[1] + d[2]);
        else *(f4v *)sums[wave][i * 4 * GP + g][h] = d;
      }
      __builtin_amdgcn_sched_barrier(0);
    }

  auto tile = [&](const FewWeights<HQ, GP> &w, int turn) {
    float acc[OUT];
#pragma unroll
    for (int r = 0; r < OUT; r++) acc[r] = 0.0f;
    asm volatile("" ::: "memory");  // the sums stay in LDS from tile to tile
#pragma unroll
    for (int i = 0; i < HQ; i++)
#pragma unroll
      for (int g = 0; g < 4 * GP; g++) {  // groups of the quad
        f4v d = {0, 0, 0, 0};
#pragma unroll
        for (int j = g * 4 / GP; j < (g + 1) * 4 / GP; j++)  // 32 k of the quad's 512
          d = Op<X>::mma(a[i][j / 4][j % 4], weights<X>(w.q[i][j / 4][j % 4]), d);
        const float s = w.g[i].scale(g, c.s16), z = w.g[i].zero(g);
        if (SPLIT) d[0] += d[1] + d[2];
#pragma unroll
        for (int r = 0; r < OUT; r++)
          acc[r] = fmaf(s, fmaf(-z, sums[wave][i * 4 * GP + g][h][r], d[r]), acc[r]);
        if (g % GP == GP - 1) __builtin_amdgcn_sched_barrier(0);  // registers of one chunk
      }
#pragma unroll
    for (int r = 0; r < OUT; r++)
      red[turn & 1][wave][r][lane] = acc[r];
  };
  auto join = [&](int rt, int turn) {
    __syncthreads();
    // 64 sums at a time, by waves in turn; two buffers: a wave that writes the other one
    // has passed this barrier, and one that writes this one the next
    for (int o = (wave + waves - turn % waves) % waves; o < OUT; o += waves) {
      const int64_t t = SPLIT ? h : 4 * o + h;
      const int n = (int)linear4_row(rt, col);
      float v = 0.0f;
#pragma unroll 4
      for (int w = 0; w < waves; w++) v += red[turn & 1][w][o][lane];
      if (t < c.T && n < c.d_out) put(c, t, n, v);
    }
  };
  if constexpr (RING == 1) {
    tile(ring[0], 0);
    join(blockIdx.x, 0);
  } else {
    int turn = 0;
    for (int rt0 = blockIdx.x; rt0 < c.tiles; rt0 += RING * gridDim.x) {
#pragma unroll
      for (int p = 0; p < RING; p++, turn++) {
        const int rt = rt0 + p * gridDim.x;
        if (p && rt >= c.tiles) return;
        tile(ring[p], turn);
        if (rt + RING * (int)gridDim.x < c.tiles)
          ring[p].load(c, rt + RING * gridDim.x, wave, waves, lane);
        join(rt, turn);
      }
    }
  }
}

// ---- many tokens --------------------------------------------------------------
// A block takes 16 RT WN rows of W and 16 CT tokens; WK of its waves share a row's k, a
// run of its chunks each, one a step. x goes through LDS in the operands' order, a step
// ahead: copied there as it is (DMA: rows of whole chunks, aligned to 16 bytes), or by way
// of registers (fp32 becomes its three parts). Weights go straight to the lanes that use
// them, and a chunk's operands stay in registers while its token tiles pass; scales and
// zero points come for several chunks at once, as every load costs the same address cycles.
//
// What the zero points take off, s (z - 7.5) sum x, follows a step behind: the waves that share
// a chunk find the sums of its token tiles on the MFMAs (x times halves), each those of the
// tiles that it comes to first, and leave them in LDS.
//
// 2048 tokens, 8192 rows of 4096, bf16, groups of 128: 158 us, 870 TFLOP/s (a bf16 product
// of 8192^3 reaches 1266 on the same card). No one part bounds it: its vector
// instructions are 91 us of a SIMD, its MFMAs 58, and the two waves of a SIMD do not hide all of
// each other's. (With 7 instructions to unpack and 154 us: without the MFMAs 122 us, without the
// reads of LDS 126, without the copies 131, without both of these 105 of 157 then; all operands by
// way of LDS, as 16-bit numbers that one wave unpacks for all, in three buffers 156; products of
// a chunk ordered by k first 167.) fp32 x is three products: 300 tokens, 4096 rows of 1536 16 us
// in bf16, in fp32 24.
template <class X, int GP, int RT, int CT, int WN, int WK, bool DMA>
__global__ __launch_bounds__(64 * WN * WK, 2) void k_linear4_many(Linear4Call c) {
  constexpr int PARTS = Op<X>::PARTS, THREADS = 64 * WN * WK;
  constexpr int PIECES = WK * CT * 256 / THREADS;  // runs of 8 elements a thread loads a step
  static_assert(PIECES * THREADS == WK * CT * 256 && !(DMA && PARTS > 1), "whole pieces");
  static_assert(CT % WN == 0 || WN % CT == 0, "a wave's own token tiles");
  constexpr int XS = WK * PARTS * CT * 256, BUFS = DMA ? 2 : 1;
  constexpr int RED = WK > 1 ? (WK - 1) * WN * RT * CT * 64 : 1;
  constexpr int SQ = 4 / GP;  // chunks of a quad whose scales come in one load: 4 groups
  __shared__ u4v lds[BUFS * XS > RED ? BUFS * XS : RED];
  __shared__ f4v sums[2][WK][CT][GP][4];  // of x / 2 over a chunk's groups
  const int lane = threadIdx.x & 63, col = lane & 15, h = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave / WK, wk = wave % WK;
  // token tiles first (2048 tokens, 8192 rows of 4096: 160 us, with a run of neighbouring
  // tiles for each XCD 165, its rows first 162)
  const uint32_t token_tiles = (c.T + 16 * CT - 1) / (16 * CT);
  const int rt0 = (int)(blockIdx.x / token_tiles) * (RT * WN) + wn * RT;
  const int64_t t0 = (int64_t)(blockIdx.x % token_tiles) * (16 * CT);
  const int steps = (c.chunks + WK - 1) / WK;  // wave wk's chunks: from steps wk on
  // piece p of a step: [wk][ct][j][lane], run j of 32 k and (lane / 16) of 8 of a token
  const X *const x0 = (const X *)c.x + t0 * c.x_stride;
  const X *from[DMA ? 1 : PIECES];
  uint32_t offset[DMA ? PIECES : 1];
#pragma unroll
  for (int i = 0; i < PIECES; i++) {
    const int p = threadIdx.x + i * THREADS;
    const int64_t at = min((int64_t)(p / 256 % CT) * 16 + p % 16, c.T - 1 - t0) * c.x_stride;
    if constexpr (DMA) offset[i] = (uint32_t)(2 * (at + p / 64 % 4 * 32 + p % 64 / 16 * 8));
    else from[i] = x0 + at;
  }
  Eight<X> ex[DMA ? 1 : PIECES];
  auto fetch = [&](int step) {
    if constexpr (DMA) {
#pragma unroll
      for (int i = 0; i < PIECES; i++) {
        // a wave's pieces are of one chunk; one beyond the last: its scales are 0
        const int w = (64 * wave + i * THREADS) / (256 * CT);
        dma16_s(x0 + (size_t)min(steps * w + step, c.chunks - 1) * 128, offset[i],
                lds_addr(&lds[(step & 1) * XS + i * THREADS + 64 * wave]));
      }
    } else {
      const bool whole = (steps * (WK - 1) + step + 1) * 128 <= c.d_in;
#pragma unroll
      for (int i = 0; i < PIECES; i++) {
        const int p = threadIdx.x + i * THREADS;
        const int k = (steps * (p / (256 * CT)) + step) * 128 + p / 64 % 4 * 32 + p % 64 / 16 * 8;
        if (whole) ex[i].load(from[i], k);
        else ex[i].load_within(from[i], k, c.d_in);
      }
    }
  };
  u4v q[RT];
  auto load_q = [&](int step) {
    const int ch = min(steps * wk + step, c.chunks - 1);
#pragma unroll
    for (int r = 0; r < RT; r++)
      q[r] = c.q[((size_t)min(rt0 + r, c.tiles - 1) * c.chunks + ch) * 64 + lane];
  };
  uint64_t sr[RT];  // scales and zero points of 4 groups: SQ chunks
  uint32_t zr[RT];
  auto load_s = [&](int step) {
    const int ch = min(steps * wk + step, c.chunks - 1), qd = ch >> 2;
    const uint32_t at = (lane & 15) * (4 * GP) + ((ch & 3) / SQ) * 4;
#pragma unroll
    for (int r = 0; r < RT; r++) {
      const int rt = min(rt0 + r, c.tiles - 1);
      sr[r] = *(const uint64_t *)(c.s + ((size_t)rt * c.quads + qd) * (64 * GP) + at);
      zr[r] = *(const uint32_t *)(c.z + ((size_t)rt * c.z_tile + (size_t)qd * c.z_quad + at));
    }
  };
  float acc[RT][CT][4], off[GP][RT];  // off: -s (2 z - 15) of the chunk before
#pragma unroll
  for (int r = 0; r < RT; r++) {
#pragma unroll
    for (int t = 0; t < CT; t++)
#pragma unroll
      for (int i = 0; i < 4; i++) acc[r][t][i] = 0.0f;
#pragma unroll
    for (int g = 0; g < GP; g++) off[g][r] = 0.0f;
  }
  if (wn == 0)
    for (int i = lane; i < CT * GP * 4; i += 64) (&sums[1][wk][0][0][0])[i] = (f4v){0, 0, 0, 0};

  // the token tiles in each wave's own order: place t is tile (wn + t) % CT
  const uint32_t half = Op<X>::both(0.5f);
  fetch(0);
  load_s(0);
  load_q(0);
  for (int step = 0; step < steps; step++) {
    if constexpr (DMA) {
      wait_copies_and_barrier<0>();
    } else {
      if (step) __syncthreads();
#pragma unroll
      for (int i = 0; i < PIECES; i++) {
        const int p = threadIdx.x + i * THREADS;
#pragma unroll
        for (int part = 0; part < PARTS; part++)
          lds[(p / (256 * CT) * PARTS + part) * (256 * CT) + p % (256 * CT)] =
              ex[i].operand(part);
      }
      __syncthreads();
    }
    u4v b[4][RT];
    float s[GP][RT], z[GP][RT];
    const int ch = steps * wk + step, at = GP * (ch % SQ);  // the chunk's first of 4 groups
#pragma unroll
    for (int r = 0; r < RT; r++) {
#pragma unroll
      for (int g = 0; g < GP; g++) {
        const int k = at + g;
        const float v = scale_of((uint32_t)(sr[r] >> (16 * k)) & 0xffffu, c.s16);
        s[g][r] = ch < c.chunks ? v : 0.0f;
        z[g][r] = (float)(int8_t)(zr[r] >> (8 * k));
      }
#pragma unroll
      for (int j = 0; j < 4; j++) b[j][r] = weights<X>(q[r][j]);
    }
    if (step + 1 < steps) {
      fetch(step + 1);
      load_q(step + 1);
      if ((ch + 1) % SQ == 0) load_s(step + 1);
    }
    const u4v *xs = &lds[(DMA ? (step & 1) * XS : 0) + wk * (PARTS * CT * 256) + lane];
#pragma unroll
    for (int t = 0; t < CT; t++) {
      const int tile = (wn + t) % CT;
#pragma unroll
      for (int g = 0; g < GP; g++) {
        const f4v before = sums[~step & 1][wk][tile][g][h];
        f4v d[RT], sum = {0, 0, 0, 0};
#pragma unroll
        for (int r = 0; r < RT; r++) d[r] = (f4v){0, 0, 0, 0};
#pragma unroll
        for (int j = g * 4 / GP; j < (g + 1) * 4 / GP; j++)
#pragma unroll
          for (int part = 0; part < PARTS; part++) {
            const u4v a = xs[(part * CT + tile) * 256 + j * 64];
#pragma unroll
            for (int r = 0; r < RT; r++) d[r] = Op<X>::mma(a, b[j][r], d[r]);
            if (t % WN == 0) sum = Op<X>::mma(a, (u4v){half, half, half, half}, sum);
          }
        if (t % WN == 0 && col == 0) sums[step & 1][wk][tile][g][h] = sum;
#pragma unroll
        for (int r = 0; r < RT; r++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            acc[r][t][i] = fmaf(off[g][r], before[i], acc[r][t][i]);
            acc[r][t][i] = fmaf(s[g][r], d[r][i], acc[r][t][i]);
          }
      }
    }
#pragma unroll
    for (int g = 0; g < GP; g++)
#pragma unroll
      for (int r = 0; r < RT; r++) off[g][r] = -s[g][r] * z[g][r];
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < CT; t++)
#pragma unroll
    for (int g = 0; g < GP; g++) {
      const f4v before = sums[~steps & 1][wk][(wn + t) % CT][g][h];
#pragma unroll
      for (int r = 0; r < RT; r++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[r][t][i] = fmaf(off[g][r], before[i], acc[r][t][i]);
    }
  if constexpr (WK > 1) {  // the waves' parts of k
    if (wk)
#pragma unroll
      for (int r = 0; r < RT; r++)
#pragma unroll
        for (int t = 0; t < CT; t++)
          lds[(((wk - 1) * WN + wn) * RT * CT + r * CT + t) * 64 + lane] =
              __builtin_bit_cast(u4v, *(f4v *)acc[r][t]);
    __syncthreads();
    if (wk) return;
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
      for (int t = 0; t < CT; t++)
        for (int w = 1; w < WK; w++) {
          const f4v o = __builtin_bit_cast(
              f4v, lds[(((w - 1) * WN + wn) * RT * CT + r * CT + t) * 64 + lane]);
#pragma unroll
          for (int i = 0; i < 4; i++) acc[r][t][i] += o[i];
        }
  }
  const int n = (int)linear4_row(rt0, col);
#pragma unroll
  for (int t = 0; t < CT; t++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int64_t token = t0 + 16 * ((wn + t) % CT) + 4 * h + i;
      if (token >= c.T) continue;
      float v[RT];
#pragma unroll
      for (int r = 0; r < RT; r++) v[r] = acc[r][t][i];
      if (n + RT <= c.d_out) {
        if (c.y_type == HY3X_F32) put_run<float>(c, token, n, v);
        else if (c.y_type == HY3X_F16) put_run<__half>(c, token, n, v);
        else put_run<__hip_bfloat16>(c, token, n, v);
      } else {
#pragma unroll
        for (int r = 0; r < RT; r++)
          if (n + r < c.d_out) put(c, token, n + r, v[r]);
      }
    }
}

template <class X, int GP, int RT, int CT, int WN, int WK, bool DMA>
void many(const Linear4Call &c, hipStream_t st) {
  const int64_t blocks = (int64_t)((c.T + 16 * CT - 1) / (16 * CT)) *
                         ((c.tiles + RT * WN - 1) / (RT * WN));
  k_linear4_many<X, GP, RT, CT, WN, WK, DMA><<<(uint32_t)blocks, 64 * WN * WK, 0, st>>>(c);
}
template <class X, int GP, int HQ, int NR, int RING>
void few(const Linear4Call &c, int waves, int blocks, hipStream_t st) {
  k_linear4_few<X, GP, HQ, NR, RING><<<blocks, 64 * waves, 0, st>>>(c);
}
// Whether x in registers serves this call, and if so its launch. Where all row tiles fit the
// card at once (16 waves on each of 256 CUs) each has a block and no ring; longer ones have
// a ring where the waves are enough for the card (from 5 quads), and two quads a wave only
// where the registers are (groups of 128, up to 4 tokens). us for one bf16 token, then of the
// next kernel's best shape: 4096 rows of 4096 4.7 and 5.5 (once), 8192 of 4096 6.8 and 7.7
// (once), 4096 of 8192 6.8 and 8.7 (once), 120832 of 4096 46.0 and 53.3 (ring); 8192 of 8192
// 12.3 and 11.3 (two quads a wave, what it costs at its worst).
template <class X, int GP, int NR>
bool few(const Linear4Call &c, hipStream_t st) {
  constexpr int RING = few_waves<X, 2>();
  if constexpr (Op<X>::PARTS == 1) {
    constexpr int ONCE = few_waves<X, 1>();
    if (c.quads <= ONCE && (int64_t)c.tiles * c.quads <= 256 * ONCE) {
      few<X, GP, 1, NR, 1>(c, c.quads, c.tiles, st);
      return true;
    }
    if constexpr (GP == 1 && NR == 1)
      if (c.quads > RING && c.quads <= 2 * RING) {
        few<X, GP, 2, NR, 2>(c, (c.quads + 1) / 2, std::min(c.tiles, 256), st);
        return true;
      }
  }
  if (c.quads > 4 && c.quads <= RING) {
    few<X, GP, 1, NR, 3>(c, c.quads, std::min(c.tiles, 256), st);
    return true;
  }
  return false;
}

// The tile's shape by the size of the result: small tiles and a split of k where blocks are
// few, large ones, which read and unpack less, where they are many; the limits of those with 8
// waves are where each CU has a block (2124: two). us, shapes as RT CT WN WK, the chosen one and
// the next best, groups of 128 (in brackets: of 32, whose sums and scales leave no registers for
// 4 x 4 tiles); tokens x rows of d_in, 16-bit x:
//   16 x 4096 of 1536   1124  5.4, 1118  5.7    24 x 4096 of 1536   2124  6.3, 2142  8.0
//   16 x 4096 of 4096   1118  7.7, 2118  8.9    24 x 4096 of 4096   2124 11.0, 4118 11.4
//   16 x 8192 of 4096   2118 10.1, 1124 10.6    24 x 4096 of 8192   4118 17.1, 2124 18.3
//   16 x 16384 of 4096  1124 13.0, 2118 14.7    64 x 8192 of 4096   2124 16.5, 2224 17.0
//   16 x 120832 of 4096 4141 57.4, 1124 80.8    200 x 4096 of 4096  2242 22.0, 2142 25.3
//   300 x 4096 of 1536  2241 16.6, 2442 16.4        (1242 33.1, 2242 33.3)
//   300 x 8192 of 4096  2241 45.0, 2242 45.4    512 x 4096 of 4096  2442 31.8, 2241 33.9
//   512 x 8192 of 4096  2441 55.9, 2281 61.4        (2442 45.4, 2241 52.1)
//   32 x 65536 of 4096  2241 40.9, 2442 54.6    528 x 4096 of 4096  2241 45.0, 2242 43.9
//   768 x 4096 of 4096  2241 46.2, 2441 48.8    832 x 4096 of 4096  2441 48.5, 4241 56.8
//       (2241 66.0, 2441 73.9)                      (2441 74.4, 2241 90.9)
//   768 x 8192 of 4096  2441 71.9, 4441 83.1    784 x 8192 of 4096  4441 78.9, 2441 90.8
//   32 x 120832 of 4096 4241 65.6, 2241 70.5    40 x 120832 of 4096 4441 87.3, 2441 93.0
//       (2241  100, 2441  139)                      (2441  141, 2241  164)
//   2048 x 8192 of 4096 4441  157, 2441  175; by 64 2441 199, 2241 243
// groups of 64:
//   256 x 4096 of 4096  2242 24.6, 2241 30.6    512 x 4096 of 4096  2442 35.9, 2242 37.6
//   768 x 4096 of 4096  2241 53.2, 2242 54.2    448 x 8192 of 4096  2441 56.8, 2242 66.5
// 16-bit x that goes by way of registers (larger tiles share that work):
//   64 x 8192 of 4096   4124 24.4, 2124 25.6    400 x 4096 of 4096  2241 48.3, 2442 53.2
// fp32 x:
//   64 x 4096 of 8192   2124 33.5, 4118 33.1    100 x 4096 of 4096  4124 26.5, 2124 33.5
//   150 x 4096 of 4096  4142 40.7, 4124 47.0    256 x 4096 of 4096  4142 40.4, 2141 49.0
//   264 x 4096 of 4096  2141 57.3, 2281 60.7    320 x 4096 of 4096  2141 57.0, 2281 60.8
//   352 x 4096 of 4096  2281 60.9, 2141 59.2    400 x 4096 of 4096  2281 61.1, 2241 66.5
//   512 x 4096 of 4096  2281 63.5, 2241 68.7    300 x 8192 of 4096  2241 89.1, 2141 95.9
//   512 x 8192 of 4096  4241  110, 2241  128
// and, up to where 2141 has three blocks on each CU, groups of 32 (of 64 already 352 x 4096
// 2281 64.7, 2141 66.3):
//   384 x 4096 of 4096  (2141 74.8, 2281 82.4)  400 x 4096 of 4096  (2281 82.7, 2141  105)
template <class X, int GP, bool DMA>
void by_size(const Linear4Call &c, hipStream_t st) {
  constexpr bool SPLIT = Op<X>::PARTS == 3;
  constexpr int RT = GP == 4 ? 2 : 4;
  const int64_t size = (int64_t)((c.T + 15) / 16) * c.tiles;  // in tiles of 16 x 16 outputs
  if (c.T <= 16) {
    if (size > 2048) return many<X, GP, 4, 1, 4, 1, DMA>(c, st);
    if (size > 768 || c.chunks < 24) return many<X, GP, 1, 1, 2, 4, DMA>(c, st);
    if (size > 384) return many<X, GP, 2, 1, 1, 8, DMA>(c, st);
    return many<X, GP, 1, 1, 1, 8, DMA>(c, st);
  }
  if constexpr (SPLIT) {
    if (size <= 1536) return many<X, GP, 2, 1, 2, 4, DMA>(c, st);
    if (size <= 2048) return many<X, GP, 4, 1, 2, 4, DMA>(c, st);
    if (size <= 4096) return many<X, GP, 4, 1, 4, 2, DMA>(c, st);
    if (size <= (GP == 4 ? 6144 : 5120)) return many<X, GP, 2, 1, 4, 1, DMA>(c, st);
    if (size <= 8192) return many<X, GP, 2, 2, 8, 1, DMA>(c, st);
    if (size <= 12288) return many<X, GP, 2, 2, 4, 1, DMA>(c, st);
    return many<X, GP, RT, 2, 4, 1, DMA>(c, st);
  } else {
    if (size <= 1536 && c.chunks >= 48) return many<X, GP, 4, 1, 1, 8, DMA>(c, st);
    if (size <= (DMA ? 2048 : 1536)) return many<X, GP, 2, 1, 2, 4, DMA>(c, st);
    if constexpr (DMA) {
      if (size <= 4096) return many<X, GP, GP == 4 ? 1 : 2, 2, 4, 2, DMA>(c, st);
      if (size <= 8192 && c.T > 32 && (GP == 4 || c.chunks >= 24))
        return many<X, GP, 2, 4, 4, 2, DMA>(c, st);
    } else {
      if (size <= 2048) return many<X, GP, 4, 1, 2, 4, DMA>(c, st);
      if (size <= 4096) return many<X, GP, 2, 2, 4, 2, DMA>(c, st);
    }
    if (size <= 12288) return many<X, GP, 2, 2, 4, 1, DMA>(c, st);
    if (c.T <= 32) return many<X, GP, RT, 2, 4, 1, DMA>(c, st);
    if (size <= 24576 && c.T > 64) return many<X, GP, 2, 4, 4, 1, DMA>(c, st);
    return many<X, GP, GP == 1 ? 4 : 2, 4, 4, 1, DMA>(c, st);
  }
}

// x in registers up to 4 tokens, for 16-bit x up to 16: there one wave's 4 sums a lane cost it
// 4 times the FMAs, and it is the faster one only for few row tiles, which are all there at
// once, and for many: 16 tokens, 4096 rows of 4096 7.1 us and 7.7, 8192 of 4096 11.2 and 10.0,
// 16384 13.5 and 12.6, 120832 55.0 and 57.4. With groups of 32 the FMAs of 16 tokens outweigh
// the bytes (4096 of 4096, when it was built, 17.7 and 9.2). fp32 x has the ring alone: one
// token, 8192 rows of 4096 12.5 and 11.8, 16384 15.9 and 19.9, 120832 51.0 and 70.9; its
// groups of 32 do not fit the registers.
template <class X, int GP>
void launch_group(const Linear4Call &c, hipStream_t st) {
  constexpr bool SPLIT = Op<X>::PARTS == 3;
  if (c.T <= 4) {
    if constexpr (!SPLIT || GP < 4)
      if (!SPLIT || c.tiles > 768)
        if (few<X, GP, 1>(c, st)) return;
  } else if (c.T <= 16 && (c.tiles <= 256 || c.tiles > 1024)) {
    if constexpr (!SPLIT && GP < 4)
      if (few<X, GP, 4>(c, st)) return;
  }
  // copies to LDS (2048 tokens, 8192 rows of 4096: 158 us; rows that begin at odd
  // elements, by way of registers, 237)
  if constexpr (!SPLIT)  // 32-bit offsets of 64 rows
    if (c.d_in % 128 == 0 && (uintptr_t)c.x % 16 == 0 && c.x_stride % 8 == 0 &&
        c.x_stride <= 1 << 24)
      return by_size<X, GP, true>(c, st);
  by_size<X, GP, false>(c, st);
}

}  // namespace linear4

template <class X>
void launch_linear4(const Linear4Call &c, hipStream_t st) {
  if (c.group == 128) linear4::launch_group<X, 1>(c, st);
  else if (c.group == 64) linear4::launch_group<X, 2>(c, st);
  else linear4::launch_group<X, 4>(c, st);
}

}  // namespace hy3x
