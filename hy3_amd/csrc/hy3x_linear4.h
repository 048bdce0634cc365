// hy3x_linear4.h -- products of 4-bit weights: their layout, and a checked call of
// their kernels (hy3x_linear4_kernels.h, instances by x's type in
// hy3x_linear4_{f32,f16,bf16}.hip; the entry points are hy3x_linear4.hip's).
//
//   W[n][k] = s[n][k / group] (q[n][k] - z[n][k / group])
//   y[t][n] = base[t][n] + sum_k W[n][k] x[t][k]        (fp32 sums, y rounded once)
//
// Weights as the MFMAs read them:
//   q  [row tile][chunk of 128 k][lane][4 dwords]: dword j of lane l holds k =
//      128 c + 32 j + 8 (l / 16) + i of the tile's row l % 16, elements i and i + 4 in
//      byte i, each as sign and magnitude of the odd number 2 q - 15 = +-(2 m + 1): element
//      i < 4 has its sign in bit 7 and m in bits 3 .. 1, i >= 4 its sign in bit 0 and m in
//      bits 6 .. 4;
//   s  [row tile][quad of chunks][row][4 GP] (GP groups in a chunk), 0 beyond d_in
//      and d_out; 2 z - 15 the same, in bytes. Without zero points z is 8 everywhere, and
//      one quad is read for all (z_tile and z_quad 0).
// Row i of tile 4 b + r is row 64 b + 4 i + r of W: the lane that has column i of four
// tiles has four outputs that follow each other.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/hy3x_moe.h"

namespace hy3x {

__host__ __device__ inline int64_t linear4_row(int64_t tile, int i) {
  return (tile >> 2) * 64 + 4 * i + (tile & 3);
}

// q as element i of its lane's dword.
__host__ __device__ inline uint32_t linear4_code(uint32_t q, int i) {
  const uint32_t below = q < 8, m = (below ? ~q : q) & 7;
  return (i < 4 ? below << 7 | m << 1 : below | m << 4) << (8 * (i & 3));
}

typedef float f4v __attribute__((ext_vector_type(4)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));

struct Linear4Call {
  const u4v *q;
  const uint16_t *s;
  const uint8_t *z;
  uint32_t z_tile, z_quad;  // bytes from a row tile's zero points to the next, from a quad's
  int d_out, d_in, tiles, chunks, quads, group;
  bool s16;  // scales are fp16
  const void *x, *base;
  void *y;
  int64_t x_stride, base_stride, y_stride;
  int T, y_type;
};

template <class X>  // x's elements: float, __half or __hip_bfloat16
void launch_linear4(const Linear4Call &c, hipStream_t st);

}  // namespace hy3x
