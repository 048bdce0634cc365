// hy3x_linear4.h -- products of 4-bit weights: their layout, and a checked call of
// their kernels (hy3x_linear4_kernels.h, instances by x's type in
// hy3x_linear4_{f32,f16,bf16}.hip; the entry points are hy3x_linear4.hip's).
//
//   W[n][k] = s[n][k / group] (q[n][k] - z[n][k / group])
//   y[t][n] = base[t][n] + sum_k W[n][k] x[t][k]        (fp32 sums, y rounded once)
//
// Weights as the MFMAs read them:
//   q  [row tile][chunk of 128 k][lane][4 dwords]: dword j of lane l holds k =
//      128 c + 32 j + 8 (l / 16) + i of the tile's row l % 16, element i < 4 in the
//      low half of byte i, i >= 4 in the high half of byte i - 4;
//   s  [row tile][quad of chunks][row][4 GP] (GP groups in a chunk), 0 beyond d_in
//      and d_out; z the same, in bytes. Without zero points all are 8, and one quad
//      is read for all (z_tile and z_quad 0).
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
