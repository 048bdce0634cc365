// hy3x_adapted.hip -- the steps of a forward that only a layer with adapters or
// a routing rule of its own has; all are small beside the experts.
#include "hy3x_kernels.h"

namespace hy3x {

// After hy3x_route_experts: the weights with the forward's scale, and the
// token's bit and place in each of its experts' dispatch bitmaps, as k_topk
// leaves them.
__global__ __launch_bounds__(256) void k_mark_routes(const int32_t *__restrict__ ids,
                                                     const float *__restrict__ wpre, float scale,
                                                     int T, int K, float *__restrict__ wout,
                                                     uint32_t *__restrict__ bits, int wt,
                                                     uint8_t *__restrict__ ranks) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= T * K) return;
  const int t = i / K, e = ids[i];
  wout[i] = wpre[i] * scale;
  atomicOr(&bits[(size_t)e * wt + (t >> 5)], 1u << (t & 31));
  ranks[(size_t)e * wt * 32 + t] = (uint8_t)(i % K);
}

// The shared expert's gate and up with their adapters added, raw[t][gate | up]:
// h = silu(gate) up, rounded to fp16 for the down GEMM as every gate/up kernel
// rounds it, and in fp32 in gate's place for the down adapters.
__global__ __launch_bounds__(256) void k_shared_swiglu(float *__restrict__ raw, int T,
                                                       __half *__restrict__ h16m) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= T * F) return;
  const int t = i / F, r = i % F;
  float *g = raw + (size_t)t * (2 * F) + r;
  const float gate = g[0], up = g[F];
  h16m[(size_t)t * F + perm8(r)] = swiglu_h(gate, up);
  g[0] = silu(gate) * up;
}

}  // namespace hy3x
