// hy3x_experts.hip -- routing to experts as an operator of its own
// (hy3x_route_experts): the best k of E experts for each row of logits.
//
//   s_e   = 1 / (1 + exp(-l_e))  or  exp(l_e - max) / sum exp(l_e - max)
//   key_e = s_e + bias_e in 64 bits; without a bias the logit (s grows with l)
//   group score = its best key, or the sum of its best two s_e + bias_e
//   ids = the k best keys of the best topk_group groups, ties to the lower index
//   w_j = s_ids[j] / (sum_j s_ids[j] + 1e-20) * scale
//
// The keys are 64-bit because a choice has no tolerance: two fp32 sums
// s + bias closer than their rounding errors would come out in an order that
// depends on how exp was evaluated.
//
// One wave per row; expert lane + 64 m is the lane's value m. A row's keys are
// compared as 64-bit integers that order as the doubles do, with 1 for a
// masked expert and 0 for one of a group that was dropped.
#include <hip/hip_bf16.h>
#include <math.h>

#include "../../include/hy3x_moe.h"
#include "hy3x_common.h"
#include "hy3x_error.h"

namespace hy3x {
namespace {

constexpr int ROUTE_WAVES = 4;

// Orders as the double does: larger value, larger integer; above 1 for every
// number, as the integers 0 and 1 are those of two NaNs.
__device__ __forceinline__ uint64_t ordered(double v) {
  const int64_t b = __builtin_bit_cast(int64_t, v + 0.0);  // -0 counts as 0
  return (uint64_t)(b ^ ((b >> 63) | INT64_MIN));
}
__device__ __forceinline__ double from_ordered(uint64_t k) {
  const int64_t b = (int64_t)k;
  return __builtin_bit_cast(double, b < 0 ? (b & INT64_MAX) : ~b);
}

template <class T>
struct Limits;
template <>
struct Limits<float> {
  static constexpr float max = 3.402823466e+38f;
};
template <>
struct Limits<__half> {
  static constexpr float max = 65504.0f;
};
template <>
struct Limits<__hip_bfloat16> {
  static constexpr float max = 3.38953139e+38f;  // 255 * 2^120
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__hip_bfloat16 v) { return __bfloat162float(v); }

template <class T, int V>
__global__ __launch_bounds__(64 * ROUTE_WAVES) void k_route_experts(
    const hy3x_route_spec spec, const T *__restrict__ logits, int64_t stride,
    const float *__restrict__ bias, int n_row, int32_t *__restrict__ ids, float *__restrict__ w) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int t = blockIdx.x * ROUTE_WAVES + wave;
  const int E = spec.n_expert, K = spec.k, G = spec.n_group;
  extern __shared__ double keys_l[];
  double *kl = keys_l + (size_t)wave * E;
  const bool live = t < n_row;
  const T *row = logits + (live ? t : 0) * stride;
  float l[V];
  bool on[V];
#pragma unroll
  for (int m = 0; m < V; m++) {
    const int e = lane + 64 * m;
    const float b = bias && e < E ? bias[e] : 0.0f;
    l[m] = e < E ? fminf(to_f32(row[e]), Limits<T>::max) : -INFINITY;
    on[m] = e < E && l[m] > -Limits<T>::max && b > -INFINITY && to_f32(row[e]) == to_f32(row[e]);
  }
  double s[V];
  if (spec.score == HY3X_SCORE_SIGMOID) {
#pragma unroll
    for (int m = 0; m < V; m++) s[m] = on[m] ? 1.0 / (1.0 + exp(-(double)l[m])) : 0.0;
  } else {
    float top = -INFINITY;
#pragma unroll
    for (int m = 0; m < V; m++) top = on[m] ? fmaxf(top, l[m]) : top;
    for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    double sum = 0.0;
#pragma unroll
    for (int m = 0; m < V; m++) {
      s[m] = on[m] ? exp((double)l[m] - (double)top) : 0.0;
      sum += s[m];
    }
    for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
#pragma unroll
    for (int m = 0; m < V; m++) s[m] = on[m] ? s[m] / sum : 0.0;
  }
  uint64_t key[V];
#pragma unroll
  for (int m = 0; m < V; m++) {
    const int e = lane + 64 * m;
    const double b = bias && e < E ? (double)bias[e] : 0.0;
    key[m] = e >= E ? 0 : on[m] ? ordered(bias ? s[m] + b : (double)l[m]) : 1;
    if (G > 1 && e < E)
      kl[e] = !on[m] ? __builtin_nan("") : spec.group_score == HY3X_GROUP_TOP2 ? s[m] + b
                                         : from_ordered(key[m]);
  }
  if (G > 1) {
    __syncthreads();
    const int size = E / G;
    uint64_t score = 0;
    if (lane < G) {
      double best = 0.0, second = 0.0;
      int n = 0;
      for (int j = 0; j < size; j++) {
        const double v = kl[lane * size + j];
        if (v != v) continue;
        if (n == 0 || v > best) {
          second = best;
          best = v;
        } else if (n == 1 || v > second) {
          second = v;
        }
        n++;
      }
      if (n) score = ordered(spec.group_score == HY3X_GROUP_TOP2 && n > 1 ? best + second : best);
    }
    int before = 0;  // groups ahead of this lane's
    for (int g = 0; g < G; g++) {
      const uint64_t o = __shfl(score, g, 64);
      before += o > score || (o == score && g < lane);
    }
    const uint64_t keep = __ballot(lane < G && before < spec.topk_group);
#pragma unroll
    for (int m = 0; m < V; m++) {
      const int e = lane + 64 * m;
      if (e < E && !(keep >> (e / size) & 1)) key[m] = 0;
    }
  }
  if (!live) return;
  double mine = 0.0, sum = 0.0;
  int my_e = 0;
  for (int k = 0; k < K; k++) {
    uint64_t bk = 0;
    int be = E;
    double bs = 0.0;
#pragma unroll
    for (int m = 0; m < V; m++)
      if (key[m] > bk) {
        bk = key[m];
        be = lane + 64 * m;
        bs = s[m];
      }
    for (int o = 32; o >= 1; o >>= 1) {
      const uint64_t ok = __shfl_xor(bk, o, 64);
      const int oe = __shfl_xor(be, o, 64);
      const double os = __shfl_xor(bs, o, 64);
      if (ok > bk || (ok == bk && oe < be)) {
        bk = ok;
        be = oe;
        bs = os;
      }
    }
#pragma unroll
    for (int m = 0; m < V; m++)
      if (be == lane + 64 * m) key[m] = 0;
    sum += bs;
    if (lane == k) {
      mine = bs;
      my_e = be;
    }
  }
  if (lane < K) {
    const double v = spec.renorm ? mine / (sum + 1e-20) : mine;
    ids[(int64_t)t * K + lane] = my_e;
    w[(int64_t)t * K + lane] = (float)(v * (double)spec.scale);
  }
}

template <class T>
void launch(const hy3x_route_spec &spec, const void *logits, int64_t stride, const float *bias,
            int n_row, int32_t *ids, float *w, hipStream_t st) {
  const dim3 grid((n_row + ROUTE_WAVES - 1) / ROUTE_WAVES), block(64 * ROUTE_WAVES);
  const size_t lds = spec.n_group > 1 ? (size_t)ROUTE_WAVES * spec.n_expert * sizeof(double) : 0;
  const T *lg = (const T *)logits;
#define HY3X_ROUTE(V)                                                                   \
  if (spec.n_expert <= 64 * V) {                                                        \
    k_route_experts<T, V><<<grid, block, lds, st>>>(spec, lg, stride, bias, n_row, ids, w); \
    return;                                                                             \
  }
  HY3X_ROUTE(1)
  HY3X_ROUTE(2)
  HY3X_ROUTE(3)
  HY3X_ROUTE(4)
  HY3X_ROUTE(8)
  HY3X_ROUTE(16)
#undef HY3X_ROUTE
}

}  // namespace

int check_route_spec(const hy3x_route_spec *s) {
  if (!s) return op_fail(HY3X_E_ARG, "NULL routing spec");
  if (s->n_expert < 1 || s->n_expert > HY3X_ROUTE_MAX_EXPERT)
    return op_fail(HY3X_E_ARG, "n_expert %d outside [1,%d]", s->n_expert, HY3X_ROUTE_MAX_EXPERT);
  if (s->n_group < 1 || s->n_group > HY3X_ROUTE_MAX_GROUP || s->n_expert % s->n_group)
    return op_fail(HY3X_E_ARG, "n_group %d: outside [1,%d] or no divisor of n_expert %d",
                   s->n_group, HY3X_ROUTE_MAX_GROUP, s->n_expert);
  if (s->topk_group < 1 || s->topk_group > s->n_group)
    return op_fail(HY3X_E_ARG, "topk_group %d outside [1,%d]", s->topk_group, s->n_group);
  const int reach = s->topk_group * (s->n_expert / s->n_group);
  if (s->k < 1 || s->k > HY3X_ROUTE_MAX_K || s->k > reach)
    return op_fail(HY3X_E_ARG, "k %d outside [1,%d], or above the %d experts of the kept groups",
                   s->k, HY3X_ROUTE_MAX_K, reach);
  if (s->score != HY3X_SCORE_SIGMOID && s->score != HY3X_SCORE_SOFTMAX)
    return op_fail(HY3X_E_ARG, "score %d unknown", s->score);
  if (s->group_score != HY3X_GROUP_MAX && s->group_score != HY3X_GROUP_TOP2)
    return op_fail(HY3X_E_ARG, "group_score %d unknown", s->group_score);
  return HY3X_OK;
}

}  // namespace hy3x

using namespace hy3x;

extern "C" int hy3x_route_experts(const hy3x_route_spec *spec, const void *logits, int type,
                                  int64_t row_stride, const float *bias, int T, int32_t *ids,
                                  float *w, void *stream) {
  const int rc = check_route_spec(spec);
  if (rc) return rc;
  if (type != HY3X_F32 && type != HY3X_F16 && type != HY3X_BF16)
    return op_fail(HY3X_E_ARG, "logits type %d unknown", type);
  if (T < 0 || T > HY3X_ROUTE_MAX_TOKENS)
    return op_fail(HY3X_E_ARG, "T=%d outside [0,%d]", T, HY3X_ROUTE_MAX_TOKENS);
  if (row_stride < spec->n_expert)
    return op_fail(HY3X_E_ARG, "row_stride %lld below n_expert %d", (long long)row_stride,
                   spec->n_expert);
  if (T == 0) return HY3X_OK;
  if (!logits || !ids || !w) return op_fail(HY3X_E_ARG, "NULL logits, ids or w");
  const size_t size = type == HY3X_F32 ? 4 : 2;
  if ((uintptr_t)logits % size || (uintptr_t)bias % 4 || (uintptr_t)ids % 4 || (uintptr_t)w % 4)
    return op_fail(HY3X_E_ARG, "a pointer is not aligned to its elements");
  hipStream_t st = (hipStream_t)stream;
  if (type == HY3X_F32)
    launch<float>(*spec, logits, row_stride, bias, T, ids, w, st);
  else if (type == HY3X_F16)
    launch<__half>(*spec, logits, row_stride, bias, T, ids, w, st);
  else
    launch<__hip_bfloat16>(*spec, logits, row_stride, bias, T, ids, w, st);
  OP_HIP_TRY(hipGetLastError());
  return HY3X_OK;
}
