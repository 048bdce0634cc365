// hy3x_logprobs.hip -- log-probabilities of given tokens, entropy and the most
// probable tokens of rows of logits (hy3x_logprobs):
//
//   m = max l,  S = sum_v e^(l_v - m),  log p_v = (l_v - m) - log S
//   H = log S - (sum_v (l_v - m) e^(l_v - m)) / S
//
// Both terms of H are at least 0, so it keeps its precision where one token has
// nearly all of the mass.
#include <hip/hip_bf16.h>

#include "../../include/hy3x_moe.h"
#include "hy3x_common.h"
#include "hy3x_error.h"
#include "hy3x_ops.h"

namespace hy3x {
namespace {

__device__ __forceinline__ float elem(float v) { return v; }
__device__ __forceinline__ float elem(__half v) { return __half2float(v); }
__device__ __forceinline__ float elem(__hip_bfloat16 v) { return __bfloat162float(v); }
template <class X>
struct Range;
template <>
struct Range<float> {
  static constexpr float HIGH = 3.4028234663852886e38f;
};
template <>
struct Range<__half> {
  static constexpr float HIGH = 65504.0f;
};
template <>
struct Range<__hip_bfloat16> {
  static constexpr float HIGH = 3.3895313892515355e38f;
};

struct Call {
  const void *logits;
  int64_t stride;
  int V, T, top;
  const int32_t *tokens;
  float *logp, *entropy, *top_logp;
  int32_t *top_ids;
};

// A logit as it counts: masked ones (NaN, -inf, the type's lowest) are -inf, +inf
// the largest finite value.
template <class X>
__device__ __forceinline__ float logit(const X *row, int v) {
  const float l = elem(row[v]);
  return l > -Range<X>::HIGH ? fminf(l, Range<X>::HIGH) : -INFINITY;
}

// One block per row.
template <class X>
__global__ __launch_bounds__(256) void k_logprobs(Call c) {
  __shared__ float red[4];
  __shared__ double redd[4][2];
  __shared__ float bestv[4];
  __shared__ int besti[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int64_t t = blockIdx.x; t < c.T; t += gridDim.x) {
    const X *row = (const X *)c.logits + t * c.stride;
    float m = -INFINITY;
    for (int v = tid; v < c.V; v += 256) m = fmaxf(m, logit(row, v));
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    if (lane == 0) red[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    double S = 0.0, E = 0.0;
    for (int v = tid; v < c.V; v += 256) {
      const float l = logit(row, v);
      if (l > -INFINITY) {
        const double d = (double)l - m, e = exp(d);
        S += e;
        E += e * d;
      }
    }
    for (int o = 32; o; o >>= 1) {
      S += __shfl_xor(S, o, 64);
      E += __shfl_xor(E, o, 64);
    }
    if (lane == 0) redd[wave][0] = S, redd[wave][1] = E;
    __syncthreads();
    S = redd[0][0] + redd[1][0] + redd[2][0] + redd[3][0];
    E = redd[0][1] + redd[1][1] + redd[2][1] + redd[3][1];
    const double lse = log(S);
    auto logp = [&](float l) { return l > -INFINITY ? (float)(((double)l - m) - lse) : -INFINITY; };
    if (tid == 0) {
      const int token = c.tokens[t];
      c.logp[t] = token >= 0 && token < c.V ? logp(logit(row, token)) : 0.0f;
      if (c.entropy) c.entropy[t] = m > -INFINITY ? (float)(lse - E / S) : 0.0f;
    }
    float lastv = INFINITY;
    int lasti = -1;
    for (int k = 0; k < c.top; k++) {
      float bv = -INFINITY;
      int bi = 0x7fffffff;
      for (int v = tid; v < c.V; v += 256) {
        const float l = logit(row, v);
        if ((l < lastv || (l == lastv && v > lasti)) && (l > bv || (l == bv && v < bi))) {
          bv = l;
          bi = v;
        }
      }
      for (int o = 32; o; o >>= 1) {
        const float ov = __shfl_xor(bv, o, 64);
        const int oi = __shfl_xor(bi, o, 64);
        if (ov > bv || (ov == bv && oi < bi)) bv = ov, bi = oi;
      }
      __syncthreads();
      if (lane == 0) bestv[wave] = bv, besti[wave] = bi;
      __syncthreads();
      for (int w = 0; w < 4; w++)
        if (bestv[w] > bv || (bestv[w] == bv && besti[w] < bi)) bv = bestv[w], bi = besti[w];
      if (tid == 0) {
        c.top_ids[t * c.top + k] = bi;
        c.top_logp[t * c.top + k] = logp(bv);
      }
      lastv = bv;
      lasti = bi;
    }
    __syncthreads();
  }
}

template <class X>
void launch(const Call &c, hipStream_t st) {
  k_logprobs<X><<<c.T < 65536 ? c.T : 65536, 256, 0, st>>>(c);
}

}  // namespace
}  // namespace hy3x

using namespace hy3x;

extern "C" {

int64_t hy3x_logprobs_workspace(int T, int V, int n_top) {
  if (T < 0 || T > HY3X_LOGPROBS_MAX_TOKENS || V < 1 || V > HY3X_LOGPROBS_MAX_VOCAB ||
      n_top < 0 || n_top > HY3X_LOGPROBS_MAX_TOP || n_top > V)
    return op_fail(HY3X_E_ARG, "T=%d, V=%d or n_top=%d out of range", T, V, n_top);
  return 0;
}

int hy3x_logprobs(const void *logits, int type, int64_t row_stride, int V, const int32_t *tokens,
                  int T, int n_top, float *logp, float *entropy, int32_t *top_ids, float *top_logp,
                  void *workspace, int64_t workspace_bytes, void *stream) {
  if (type < HY3X_F32 || type > HY3X_BF16)
    return op_fail(HY3X_E_ARG, "logits type %d is none of HY3X_F32, HY3X_F16, HY3X_BF16", type);
  if (V < 1 || V > HY3X_LOGPROBS_MAX_VOCAB)
    return op_fail(HY3X_E_ARG, "V=%d outside [1,%d]", V, HY3X_LOGPROBS_MAX_VOCAB);
  if (T < 0 || T > HY3X_LOGPROBS_MAX_TOKENS)
    return op_fail(HY3X_E_ARG, "T=%d outside [0,%d]", T, HY3X_LOGPROBS_MAX_TOKENS);
  if (n_top < 0 || n_top > HY3X_LOGPROBS_MAX_TOP || n_top > V)
    return op_fail(HY3X_E_ARG, "n_top=%d outside [0,%d] or above V", n_top,
                   HY3X_LOGPROBS_MAX_TOP);
  if (row_stride < V || row_stride > (int64_t)1 << 32)
    return op_fail(HY3X_E_ARG, "row stride %lld below the row's length, or above 2^32",
                   (long long)row_stride);
  if (T == 0) return HY3X_OK;
  if (!logits || !tokens || !logp) return op_fail(HY3X_E_ARG, "NULL logits, tokens or logp");
  if (n_top && (!top_ids || !top_logp))
    return op_fail(HY3X_E_ARG, "n_top=%d without top_ids and top_logp", n_top);
  const int64_t room = hy3x_logprobs_workspace(T, V, n_top);
  if (room && (!workspace || workspace_bytes < room))
    return op_fail(HY3X_E_ARG, "a workspace of %lld bytes is needed", (long long)room);
  const int64_t es = type == HY3X_F32 ? 4 : 2;
  if ((uintptr_t)logits % es || (uintptr_t)tokens % 4 || (uintptr_t)logp % 4 ||
      (uintptr_t)entropy % 4 || (n_top && ((uintptr_t)top_ids % 4 || (uintptr_t)top_logp % 4)) ||
      (room && (uintptr_t)workspace % 16))
    return op_fail(HY3X_E_ARG, "a pointer is not aligned to its elements");
  const struct {
    const char *name;
    const void *p;
    int64_t bytes;
    bool written;
  } mem[] = {{"logits", logits, ((T - 1) * row_stride + V) * es, false},
             {"tokens", tokens, (int64_t)T * 4, false},
             {"logp", logp, (int64_t)T * 4, true},
             {"entropy", entropy, entropy ? (int64_t)T * 4 : 0, true},
             {"top_ids", top_ids, (int64_t)T * n_top * 4, true},
             {"top_logp", top_logp, (int64_t)T * n_top * 4, true},
             {"workspace", workspace, room, true}};
  for (const auto &a : mem)
    for (const auto &b : mem)
      if (&a < &b && (a.written || b.written) && a.bytes && b.bytes &&
          (uintptr_t)a.p < (uintptr_t)b.p + (uintptr_t)b.bytes &&
          (uintptr_t)b.p < (uintptr_t)a.p + (uintptr_t)a.bytes)
        return op_fail(HY3X_E_ARG, "%s overlaps %s", a.name, b.name);
  Call c;
  c.logits = logits;
  c.stride = row_stride;
  c.V = V;
  c.T = T;
  c.top = n_top;
  c.tokens = tokens;
  c.logp = logp;
  c.entropy = entropy;
  c.top_logp = top_logp;
  c.top_ids = top_ids;
  const hipStream_t st = (hipStream_t)stream;
  if (type == HY3X_F32) launch<float>(c, st);
  else if (type == HY3X_F16) launch<__half>(c, st);
  else launch<__hip_bfloat16>(c, st);
  OP_HIP_TRY(hipGetLastError());
  return HY3X_OK;
}

}  // extern "C"
