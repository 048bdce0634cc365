// hy3x_experts.hip -- routing to experts as an operator of its own
// (hy3x_route_experts): the best k of E experts for each row of logits.
//
//   s_e   = 1 / (1 + exp(-l_e))  or  exp(l_e - max) / sum exp(l_e - max)
//   key_e = s_e + bias_e in 64 bits; without a bias the logit (s grows with l)
//   group score = its best key, or the sum of its best two s_e + bias_e
//   ids = the k best keys of the best topk_group groups, ties to the lower index
//   w_j = s_ids[j] / (sum_j s_ids[j] + 1e-20) * scale
//
// One wave per row. With G > 1 groups a group has its own LG = 2^n lanes, so
// that its score is a reduction inside them; each lane holds V consecutive
// experts, and lanes ascend with the experts: the first lane's first slot that
// holds a maximum is the lowest index of a tie.
//
// A choice has no tolerance: two keys s + bias closer than the rounding errors
// of an fp32 evaluation come out in an order that depends on how exp was
// evaluated. So keys are fp32 first (as integers that order as the floats do,
// k + 1 rounds of a wave-wide maximum), and the row is decided there if each
// chosen key lies further from the next one than both can be wrong (margin()).
// Otherwise the candidates, every key within the margin of the k-th, get
// 64-bit keys, a lane each, and are ranked by counting (experts of the same
// logit and bias need none: they are equal). A row with more candidates than
// lanes is decided by 64-bit keys throughout (choose64). Groups whose scores are
// that close at the border, or are sums that cancel, are scored in 64 bits
// (groups64). Without a bias the keys are the logits, which are exact: no
// margin, and ties are ties.
//
// What bounds it (us of the kernel, MI355X): few rows the load and k rounds that
// wait for each other (one row of 192: 2.8 us; 512: 4.2, its end a row with
// candidates); 4096 rows, 4 a SIMD, still this latency: of 8.2 us for 256 experts in
// 8 groups the 512 vector instructions a row are 3.4, the others the groups' shuffles
// and lane reads, the rounds and the rows with candidates; 16383 rows of 251 mostly
// vector instructions (401 a row, 10.7 us of 15.9), not bytes (8 MB). With 64-bit
// keys for every row these were 8.2, 10.2, 22.8 and 48.7. A wave per row in blocks
// of 4 waves: blocks of 1, 8 or 16 are no faster; waves that take rows in turn, the
// next row's loads in flight, were slower (10.4 against 9.3 at 4096 rows, 22.4
// against 18.8 at 16383). 64 registers, 8 waves a SIMD, where lanes hold 2 to 4
// experts: 16.5 us against 17.0 with 72.
#include <hip/hip_bf16.h>
#include <math.h>

#include "../../include/hy3x_moe.h"
#include "hy3x_common.h"
#include "hy3x_error.h"
#include "hy3x_ops.h"

namespace hy3x {
namespace {

constexpr int ROUTE_WAVES = 4;

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

// Keys as integers that order as the numbers do (-0 as 0). MASKED, for a
// masked expert, lies below every number, GONE (taken, or of a dropped group)
// below that.
template <class U>
constexpr U GONE = 0;
template <class U>
constexpr U MASKED = 1;
__device__ __forceinline__ uint32_t ordered(float v) {
  const int32_t b = __builtin_bit_cast(int32_t, v + 0.0f);
  return (uint32_t)(b ^ ((b >> 31) | INT32_MIN));
}
__device__ __forceinline__ uint64_t ordered(double v) {
  const int64_t b = __builtin_bit_cast(int64_t, v + 0.0);
  return (uint64_t)(b ^ ((b >> 63) | INT64_MIN));
}
__device__ __forceinline__ float number(uint32_t k) {
  const int32_t b = (int32_t)k;
  return __builtin_bit_cast(float, b < 0 ? (b & INT32_MAX) : ~b);
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = max(v, (uint32_t)dppi<DPP_XOR1>((int)v));
  v = max(v, (uint32_t)dppi<DPP_XOR2>((int)v));
  v = max(v, (uint32_t)dppi<DPP_HALF_MIRROR>((int)v));
  v = max(v, (uint32_t)dppi<DPP_MIRROR>((int)v));
  // 0 where a row takes no broadcast: one instruction with the maximum
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, DPP_BCAST15, 0xA, 0xF, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, DPP_BCAST31, 0xC, 0xF, false));
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// Lane i's value, i the same in all lanes.
__device__ __forceinline__ uint64_t lane_of(uint64_t v, int i) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, i);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), i);
  return (uint64_t)hi << 32 | lo;
}

// One row as its wave reads it.
template <class T>
struct Row {
  const T *logits;
  const float *bias;
  int softmax;
  float top;  // softmax: the largest logit that is not masked

  __device__ __forceinline__ float logit(int e) const {
    return fminf(to_f32(logits[e]), Limits<T>::max);  // a NaN: see masked()
  }
  __device__ __forceinline__ bool masked(int e) const {
    return !(to_f32(logits[e]) > -Limits<T>::max) || (bias && !(bias[e] > -INFINITY));
  }
  // the score of logit l, in 64 bits; sum: the softmax's
  __device__ __forceinline__ double score64(float l, double sum) const {
    const double x = softmax ? (double)l - (double)top : -(double)l;
    const double e = exp(x);
    return softmax ? e / sum : 1.0 / (1.0 + e);
  }
  __device__ __forceinline__ uint64_t key64(int e, double sum) const {
    if (masked(e)) return MASKED<uint64_t>;
    return ordered(bias ? score64(logit(e), sum) + (double)bias[e] : (double)logit(e));
  }
};

// The lanes of groups: LG = 2^shift lanes each, `size` experts, V per lane.
struct Lanes {
  int size, shift, lane, group, first, n;  // this lane: experts first .. first + n - 1
  __device__ __forceinline__ Lanes(const hy3x_route_spec &s, int v) {
    lane = threadIdx.x & 63;
    size = s.n_expert / s.n_group;
    shift = 31 - __builtin_clz(64 / s.n_group);
    group = lane >> shift;
    const int at = (lane & ((1 << shift) - 1)) * v;
    first = group * size + at;
    n = group < s.n_group ? min(max(size - at, 0), v) : 0;
  }
};

// This lane's logits one after another, NaN for masked ones and slots without an
// expert: l as the kernel holds it, moved up (no indexed registers), or, of many,
// read again.
template <class T, int V>
struct Each {
  static constexpr bool HELD = V <= 8;
  float c[HELD ? V : 1];
  const Row<T> &row;
  const Lanes &L;
  int j = 0;
  __device__ __forceinline__ Each(const Row<T> &r, const Lanes &lanes, const float (&l)[V])
      : row(r), L(lanes) {
#pragma unroll
    for (int i = 0; i < (HELD ? V : 0); i++) c[i] = l[i];
  }
  __device__ __forceinline__ float next() {
    if constexpr (HELD) {
      const float x = c[0];
#pragma unroll
      for (int i = 0; i + 1 < V; i++) c[i] = c[i + 1];
      return x;
    } else {
      const int e = L.first + j;
      return j++ < L.n && !row.masked(e) ? row.logit(e) : NAN;
    }
  }
};

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

template <class T, int V>
__device__ __forceinline__ double sum64(const Row<T> &row, const Lanes &L, const float (&l)[V]) {
  if (!row.softmax) return 0.0;
  double sum = 0.0;
  Each<T, V> each(row, L, l);
#pragma unroll 1  // one copy of exp in the code
  for (int j = 0; j < V; j++) {
    const float x = each.next();
    if (x == x) sum += exp((double)x - (double)row.top);
  }
  return wave_sum64(sum);
}

// How many groups come ahead of this lane's, by 64-bit scores.
template <class T, int V>
__device__ __forceinline__ int groups64(const hy3x_route_spec &spec, const Row<T> &row,
                                        const Lanes &L, const float (&l)[V]) {
  const bool top2 = spec.group_score == HY3X_GROUP_TOP2;
  const double sum = sum64(row, L, l);
  double b0 = -INFINITY, b1 = -INFINITY;
  int live = 0;
  Each<T, V> each(row, L, l);
#pragma unroll 1
  for (int j = 0; j < V; j++) {
    const float x = each.next();
    if (x != x) continue;
    const double s = !top2 && !row.bias
                         ? (double)x
                         : row.score64(x, sum) + (row.bias ? (double)row.bias[L.first + j] : 0.0);
    b1 = fmax(b1, fmin(b0, s));
    b0 = fmax(b0, s);
    live++;
  }
  for (int o = 1; o < 1 << L.shift; o <<= 1) {
    const double o0 = __shfl_xor(b0, o, 64), o1 = __shfl_xor(b1, o, 64);
    b1 = fmax(fmax(b1, o1), fmin(b0, o0));
    b0 = fmax(b0, o0);
    live += __shfl_xor(live, o, 64);
  }
  const uint64_t best = !live ? GONE<uint64_t> : ordered(top2 && live > 1 ? b0 + b1 : b0);
  int before = 0;
  for (int g = 0; g < spec.n_group; g++) {
    const uint64_t o = lane_of(best, g << L.shift);
    before += o > best || (o == best && g < L.group);
  }
  return before;
}

// The choice by 64-bit keys alone, lane k < K returning the k-th expert: for
// rows with more candidates than lanes. It forms every key again in each round
// and keeps none.
template <class T, int V>
__device__ __forceinline__ int choose64(const hy3x_route_spec &spec, const Row<T> &row,
                                        const Lanes &L, const float (&l)[V]) {
  const double sum = sum64(row, L, l);
  const bool stays = spec.n_group == 1 || groups64(spec, row, L, l) < spec.topk_group;
  uint32_t taken = 0;
  int mine = 0;
  for (int k = 0; k < spec.k; k++) {
    uint64_t bk = GONE<uint64_t>;
    int be = INT32_MAX;
    for (int j = 0; stays && j < L.n; j++) {
      const uint64_t key = taken >> j & 1 ? GONE<uint64_t> : row.key64(L.first + j, sum);
      if (key > bk) {
        bk = key;
        be = L.first + j;
      }
    }
    for (int o = 32; o >= 1; o >>= 1) {
      const uint64_t ok = __shfl_xor(bk, o, 64);
      const int oe = __shfl_xor(be, o, 64);
      if (ok > bk || (ok == bk && oe < be)) {
        bk = ok;
        be = oe;
      }
    }
    if (be >= L.first && be < L.first + L.n) taken |= 1u << (be - L.first);
    if (L.lane == k) mine = be;
  }
  return mine;
}

// How far two fp32 keys s + bias near `key` can be from their 64-bit order: the
// sum's rounding (2^-24 of it each) and the scores' errors, with `most` the
// largest score. exp(x) by v_exp_f32 is off by (1.5 |x| + 4) 2^-24 of itself (the
// product x log2(e) and 2 ulp), which |x| exp(-|x|) <= 0.37 bounds: sigmoid, with
// 1 + e and rcp (1 ulp), is off by less than 2^-21; softmax, with l - top and the
// up to 32 + 6 roundings of its sum, by less than 2^-18 of `most`. Two keys, and
// doubled once more. The last term: scores that underflow.
__device__ __forceinline__ float margin(bool softmax, float most, float key) {
  return (softmax ? 0x1p-16f : 0x1p-19f) * most + 0x1p-22f * fabsf(key) + 0x1p-120f;
}

// Weights of the chosen experts (lane k: the k-th) and the row's outputs.
// ls: the lane's logits; sum: the softmax's; live, l: the expert is not masked, its
// logit. fp32, except where a score lies near or below its normal numbers.
template <class T, int V>
__device__ __forceinline__ void finish(const hy3x_route_spec &spec, const Row<T> &row,
                                       const Lanes &L, const float (&ls)[V], float sum,
                                       int mine, bool live, float l, int64_t t, int32_t *ids,
                                       float *w) {
  static_assert(HY3X_ROUTE_MAX_K <= 16, "a row of 16 lanes holds the chosen");
  const int lane = L.lane, K = spec.k;
  live = live && lane < K;
  const float x = live ? l - (row.softmax ? row.top : 0.0f) : 0.0f;
  float v = 0.0f;
  if (__ballot(x < -80.0f)) {
    const double s64 = sum64(row, L, ls);
    double s = live ? row.score64(l, s64) : 0.0;
    if (spec.renorm) s /= wave_sum64(s) + 1e-20;
    v = (float)(s * (double)spec.scale);
  } else {
    // softmax: e / sum, or e / (sum of the chosen e + 1e-20 sum)
    const float s = !live ? 0.0f : row.softmax ? expf(x) : 1.0f / (1.0f + expf(-x));
    const float all = row.softmax ? sum : 1.0f;
    const float by = spec.renorm ? row16_sum(s) + 1e-20f * all : all;
    if (live) v = s / by * spec.scale;
  }
  if (lane < K) {
    ids[t * K + lane] = mine;
    w[t * K + lane] = v;
  }
}

template <class T, int V>
__global__ __launch_bounds__(64 * ROUTE_WAVES, V > 1 && V <= 4 ? 8 : 1) void k_route_experts(
    const hy3x_route_spec spec, const T *__restrict__ logits, int64_t stride,
    const float *__restrict__ bias, int n_row, int32_t *__restrict__ ids, float *__restrict__ w) {
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * ROUTE_WAVES + (threadIdx.x >> 6);
  if (t >= n_row) return;  // whole waves; no barriers below
  const int K = spec.k, G = spec.n_group;
  const bool softmax = spec.score == HY3X_SCORE_SOFTMAX, top2 = spec.group_score == HY3X_GROUP_TOP2;
  Row<T> row{logits + t * stride, bias, softmax, 0.0f};
  const Lanes L(spec, V);
  float l[V], b[V];
  if (L.size % V == 0) {  // whole lanes: V elements at once
    const int e = min(L.first, spec.n_expert - V);
    T lv[V];
    __builtin_memcpy(lv, row.logits + e, sizeof(lv));
    if (bias) __builtin_memcpy(b, bias + e, sizeof(b));
#pragma unroll
    for (int j = 0; j < V; j++) l[j] = to_f32(lv[j]);
  } else {
    int e[V];
#pragma unroll
    for (int j = 0; j < V; j++) e[j] = min(L.first + j, spec.n_expert - 1);
#pragma unroll
    for (int j = 0; j < V; j++) l[j] = to_f32(row.logits[e[j]]);
    if (bias)
#pragma unroll
      for (int j = 0; j < V; j++) b[j] = bias[e[j]];
  }
  if (!bias)
#pragma unroll
    for (int j = 0; j < V; j++) b[j] = 0.0f;
  uint32_t key[V];
  float sum = 1.0f, most = 1.0f;  // the softmax's sum; no score is larger than `most`
  {
    float s[V];
    bool on[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
      on[j] = j < L.n && l[j] > -Limits<T>::max && b[j] > -INFINITY;
      l[j] = on[j] ? fminf(l[j], Limits<T>::max) : NAN;
    }
    if (softmax) {
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < V; j++) top = on[j] ? max(top, ordered(l[j])) : top;
      row.top = number(wave_max(top));
      sum = 0.0f;
#pragma unroll
      for (int j = 0; j < V; j++) {
        s[j] = on[j] ? __expf(l[j] - row.top) : 0.0f;
        sum += s[j];
      }
      sum = wave_total(sum);
      most = __builtin_amdgcn_rcpf(sum);
#pragma unroll
      for (int j = 0; j < V; j++) s[j] *= most;
    } else if (bias || (G > 1 && top2)) {
#pragma unroll
      for (int j = 0; j < V; j++) s[j] = __builtin_amdgcn_rcpf(1.0f + __expf(-l[j]));
    }
#pragma unroll
    for (int j = 0; j < V; j++)
      key[j] = j >= L.n ? GONE<uint32_t>
               : !on[j] ? MASKED<uint32_t>
                        : ordered(bias ? s[j] + b[j] : l[j]);
    if (G > 1) {
      // the group's best key, or its best two s + bias, in each of its lanes
      uint32_t a0 = GONE<uint32_t>, a1 = GONE<uint32_t>;
#pragma unroll
      for (int j = 0; j < V; j++) {
        const uint32_t k = !on[j] ? GONE<uint32_t> : top2 ? ordered(s[j] + b[j]) : key[j];
        a1 = max(a1, min(a0, k));
        a0 = max(a0, k);
      }
      for (int o = 1; o < 1 << L.shift; o <<= 1) {
        const uint32_t o0 = __shfl_xor(a0, o, 64), o1 = __shfl_xor(a1, o, 64);
        a1 = max(max(a1, o1), min(a0, o0));
        a0 = max(a0, o0);
      }
      // A sum rounds as its two keys do, so margin() of the sum covers it unless they
      // cancel: a steering bias of +1e6 and one of -1e6 leave a sum of 1 off by 0.1.
      bool cancel = false;
      if (top2 && a1 > MASKED<uint32_t>) {
        const float k0 = number(a0), k1 = number(a1), both = k0 + k1;
        cancel = fabsf(k0) + fabsf(k1) > fabsf(both) + most;
        a0 = ordered(both);
      }
      int before = 0;  // groups ahead of this lane's
      for (int g = 0; g < G; g++) {
        const uint32_t o = (uint32_t)__builtin_amdgcn_readlane((int)a0, g << L.shift);
        before += o > a0 || (o == a0 && g < L.group);
      }
      if (spec.topk_group < G && (bias || top2)) {
        auto at = [&](int place) {  // the score of the group at that place
          return (uint32_t)__builtin_amdgcn_readlane(
              (int)a0, __builtin_ctzll(__ballot(L.group < G && before == place)));
        };
        const uint32_t in = at(spec.topk_group - 1), out = at(spec.topk_group);
        if (__ballot(cancel) ||
            (out > MASKED<uint32_t> &&
             !(number(in) - number(out) > 2.0f * margin(softmax, most, number(in)))))
          before = groups64(spec, row, L, l);
      }
      const bool stays = L.group < G && before < spec.topk_group;
#pragma unroll
      for (int j = 0; j < V; j++) key[j] = stays ? key[j] : GONE<uint32_t>;
    }
  }

  // rounds of the largest key left: lane k receives the k-th and its expert
  uint32_t my_key = GONE<uint32_t>;
  int mine = 0;
  float my_l = 0.0f;  // its logit
  auto round = [&](int k) {
    uint32_t v = key[0];
#pragma unroll
    for (int j = 1; j < V; j++) v = max(v, key[j]);
    const uint32_t M = wave_max(v);
    const int wl = __builtin_ctzll(__ballot(v == M));
    int slot = 0;
#pragma unroll
    for (int j = V - 1; j > 0; j--) slot = key[j] == M ? j : slot;
    slot = key[0] == M ? 0 : slot;
#pragma unroll
    for (int j = 0; j < V; j++) key[j] = lane == wl && slot == j ? GONE<uint32_t> : key[j];
    const int e = __builtin_amdgcn_readlane(L.first + slot, wl);
    if (lane == k) {
      my_key = M;
      mine = e;
    }
    return M;
  };
  uint32_t kth = GONE<uint32_t>;   // the last chosen
  uint32_t head = GONE<uint32_t>;  // this lane's largest left
  if constexpr (V <= 8) {
    // each lane's keys sorted once: a round is the maximum of the heads, and
    // its lane's keys move up; the expert is found from the unsorted keys
    uint32_t q[V];
#pragma unroll
    for (int j = 0; j < V; j++) q[j] = key[j];
#pragma unroll
    for (int i = 0; i < V; i++)  // odd-even transposition, descending
#pragma unroll
      for (int j = i & 1; j + 1 < V; j += 2) {
        const uint32_t x = q[j], y = q[j + 1];
        q[j] = max(x, y);
        q[j + 1] = min(x, y);
      }
    int where = 0;  // the lane, and 64 times how many equal keys it gave before
    int last = -1, again = 0;
    for (int k = 0; k < K; k++) {
      const uint32_t M = wave_max(q[0]);
      const int wl = __builtin_ctzll(__ballot(q[0] == M));
#pragma unroll
      for (int j = 0; j < V; j++) {
        const uint32_t own = q[j], up = j + 1 < V ? q[j + 1] : GONE<uint32_t>;
        q[j] = lane == wl ? up : own;
      }
      again = M == kth && wl == last ? again + 64 : 0;
      kth = M;
      last = wl;
      if (lane == k) {
        my_key = M;
        where = wl + again;
      }
    }
    const int from = where & 63, nth = where >> 6;
    head = q[0];
    int seen = 0, slot = 0;
#pragma unroll
    for (int j = 0; j < V; j++) {
      const bool hit = (uint32_t)__shfl((int)key[j], from, 64) == my_key;
      const float lj = __shfl(l[j], from, 64);
      my_l = hit && seen == nth ? lj : my_l;
      slot = hit && seen == nth ? j : slot;
      seen += hit;
    }
    mine = __shfl(L.first, from, 64) + slot;
  } else {
    for (int k = 0; k < K; k++) kth = round(k);
    my_l = row.logit(mine);
#pragma unroll
    for (int j = 0; j < V; j++) head = max(head, key[j]);
  }
  bool live = my_key > MASKED<uint32_t>;
  if (bias) {
    // close to the next chosen, or left over and close to the last
    const float edge = margin(softmax, most, number(kth));
    const uint32_t next = __shfl(my_key, lane + 1, 64);
    bool close = lane < K - 1 && next > MASKED<uint32_t> &&
                 number(my_key) - number(next) <= margin(softmax, most, number(my_key));
    auto left = [&](uint32_t k) {
      return k > MASKED<uint32_t> && !(number(kth) - number(k) > edge);
    };
    if (__ballot(close || left(head))) {
      if constexpr (V <= 8)
        for (int k = 0; k < K; k++) {
          const int e = __builtin_amdgcn_readlane(mine, k);
#pragma unroll
          for (int j = 0; j < V; j++)
            key[j] = e == L.first + j && j < L.n ? GONE<uint32_t> : key[j];
        }
      // experts of the same logit and bias are equal in any arithmetic
      if constexpr (V <= 8)
#pragma unroll
        for (int j = 0; j < V; j++) b[j] = bias[min(L.first + j, spec.n_expert - 1)];
      const float lm = my_l, bm = bias[mine];
      const float ln = __shfl(lm, lane + 1, 64), bn = __shfl(bm, lane + 1, 64);
      const float lk = __shfl(lm, K - 1, 64), bk = __shfl(bm, K - 1, 64);
      bool any = close && (lm != ln || bm != bn);
#pragma unroll
      for (int j = 0; j < V; j++)
        if (left(key[j])) any |= l[j] != lk || (V <= 8 ? b[j] : bias[L.first + j]) != bk;
      if (__ballot(any)) {
        // candidates: the k chosen and all that lies close to the last of them
        int n = K;
        for (uint32_t M; n < 64 && (M = round(n)) > MASKED<uint32_t> &&
                         !(number(kth) - number(M) > edge);)
          n++;
        if (n == 64) {
          mine = choose64(spec, row, L, l);
        } else {
          const double s64 = sum64(row, L, l);
          const uint64_t k64 = lane < n ? row.key64(mine, s64) : GONE<uint64_t>;
          int rank = lane < n ? 0 : lane;
          for (int i = 0; i < n; i++) {
            const uint64_t o = lane_of(k64, i);
            const int oe = __builtin_amdgcn_readlane(mine, i);
            if (lane < n) rank += o > k64 || (o == k64 && oe < mine);
          }
          mine = __builtin_amdgcn_ds_permute(4 * rank, mine);
        }
        my_l = row.logit(mine);
        live = !row.masked(mine);
      }
    }
  }
  finish(spec, row, L, l, sum, mine, live, my_l, t, ids, w);
}

template <class T>
void launch(const hy3x_route_spec &spec, const void *logits, int64_t stride, const float *bias,
            int n_row, int32_t *ids, float *w, hipStream_t st) {
  const dim3 grid((n_row + ROUTE_WAVES - 1) / ROUTE_WAVES), block(64 * ROUTE_WAVES);
  int lanes = 1;  // of a group
  while (2 * lanes * spec.n_group <= 64) lanes *= 2;
  const int v = (spec.n_expert / spec.n_group + lanes - 1) / lanes;  // at most 32
#define HY3X_ROUTE(V)                                                                   \
  if (v <= V) {                                                                         \
    k_route_experts<T, V><<<grid, block, 0, st>>>(spec, (const T *)logits, stride, bias, \
                                                  n_row, ids, w);                       \
    return;                                                                             \
  }
  HY3X_ROUTE(1)
  HY3X_ROUTE(2)
  HY3X_ROUTE(3)
  HY3X_ROUTE(4)
  HY3X_ROUTE(6)
  HY3X_ROUTE(8)
  HY3X_ROUTE(16)
  HY3X_ROUTE(32)
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

void launch_route(const hy3x_route_spec &spec, const void *logits, int type, int64_t row_stride,
                  const float *bias, int T, int32_t *ids, float *w, hipStream_t st) {
  if (type == HY3X_F32)
    launch<float>(spec, logits, row_stride, bias, T, ids, w, st);
  else if (type == HY3X_F16)
    launch<__half>(spec, logits, row_stride, bias, T, ids, w, st);
  else
    launch<__hip_bfloat16>(spec, logits, row_stride, bias, T, ids, w, st);
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
  if (row_stride < spec->n_expert || row_stride > (int64_t)1 << 32)
    return op_fail(HY3X_E_ARG, "row_stride %lld outside [n_expert %d, 2^32]",
                   (long long)row_stride, spec->n_expert);
  if (T == 0) return HY3X_OK;
  if (!logits || !ids || !w) return op_fail(HY3X_E_ARG, "NULL logits, ids or w");
  const size_t size = type == HY3X_F32 ? 4 : 2;
  if ((uintptr_t)logits % size || (uintptr_t)bias % 4 || (uintptr_t)ids % 4 || (uintptr_t)w % 4)
    return op_fail(HY3X_E_ARG, "a pointer is not aligned to its elements");
  // no output may lie on anything else
  struct Span {
    uintptr_t at, end;
    Span(const void *p, int64_t bytes) : at((uintptr_t)p), end(at + (p ? (uintptr_t)bytes : 0)) {}
    bool meets(const Span &o) const { return at < o.end && o.at < end; }
  };
  const int64_t chosen = (int64_t)T * spec->k * 4;
  const Span in(logits, ((int64_t)(T - 1) * row_stride + spec->n_expert) * (int64_t)size),
      by(bias, 4 * spec->n_expert), i(ids, chosen), o(w, chosen);
  if (i.meets(in) || i.meets(by) || i.meets(o) || o.meets(in) || o.meets(by))
    return op_fail(HY3X_E_ARG, "ids or w overlaps another buffer");
  launch_route(*spec, logits, type, row_stride, bias, T, ids, w, (hipStream_t)stream);
  OP_HIP_TRY(hipGetLastError());
  return HY3X_OK;
}
