// hy3x_logprobs.hip -- log-probabilities of given tokens, entropy and the most
// probable tokens of rows of logits (hy3x_logprobs):
//
//   m = max l,  S = sum_v e^(l_v - m),  E = sum_v (l_v - m) e^(l_v - m)
//   log p_v = (l_v - m) - log S,   H = log S - E / S
//
// Both terms of H are at least 0, so it keeps its precision where one token has
// nearly all of the mass.
//
// One pass: a lane keeps the maximum of the logits it has met and the two sums relative
// to it (a larger maximum scales them down), in fp32; lanes, waves and the parts of a row
// meet in 64 bits. Few rows are split into parts, which a second launch joins.
//
// The most probable tokens: a wave keeps its best in falling order, one a lane, and looks
// at single logits only where one of 64 lanes has met a batch whose maximum passes the
// last of them. The first batch would put every logit there: a bound is found first, with
// at least as many lanes at or above it as tokens are wanted.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>

#include "../../include/hy3x_moe.h"
#include "hy3x_error.h"
#include "hy3x_ops.h"

namespace hy3x {
namespace {

__device__ __forceinline__ float elem(float v) { return v; }
__device__ __forceinline__ float elem(__half v) { return __half2float(v); }
__device__ __forceinline__ float elem(__hip_bfloat16 v) { return __bfloat162float(v); }
template <class X>
struct Type;
template <>
struct Type<float> {
  static constexpr float HIGH = 3.4028234663852886e38f;  // largest finite value
  static constexpr uint32_t MASKED = 0xff800000u;        // -inf
};
template <>
struct Type<__half> {
  static constexpr float HIGH = 65504.0f;
  static constexpr uint32_t MASKED = 0xfc00fc00u;
};
template <>
struct Type<__hip_bfloat16> {
  static constexpr float HIGH = 3.3895313892515355e38f;
  static constexpr uint32_t MASKED = 0xff80ff80u;
};

// e^(-FAR) is 0 in fp32: what lies further below a maximum counts as this far, so that a
// masked logit, -inf or NaN (which max passes over), adds 0 to both sums.
constexpr float FAR = 200.0f;
constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr int MAX_PARTS = 64;  // of a row: a lane for each in k_join
constexpr int NO_ID = 0x7fffffff;

struct Stats {  // of a part of a row; m: the type's lowest value where all is masked
  double S, E;
  float m;
  int unused[3];
};
struct Entry {
  float v;
  int id;
};

struct Call {
  const void *logits;
  int64_t stride;
  int V, T, top, parts, part;  // part: logits of one
  const int32_t *tokens;
  float *logp, *entropy, *top_logp;
  int32_t *top_ids;
  Stats *stats;   // [T x parts]
  Entry *lists;   // [T x parts x top]
};

__device__ __forceinline__ bool better(float v, int id, float w, int jd) {
  return v > w || (v == w && id < jd);
}
__device__ __forceinline__ float lane_value(float v, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}

// Integers in the order of the floats, -0 as 0; the float just below one.
__device__ __forceinline__ int order_of(float v) {
  const int b = __float_as_int(v + 0.0f);
  return b ^ (b >> 31 & 0x7fffffff);
}
__device__ __forceinline__ float below(int order) {
  int o = order - 1;
  if (o == -1) o = -2;  // -0
  return __int_as_float(o ^ (o >> 31 & 0x7fffffff));
}
// A value that at least n of the wave's v reach (-inf if fewer are finite): bisected, in
// their order.
__device__ __forceinline__ int reached_by(float v, int n) {
  const int k = order_of(v), none = order_of(-INFINITY);
  if (__popcll(__ballot(k > none)) < n) return none;
  int lo = none, hi = order_of(INFINITY);
  for (int i = 0; i < 20; i++) {
    const int mid = (lo & hi) + ((lo ^ hi) >> 1);
    if (__popcll(__ballot(k >= mid)) >= n) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The wave's best in falling order, one a lane.
struct Best {
  float v = -INFINITY, last;  // last: what a logit has to pass
  int id = NO_ID;
  __device__ __forceinline__ void put(float x, int i, int n, int lane) {
    const int at = __popcll(__ballot(better(v, id, x, i)));
    if (at >= n) return;
    const float up = __int_as_float(
        __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x138, 0xf, 0xf, false));
    const int upi = __builtin_amdgcn_update_dpp(0, id, 0x138, 0xf, 0xf, false);
    v = lane < at ? v : lane == at ? x : up;
    id = lane < at ? id : lane == at ? i : upi;
    last = fmaxf(last, lane_value(v, n - 1));
  }
};

// S and E of lanes, relative to their own maxima, to sums over the wave relative to the
// wave's.
__device__ __forceinline__ void meet(float &m, double &S, double &E) {
  float top = m;
  for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  const double d = fmax((double)m - top, (double)-FAR), f = exp(d);
  E = (E + S * d) * f;
  S *= f;
  for (int o = 32; o; o >>= 1) {
    S += __shfl_xor(S, o, 64);
    E += __shfl_xor(E, o, 64);
  }
  m = top;
}

// The row's results from its statistics and its candidates (value, id; -inf: none), which
// stand in LDS. Every thread of the block calls it.
template <class X>
__device__ void finish(const Call &c, int t, float m, double S, double E, float given,
                       const Entry *cand, int n_cand) {
  const X *row = (const X *)c.logits + t * c.stride;
  const bool some = m > -Type<X>::HIGH;
  const double lse = some ? log(S) : 0.0;
  auto logp = [&](float l) {
    return l > -Type<X>::HIGH ? (float)(((double)fminf(l, Type<X>::HIGH) - m) - lse) : -INFINITY;
  };
  if (threadIdx.x == 0) {
    const int token = c.tokens[t];
    c.logp[t] = token >= 0 && token < c.V ? logp(given) : 0.0f;
    if (c.entropy) c.entropy[t] = some ? (float)(lse - E / S) : 0.0f;
  }
  if (!c.top) return;
  __shared__ int live;
  if (threadIdx.x == 0) live = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n_cand; i += blockDim.x) {
    const Entry e = cand[i];
    if (e.id == NO_ID) continue;
    int rank = 0;
    for (int j = 0; j < n_cand; j++) rank += better(cand[j].v, cand[j].id, e.v, e.id);
    atomicAdd(&live, 1);
    if (rank < c.top) {
      c.top_ids[(int64_t)t * c.top + rank] = e.id;
      c.top_logp[(int64_t)t * c.top + rank] = logp(e.v);
    }
  }
  __syncthreads();
  // masked tokens in the places that are left, in index order
  if (live < c.top && threadIdx.x < 64) {
    int at = live;
    for (int v = 0; v < c.V && at < c.top; v += 64) {
      const int id = v + threadIdx.x;
      const bool off = id < c.V && !(elem(row[min(id, c.V - 1)]) > -Type<X>::HIGH);
      const uint64_t all = __ballot(off);
      const int mine = at + __popcll(all & ((1ull << threadIdx.x) - 1));
      if (off && mine < c.top) {
        c.top_ids[(int64_t)t * c.top + mine] = id;
        c.top_logp[(int64_t)t * c.top + mine] = -INFINITY;
      }
      at += __popcll(all);
    }
  }
}

template <class X>
__device__ __forceinline__ float given_logit(const Call &c, int t) {
  const int token = c.tokens[t];
  return elem(((const X *)c.logits)[t * c.stride + min(max(token, 0), c.V - 1)]);
}

// A part of a row.
template <class X, bool TOP>
__global__ __launch_bounds__(THREADS) void k_logprobs(Call c) {
  constexpr int N = 16 / sizeof(X), U = sizeof(X) == 4 ? 4 : 2, BATCH = THREADS * N * U;
  constexpr float HIGH = Type<X>::HIGH;
  __shared__ Stats part[WAVES];
  __shared__ Entry cand[TOP ? WAVES * HY3X_LOGPROBS_MAX_TOP : 1];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int t = blockIdx.x / c.parts, p = blockIdx.x % c.parts;
  const int first = p * c.part, end = min(c.V, first + c.part);
  const X *row = (const X *)c.logits + t * c.stride;
  const float given = c.parts == 1 ? given_logit<X>(c, t) : 0.0f;

  struct Raw {
    uint32_t w[U][4];
    __device__ __forceinline__ void load(const X *row, int at, int end, int tid) {
      if (at + BATCH <= end) {
#pragma unroll
        for (int u = 0; u < U; u++)
          __builtin_memcpy(w[u], row + at + (u * THREADS + tid) * N, 16);
      } else {
#pragma unroll
        for (int u = 0; u < U; u++) {
          const int k = at + (u * THREADS + tid) * N;
          if (k + N <= end) {
            __builtin_memcpy(w[u], row + k, 16);
          } else {
            X e[N];
#pragma unroll
            for (int i = 0; i < N; i++) {
              const uint32_t none = Type<X>::MASKED;
              __builtin_memcpy(&e[i], &none, sizeof(X));
              if (k + i < end) e[i] = row[k + i];
            }
            __builtin_memcpy(w[u], e, 16);
          }
        }
      }
    }
    __device__ __forceinline__ float at(int j) const {
      const uint32_t x = sizeof(X) == 4 ? w[j / 4][j % 4] : w[j / 8][j % 8 / 2];
      if constexpr (sizeof(X) == 4) return __uint_as_float(x);
      else return elem(__builtin_bit_cast(X, (uint16_t)(x >> (16 * (j & 1)))));
    }
  };
  Raw next;
  next.load(row, first, end, tid);
  float m = -HIGH, S = 0.0f, E = 0.0f;
  Best best;
  best.last = -HIGH;
  for (int at = first; at < end; at += BATCH) {
    float v[N * U];
#pragma unroll
    for (int j = 0; j < N * U; j++) v[j] = next.at(j);
    if (at + BATCH < end) next.load(row, at + BATCH, end, tid);
    float top = -INFINITY;  // not NaN where all of them are
#pragma unroll
    for (int j = 0; j < N * U; j++) top = fmaxf(top, v[j]);
    if (__ballot(top > HIGH)) {  // +inf
#pragma unroll
      for (int j = 0; j < N * U; j++) v[j] = v[j] > HIGH ? HIGH : v[j];
      top = fminf(top, HIGH);
    }
    if constexpr (TOP) {
      if (at == first) {
        const int bound = reached_by(top, c.top);
        if (bound != order_of(-INFINITY)) best.last = fmaxf(best.last, below(bound));
      }
      if (__ballot(top > best.last)) {
        const float last = best.last;  // a later batch's equals have higher indices
#pragma unroll
        for (int j = 0; j < N * U; j++) {
          uint64_t hits = __ballot(v[j] > last);
          while (hits) {
            const int l = __builtin_ctzll(hits);
            hits &= hits - 1;
            best.put(lane_value(v[j], l),
                     at + (j / N * THREADS + 64 * wave + l) * N + j % N, c.top, lane);
          }
        }
      }
    }
    const float to = fmaxf(m, top), d = fmaxf(m - to, -FAR), f = __expf(d);
    E = fmaf(S, d, E) * f;
    S *= f;
    m = to;
#pragma unroll
    for (int j = 0; j < N * U; j++) {
      const float x = fmaxf(v[j] - m, -FAR), e = __expf(x);
      S += e;
      E = fmaf(e, x, E);
    }
  }
  double Sd = S, Ed = E;
  meet(m, Sd, Ed);
  if (lane == 0) part[wave] = {Sd, Ed, m, {}};
  if (TOP && lane < c.top) cand[wave * c.top + lane] = {best.v, best.id};
  __syncthreads();
  m = part[lane % WAVES].m;
  Sd = lane < WAVES ? part[lane % WAVES].S : 0.0;
  Ed = lane < WAVES ? part[lane % WAVES].E : 0.0;
  meet(m, Sd, Ed);
  if (c.parts == 1) {
    finish<X>(c, t, m, Sd, Ed, given, cand, TOP ? WAVES * c.top : 0);
    return;
  }
  if (tid == 0) c.stats[blockIdx.x] = {Sd, Ed, m, {}};
  if (TOP && tid < WAVES * c.top) {
    const Entry e = cand[tid];
    int rank = 0;
    for (int j = 0; j < WAVES * c.top; j++) {
      // empty places are equal: in the order of the threads
      const Entry o = cand[j];
      rank += better(o.v, o.id, e.v, e.id) || (o.v == e.v && o.id == e.id && j < tid);
    }
    if (rank < c.top) c.lists[(int64_t)blockIdx.x * c.top + rank] = e;
  }
}

// The parts of a row.
template <class X>
__global__ __launch_bounds__(THREADS) void k_join(Call c) {
  __shared__ Entry cand[MAX_PARTS * HY3X_LOGPROBS_MAX_TOP];
  __shared__ int n_cand;
  const int t = blockIdx.x, lane = threadIdx.x & 63;
  const float given = given_logit<X>(c, t);
  const bool in = lane < c.parts;
  const Stats part = c.stats[(int64_t)t * c.parts + (in ? lane : 0)];
  float m = part.m;
  double S = in ? part.S : 0.0, E = in ? part.E : 0.0;
  meet(m, S, E);
  if (threadIdx.x == 0) n_cand = 0;
  __syncthreads();
  if (c.top) {
    // at least c.top candidates reach what `lists` of the lists' `deep` first ones reach
    const Entry *all = c.lists + (int64_t)t * c.parts * c.top;
    const int deep = (c.top + c.parts - 1) / c.parts, lists = (c.top + deep - 1) / deep;
    const int bound = reached_by(in ? all[lane * c.top + deep - 1].v : -INFINITY, lists);
    for (int i = threadIdx.x; i < c.parts * c.top; i += THREADS) {
      const Entry e = all[i];
      if (e.id != NO_ID && order_of(e.v) >= bound) cand[atomicAdd(&n_cand, 1)] = e;
    }
    __syncthreads();
  }
  finish<X>(c, t, m, S, E, given, cand, n_cand);
}

// Parts of a row: enough blocks for the card, of no less than PART logits each.
constexpr int PART = 2048, BLOCKS = 1024;
int parts_of(int T, int V) {
  const int most = std::min(MAX_PARTS, (V + PART - 1) / PART);
  return std::max(1, std::min(most, BLOCKS / std::max(T, 1)));
}

template <class X>
void launch(const Call &c, hipStream_t st) {
  const uint32_t blocks = (uint32_t)c.T * c.parts;
  if (c.top) k_logprobs<X, true><<<blocks, THREADS, 0, st>>>(c);
  else k_logprobs<X, false><<<blocks, THREADS, 0, st>>>(c);
  if (c.parts > 1) k_join<X><<<c.T, THREADS, 0, st>>>(c);
}

}  // namespace
}  // namespace hy3x

using namespace hy3x;

extern "C" {

int64_t hy3x_logprobs_workspace(int T, int V, int n_top) {
  if (T < 0 || T > HY3X_LOGPROBS_MAX_TOKENS || V < 1 || V > HY3X_LOGPROBS_MAX_VOCAB ||
      n_top < 0 || n_top > HY3X_LOGPROBS_MAX_TOP || n_top > V)
    return op_fail(HY3X_E_ARG, "T=%d, V=%d or n_top=%d out of range", T, V, n_top);
  const int64_t parts = parts_of(T, V);
  return parts == 1 ? 0 : T * parts * (int64_t)(sizeof(Stats) + n_top * sizeof(Entry));
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
  c.parts = parts_of(T, V);
  c.part = ((V + c.parts - 1) / c.parts + 7) & ~7;  // whole 16 bytes
  c.parts = (V + c.part - 1) / c.part;
  c.stats = (Stats *)workspace;
  c.lists = (Entry *)(c.stats + (int64_t)T * c.parts);
  const hipStream_t st = (hipStream_t)stream;
  if (type == HY3X_F32) launch<float>(c, st);
  else if (type == HY3X_F16) launch<__half>(c, st);
  else launch<__hip_bfloat16>(c, st);
  OP_HIP_TRY(hipGetLastError());
  return HY3X_OK;
}

}  // extern "C"
