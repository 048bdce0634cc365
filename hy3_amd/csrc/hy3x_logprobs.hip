// hy3x_logprobs.hip -- log-probabilities of given tokens, entropy and the most
// probable tokens of rows of logits (hy3x_logprobs):
//
//   m = max l,  S = 1 + R = sum_v e^(l_v - m),  E = sum_v (l_v - m) e^(l_v - m)
//   log p_v = (l_v - m) - log S,   H = log S - E / S
//
// Both terms of H are at least 0, so where one token has nearly all of the mass it keeps the
// precision of R, of what the others have. fp32 sums that hold the 1 would lose R below 2^-24
// (and keep three digits of it at 2^-14): where R is below PEAK, the logits of the lane that
// has the largest one are summed again without it, by all threads (2048 rows of 120832 bf16
// logits, a few in a hundred of them such rows, 102 us with it and without; 511 of 50021 22.6
// and 22.5; by one wave alone 104 and 23.4).
//
// One pass: a lane keeps the maximum of the logits it has met and the two sums relative
// to it (a larger maximum scales them down), in fp32; lanes, waves and the parts of a row
// meet in 64 bits. Few rows are split into parts, which a second launch joins.
//
// The most probable tokens: a lane remembers the largest maximum of its batches, which
// batch it was, and the second largest. When all have been met, a value is found that as
// many lanes' maxima reach as tokens are wanted. The batches of the lanes above it are
// read again (all of a lane's where its second reaches it too), and what reaches it,
// little more than is wanted, is ranked: a candidate's place is the number of better
// ones. Rows where too many logits reach it (equal ones) are gone through again, the
// wave's best in its lanes.
//
// Bytes bound many long rows: 2048 of 120832 bf16 logits 97 us, 5.1 TB/s, a copy's rate (plain
// reads reach 6.2). Where each CU has a row or two, waits bound it, 55 % of the waves' cycles: 511
// rows of 50021 fp16 16.6 us, with 20 alternatives 22.4, 2.3 TB/s, of which the 11 vector
// instructions a logit (14 with alternatives) are 9; what comes after the pass (the bound, the
// candidates' reads, their ranks, the logarithm) is a chain that nothing overlaps. Few rows are
// chains alone (a lane's loads, that end, the join): one row of 120832 with 20, 59 parts, 7.0 and
// 4.3 us.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>

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

// e^(-FAR) is 0 in fp32 (its least number is e^-103): what lies further below a maximum
// counts as this far, so that a masked logit, -inf or NaN (which max passes over), adds 0 to
// both sums. (Where a lane has met nothing but the type's lowest value, these count as 1 each
// until a larger maximum takes their sums to 0 with it, in fp16 at most to e^-32 of them, its
// least step being 32; if none comes the row has nothing left, and its sums are not used.)
constexpr float FAR = 200.0f;
constexpr double PEAK = 0.0625;  // from there on R has lost at most 4 bits of a lane's sum
constexpr int MAX_PARTS = 64;    // of a row: a lane for each in k_join

struct Stats {  // of a part of a row; m: the type's lowest value where all is masked
  double R, E;
  float m, unused;
};
// A logit and its index as one number: the better one is the larger one. 0: none.
typedef unsigned long long Entry;

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

template <int CTRL>
__device__ __forceinline__ double moved(double v) {  // between lanes of 16
  const long long b = __double_as_longlong(v);
  const uint32_t lo = dppi<CTRL>((int)b), hi = dppi<CTRL>((int)(b >> 32));
  return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
__device__ __forceinline__ double lane_value(double v, int lane) {
  const long long b = __double_as_longlong(v);
  const uint32_t lo = __builtin_amdgcn_readlane((int)b, lane),
                 hi = __builtin_amdgcn_readlane((int)(b >> 32), lane);
  return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
__device__ __forceinline__ float lane_value(float v, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}
__device__ __forceinline__ double sum_of_wave(double v) {
  v += moved<DPP_XOR1>(v);
  v += moved<DPP_XOR2>(v);
  v += moved<DPP_HALF_MIRROR>(v);
  v += moved<DPP_MIRROR>(v);
  return (lane_value(v, 0) + lane_value(v, 16)) + (lane_value(v, 32) + lane_value(v, 48));
}
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp<DPP_XOR1>(v));
  v = fmaxf(v, dpp<DPP_XOR2>(v));
  v = fmaxf(v, dpp<DPP_HALF_MIRROR>(v));
  v = fmaxf(v, dpp<DPP_MIRROR>(v));
  return fmaxf(fmaxf(lane_value(v, 0), lane_value(v, 16)),
               fmaxf(lane_value(v, 32), lane_value(v, 48)));
}

// Integers in the order of the floats, -0 as 0; the float of one, and the one just below.
__device__ __forceinline__ int order_of(float v) {
  const int b = __float_as_int(v + 0.0f);
  return b ^ (b >> 31 & 0x7fffffff);
}
__device__ __forceinline__ float in_order(int o) {
  return __int_as_float(o ^ (o >> 31 & 0x7fffffff));
}
__device__ __forceinline__ float below(int o) {
  return in_order(o == 0 ? -2 : o - 1);  // -1 stands for -0
}
__device__ __forceinline__ Entry entry(float v, int id) {
  return (Entry)((uint32_t)order_of(v) ^ 0x80000000u) << 32 | (uint32_t)~id;
}
__device__ __forceinline__ float value_of(Entry e) {
  return in_order((int)((uint32_t)(e >> 32) ^ 0x80000000u));
}
__device__ __forceinline__ int id_of(Entry e) { return (int)~(uint32_t)e; }
// How many of n entries in LDS are better.
__device__ __forceinline__ int better_than(Entry e, const Entry *all, int n) {
  int place = 0, k = 0;
  for (; k + 8 <= n; k += 8) {
    Entry o[8];
#pragma unroll
    for (int j = 0; j < 8; j++) o[j] = all[k + j];
#pragma unroll
    for (int j = 0; j < 8; j++) place += o[j] > e;
  }
  for (; k < n; k++) place += all[k] > e;
  return place;
}

// A value that at least n of the wave's v reach (-inf if fewer are finite), near the
// largest such: its place in their order, quartered.
__device__ __forceinline__ int reached_by(float v, int n) {
  const int k = order_of(v), none = order_of(-INFINITY);
  if (__popcll(__ballot(k > none)) < n) return none;
  int lo = order_of(-wave_max(-v)), hi = order_of(wave_max(v));
  for (int i = 0; i < 6; i++) {
    const int mid = (lo & hi) + ((lo ^ hi) >> 1);
    const int low = (lo & mid) + ((lo ^ mid) >> 1), high = (mid & hi) + ((mid ^ hi) >> 1);
    const int a = __popcll(__ballot(k >= low)), b = __popcll(__ballot(k >= mid)),
              c = __popcll(__ballot(k >= high));
    hi = a < n ? low : b < n ? mid : c < n ? high : hi;
    lo = c >= n ? high : b >= n ? mid : a >= n ? low : lo;
  }
  return lo;
}

constexpr int MAX_TOP = HY3X_LOGPROBS_MAX_TOP;
constexpr int CANDIDATES = 384;  // normally 1 to 3 times the tokens that are wanted
constexpr int AGAIN = 512;       // batches of a lane that are read again
constexpr int ROUND = 4;         // logits of a lane that are ranked at once
struct Ranking {                 // a wave's, in LDS
  Entry all[MAX_TOP + 64 * ROUND], sorted[MAX_TOP];
};

// The wave's best in falling order, one a lane.
struct Best {
  Entry e = 0;
  float last;  // what a logit has to pass
  int size = 0;
  // with `more` entries from room.all[MAX_TOP] on, the best n
  __device__ __forceinline__ void rank(Ranking &room, int more, int n, int lane) {
    if (lane < size) room.all[MAX_TOP - size + lane] = e;
    const Entry *all = room.all + MAX_TOP - size;
    const int count = size + more;
    for (int c = 0; c < count; c += 64) {
      const Entry o = all[min(c + lane, count - 1)];
      const int place = better_than(o, all, count);
      if (c + lane < count && place < n) room.sorted[place] = o;
    }
    size = min(count, n);
    e = room.sorted[lane % MAX_TOP];
    if (lane >= size) e = 0;
    if (size == n) last = lane_value(value_of(e), n - 1);
  }
};

// A lane's maximum and sums relative to it, to sums relative to `top`.
__device__ __forceinline__ void rescale(float m, float top, float &S, float &E) {
  const float d = fmaxf(m - top, -FAR), f = __expf(d);
  E = fmaf(S, d, E) * f;
  S *= f;
}

// The row's results from its statistics and its candidates, which stand in LDS (some may
// be none). Every thread of the block calls it.
template <class X>
__device__ void finish(const Call &c, int t, int token, float given, float m, double R, double E,
                       const Entry *cand, int n_cand, int live) {
  const X *row = (const X *)c.logits + t * c.stride;
  const bool some = m > -Type<X>::HIGH;
  const double lse = !some ? 0.0 : R < PEAK ? log1p(R) : log(1.0 + R);
  auto logp = [&](float l) {
    return l > -Type<X>::HIGH ? (float)(((double)fminf(l, Type<X>::HIGH) - m) - lse) : -INFINITY;
  };
  if (threadIdx.x == 0) {
    c.logp[t] = token >= 0 && token < c.V ? logp(given) : 0.0f;
    if (c.entropy) c.entropy[t] = some ? (float)(lse - E / (1.0 + R)) : 0.0f;
  }
  if (!c.top) return;
  for (int i = threadIdx.x; i < n_cand; i += blockDim.x) {
    const Entry e = cand[i];
    if (!e) continue;
    const int place = better_than(e, cand, n_cand);
    if (place < c.top) {
      c.top_ids[(int64_t)t * c.top + place] = id_of(e);
      c.top_logp[(int64_t)t * c.top + place] = logp(value_of(e));
    }
  }
  // masked tokens in the places that are left, in index order
  if (threadIdx.x < 64) {
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
__device__ __forceinline__ float given_logit(const Call &c, int t, int token) {
  return elem(((const X *)c.logits)[t * c.stride + min(max(token, 0), c.V - 1)]);
}

// A lane's logits of a batch: U times N that follow each other.
template <class X, int WAVES>
struct Batch {
  static constexpr int THREADS = 64 * WAVES, N = 16 / sizeof(X), U = sizeof(X) == 4 ? 4 : 2;
  static constexpr int COUNT = N * U, SIZE = THREADS * COUNT;
  uint32_t w[U][4];
  // index of logit j in the batch
  static __device__ __forceinline__ int place(int j, int tid) {
    return (j / N * THREADS + tid) * N + j % N;
  }
  // of the batch from `at`; what lies beyond `end` is masked
  __device__ __forceinline__ void load(const X *row, int at, int end, int tid) {
    if (at + SIZE <= end) {
#pragma unroll
      for (int u = 0; u < U; u++) __builtin_memcpy(w[u], row + at + place(u * N, tid), 16);
    } else {
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int k = at + place(u * N, tid);
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
  // logit j; +inf as the largest finite value where the caller says that there is one
  __device__ __forceinline__ float at(int j) const {
    const uint32_t x = sizeof(X) == 4 ? w[j / 4][j % 4] : w[j / 8][j % 8 / 2];
    if constexpr (sizeof(X) == 4) return __uint_as_float(x);
    else return elem(__builtin_bit_cast(X, (uint16_t)(x >> (16 * (j & 1)))));
  }
};

// The waves' best of a part, through its batches, whatever there is.
template <class X, int WAVES>
__device__ void best_of_all(const X *row, int first, int end, int n, Ranking &room, Entry *cand) {
  using B = Batch<X, WAVES>;
  const int tid = threadIdx.x, lane = tid & 63;
  Best best;
  best.last = -Type<X>::HIGH;
  for (int at = first; at < end; at += B::SIZE) {
    B batch;
    batch.load(row, at, end, tid);
    float v[B::COUNT], top = -INFINITY;
#pragma unroll
    for (int j = 0; j < B::COUNT; j++) {
      v[j] = batch.at(j) > Type<X>::HIGH ? Type<X>::HIGH : batch.at(j);
      top = fmaxf(top, v[j]);
    }
    const uint64_t over = __ballot(top > best.last);
    if (!over) continue;
    // an equal logit of a later batch has a higher index and comes after the last
    float last = best.last;
    if (__popcll(over) >= n) last = fmaxf(last, below(reached_by(top, n)));
    for (int round = 0; round < B::COUNT / ROUND; round++) {
      int more = 0;
#pragma unroll
      for (int j = 0; j < ROUND; j++) {
        float x = v[j];
        int id = at + B::place(j, tid);
#pragma unroll
        for (int r = 1; r < B::COUNT / ROUND; r++) {
          x = round == r ? v[r * ROUND + j] : x;
          id = round == r ? at + B::place(r * ROUND + j, tid) : id;
        }
        const uint64_t hits = __ballot(x > last);
        if (x > last)
          room.all[MAX_TOP + more + __popcll(hits & ((1ull << lane) - 1))] = entry(x, id);
        more += __popcll(hits);
      }
      if (more) best.rank(room, more, n, lane);
    }
  }
  if (lane < n) cand[tid / 64 * n + lane] = best.e;
}

// This thread's share of the sum over thread `of`'s logits of a part, relative to the largest
// one, `top`, and without it.
template <class X, int WAVES>
__device__ __forceinline__ float others(const X *row, int first, int end, float top, int of) {
  using B = Batch<X, WAVES>;
  const int items = (end - first + B::SIZE - 1) / B::SIZE * B::COUNT;
  float sum = 0.0f;
#pragma unroll 4
  for (int i = threadIdx.x; i < items; i += B::THREADS) {
    const int id = first + i / B::COUNT * B::SIZE + B::place(i % B::COUNT, of);
    const float v = id < end ? elem(row[id]) : -INFINITY;
    sum += v < top && v > -Type<X>::HIGH ? __expf(fmaxf(v - top, -FAR)) : 0.0f;
  }
  return sum;
}

// A part of a row.
template <class X, bool TOP, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_logprobs(Call c) {
  using B = Batch<X, WAVES>;
  constexpr int THREADS = B::THREADS;
  constexpr float HIGH = Type<X>::HIGH;
  __shared__ float high[WAVES], reach[WAVES];
  __shared__ double sums[WAVES][2];
  __shared__ Entry cand[TOP ? CANDIDATES : 1];
  __shared__ Ranking room[TOP ? WAVES : 1];
  __shared__ int again[TOP ? AGAIN : 1];  // batch of the part and thread
  __shared__ int n_cand, n_again, peak;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int t = blockIdx.x / c.parts, p = blockIdx.x % c.parts;
  const int first = p * c.part, end = min(c.V, first + c.part);
  const X *row = (const X *)c.logits + t * c.stride;
  const int token = c.parts == 1 ? c.tokens[t] : 0;
  const float given = c.parts == 1 ? given_logit<X>(c, t, token) : 0.0f;

  B next;
  next.load(row, first, end, tid);
  float m = -HIGH, S = 0.0f, E = 0.0f;
  float best = -INFINITY, second = -INFINITY;  // of the batches' maxima
  int best_at = first;
  for (int at = first; at < end; at += B::SIZE) {
    float v[B::COUNT];
#pragma unroll
    for (int j = 0; j < B::COUNT; j++) v[j] = next.at(j);
    if (at + B::SIZE < end) next.load(row, at + B::SIZE, end, tid);
    float top = -INFINITY;  // not NaN where all of them are
#pragma unroll
    for (int j = 0; j < B::COUNT; j++) top = fmaxf(top, v[j]);
    if (__ballot(top > HIGH)) {  // +inf
#pragma unroll
      for (int j = 0; j < B::COUNT; j++) v[j] = v[j] > HIGH ? HIGH : v[j];
      top = fminf(top, HIGH);
    }
    if (TOP) {
      second = fmaxf(second, fminf(best, top));
      best_at = top > best ? at : best_at;
      best = fmaxf(best, top);
    }
    const float to = fmaxf(m, top);
    rescale(m, to, S, E);
    m = to;
    float Sb = 0.0f, Eb = 0.0f;  // of the batch: a row's sums round once a batch
#pragma unroll
    for (int j = 0; j < B::COUNT; j++) {
      const float x = fmaxf(v[j] - m, -FAR), e = __expf(x);
      Sb += e;
      Eb = fmaf(e, x, Eb);
    }
    S += Sb;
    E += Eb;
  }
  // the block's maximum, then the sums
  const float wave_high = wave_max(m);  // every lane takes part
  if (lane == 0) high[wave] = wave_high;
  if (TOP) {
    const int bound = reached_by(best, (c.top + WAVES - 1) / WAVES);
    if (lane == 0) reach[wave] = in_order(bound);
    if (tid == 0) n_cand = n_again = 0;
  }
  __syncthreads();
  float top = high[0];
#pragma unroll
  for (int w = 1; w < WAVES; w++) top = fmaxf(top, high[w]);
  rescale(m, top, S, E);
  const double Sw = sum_of_wave((double)S), Ew = sum_of_wave((double)E);
  if (lane == 0) sums[wave][0] = Sw, sums[wave][1] = Ew;
  if (TOP) {
    float bound = reach[0];
#pragma unroll
    for (int w = 1; w < WAVES; w++) bound = fminf(bound, reach[w]);
    bound = fmaxf(bound, below(order_of(-HIGH) + 2));  // of what is not masked
    if (best >= bound) {
      const bool all = second >= bound;
      const int batches = all ? (end - first + B::SIZE - 1) / B::SIZE : 1;
      const int at = all ? 0 : (best_at - first) / B::SIZE, to = atomicAdd(&n_again, batches);
      for (int i = 0; i < batches && to + i < AGAIN; i++) again[to + i] = (at + i) * THREADS + tid;
    }
    __syncthreads();
    const int items = min(n_again, AGAIN) * B::COUNT;
#pragma unroll 4
    for (int i = tid; i < items; i += THREADS) {
      const int a = again[i / B::COUNT];
      const int id = first + a / THREADS * B::SIZE + B::place(i % B::COUNT, a % THREADS);
      const float x = id < end ? elem(row[id]) : -INFINITY;
      if (x >= bound) {
        const int to = atomicAdd(&n_cand, 1);
        if (to < CANDIDATES) cand[to] = entry(fminf(x, HIGH), id);
      }
    }
  }
  __syncthreads();
  double Rd = -1.0, Ed = 0.0;
#pragma unroll
  for (int w = 0; w < WAVES; w++) Rd += sums[w][0], Ed += sums[w][1];
  if (Rd < PEAK && top > -HIGH) {  // only one logit is the largest
    if (m == top) peak = tid;
    __syncthreads();
    const double rest = (double)others<X, WAVES>(row, first, end, top, peak) +
                        (tid == peak ? 0.0 : (double)S);
    const double Rw = sum_of_wave(rest);
    if (lane == 0) sums[wave][0] = Rw;
    __syncthreads();
    Rd = 0.0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) Rd += sums[w][0];
  }
  int count = TOP ? n_cand : 0, live = count;
  if (TOP && (count > CANDIDATES || n_again > AGAIN)) {
    __syncthreads();
    best_of_all<X, WAVES>(row, first, end, c.top, room[wave], cand);
    count = WAVES * c.top;
    __syncthreads();
    live = better_than(0, cand, count);
  }
  if (c.parts == 1) {
    finish<X>(c, t, token, given, top, Rd, Ed, cand, count, live);
    return;
  }
  if (tid == 0) c.stats[blockIdx.x] = {Rd, Ed, top, 0.0f};
  if (TOP) {
    Entry *list = c.lists + (int64_t)blockIdx.x * c.top;
    for (int i = tid; i < count; i += THREADS) {
      const Entry e = cand[i];
      const int place = better_than(e, cand, count);
      if (e && place < c.top) list[place] = e;
    }
    if (tid < c.top && tid >= live) list[tid] = 0;
  }
}

// The parts of a row.
constexpr int JOIN = 256;  // threads
template <class X>
__global__ __launch_bounds__(JOIN) void k_join(Call c) {
  __shared__ Entry cand[MAX_PARTS * HY3X_LOGPROBS_MAX_TOP];
  __shared__ int n_cand;
  const int t = blockIdx.x, lane = threadIdx.x & 63;
  const bool in = lane < c.parts;
  const Stats part = c.stats[(int64_t)t * c.parts + (in ? lane : 0)];
  // at least c.top candidates reach what `lists` of the lists' `deep` first ones reach
  const Entry *all = c.lists + (int64_t)t * c.parts * c.top;
  const int count = c.parts * c.top;
  const int deep = (c.top + c.parts - 1) / c.parts, lists = c.top ? (c.top + deep - 1) / deep : 0;
  Entry mine[MAX_PARTS * MAX_TOP / JOIN], first = 0;  // on their way together
  if (c.top) {
    if (in) first = all[lane * c.top + deep - 1];
#pragma unroll
    for (int i = 0; i < MAX_PARTS * MAX_TOP / JOIN; i++) {
      const int at = threadIdx.x + i * JOIN;
      mine[i] = 0;
      if (at < count) mine[i] = all[at];
    }
  }
  const int token = c.tokens[t];
  const float given = given_logit<X>(c, t, token);
  const float m = wave_max(part.m);
  const float d = fmaxf(part.m - m, -FAR), f = in ? __expf(d) : 0.0f;
  // one of the largest logits is the row's 1
  const int lead = __builtin_ctzll(__ballot(in && part.m == m));
  const double S = 1.0 + part.R, E = sum_of_wave((part.E + S * d) * f);
  const double R = sum_of_wave(lane == lead ? part.R : S * f);
  if (threadIdx.x == 0) n_cand = 0;
  __syncthreads();
  if (c.top) {
    const int bound = reached_by(first ? value_of(first) : -INFINITY, lists);
#pragma unroll
    for (int i = 0; i < MAX_PARTS * MAX_TOP / JOIN; i++)
      if (mine[i] && order_of(value_of(mine[i])) >= bound) cand[atomicAdd(&n_cand, 1)] = mine[i];
    __syncthreads();
  }
  finish<X>(c, t, token, given, m, R, E, cand, n_cand, n_cand);
}

// Rows in parts: rows that are fewer than the CUs, over a long vocabulary; parts have no less
// than PART logits. A row as a whole takes 75 us for a million logits more, whatever their type,
// and the card's rate for all parts is twice as high (in logits) for 16-bit ones. us of whole
// rows (8 waves each) and of parts and their join, 5 alternatives:
//   fp32     1 row of 32003   8.3   9.8    16-bit   8 rows of 32003  10.2  11.6
//            8 of 64000      12.7  11.4             8 of 64000      13.1  11.5
//           64 of 64000      13.7  13.3            64 of 64000      14.1  13.2
//          100 of 64000      13.7  15.1           128 of 64000      14.2  14.7
//           64 of 120832     18.1  15.8           128 of 120832     19.6  18.5
//          100 of 120832     19.8  20.0           160 of 120832     21.0  21.2
//          128 of 120832     20.0  22.3           200 of 120832     21.2  22.9
//           90 of 260000     32.6  27.3           200 of 260000     35.0  33.2
//          160 of 260000     33.7  38.1           255 of 260000     35.6  36.9
constexpr int PART = 2048, BLOCKS = 1024;
int most_split(int V, int type) {  // rows
  return type == HY3X_F32 ? 160 - (6000000 + V - 1) / V : 260 - (12000000 + V - 1) / V;
}
int parts_of(int T, int V, int type) {
  if (T < 1 || T > most_split(V, type)) return 1;
  return std::min({MAX_PARTS, (V + PART - 1) / PART, BLOCKS / T});
}
// Bytes of workspace of a call.
int64_t room_of(int T, int V, int type, int n_top) {
  const int64_t parts = parts_of(T, V, type);
  return parts == 1 ? 0 : T * parts * (int64_t)(sizeof(Stats) + n_top * sizeof(Entry));
}
// Whole rows: 8 waves each where the rows are long and each has a CU (up to 256), longer 16-bit
// rows also where two have one (up to 512). us with 4 waves and with 8, 5 alternatives:
//   fp32   256 rows of 20003 10.2 10.0    16-bit  256 rows of 20003 10.2 10.3
//          256 of 32003      13.3 11.9            256 of 24576      10.4 10.2
//          256 of 120832     29.6 27.8            256 of 50021      15.7 14.0
//          270 of 32003      13.4 14.5            256 of 120832     31.2 22.6
//          270 of 120832     30.3 33.8            333 of 50021      19.2 19.2
//          511 of 50021      23.8 25.8            333 of 64000      21.9 21.1
//          511 of 120832     47.1 45.0            511 of 120832     37.0 32.4
//          800 of 120832     81.5 80.2            560 of 64000      27.3 28.2
constexpr int CUS = 256, EIGHT = 24576, EIGHT_FOR_TWO = 65536;
bool eight_waves(int T, int V, int type) {
  return (T <= CUS && V >= EIGHT) || (T <= 2 * CUS && V >= EIGHT_FOR_TWO && type != HY3X_F32);
}
constexpr int ROWS = 1 << 23;  // of a launch, which has less than 2^32 threads

template <class X, int WAVES>
void launch_waves(const Call &c, hipStream_t st) {
  const uint32_t blocks = (uint32_t)c.T * c.parts;
  if (c.top) k_logprobs<X, true, WAVES><<<blocks, 64 * WAVES, 0, st>>>(c);
  else k_logprobs<X, false, WAVES><<<blocks, 64 * WAVES, 0, st>>>(c);
}
template <class X>
void launch(const Call &c, hipStream_t st) {
  constexpr int TYPE = sizeof(X) == 4 ? HY3X_F32 : HY3X_F16;
  if (c.parts == 1 && eight_waves(c.T, c.V, TYPE)) launch_waves<X, 8>(c, st);
  else launch_waves<X, 4>(c, st);
  if (c.parts > 1) k_join<X><<<c.T, JOIN, 0, st>>>(c);
}

}  // namespace
}  // namespace hy3x

using namespace hy3x;

extern "C" {

int64_t hy3x_logprobs_workspace(int T, int V, int n_top) {
  if (T < 0 || T > HY3X_LOGPROBS_MAX_TOKENS || V < 1 || V > HY3X_LOGPROBS_MAX_VOCAB ||
      n_top < 0 || n_top > HY3X_LOGPROBS_MAX_TOP || n_top > V)
    return op_fail(HY3X_E_ARG, "T=%d, V=%d or n_top=%d out of range", T, V, n_top);
  // the most parts that up to T rows of either type have together
  const int rows = std::min(T, std::max({most_split(V, HY3X_F32), most_split(V, HY3X_F16), 0}));
  const int parts = std::min(rows * std::min(MAX_PARTS, (V + PART - 1) / PART), BLOCKS);
  return parts * (int64_t)(sizeof(Stats) + n_top * sizeof(Entry));
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
  const int64_t room = room_of(T, V, type, n_top);
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
  c.top = n_top;
  c.tokens = tokens;
  c.logp = logp;
  c.entropy = entropy;
  c.top_ids = top_ids;
  c.top_logp = top_logp;
  c.parts = parts_of(T, V, type);
  c.part = ((V + c.parts - 1) / c.parts + 7) & ~7;  // whole 16 bytes
  c.parts = (V + c.part - 1) / c.part;
  c.stats = (Stats *)workspace;
  c.lists = (Entry *)(c.stats + (int64_t)T * c.parts);
  const hipStream_t st = (hipStream_t)stream;
  for (int t = 0; t < T; t += ROWS) {
    c.T = std::min(T - t, ROWS);
    if (type == HY3X_F32) launch<float>(c, st);
    else if (type == HY3X_F16) launch<__half>(c, st);
    else launch<__hip_bfloat16>(c, st);
    OP_HIP_TRY(hipGetLastError());
    c.logits = (const uint8_t *)c.logits + c.T * row_stride * es;
    c.tokens += c.T;
    c.logp += c.T;
    if (entropy) c.entropy += c.T;
    if (n_top) c.top_ids += (int64_t)c.T * n_top, c.top_logp += (int64_t)c.T * n_top;
  }
  return HY3X_OK;
}

}  // extern "C"
