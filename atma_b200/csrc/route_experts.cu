// Which experts a token goes to, with what weights, and the tokens in the order of their experts.
//
//   score = sigmoid(z) or softmax(z);  key = score + bias;  a group's key = the sum of its two best keys
//   the best groups stay; of their experts the k with the largest keys, falling, the lower index first where keys are equal
//   weight = score (/ the sum over the k) * scale
//
// A choice is only as good as the difference between the keys that it turns on, and fp32 keys are off by some 1e-7.  So a warp takes
// a token in fp32 first, and where two neighbours among the sorted best (and the first one left out, and the groups likewise) are
// nearer to one another than their errors can reach, those are decided again with keys in fp64.  Without a bias and groups both scores
// grow with the logit, which is then the key itself and exact.  Weights are fp32 scores over their sum, and fp64 ones where the chosen scores
// are below what fp32 holds: sigmoids of logits below -87, softmax beside a far larger logit that a bias or its group keeps out.
//
// Bound by instructions, 971 a token: 16384 tokens of 256 experts in 8 groups, top 8, 28 us and 9 for the order (18 MB: 2.8); 75 and 15 with a
// scan of the lane's keys in every round and whole tokens again in fp64, which held up their CTAs by 10 us each.  That scan (choose) is what
// groups of no 1, 2, 4, .. whole lanes still take, and 32 choices or more: 160 experts in 8 groups, top 6, 85 us.  A CTA of 1024 threads leaves
// a thread 64 registers; with eight experts a lane 308 bytes of it are spilled, with sixteen 556, and most of that around the calls of
// what few tokens need.
// A warp holds a token's experts, V of them a lane, neighbours in neighbouring places.  Largest values come by redux over the keys as
// ordered integers.  A NaN counts as the smallest logit, so that every choice is an expert; infinities as the largest finite values.
//
// The order: a CTA's tokens are a chunk; it leaves how many of them go to every expert (route), and a second launch adds up the chunks in
// front and gives every (token, choice) its place among its expert's, by counts and ranks alone (order): the same result at every run.
// One chunk does both in the first launch.
#include "common.cuh"
#include "early.cuh"
#include "../../include/atma_decoder.h"

#include <cfloat>

namespace atma {

namespace {

constexpr int kRouteThreads = 1024, kRouteWarps = kRouteThreads / 32;
constexpr int kMaxExperts = 512;
// Twice what keys are off by, relative to |key| + 1.  Sigmoid: 2 units of e^-z, which s (1 - s) <= 1 / 4 damps, one unit each of 1 + e^-z, its
// reciprocal and the sum with the bias, 2.5e-7 + 6e-8 |key|.  Softmax: up to 22 roundings of the sum, which all keys share, as well.
constexpr float kKeyError = 4e-6f, kSigmoidError = 1e-6f;

// How far the sum of a group's two best keys may be off: half of `error` for either key and |key| + 1, not for their sum, where keys of
// opposite signs cancel.  The sum's own rounding is in what kSigmoidError and kKeyError leave of every key.  One key: second = 0.
__device__ __forceinline__ float group_reach(float best, float second, float error) {
  return fmaf(.5f * error, fabsf(best), fmaf(.5f * error, fabsf(second), error));
}

struct RouteArgs {
  const float* logits; int64_t l_rs;
  const float* bias;
  int32_t* ids;
  float* weights;
  int32_t* counts;                          // [chunks][experts]
  int32_t *order, *place, *starts;
  int tokens, experts, k, groups, top_groups, chunk, chunks;
  float scale;
  bool sigmoid, renormalize;
  bool vec;                                 // rows start on 16-byte boundaries
  bool lanes;                               // choose_fast: groups are 1, 2, 4, .. whole lanes, k is below 32
};

// floats and doubles as integers in the same order; 0 is below all of them
__device__ __forceinline__ uint32_t ordered(float f) {
  const uint32_t u = __float_as_uint(f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t ordered(double f) {
  const uint64_t u = (uint64_t)__double_as_longlong(f);
  return u >> 63 ? ~u : u | (1ull << 63);
}
__device__ __forceinline__ float value_of(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }
__device__ __forceinline__ double value_of(uint64_t u) { return __longlong_as_double((long long)(u >> 63 ? u & ~(1ull << 63) : ~u)); }
__device__ __forceinline__ uint32_t warp_most(uint32_t u) { return __reduce_max_sync(0xffffffffu, u); }
__device__ __forceinline__ uint64_t warp_most(uint64_t u) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(u >> 32));
  return (uint64_t)hi << 32 | __reduce_max_sync(0xffffffffu, (uint32_t)(u >> 32) == hi ? (uint32_t)u : 0u);
}

template <typename F> struct Ordered;
template <> struct Ordered<float> { using type = uint32_t; };
template <> struct Ordered<double> { using type = uint64_t; };

__device__ __forceinline__ float exp_of(float x) { return expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }

// The exponential is 1 at most: e^-z has no fp32 value below z = -88, where the result still has one.
__device__ __forceinline__ float sigmoid_of(float z) {
  const float e = expf(-fabsf(z));
  return (z < 0.f ? e : 1.f) / (1.f + e);
}
__device__ __forceinline__ double sigmoid_of(double z) { return 1. / (1. + exp(-z)); }

template <typename F>
__device__ __forceinline__ F warp_add(F v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The scores of a lane's experts.
template <typename F, int V>
__device__ __forceinline__ void scores_of(const float (&z)[V], int e0, int experts, bool sigmoid, F (&s)[V]) {
  if (sigmoid) {
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = sigmoid_of(F(z[v]));
    return;
  }
  float m = -FLT_MAX;
#pragma unroll
  for (int v = 0; v < V; ++v) m = fmaxf(m, z[v]);            // behind the last expert z is -FLT_MAX
  m = value_of(warp_most(ordered(m)));
  F sum = 0;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    s[v] = e0 + v < experts ? exp_of(F(z[v]) - F(m)) : F(0);
    sum += s[v];
  }
  sum = warp_add(sum);
#pragma unroll
  for (int v = 0; v < V; ++v) s[v] /= sum;
}

// Takes experts out whose group is not among the best; false where fp32 keys do not settle which those are.
template <typename F, int V>
__device__ __forceinline__ bool keep_groups(typename Ordered<F>::type (&key)[V], int e0, const RouteArgs& a) {
  using U = typename Ordered<F>::type;
  const int lane = threadIdx.x & 31, size = a.experts / a.groups;
  U mine[2] = {0, 0};                                        // keys of groups `lane` and `lane + 32`
  float reach[2] = {0.f, 0.f};                               // fp32: how far they may be off; nothing where a key is infinite
  bool settled = true;
  for (int g = 0; g < a.groups; ++g) {
    U best = 0, second = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const U u = e0 + v >= g * size && e0 + v < (g + 1) * size ? key[v] : U(0);
      second = u > best ? best : (u > second ? u : second);
      best = u > best ? u : best;
    }
    const U most = warp_most(best);
    const uint32_t holders = __ballot_sync(0xffffffffu, best == most);
    const U next = warp_most(lane == __ffs(holders) - 1 ? second : best);
    // a group of one expert has no second; inf and -inf are inf
    const F sum = next == 0 || value_of(most) == F(INFINITY) ? value_of(most) : value_of(most) + value_of(next);
    if (lane == (g & 31)) mine[g >> 5] = ordered(sum);
    if constexpr (std::is_same<F, float>::value) {
      const float r = group_reach(value_of(most), next == 0 ? 0.f : value_of(next), kKeyError);
      if (fabsf(sum) <= FLT_MAX) {
        if (lane == (g & 31)) reach[g >> 5] = r;
      } else if (r <= FLT_MAX) {                             // finite keys whose sum is not
        settled = false;
      }
    }
  }
  uint64_t left = 0;
  float lowest = INFINITY;                                   // what a group that stays has at least
  for (int n = 0; n <= a.top_groups && n < a.groups; ++n) {
    if (n == a.top_groups) {                                 // the others go: may one of them have as much?
      if constexpr (std::is_same<F, float>::value) {
        const float highest = fmaxf(mine[0] == 0 ? -INFINITY : value_of(mine[0]) + reach[0], mine[1] == 0 ? -INFINITY : value_of(mine[1]) + reach[1]);
        settled = settled && lowest > value_of(warp_most(ordered(highest)));
      }
      break;
    }
    const U most = warp_most(mine[0] > mine[1] ? mine[0] : mine[1]);
    const uint32_t low = __ballot_sync(0xffffffffu, mine[0] == most), high = __ballot_sync(0xffffffffu, mine[1] == most);
    const int g = low ? __ffs(low) - 1 : 31 + __ffs(high);
    if constexpr (std::is_same<F, float>::value) lowest = fminf(lowest, value_of(most) - __shfl_sync(0xffffffffu, reach[g >> 5], g & 31));
    left |= 1ull << g;
    if (lane == (g & 31)) mine[g >> 5] = 0;
  }
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (e0 + v < a.experts && !(left >> ((e0 + v) / size) & 1)) key[v] = 0;        // below -inf, which a bias may give experts that stay
  return settled;
}

struct Chosen { int id[2]; float score[2]; };                // lane j's choices j and j + 32; id[0] = -1: not settled

__device__ __forceinline__ float logit_of(float f) { return fminf(fmaxf(f, -FLT_MAX), FLT_MAX); }      // a NaN becomes -FLT_MAX

// The k best of a token with keys of type F.  Out of line, and with the logits read again: few tokens come here.
template <typename F, int V>
__device__ __noinline__ Chosen choose(const float* row, int e0, const RouteArgs& a) {
  using U = typename Ordered<F>::type;
  const int lane = threadIdx.x & 31;
  const bool exact = a.bias == nullptr && a.groups == 1;     // keys are the logits
  float z[V];
  F s[V];
  U key[V];
#pragma unroll
  for (int v = 0; v < V; ++v) z[v] = e0 + v < a.experts ? logit_of(row[e0 + v]) : -FLT_MAX;
  scores_of<F, V>(z, e0, a.experts, a.sigmoid, s);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = e0 + v;
    F f = exact ? F(z[v]) : s[v];
    if (a.bias != nullptr && e < a.experts) {
      const float b = a.bias[e];
      f += F(isnan(b) ? -INFINITY : b);
    }
    key[v] = e < a.experts ? ordered(f) : U(0);
  }
  bool settled = true;
  if (a.groups > 1) settled = keep_groups<F, V>(key, e0, a);
  Chosen c = {{0, 0}, {0.f, 0.f}};
  U last = 0;
  const bool check = std::is_same<F, float>::value && !exact;
  const int rounds = check && a.k < a.experts ? a.k + 1 : a.k;
  for (int n = 0; n < rounds; ++n) {
    U best = 0;
    F at = 0;
    int where = 0;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (key[v] > best) { best = key[v]; at = s[v]; where = v; }
    const U most = warp_most(best);
    if (check && n > 0 && most != 0) {                       // 0: none is left
      const float p = (float)value_of(last), q = (float)value_of(most);
      settled = settled && p - q > kKeyError * (fabsf(p) + 1.f);       // also where both are -inf
    }
    last = most;
    if (n == a.k) break;
    const int holder = __ffs(__ballot_sync(0xffffffffu, best == most)) - 1;
    const int e = __shfl_sync(0xffffffffu, e0 + where, holder);
    const float got = (float)__shfl_sync(0xffffffffu, at, holder);
    if (lane == (n & 31)) {
      if (n < 32) { c.id[0] = e; c.score[0] = got; } else { c.id[1] = e; c.score[1] = got; }
    }
    if (lane == holder) {
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (v == where) key[v] = 0;
    }
  }
  if (!settled) c.id[0] = -1;               // the same for all lanes
  return c;
}

// 1 / (1 + 2^(-z log2(e))), each step to two units in its last place; zero below z = -87 or so.
__device__ __forceinline__ float sigmoid_fast(float z) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return r;
}

// A lane's words in falling order: odd-even merge sort.
template <int V>
__device__ __forceinline__ void sort_words(uint32_t (&w)[V]) {
#pragma unroll
  for (int p = 1; p < V; p *= 2)
#pragma unroll
    for (int d = p; d > 0; d /= 2)
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i >= d % p && (i - d % p) % (2 * d) < d && i + d < V && i / (2 * p) == (i + d) / (2 * p)) {
          const uint32_t hi = max(w[i], w[i + d]), lo = min(w[i], w[i + d]);
          w[i] = hi; w[i + d] = lo;
        }
}

// A key in fp64; m: the largest logit, total: the sum of all exp(z - m).
__device__ __forceinline__ double key_in_64(const float* row, int e, float m, double total, const RouteArgs& a) {
  const double z = logit_of(row[e]);
  if (a.bias == nullptr && a.groups == 1) return z;
  const double s = a.sigmoid ? sigmoid_of(z) : exp(z - (double)m) / total;
  if (a.bias == nullptr) return s;
  const float b = a.bias[e];
  return s + (isnan(b) ? -INFINITY : b);
}
__device__ __forceinline__ double total_in_64(const float* row, float m, const RouteArgs& a) {
  double total = 0.;
  if (!a.sigmoid)
#pragma unroll 1
    for (int i = threadIdx.x & 31; i < a.experts; i += 32) total += exp((double)logit_of(row[i]) - (double)m);
  return warp_add(total);
}

// Weights of a token whose chosen scores are not, or hardly, fp32 values: the scores over their sum in fp64 (softmax: the sum over all experts
// is in both and left out), zero where that sum is.  Two choices a lane, where they are used.
struct Two { float v[2]; };
__device__ __noinline__ Two weights_in_64(const float* row, int e0, int e1, bool used0, bool used1, const RouteArgs& a) {
  float m = -FLT_MAX;
  if (!a.sigmoid) {
#pragma unroll 1
    for (int i = threadIdx.x & 31; i < a.experts; i += 32) m = fmaxf(m, logit_of(row[i]));
    m = value_of(warp_most(ordered(m)));
  }
  const double x = logit_of(row[e0]), y = logit_of(row[e1]);
  const double s = !used0 ? 0. : a.sigmoid ? sigmoid_of(x) : exp(x - (double)m), t = !used1 ? 0. : a.sigmoid ? sigmoid_of(y) : exp(y - (double)m);
  const double sum = warp_add(s + t);
  return {{sum > 0. ? (float)(s / sum) : 0.f, sum > 0. ? (float)(t / sum) : 0.f}};
}

// Of n taken experts, one a lane, how many have a larger key, in fp64.  Out of line, like the next one: one token in some dozens comes
// here, and a long way through cold code would hold up its CTA.
__device__ __noinline__ int rank_in_64(const float* row, int e, int n, float m, const RouteArgs& a) {
  const double f = key_in_64(row, e, m, total_in_64(row, m, a), a);
  int above = 0;
  for (int i = 0; i < n; ++i) {
    const double g = __shfl_sync(0xffffffffu, f, i);
    const int h = __shfl_sync(0xffffffffu, e, i);
    above += g > f || (g == f && h < e);
  }
  return (threadIdx.x & 31) < n ? above : 32;
}
// Whether this lane's group goes, in fp64 (groups of whole lanes, V experts each).
template <int V>
__device__ __noinline__ bool group_goes_in_64(const float* row, int e0, float m, const RouteArgs& a) {
  const int lanes = a.experts / a.groups / V, mine = (threadIdx.x & 31) & -lanes;
  const double total = total_in_64(row, m, a);
  double best = -INFINITY, second = -INFINITY;
#pragma unroll 2
  for (int v = 0; v < V; ++v)
    if (e0 + v < a.experts) {
      const double f = key_in_64(row, e0 + v, m, total, a);
      second = fmax(second, fmin(best, f));
      best = fmax(best, f);
    }
#pragma unroll 1
  for (int o = 1; o < lanes; o <<= 1) {
    const double b = __shfl_xor_sync(0xffffffffu, best, o), c = __shfl_xor_sync(0xffffffffu, second, o);
    second = fmax(fmax(second, c), fmin(best, b));
    best = fmax(best, b);
  }
  const double both = V * lanes == 1 || best == INFINITY ? best : best + second;      // inf and -inf are inf
  int above = 0;
#pragma unroll 1
  for (int from = 0; from < a.groups * lanes; from += lanes) {
    const double other = __shfl_sync(0xffffffffu, both, from);
    above += other > both || (other == both && from < mine);
  }
  return above >= a.top_groups;
}

// The same in fp32 where every lane's experts are of one group (or there are none), a group is 1, 2, 4, .. lanes and k is small.
//
// Keys come from instructions that round more; what they are off by stays below kKeyError, since s (1 - s) |z| and |d| exp(-|d|),
// d = z - max, are below 0.4.  A key and its expert are one word: the key as an ordered integer without its last bits, the expert there,
// lower ones larger.  A lane sorts its words once, and a round is one redux over the lanes' first ones.  Rounds go on until k words are
// taken and the next key is surely below the last; if some of the taken are nearer to one another than that, each lane computes one
// taken expert's key in fp64 and counts those above it.  Lane `rank` of the result: choice `rank`.  kFull: no lane has places without an expert.
template <int V, bool kFull>
__device__ __forceinline__ bool choose_fast(const float (&z)[V], const float (&bias)[V], int e0, const RouteArgs& a, const float* row, int* rank, int* id, float* score) {
  constexpr uint32_t kPlace = V <= 8 ? 255 : 511;
  const int lane = threadIdx.x & 31, own = kFull ? V : a.experts - e0;             // the lane's experts, if they are fewer than V
  const bool exact = a.bias == nullptr && a.groups == 1;     // keys are the logits
  const float width = exact ? 0.f : a.sigmoid ? kSigmoidError : kKeyError;
  float key[V], m = 0.f, sum = 1.f;
  if (!a.sigmoid) {
    m = z[0];
#pragma unroll
    for (int v = 1; v < V; ++v) m = fmaxf(m, z[v]);          // behind the last expert z is -FLT_MAX
    m = value_of(warp_most(ordered(m)));
    sum = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      key[v] = v < own ? expf(z[v] - m) : 0.f;
      sum += key[v];
    }
    sum = warp_add(sum);
    const float r = 1.f / sum;
#pragma unroll
    for (int v = 0; v < V; ++v) key[v] *= r;
  } else if (!exact) {
#pragma unroll
    for (int v = 0; v < V; ++v) key[v] = sigmoid_fast(z[v]);
  }
  if (exact) {
#pragma unroll
    for (int v = 0; v < V; ++v) key[v] = z[v];
  } else if (a.bias != nullptr) {
#pragma unroll
    for (int v = 0; v < V; ++v) key[v] = fmaxf(key[v] + bias[v], -FLT_MAX);         // a NaN becomes -FLT_MAX here
  }
  bool out = false;                         // this lane's group goes
  if (a.groups > 1) {                       // V divides a group here: own is V or less than 1
    const int lanes = a.experts / a.groups / V, mine = lane & -lanes;
    float best = key[0], second = -INFINITY;
#pragma unroll
    for (int v = 1; v < V; ++v) {
      second = fmaxf(second, fminf(best, key[v]));
      best = fmaxf(best, key[v]);
    }
    for (int o = 1; o < lanes; o <<= 1) {
      const float b = __shfl_xor_sync(0xffffffffu, best, o), c = __shfl_xor_sync(0xffffffffu, second, o);
      second = fmaxf(fmaxf(second, c), fminf(best, b));
      best = fmaxf(best, b);
    }
    const float both = second == -INFINITY ? best : best + second;
    const float reach = group_reach(best, second == -INFINITY ? 0.f : second, width);
    int above = 0;                          // groups that are better than this lane's
    float nearest = INFINITY;               // of the distances from another one, less what that one may be off by
#pragma unroll 4
    for (int from = 0; from < a.groups * lanes; from += lanes) {
      const float other = __shfl_sync(0xffffffffu, both, from), its = __shfl_sync(0xffffffffu, reach, from);
      above += other > both;
      nearest = fminf(nearest, from == mine ? INFINITY : fabsf(other - both) - its);
    }
    // two infinities are as near as can be
    const bool settled = (nearest > reach && fabsf(both) <= FLT_MAX) || lane >= a.groups * lanes;
    out = above >= a.top_groups;
    if (!__all_sync(0xffffffffu, settled)) out = group_goes_in_64<V>(row, e0, m, a);
  }
  uint32_t word[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    word[v] = (ordered(key[v]) & ~kPlace) | (kPlace - (uint32_t)(e0 + v));
    if (out || (!kFull && v >= own)) word[v] = 0;            // not to be had: below all others
  }
  sort_words<V>(word);
  auto take = [&]() {                       // the largest word that is left
    const uint32_t most = warp_most(word[0]);
    if (word[0] == most) {
#pragma unroll
      for (int v = 0; v + 1 < V; ++v) word[v] = word[v + 1];
      word[V - 1] = 0;
    }
    return most;
  };
  auto apart = [&](uint32_t above, uint32_t below) {         // what the key above is at least, and the one below at most
    const float p = value_of(above & ~kPlace), q = value_of(below | kPlace);
    return below == 0 || (exact ? (above & ~kPlace) > (below | kPlace) : p - q > width * (fabsf(p) + 1.f));
  };
  uint32_t taken = 0;                       // lane n: word n
  for (int n = 0; n <= a.k; ++n) {
    const uint32_t most = take();
    if (lane == n) taken = most;
  }
  int n = a.k;                              // words that are surely above the next one
  const uint32_t next = __shfl_down_sync(0xffffffffu, taken, 1);
  const uint32_t near = __ballot_sync(0xffffffffu, lane < a.k && !apart(taken, next));
  if (near >> (a.k - 1)) {
    uint32_t last = __shfl_sync(0xffffffffu, taken, n);
    do {
      if (++n == 32) return false;
      const uint32_t most = take();
      if (lane == n) taken = most;
      if (apart(last, most)) break;
      last = most;
    } while (true);
  }
  const int e = lane < n ? (int)(kPlace - (taken & kPlace)) : 0;
  const float x = logit_of(row[e]);
  *id = e;
  *rank = lane < n ? lane : 32;
  *score = a.sigmoid ? sigmoid_of(x) : expf(x - m) / sum;
  if (near) *rank = rank_in_64(row, e, n, m, a);             // the same for all lanes
  return true;
}

// ---- places ----------------------------------------------------------------------------------------------
struct OrderShared {
  int32_t base[kMaxExperts];                // the next place of every expert
  int32_t scan[kRouteWarps];
  uint16_t counts[kRouteWarps][kMaxExperts];
};

// Sum over the threads in front of this one.
__device__ __forceinline__ int scan_exclusive(int v, int32_t* s_scan, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int in = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, in, o);
    if (lane >= o) in += t;
  }
  if (lane == 31) s_scan[warp] = in;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < kRouteWarps; ++w) {
    if (w < warp) before += s_scan[w];
    all += s_scan[w];
  }
  __syncthreads();
  *total = all;
  return before + in - v;
}

// Places of the entries of tokens [t0, t1): `before` and `total` are thread e's counts of expert e in the chunks in front and in all.
__device__ void place_entries(OrderShared& s, const RouteArgs& a, int t0, int t1, int before, int total, bool write_starts) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int all;
  const int start = scan_exclusive(total, s.scan, &all);
  if (tid < a.experts) {
    s.base[tid] = start + before;
    if (write_starts) a.starts[tid] = start;
  }
  if (write_starts && tid == 0) a.starts[a.experts] = all;
  const int first = t0 * a.k, entries = t1 * a.k;
  for (int i0 = first; i0 < entries; i0 += kRouteThreads) {
    for (int e = lane; e < a.experts; e += 32) s.counts[warp][e] = 0;
    __syncthreads();                                         // base is there too
    const int i = i0 + tid;
    const int e = i < entries ? a.ids[i] : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, e);
    const int rank = __popc(same & ((1u << lane) - 1));
    if (e >= 0 && rank == 0) s.counts[warp][e] = (uint16_t)__popc(same);
    __syncthreads();
    int batch = 0;                                           // thread e's: the batch's entries of expert e
    if (tid < a.experts)
      for (int w = 0; w < kRouteWarps; ++w) {                // counts become the warps' first places
        const int n = s.counts[w][tid];
        s.counts[w][tid] = (uint16_t)batch;
        batch += n;
      }
    __syncthreads();
    if (e >= 0) {
      const int at = s.base[e] + s.counts[warp][e] + rank;
      a.order[at] = i;
      a.place[i] = at;
    }
    __syncthreads();
    if (tid < a.experts) s.base[tid] += batch;
  }
}

template <int V, bool kFull>
__global__ void __launch_bounds__(kRouteThreads)
route_experts_kernel(const __grid_constant__ RouteArgs a) {
  early_start();
  __shared__ int32_t s_counts[kMaxExperts];
  extern __shared__ uint8_t s_more[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, e0 = lane * V;
  for (int e = tid; e < a.experts; e += kRouteThreads) s_counts[e] = 0;
  __syncthreads();
  const int t0 = blockIdx.x * a.chunk, t1 = min(a.tokens, t0 + a.chunk);
  float bias[V], next[V];
#pragma unroll
  for (int v = 0; v < V; ++v) bias[v] = a.bias != nullptr && (kFull || e0 + v < a.experts) ? a.bias[e0 + v] : 0.f;
  auto bring = [&](int t) {                 // a token's logits, one token ahead
    const float* row = a.logits + (int64_t)t * a.l_rs;
    if (V % 4 == 0 && a.vec && (kFull || e0 + V <= a.experts)) {
#pragma unroll
      for (int v = 0; v < V; v += 4) {
        const float4 f = *reinterpret_cast<const float4*>(row + e0 + v);
        next[v] = f.x; next[(v + 1) % V] = f.y; next[(v + 2) % V] = f.z; next[(v + 3) % V] = f.w;
      }
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) next[v] = kFull || e0 + v < a.experts ? row[e0 + v] : -FLT_MAX;
    }
  };
  if (t0 + warp < t1) bring(t0 + warp);
  for (int t = t0 + warp; t < t1; t += kRouteWarps) {
    const float* row = a.logits + (int64_t)t * a.l_rs;
    float z[V];
#pragma unroll
    for (int v = 0; v < V; ++v) z[v] = logit_of(next[v]);
    if (t + kRouteWarps < t1) bring(t + kRouteWarps);
    // choices of this lane and the places they go to; places behind k are not taken
    int id[2] = {0, 0}, rank[2] = {lane, a.k};
    float score[2] = {0.f, 0.f};
    if (!a.lanes || !choose_fast<V, kFull>(z, bias, e0, a, row, rank, id, score)) {
      Chosen c = {{-1, 0}, {0.f, 0.f}};
      if (!a.lanes) c = choose<float, V>(row, e0, a);
      if (__any_sync(0xffffffffu, c.id[0] < 0)) c = choose<double, V>(row, e0, a);
      rank[0] = lane;
      rank[1] = lane + 32;
      id[0] = c.id[0]; id[1] = c.id[1];
      score[0] = c.score[0]; score[1] = c.score[1];
    }
    if (a.renormalize) {
      const bool used[2] = {rank[0] < a.k, rank[1] < a.k};
      const float sum = warp_sum((used[0] ? score[0] : 0.f) + (used[1] ? score[1] : 0.f));
      // a score below fp32's least normal value has fewer bits, or none; over a sum from 2^-20 on that is less than 2^-129 of a weight
      if (sum < 0x1p-20f && __any_sync(0xffffffffu, (used[0] && score[0] < FLT_MIN) || (used[1] && score[1] < FLT_MIN))) {
        const Two w = weights_in_64(row, id[0], id[1], used[0], used[1], a);
        score[0] = w.v[0]; score[1] = w.v[1];
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) score[i] /= sum;
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (rank[i] < a.k) {
        a.ids[(int64_t)t * a.k + rank[i]] = id[i];
        a.weights[(int64_t)t * a.k + rank[i]] = score[i] * a.scale;
        atomicAdd(&s_counts[id[i]], 1);                      // whole numbers: any order gives the same
      }
  }
  __syncthreads();
  if (a.chunks == 1) {
    const int n = tid < a.experts ? s_counts[tid] : 0;
    place_entries(*reinterpret_cast<OrderShared*>(s_more), a, t0, t1, 0, n, true);
  } else {
    for (int e = tid; e < a.experts; e += kRouteThreads) a.counts[(int64_t)blockIdx.x * a.experts + e] = s_counts[e];
  }
}

__global__ void __launch_bounds__(kRouteThreads)
order_experts_kernel(const RouteArgs a) {
  early_start();
  extern __shared__ uint8_t s_more[];
  // the chunks' counts, by as many threads an expert as there are, 16 loads of each under way
  const int tid = threadIdx.x, each = kRouteThreads / a.experts, e = tid % a.experts, part = tid / a.experts;
  int32_t* s_sum = reinterpret_cast<int32_t*>(s_more);       // [2][kMaxExperts]
  for (int i = tid; i < 2 * kMaxExperts; i += kRouteThreads) s_sum[i] = 0;
  __syncthreads();
  int before = 0, total = 0;
  if (part < each) {
#pragma unroll 16
    for (int c = part; c < a.chunks; c += each) {
      const int n = a.counts[(int64_t)c * a.experts + e];
      if (c < (int)blockIdx.x) before += n;
      total += n;
    }
    atomicAdd(&s_sum[e], before);
    atomicAdd(&s_sum[kMaxExperts + e], total);
  }
  __syncthreads();
  before = tid < a.experts ? s_sum[tid] : 0;
  total = tid < a.experts ? s_sum[kMaxExperts + tid] : 0;
  __syncthreads();                                           // the memory is place_entries' next
  const int t0 = blockIdx.x * a.chunk;
  place_entries(*reinterpret_cast<OrderShared*>(s_more), a, t0, min(a.tokens, t0 + a.chunk), before, total, blockIdx.x == 0);
}

// Tokens of a chunk: as few as give every SM one, 32 at least.
int route_chunk(int tokens) {
  const int sms = sm_count_of_current_device(), n = (tokens + sms - 1) / sms;
  if (tokens <= 128) return 128;                             // one launch takes less than two
  return n <= 32 ? 32 : (n + 15) / 16 * 16;
}

template <int V>
int launch_route(RouteArgs a, cudaStream_t st) {
  const int size = a.experts / a.groups;
  a.lanes = a.k < 32 && (a.groups == 1 || (size % V == 0 && (size / V & (size / V - 1)) == 0));
  auto kernel = a.experts == 32 * V ? route_experts_kernel<V, true> : route_experts_kernel<V, false>;
  const size_t more = a.chunks == 1 ? sizeof(OrderShared) : 0;
  launch_early(0, kernel, a.chunks, kRouteThreads, more, st, a);
  return launch_status("route_experts");
}

}  // namespace
}  // namespace atma

using namespace atma;

extern "C" int64_t atma_route_scratch_ints(int tokens, int experts) {
  if (tokens <= 0 || experts <= 0) return 0;
  const int chunk = route_chunk(tokens), chunks = (tokens + chunk - 1) / chunk;
  return chunks == 1 ? 0 : (int64_t)chunks * experts;
}

extern "C" int atma_route_experts(const float* logits, int64_t l_rs, const float* bias, int32_t* ids, float* weights, int32_t* order,
                                  int32_t* place, int32_t* starts, int32_t* scratch, int tokens, int experts, int k, int sigmoid,
                                  int groups, int top_groups, int renormalize, float scale, void* stream) {
  ATMA_REQUIRE(experts > 0 && experts <= kMaxExperts, "route_experts: %d experts, at most %d are served", experts, kMaxExperts);
  ATMA_REQUIRE(tokens >= 0 && k > 0 && (int64_t)tokens * k <= INT32_MAX - kRouteThreads, "route_experts: bad shape");
  ATMA_REQUIRE(groups > 0 && groups <= 64 && experts % groups == 0 && top_groups > 0 && top_groups <= groups,
               "route_experts: %d of %d groups of %d experts", top_groups, groups, experts);
  ATMA_REQUIRE(k <= 64 && k <= experts / groups * top_groups, "route_experts: %d experts of %d", k, experts / groups * top_groups);
  ATMA_REQUIRE(starts != nullptr, "route_experts: null tensors");
  cudaStream_t st = (cudaStream_t)stream;
  if (tokens == 0) {
    ATMA_CUDA_OK(cudaMemsetAsync(starts, 0, (experts + 1) * sizeof(int32_t), st));
    return ATMA_OK;
  }
  ATMA_REQUIRE(logits != nullptr && ids != nullptr && weights != nullptr && order != nullptr && place != nullptr && l_rs >= experts,
               "route_experts: null tensors or overlapping rows");
  const int chunk = route_chunk(tokens), chunks = (tokens + chunk - 1) / chunk;
  ATMA_REQUIRE(chunks == 1 || scratch != nullptr, "route_experts: no scratch memory");
  const RouteArgs a{logits, l_rs, bias, ids, weights, scratch, order, place, starts, tokens, experts, k, groups, top_groups, chunk, chunks, scale,
                    sigmoid != 0, renormalize != 0, (reinterpret_cast<uintptr_t>(logits) & 15) == 0 && l_rs % 4 == 0, false};
  int rc;
  if (experts <= 32) rc = launch_route<1>(a, st);
  else if (experts <= 64) rc = launch_route<2>(a, st);
  else if (experts <= 128) rc = launch_route<4>(a, st);
  else if (experts <= 256) rc = launch_route<8>(a, st);
  else rc = launch_route<16>(a, st);
  if (rc != ATMA_OK || chunks == 1) return rc;
  launch_early(0, order_experts_kernel, dim3(chunks), dim3(kRouteThreads), sizeof(OrderShared), st, a);
  return launch_status("order_experts");
}
