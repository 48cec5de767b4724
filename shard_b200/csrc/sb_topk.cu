// Routing from a caller's logits (expert groups, selection bias, several score functions), and the
// expert order of the routed pairs that the grouped fp4 product reads.
//
// topk_kernel: one warp per token, lane l holds experts C l .. C l + C - 1. Selection values are exact
// without a bias (the scores ascend with the logits, so the logits themselves are compared). With a
// bias, or for groups scored by a sum, they are fp32 sums of rounded scores: the gaps that decide are
// compared with the error bounds of the values on their two sides, and where one is smaller the candidates in doubt
// are compared again in 64 bits (a fraction of a percent of the tokens; selecting those tokens anew from 64-bit
// scores of all experts took 20 us of 38). So a selection never hangs on how an exponential rounds.
//
// order_kernel: a stable counting sort of the pairs by expert, in blocks of 2048 pairs, no atomics
// on anything the outputs depend on. Up to eight blocks form a cluster that reads one another's counts in
// shared memory; more leave them in memory by a kernel before, and many have them summed by one between.
#include <cfloat>

#include "sb_device.cuh"
#include "sb_fp4.h"
#include "sb_launch.h"

namespace sb {
namespace topk {

// order-preserving keys; 0: no candidate, 1: a masked expert
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// the two best of (b1 >= b2) and (c1 >= c2)
template <typename V>
__device__ __forceinline__ void merge(V& b1, V& b2, V c1, V c2) {
  const V low = b1 < c1 ? b1 : c1, two = b2 > c2 ? b2 : c2;
  b1 = b1 > c1 ? b1 : c1;
  b2 = low > two ? low : two;
}

__device__ __forceinline__ float rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// sqrt(softplus(l)). Below FAR e^l is a subnormal number or 0, whose root is not: e^(l / 2) is the score to within e^l of itself.
constexpr float FAR = -80.f;
__device__ __forceinline__ float sqrtsoftplus(float l) {
  const float t = expf(l < FAR ? 0.5f * l : -fabsf(l));
  return l < FAR ? t : sqrtf(fmaxf(l, 0.f) + log1pf(t));
}

// The score of a logit: for the selection (each within a few 2^-24 of itself, softmax of the row's largest; sigmoids below
// 2^-126 count as 0), as an output, and in 64 bits; mx, sum: the row's softmax statistics.
__device__ __forceinline__ float score32(int func, float l, float mx, float rsum) {
  if (func == SCORE_SOFTMAX) return l > -INFINITY ? __expf(l - mx) * rsum : 0.f;
  if (func == SCORE_SIGMOID) return rcp(1.f + expf(-l));
  return sqrtsoftplus(l);
}
__device__ __forceinline__ float score_weight(int func, float l, float mx, float sum) {
  if (func == SCORE_SOFTMAX) return __fdiv_rn(expf(l - mx), sum);
  if (func == SCORE_SIGMOID) return l < FAR ? expf(l) : __fdiv_rn(1.f, 1.f + expf(-l));   // (expf(-l) may be inf there)
  return sqrtsoftplus(l);
}
__device__ __noinline__ double score64(int func, float l, double mx, double sum) {
  const double x = (double)l;
  if (func == SCORE_SOFTMAX) return exp(x - mx) / sum;
  if (func == SCORE_SIGMOID) return 1.0 / (1.0 + exp(-x));
  return l < FAR ? exp(0.5 * x) : sqrt(fmax(x, 0.0) + log1p(exp(-fabs(x))));
}

__device__ __forceinline__ float logit(const float* p) { return *p; }
__device__ __forceinline__ float logit(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float logit(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// NaN: masked, like -inf and the type's lowest value; +inf counts as the largest fp32 value
__device__ __forceinline__ float clean(float l, float lowest) {
  return l > lowest ? fminf(l, FLT_MAX) : -INFINITY;
}

template <int C, typename T>
__device__ __forceinline__ void load_row(const TopkArgs& a, const T* row, int lane, float lowest, float (&l)[C]) {
  constexpr int PER = 16 / (int)sizeof(T);
  if (C % PER == 0 && a.vec) {
#pragma unroll
    for (int i = 0; i < C; i += PER) {
      const int e = lane * C + i;
      uint4 w = make_uint4(0u, 0u, 0u, 0u);
      if (e < a.experts) w = __ldg(reinterpret_cast<const uint4*>(row + e));   // experts % PER == 0 with vec
      const T* p = reinterpret_cast<const T*>(&w);
#pragma unroll
      for (int j = 0; j < PER; ++j) l[i + j] = e < a.experts ? clean(logit(p + j), lowest) : -INFINITY;
    }
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int e = lane * C + i;
      l[i] = e < a.experts ? clean(logit(row + e), lowest) : -INFINITY;
    }
  }
}

template <int C>
__device__ __forceinline__ float row_max(const float (&l)[C]) {
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < C; ++i) mx = fmaxf(mx, l[i]);
  return warp_max(mx);
}

// A token's selection with a bias, in 64 bits: lane j < k gets the expert of rank j. Out of line: it is rare, and its
// registers are not the others'.
template <int C, typename T>
__device__ __noinline__ int select_exact(const TopkArgs& a, const T* row, int lane, float lowest) {
  float l[C];
  load_row<C, T>(a, row, lane, lowest, l);
  const double NONE = -(double)INFINITY, mx = (double)row_max<C>(l);
  double sum = 0.0;
#pragma unroll 1
  for (int i = 0; i < C; ++i) sum += l[i] > -INFINITY ? exp((double)l[i] - mx) : 0.0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  double v[C];             // what the experts, and their groups, are compared by
#pragma unroll 1
  for (int i = 0; i < C; ++i) {
    const int e = lane * C + i;
    v[i] = NONE;
    if (e < a.experts && l[i] > -INFINITY) {
      const double t = score64(a.score, l[i], mx, sum) + (double)a.bias[e];
      v[i] = t == t ? t : NONE;
    }
  }
  uint32_t kept = 0xffffffffu;
  const int size = a.size;
  if (a.groups > 1) {
    double gs = NONE;   // lane g: the score of group g
    for (int g = 0; g < a.groups; ++g) {
      double b1 = NONE, b2 = NONE;
#pragma unroll 1
      for (int i = 0; i < C; ++i) {
        const int e = lane * C + i;
        if (e >= g * size && e < (g + 1) * size) merge(b1, b2, v[i], NONE);
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double c1 = __shfl_xor_sync(0xffffffffu, b1, o), c2 = __shfl_xor_sync(0xffffffffu, b2, o);
        merge(b1, b2, c1, c2);
      }
      if (lane == g) gs = a.group_two && b2 > NONE ? b1 + b2 : b1;
    }
    int rank = 0;
    for (int g = 0; g < a.groups; ++g) {
      const double x = __shfl_sync(0xffffffffu, gs, g);
      rank += x > gs || (x == gs && g < lane) ? 1 : 0;
    }
    kept = __ballot_sync(0xffffffffu, lane < a.groups && rank < a.kept);
  }
  int mine = 0;
  uint32_t taken = 0u;   // this lane's experts already chosen
  for (int j = 0; j < a.topk; ++j) {
    // the best left: 2 above masked, 1 masked, 0 none; then the value; then the lower id
    int cls = 0, at = 0;
    double best = NONE;
#pragma unroll 1
    for (int i = 0; i < C; ++i) {
      const int e = lane * C + i;
      const bool in = e < a.experts && ((kept >> (e / size)) & 1u) && !((taken >> i) & 1u);
      const int c = in ? (v[i] > NONE ? 2 : 1) : 0;
      if (c > cls || (c == 2 && v[i] > best)) {
        cls = c;
        best = v[i];
        at = i;
      }
    }
    const int top = __reduce_max_sync(0xffffffffu, cls);
    double b = cls == top ? best : NONE;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) b = fmax(b, __shfl_xor_sync(0xffffffffu, b, o));
    const int w = __ffs(__ballot_sync(0xffffffffu, cls == top && best == b)) - 1;
    const int e = w * C + __shfl_sync(0xffffffffu, at, w);
    if (lane == w) taken |= 1u << at;
    if (lane == j) mine = e;
  }
  return mine;
}

// Descending sorting network (odd-even merges).
template <int C>
__device__ __forceinline__ void sort_desc(uint32_t (&k)[C]) {
#pragma unroll
  for (int p = 1; p < C; p <<= 1)
#pragma unroll
    for (int q = p; q > 0; q >>= 1)
#pragma unroll
      for (int j = q % p; j + q < C; j += 2 * q)
#pragma unroll
        for (int i = 0; i < q; ++i)
          if (i + j + q < C && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
            const uint32_t x = k[i + j], y = k[i + j + q];
            k[i + j] = max(x, y);
            k[i + j + q] = min(x, y);
          }
}

// Exact values of this lane's experts in `mask` (bits: places in the lane), the two best of them.
template <int C, typename T>
__device__ __forceinline__ void best_exact(const TopkArgs& a, const T* row, int lane, float lowest, uint32_t mask, double mx,
                                           double sum, double& b1, double& b2) {
  while (__any_sync(0xffffffffu, mask != 0u)) {
    if (mask != 0u) {
      const int e = lane * C + __ffs(mask) - 1;
      mask &= mask - 1u;
      const double s = score64(a.score, clean(logit(row + e), lowest), mx, sum);
      merge(b1, b2, a.bias != nullptr ? s + (double)a.bias[e] : s, -(double)INFINITY);
    }
    __syncwarp();
  }
}

template <int C, int FUNC>
__device__ __forceinline__ void scores32(const float (&l)[C], float mx, float rsum, float (&s)[C]) {
#pragma unroll
  for (int i = 0; i < C; ++i) s[i] = score32(FUNC, l[i], mx, rsum);
}

// How far fp32 selection values may be from the real ones: a score by k times the row's largest, its sum with a bias (and that of
// two such values) by a rounding more of itself. In units of 2^-24: sigmoid 7 (the exponential 4, the sum 1, the reciprocal 2),
// sqrtsoftplus 5; softmax 4 for the exponential and its argument, 3 for the division, 20 for the exponentials in
// the sum (each 2 (2 + 1.173 d) and d for its argument, d below the largest logit; of 1024 experts at one d the mean
// is largest at d = 5.4) and C + 4 for the C + 5 additions of a lane and the warp; the factor of 6.1e-8 is 2% above
// 2^-24. Where all scores are tiny: 2.4e-38 for one that counts as 0. value +- of(value) ascends with the value, so that
// neighbours in a ranking are all that has to be compared.
struct Bound {
  float ks;   // k times the largest score
  __device__ __forceinline__ float rounding(float v) const { return 6.1e-8f * fminf(fabsf(v), FLT_MAX); }
  __device__ __forceinline__ float of(float v) const { return rounding(v) + ks; }
  // a > b for certain (never of two infinities)
  __device__ __forceinline__ bool above(float a, float b) const { return a - b > of(a) + of(b); }
};
template <int C>
__device__ __forceinline__ float bound_of_scores(int func, float largest) {
  return 6.1e-8f * (func == SCORE_SOFTMAX ? (float)(C + 32) : 8.f) * largest + 2.4e-38f;
}

template <int C>
__device__ __forceinline__ void load_bias(const TopkArgs& a, int lane, float (&b)[C]) {
  if (C % 4 == 0 && a.vec_bias) {
#pragma unroll
    for (int i = 0; i < C; i += 4) {
      const int e = lane * C + i;
      float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
      if (e < a.experts) w = __ldg(reinterpret_cast<const float4*>(a.bias + e));
      b[i] = w.x;
      b[i + (C > 1)] = w.y;
      b[i + (C > 2) * 2] = w.z;
      b[i + (C > 2) * 3] = w.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i) b[i] = lane * C + i < a.experts ? __ldg(a.bias + lane * C + i) : 0.f;
  }
}

// softmax statistics in 64 bits
template <int C>
__device__ __forceinline__ double sum_exact(const TopkArgs& a, const float (&l)[C], float mx) {
  double sum = 0.0;
  if (a.score == SCORE_SOFTMAX) {
#pragma unroll 1
    for (int i = 0; i < C; ++i) sum += l[i] > -INFINITY ? exp((double)l[i] - (double)mx) : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  return sum;
}

// The groups kept, from exact scores of the experts that can be among a group's two best: near[i], those within the bounds
// of its second best fp32 value (rare, out of line).
template <int C, typename T>
__device__ __noinline__ uint32_t kept_exact(const TopkArgs& a, const T* row, int lane, float lowest, float mx, uint32_t near) {
  const double NONE = -(double)INFINITY;
  float l[C];
  load_row<C, T>(a, row, lane, lowest, l);
  const double sum = sum_exact<C>(a, l, mx);
  double gs = NONE;
  if (a.span > 0) {
    double b1 = NONE, b2 = NONE;
    best_exact<C, T>(a, row, lane, lowest, near, (double)mx, sum, b1, b2);
    for (int o = 1; o < a.span; o <<= 1) {
      const double c1 = __shfl_xor_sync(0xffffffffu, b1, o), c2 = __shfl_xor_sync(0xffffffffu, b2, o);
      merge(b1, b2, c1, c2);
    }
    gs = __shfl_sync(0xffffffffu, a.group_two && b2 > NONE ? b1 + b2 : b1, (lane * a.span) & 31);
  } else {
    for (int g = 0; g < a.groups; ++g) {
      const int lo = min(max(g * a.size - lane * C, 0), C), hi = min(max((g + 1) * a.size - lane * C, 0), C);
      const uint32_t in = (uint32_t)((1ull << hi) - (1ull << lo));
      double b1 = NONE, b2 = NONE;
      best_exact<C, T>(a, row, lane, lowest, near & in, (double)mx, sum, b1, b2);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double c1 = __shfl_xor_sync(0xffffffffu, b1, o), c2 = __shfl_xor_sync(0xffffffffu, b2, o);
        merge(b1, b2, c1, c2);
      }
      if (lane == g) gs = a.group_two && b2 > NONE ? b1 + b2 : b1;
    }
  }
  int rank = 0;
  for (int g = 0; g < a.groups; ++g) {
    const double x = __shfl_sync(0xffffffffu, gs, g);
    rank += x > gs || (x == gs && g < lane) ? 1 : 0;
  }
  return __ballot_sync(0xffffffffu, lane < a.groups && rank < a.kept);
}

// Lanes 0 .. n - 1 hold candidates in the order of their fp32 values (cls: 2 an expert, 1 a masked one, 0 none), all
// that can be among the k best. Returns lane j's expert by exact values (rare, out of line).
template <int C, typename T>
__device__ __noinline__ int order_exact(const TopkArgs& a, const T* row, int lane, float lowest, float mx, int mine, int cls,
                                        int n) {
  float l[C];
  load_row<C, T>(a, row, lane, lowest, l);
  const double sum = sum_exact<C>(a, l, mx);
  double v = -(double)INFINITY;
  if (lane < n && cls == 2) v = score64(a.score, clean(logit(row + mine), lowest), (double)mx, sum) + (double)a.bias[mine];
  int rank = 0;
  for (int i = 0; i < n; ++i) {
    const double x = __shfl_sync(0xffffffffu, v, i);
    const int c = __shfl_sync(0xffffffffu, cls, i), e = __shfl_sync(0xffffffffu, mine, i);
    rank += c > cls || (c == cls && (x > v || (x == v && e < mine))) ? 1 : 0;
  }
  int out = mine;
  for (int i = 0; i < n; ++i) {
    const int r = __shfl_sync(0xffffffffu, lane < n ? rank : -1, i), e = __shfl_sync(0xffffffffu, mine, i);
    if (r == lane) out = e;
  }
  return out;
}

// The k best: lane j < k gets the expert of rank j. Each lane sorts its C keys once (without their ids: two
// instructions a step); a round then takes the largest head of all lanes, and lanes hold consecutive experts, so
// that of equal keys the lowest lane's is the lowest id. The places of the chosen keys in their lanes are found
// afterwards, for all of them at once.
template <int C, typename T>
__device__ __forceinline__ int select(const TopkArgs& a, const T* row, const float (&l)[C], int lane, float lowest, float mx,
                                      float sum) {
  const bool biased = a.bias != nullptr, scored = biased || (a.groups > 1 && a.group_two);
  float v[C], gv[C];
  Bound err = {0.f};
  if (scored) {
    // (one branch for the whole row, not one per expert)
    if (a.score == SCORE_SOFTMAX) scores32<C, SCORE_SOFTMAX>(l, mx, rcp(sum), gv);
    else if (a.score == SCORE_SIGMOID) scores32<C, SCORE_SIGMOID>(l, mx, 1.f, gv);
    else scores32<C, SCORE_SQRTSOFTPLUS>(l, mx, 1.f, gv);
    float largest = 0.f;
    if (a.score == SCORE_SOFTMAX) {
      largest = rcp(sum);
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) largest = fmaxf(largest, gv[i]);
      largest = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(largest)));
    }
    err.ks = bound_of_scores<C>(a.score, largest);
    if (biased) {
      float b[C];
      load_bias<C>(a, lane, b);
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const float t = gv[i] + b[i];
        v[i] = gv[i] = l[i] > -INFINITY && t == t ? t : -INFINITY;   // (a bias of -inf masks its expert)
      }
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        gv[i] = l[i] > -INFINITY ? gv[i] : -INFINITY;
        v[i] = l[i];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] = gv[i] = l[i];
  }
  uint32_t kept = 0xffffffffu;
  if (a.groups > 1) {
    float gs = -INFINITY, ge = 0.f;   // lane g: the score of group g, and its bound
    // This lane's experts that may be among their group's two best. (Four bounds of the second best: two of its own, and
    // two for an expert below it.)
    uint32_t near = 0u;
    // (halves in place of sums: two biases of the lowest value add up to -inf, which is a masked group's)
    const float part = a.group_two ? 0.5f : 1.f;
    auto group = [&](float b1, float b2, float& score, float& bound) {
      const bool two = a.group_two && b2 > -INFINITY;
      score = part * b1 + (two ? part * b2 : 0.f);
      bound = part * (err.of(b1) + (two ? err.of(b2) : 0.f)) + err.rounding(score);
    };
    if (a.span > 0) {
      float b1 = -INFINITY, b2 = -INFINITY;
#pragma unroll
      for (int i = 0; i < C; ++i) merge(b1, b2, gv[i], -INFINITY);
      for (int o = 1; o < a.span; o <<= 1) {
        const float c1 = __shfl_xor_sync(0xffffffffu, b1, o), c2 = __shfl_xor_sync(0xffffffffu, b2, o);
        merge(b1, b2, c1, c2);
      }
      group(b1, b2, gs, ge);
      gs = __shfl_sync(0xffffffffu, gs, (lane * a.span) & 31);
      ge = __shfl_sync(0xffffffffu, ge, (lane * a.span) & 31);
      const float from = b2 - 4.f * err.of(b2);
#pragma unroll
      for (int i = 0; i < C; ++i) near |= gv[i] > -INFINITY && !(gv[i] < from) ? 1u << i : 0u;
    } else {
      for (int g = 0; g < a.groups; ++g) {
        float b1 = -INFINITY, b2 = -INFINITY;
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const int e = lane * C + i;
          merge(b1, b2, e >= g * a.size && e < (g + 1) * a.size ? gv[i] : -INFINITY, -INFINITY);
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const float c1 = __shfl_xor_sync(0xffffffffu, b1, o), c2 = __shfl_xor_sync(0xffffffffu, b2, o);
          merge(b1, b2, c1, c2);
        }
        if (lane == g) group(b1, b2, gs, ge);
        const float from = b2 - 4.f * err.of(b2);
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const int e = lane * C + i;
          if (e >= g * a.size && e < (g + 1) * a.size && gv[i] > -INFINITY && !(gv[i] < from)) near |= 1u << i;
        }
      }
    }
    uint32_t gk = lane < a.groups ? key_of(gs) : 0u;
    kept = 0u;
    for (int j = 0; j < a.kept; ++j) {
      const uint32_t top = __reduce_max_sync(0xffffffffu, gk);
      const int w = __ffs(__ballot_sync(0xffffffffu, gk == top)) - 1;
      kept |= 1u << w;
      if (lane == w) gk = 0u;
    }
    if (scored && a.kept < a.groups) {
      // the least that a kept group can be, the most of the others (masked ones are what they are)
      const bool in = (kept >> lane) & 1u;
      const uint32_t low = __reduce_min_sync(0xffffffffu, in ? key_of(gs - ge) : 0xffffffffu);
      const uint32_t high = __reduce_max_sync(0xffffffffu, !in && gk > key_of(-INFINITY) ? key_of(gs + ge) : 0u);
      if (high >= low) kept = kept_exact<C, T>(a, row, lane, lowest, mx, near);
    }
  }
  uint32_t key[C], own[C];
  if (a.span > 0) {
    const bool in = (kept >> (a.groups == 1 ? 0 : lane >> a.span_log)) & 1u;
#pragma unroll
    for (int i = 0; i < C; ++i)
      own[i] = in && lane * C + i < a.experts ? (v[i] > -INFINITY ? key_of(v[i]) : 1u) : 0u;
  } else {
    int g = lane * C / a.size, left = (g + 1) * a.size - lane * C;   // the expert's group, experts left in it
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const bool in = lane * C + i < a.experts && ((kept >> g) & 1u);
      if (--left == 0) {
        ++g;
        left = a.size;
      }
      own[i] = in ? (v[i] > -INFINITY ? key_of(v[i]) : 1u) : 0u;
    }
  }
#pragma unroll
  for (int i = 0; i < C; ++i) key[i] = own[i];
  sort_desc<C>(key);
  uint32_t got = 0u;
  int from = 0;
  auto round = [&](int j) {
    const uint32_t top = __reduce_max_sync(0xffffffffu, key[0]);
    const int w = __ffs(__ballot_sync(0xffffffffu, key[0] == top)) - 1;
    if (lane == j) {
      got = top;
      from = w;
    }
    if (lane == w) {
#pragma unroll
      for (int i = 0; i + 1 < C; ++i) key[i] = key[i + 1];
      key[C - 1] = 0u;
    }
    return top;
  };
  // the place of the chosen key in its lane: of several equal ones, taken in turn, the n-th
  auto expert = [&]() {
    uint32_t at = 0u;
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (__shfl_sync(0xffffffffu, own[i], from) == got) at |= 1u << i;
    const bool several = got != 0u && (at & (at - 1u)) != 0u;
    if (__any_sync(0xffffffffu, several)) {
      const uint32_t same = __match_any_sync(0xffffffffu, several ? ((uint64_t)got << 5) | (uint64_t)from : (uint64_t)lane);
      for (int n = __popc(same & ((1u << lane) - 1u)); n > 0; --n) at &= at - 1u;
    }
    return from * C + __ffs(at) - 1;
  };
  const int rounds = biased ? a.topk + 1 : a.topk;
  for (int j = 0; j < rounds; ++j) round(j);
  int mine = expert();
  if (biased) {
    // Neighbours in the ranking, to the first one left out: far enough apart, or the same logit and bias, whose
    // order is that of their ids. Else all that may belong to the k best are ordered by their exact values.
    const uint32_t nk = __shfl_down_sync(0xffffffffu, got, 1);
    const int ne = __shfl_down_sync(0xffffffffu, mine, 1);
    const bool near = lane < a.topk && got > 1u && nk > 1u && !err.above(value_of(got), value_of(nk));
    const bool other = near && !(a.bias[mine] == a.bias[ne] && row[mine] == row[ne]);
    const uint32_t others = __ballot_sync(0xffffffffu, other), nears = __ballot_sync(0xffffffffu, near);
    if (others != 0u || ((nears >> (a.topk - 1)) & 1u)) {
      const uint32_t last = __shfl_sync(0xffffffffu, got, a.topk - 1);
      uint32_t top = __shfl_sync(0xffffffffu, got, a.topk);
      int n = rounds;
      while (n < 32 && last > 1u && top > 1u && !err.above(value_of(last), value_of(top))) top = round(n++);
      if (last > 1u && top > 1u && !err.above(value_of(last), value_of(top))) return select_exact<C, T>(a, row, lane, lowest);
      mine = expert();
      // nothing but equals of the last one behind it: the ids order them, too
      const int ml = __shfl_sync(0xffffffffu, mine, a.topk - 1);
      const bool apart = lane >= a.topk && lane < n - 1 && !(a.bias[mine] == a.bias[ml] && row[mine] == row[ml]);
      if (others == 0u && !__any_sync(0xffffffffu, apart)) return mine;
      mine = order_exact<C, T>(a, row, lane, lowest, mx, mine, lane < n ? (got > 1u ? 2 : (int)got) : 0, n);
    }
  }
  return mine;
}

// Chosen scores over their sum where fp32 scores lose bits or vanish (sigmoids of logits below -69, softmax of experts that far
// below one that is not chosen): in 64 bits, each score over e^(the largest chosen logit) before they are added (rare,
// out of line). x: the lane's chosen logit, -inf: none, or masked.
__device__ __noinline__ float far_weight(int func, float x) {
  const double top = (double)warp_max(x), c = func == SCORE_SOFTMAX ? top : fmin(top, 0.0), l = (double)x;
  double e = 0.0;
  if (x > -INFINITY) {
    if (func == SCORE_SOFTMAX) e = exp(l - c);
    else if (func == SCORE_SIGMOID) e = x < 0.f ? exp(l - c) / (1.0 + exp(l)) : 1.0 / (1.0 + exp(-l));
    else e = x < FAR ? exp(0.5 * (l - c)) : sqrt(fmax(l, 0.0) + log1p(exp(-fabs(l)))) * exp(-0.5 * c);
  }
  double sum = e;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return (float)(e / sum);
}

// One warp per token; the chain of its rounds and its instructions bound it.
template <int C, typename T>
__global__ void __launch_bounds__(128) topk_kernel(TopkArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  pdl_wait();
  pdl_trigger();
  if (t >= a.tokens) return;
  const float lowest = sizeof(T) == 4 ? -FLT_MAX : a.lowest;
  const T* row = reinterpret_cast<const T*>(a.logits) + t * a.stride;
  float l[C];
  load_row<C, T>(a, row, lane, lowest, l);
  float mx = 0.f, sum = 1.f;
  if (a.score == SCORE_SOFTMAX) {
    mx = row_max<C>(l);
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < C; ++i) sum += l[i] > -INFINITY ? __expf(l[i] - mx) : 0.f;
    sum = warp_sum(sum);
  }
  const int mine = select<C, T>(a, row, l, lane, lowest, mx, sum);
  // weights of the chosen ones, from their unbiased scores
  float w = 0.f, x = -INFINITY;
  if (lane < a.topk) {
    x = clean(logit(row + mine), lowest);
    if (x > -INFINITY) w = score_weight(a.score, x, mx, sum);
  }
  if (a.renorm) {
    if (__any_sync(0xffffffffu, x > -INFINITY && w < 1e-30f)) {
      w = far_weight(a.score, x);
    } else {
      float s = w;   // lanes 16 and above hold zeros
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      w = s > 0.f ? __fdiv_rn(w, s) : 0.f;
    }
  }
  if (lane < a.topk) {
    a.weights[t * a.topk + lane] = w * a.scale;
    a.ids[t * a.topk + lane] = mine;
  }
}

// ── expert order ───────────────────────────────────────────────────────────────────────────────
constexpr int OSTEP = 8;            // pairs of a thread
constexpr int OSEG = 32 * OSTEP;    // consecutive pairs of a warp
constexpr int OW = 8;               // warps of a block (one block of 32 for 8192 pairs: 16 us, four of 8: 7)
constexpr int OBLOCK = OW * OSEG;

// The warp's pairs' experts (-1: none), all loads in flight at once, and cnt[w][e], the pairs of expert e
// in warp w's segment.
__device__ __forceinline__ void segment(const OrderArgs& a, int* cnt, int64_t p0, int (&ex)[OSTEP]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t id[OSTEP];
#pragma unroll
  for (int i = 0; i < OSTEP; ++i) {
    const int64_t p = p0 + warp * OSEG + i * 32 + lane;
    id[i] = p < a.pairs ? a.ids[p] : -1;
  }
  for (int i = threadIdx.x; i < OW * a.experts; i += OW * 32) cnt[i] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < OSTEP; ++i) {
    ex[i] = id[i] >= 0 && id[i] < a.experts ? (int)id[i] : -1;
    if (ex[i] >= 0) atomicAdd(&cnt[warp * a.experts + ex[i]], 1);
  }
  __syncthreads();
}

__global__ void __launch_bounds__(OW * 32) order_count_kernel(OrderArgs a) {
  extern __shared__ int cnt[];
  int ex[OSTEP];
  pdl_wait();
  pdl_trigger();
  segment(a, cnt, (int64_t)blockIdx.x * OBLOCK, ex);
  for (int e = threadIdx.x; e < a.experts; e += OW * 32) {
    int s = 0;
#pragma unroll
    for (int w = 0; w < OW; ++w) s += cnt[w * a.experts + e];
    a.hist[(int64_t)blockIdx.x * a.experts + e] = s;
  }
}

// Counts [blocks][experts] to the counts of the blocks before, in place, and behind them each expert's total. A block
// takes SE experts (a row's 32 bytes), its threads SC runs of neighbouring counts.
constexpr int SE = 8, SC = 128;

__global__ void __launch_bounds__(SE * SC) order_scan_kernel(OrderArgs a) {
  __shared__ int part[SE][SC];
  const int x = threadIdx.x % SE, run = threadIdx.x / SE, e = blockIdx.x * SE + x;
  const bool in = e < a.experts;
  const int b0 = (int)((int64_t)a.blocks * run / SC), b1 = (int)((int64_t)a.blocks * (run + 1) / SC);
  int* h = a.hist + (in ? e : 0);
  pdl_wait();
  pdl_trigger();
  int sum = 0;
  if (in) {
#pragma unroll 8
    for (int b = b0; b < b1; ++b) sum += h[(int64_t)b * a.experts];
  }
  part[x][run] = sum;
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp < SE) {   // the runs of one expert
    constexpr int PER = SC / 32;
    int v[PER], mine = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      v[j] = part[warp][lane * PER + j];
      mine += v[j];
    }
    int at = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += u;
    }
    if (lane == 31 && blockIdx.x * SE + warp < a.experts)
      a.hist[(int64_t)a.blocks * a.experts + blockIdx.x * SE + warp] = at;
    at -= mine;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      part[warp][lane * PER + j] = at;
      at += v[j];
    }
  }
  __syncthreads();
  int at = part[x][run];
  for (int b = b0; in && b < b1; b += 8) {
    int v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = b + j < b1 ? h[(int64_t)(b + j) * a.experts] : 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (b + j < b1) h[(int64_t)(b + j) * a.experts] = at;
      at += v[j];
    }
  }
}

constexpr int OCLUSTER = 8;         // blocks of a cluster at most
// Up to so many blocks each adds up the counts before its own; more would read a quadratic number of them (256 experts, 64
// blocks: 9.0 us, 9.1 with the scan; 32: 7.8 and 8.8; 256: 19 and 14; 4096, 8.4 M pairs: 1194 and 114).
constexpr int OSCAN = 64;

__device__ __forceinline__ int peer_int(const int* p, int rank) {
  uint32_t r;
  int v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
  asm volatile("ld.shared::cluster.b32 %0, [%1];\n" : "=r"(v) : "r"(r) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;\n" ::: "memory");
}

template <bool CLUSTER>
__global__ void __launch_bounds__(OW * 32) order_kernel(OrderArgs a) {
  extern __shared__ int cnt[];               // [OW][experts] counts, [experts] all pairs of each, [experts] this block's
  __shared__ int wsum[OW];
  __shared__ int total;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t p0 = (int64_t)blockIdx.x * OBLOCK;
  int* all = cnt + OW * a.experts;
  int ex[OSTEP];
  // After order_count_kernel (and order_scan_kernel) this starts while they run, which in turn began when the ids were
  // written: they can be read before the wait, the counts in memory after it.
  if (CLUSTER || a.blocks == 1) pdl_wait();
  segment(a, cnt, p0, ex);
  if (!CLUSTER && a.blocks > 1) pdl_wait();
  pdl_trigger();
  if constexpr (CLUSTER) {
    int* mine = all + a.experts;
    for (int e = threadIdx.x; e < a.experts; e += OW * 32) {
      int s = 0;
#pragma unroll
      for (int w = 0; w < OW; ++w) s += cnt[w * a.experts + e];
      mine[e] = s;
    }
    cluster_sync();
  }
  // counts become each segment's first place after the expert's base (below)
  for (int e = threadIdx.x; e < a.experts; e += OW * 32) {
    int sum = 0, at = 0;
    if constexpr (CLUSTER) {
#pragma unroll
      for (int b = 0; b < OCLUSTER; ++b) {
        if (b < a.blocks) {
          const int v = peer_int(all + a.experts + e, b);
          sum += v;
          at += b < (int)blockIdx.x ? v : 0;
        }
      }
    } else if (a.scanned) {
      at = a.hist[(int64_t)blockIdx.x * a.experts + e];
      sum = a.hist[(int64_t)a.blocks * a.experts + e];
    } else if (a.blocks > 1) {
#pragma unroll 16
      for (int b = 0; b < a.blocks; ++b) {
        const int v = a.hist[(int64_t)b * a.experts + e];
        sum += v;
        at += b < (int)blockIdx.x ? v : 0;
      }
    }
    int here = 0;
#pragma unroll
    for (int w = 0; w < OW; ++w) {
      const int v = cnt[w * a.experts + e];
      cnt[w * a.experts + e] = at + here;
      here += v;
    }
    all[e] = a.blocks > 1 ? sum : here;
  }
  if constexpr (CLUSTER) cluster_sync();   // all counts are read before a block ends
  __syncthreads();
  // exclusive scan of the experts' totals
  constexpr int PER = 1024 / (OW * 32);   // experts a thread
  int four[PER], mine = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int e = threadIdx.x * PER + j;
    four[j] = e < a.experts ? all[e] : 0;
    mine += four[j];
  }
  int inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 31) wsum[warp] = inc;
  __syncthreads();
  int base = inc - mine;
  for (int w = 0; w < warp; ++w) base += wsum[w];
  if (threadIdx.x == OW * 32 - 1) total = base + mine;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int e = threadIdx.x * PER + j;
    if (e < a.experts) {
      if (blockIdx.x == 0) a.offsets[e] = base;
      all[e] = base;
    }
    base += four[j];
  }
  __syncthreads();
  if (blockIdx.x == 0 && threadIdx.x == 0) a.offsets[a.experts] = total;
  int* cursor = cnt + warp * a.experts;
  unsigned same[OSTEP];
#pragma unroll
  for (int i = 0; i < OSTEP; ++i) same[i] = __match_any_sync(0xffffffffu, ex[i]);
#pragma unroll
  for (int i = 0; i < OSTEP; ++i) {
    const int64_t p = p0 + warp * OSEG + i * 32 + lane;
    const int rank = __popc(same[i] & ((1u << lane) - 1u));
    int at = -1;
    if (ex[i] >= 0) at = cursor[ex[i]] + rank;
    __syncwarp();
    if (ex[i] >= 0 && rank == 0) cursor[ex[i]] += __popc(same[i]);
    __syncwarp();
    if (p < a.pairs) {
      if (at >= 0) {
        at += all[ex[i]];
        a.tokens[at] = (int)((unsigned)p / (unsigned)a.topk);
      }
      a.places[p] = at;
      if (p >= total) a.tokens[p] = -1;   // behind the last routed pair
    }
  }
}

template <typename T>
static cudaError_t launch_topk_t(const TopkArgs& a, cudaStream_t st) {
  const dim3 grid((unsigned)((a.tokens + 3) / 4)), block(128);
  const int c = (a.experts + 31) / 32;
  if (c <= 1) return launch_pdl(topk_kernel<1, T>, grid, block, 0, st, a);
  if (c <= 2) return launch_pdl(topk_kernel<2, T>, grid, block, 0, st, a);
  if (c <= 4) return launch_pdl(topk_kernel<4, T>, grid, block, 0, st, a);
  if (c <= 8) return launch_pdl(topk_kernel<8, T>, grid, block, 0, st, a);
  if (c <= 16) return launch_pdl(topk_kernel<16, T>, grid, block, 0, st, a);
  return launch_pdl(topk_kernel<32, T>, grid, block, 0, st, a);
}

}  // namespace topk

cudaError_t launch_topk(const TopkArgs& args, int dtype, cudaStream_t st) {
  TopkArgs a = args;
  const int es = dtype == SB_F32 ? 4 : 2, per = 16 / es;
  a.vec = (reinterpret_cast<uintptr_t>(a.logits) & 15u) == 0 && a.experts % per == 0 && (a.stride * es) % 16 == 0;
  a.lowest = dtype == SB_F16 ? -65504.f : -3.3895313892515355e38f;
  a.vec_bias = (reinterpret_cast<uintptr_t>(a.bias) & 15u) == 0 && a.experts % 4 == 0;
  // lanes per group, when groups begin with lanes and a power of two of them makes one
  int c = 1;
  while (32 * c < a.experts) c *= 2;
  a.size = a.experts / a.groups;
  const int span = a.size / c;
  a.span = a.groups == 1 ? 32 : (a.size % c == 0 && (span & (span - 1)) == 0 ? span : 0);
  a.span_log = 0;
  while ((2 << a.span_log) <= a.span) ++a.span_log;
  if (dtype == SB_F32) return topk::launch_topk_t<float>(a, st);
  if (dtype == SB_F16) return topk::launch_topk_t<__half>(a, st);
  return topk::launch_topk_t<__nv_bfloat16>(a, st);
}

int64_t order_blocks(int64_t pairs) { return (pairs + topk::OBLOCK - 1) / topk::OBLOCK; }
int64_t order_counts(int64_t pairs) {
  const int64_t b = order_blocks(pairs);
  return b > topk::OCLUSTER ? b + (b > topk::OSCAN ? 1 : 0) : 0;   // (and the totals)
}

cudaError_t launch_expert_order(const OrderArgs& args, cudaStream_t st) {
  OrderArgs a = args;
  a.blocks = (int)(a.pairs > 0 ? order_blocks(a.pairs) : 1);
  const dim3 grid(a.blocks), block(topk::OW * 32);
  const size_t smem = (size_t)(topk::OW + 2) * a.experts * sizeof(int);
  if (a.blocks > 1 && a.blocks <= topk::OCLUSTER) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.blocks;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, topk::order_kernel<true>, a);
  }
  if (a.blocks > 1) {
    cudaError_t e = launch_pdl(topk::order_count_kernel, grid, block, smem, st, a);
    a.scanned = a.blocks > topk::OSCAN;
    if (e == cudaSuccess && a.scanned)
      e = launch_pdl(topk::order_scan_kernel, dim3((a.experts + topk::SE - 1) / topk::SE), dim3(topk::SE * topk::SC), 0, st, a);
    if (e != cudaSuccess) return e;
  }
  return launch_pdl(topk::order_kernel<false>, grid, block, smem, st, a);
}

}  // namespace sb
