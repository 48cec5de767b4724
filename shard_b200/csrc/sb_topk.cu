// Routing from a caller's logits (expert groups, selection bias, several score functions), and the
// expert order of the routed pairs that the grouped fp4 product reads.
//
// topk_kernel: one warp per token, lane l holds experts C l .. C l + C - 1. Selection values are exact
// without a bias (the scores ascend with the logits, so the logits themselves are compared). With a
// bias, or for groups scored by a sum, they are fp32 sums of rounded scores: after the selection the
// gaps that decided it are compared with the error bound of those sums, and a token with a smaller
// gap is selected again in 64 bits (a fraction of a percent of them). So a selection never hangs on
// how an exponential rounds.
//
// order_kernel: a stable counting sort of the pairs by expert, in blocks of 2048 pairs, no atomics
// on anything the outputs depend on.
#include <cfloat>

#include "sb_device.cuh"
#include "sb_fp4.h"
#include "sb_launch.h"

namespace sb {
namespace topk {

// order-preserving keys; 0: no candidate, 1: a masked expert
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
__device__ __forceinline__ uint32_t warp_kmax(uint32_t k) { return __reduce_max_sync(0xffffffffu, k); }
__device__ __forceinline__ uint64_t warp_kmax(uint64_t k) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
  return ((uint64_t)hi << 32) | lo;
}
template <typename V>
struct KeyOf;
template <>
struct KeyOf<float> { using type = uint32_t; };
template <>
struct KeyOf<double> { using type = uint64_t; };

__device__ __forceinline__ float ex(float v) { return expf(v); }
__device__ __forceinline__ double ex(double v) { return exp(v); }
__device__ __forceinline__ float lg1p(float v) { return log1pf(v); }
__device__ __forceinline__ double lg1p(double v) { return log1p(v); }
__device__ __forceinline__ float sq(float v) { return sqrtf(v); }
__device__ __forceinline__ double sq(double v) { return sqrt(v); }

// score of a logit; mx, sum: the row's softmax statistics
template <typename V>
__device__ __forceinline__ V score(int func, float l, V mx, V sum) {
  const V x = (V)l;
  if (func == SCORE_SOFTMAX) return ex(x - mx) / sum;
  if (func == SCORE_SIGMOID) return (V)1 / ((V)1 + ex(-x));
  return sq((x > (V)0 ? x : (V)0) + lg1p(ex(x > (V)0 ? -x : x)));
}

template <typename V>
__device__ __forceinline__ V warp_add(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <typename V>
__device__ __forceinline__ V warp_most(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const V x = __shfl_xor_sync(0xffffffffu, v, o);
    v = x > v ? x : v;
  }
  return v;
}

__device__ __forceinline__ float logit(const float* p) { return *p; }
__device__ __forceinline__ float logit(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float logit(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// NaN: masked, like -inf and the type's lowest value; +inf counts as the largest fp32 value
__device__ __forceinline__ float clean(float l, float lowest) {
  return l > lowest ? fminf(l, FLT_MAX) : -INFINITY;
}

// The k best (lane j < k: expert of rank j). Returns whether fp32 values may have decided it wrongly.
template <typename V, int C, typename T>
__device__ __forceinline__ bool select(const TopkArgs& a, const T* row, const float (&l)[C], int lane, float mxf,
                                       int& mine) {
  using K = typename KeyOf<V>::type;
  constexpr bool FAST = sizeof(V) == 4;
  const V NONE = -(V)INFINITY;
  const bool biased = a.bias != nullptr;
  const bool sums = a.groups > 1 && a.group_two;
  bool doubt = false;
  V mx = (V)mxf, sum = (V)1, most = (V)0;
  if (a.score == SCORE_SOFTMAX && (biased || sums)) {
    sum = (V)0;
#pragma unroll
    for (int i = 0; i < C; ++i) sum += l[i] > -INFINITY ? ex((V)l[i] - mx) : (V)0;
    sum = warp_add(sum);
  }
  V v[C];      // selection values (NONE: masked or absent)
  V gv[C];     // what the groups are scored by
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int e = lane * C + i;
    v[i] = NONE;
    gv[i] = NONE;
    if (e < a.experts && l[i] > -INFINITY) {
      v[i] = (V)l[i];
      gv[i] = v[i];
      if (biased || sums) {
        const V s = score<V>(a.score, l[i], mx, sum), b = biased ? (V)a.bias[e] : (V)0;
        const V t = s + b;
        if (biased) v[i] = t == t ? t : NONE;
        gv[i] = biased ? v[i] : s;
        const V mag = s + (b < (V)0 ? -b : b);
        most = mag > most ? mag : most;
      }
    }
  }
  const V eps = FAST && (biased || sums) ? (V)2e-6f * warp_most(most) : (V)0;
  uint32_t kept = 0xffffffffu;
  if (a.groups > 1) {
    const int size = a.experts / a.groups;
    V gs = NONE;   // lane g: the score of group g
    const int span = size / C;   // lanes per group when groups begin with lanes
    if (size % C == 0 && (span & (span - 1)) == 0) {
      V b1 = NONE, b2 = NONE;
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const V x = gv[i];
        b2 = x > b1 ? b1 : (x > b2 ? x : b2);
        b1 = x > b1 ? x : b1;
      }
      for (int o = 1; o < span; o <<= 1) {
        const V c1 = __shfl_xor_sync(0xffffffffu, b1, o), c2 = __shfl_xor_sync(0xffffffffu, b2, o);
        b2 = c1 > b1 ? (b1 > c2 ? b1 : c2) : (c1 > b2 ? c1 : b2);
        b1 = c1 > b1 ? c1 : b1;
      }
      const V s = a.group_two && b2 > NONE ? b1 + b2 : b1;
      gs = __shfl_sync(0xffffffffu, s, (lane * span) & 31);
    } else {
      for (int g = 0; g < a.groups; ++g) {
        V b1 = NONE, b2 = NONE;
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const int e = lane * C + i;
          const V x = e >= g * size && e < (g + 1) * size ? gv[i] : NONE;
          b2 = x > b1 ? b1 : (x > b2 ? x : b2);
          b1 = x > b1 ? x : b1;
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const V c1 = __shfl_xor_sync(0xffffffffu, b1, o), c2 = __shfl_xor_sync(0xffffffffu, b2, o);
          b2 = c1 > b1 ? (b1 > c2 ? b1 : c2) : (c1 > b2 ? c1 : b2);
          b1 = c1 > b1 ? c1 : b1;
        }
        if (lane == g) gs = a.group_two && b2 > NONE ? b1 + b2 : b1;
      }
    }
    int rank = 0;
    for (int g = 0; g < a.groups; ++g) {
      const V x = __shfl_sync(0xffffffffu, gs, g);
      rank += x > gs || (x == gs && g < lane) ? 1 : 0;
    }
    const bool here = lane < a.groups, in = here && rank < a.kept;
    kept = __ballot_sync(0xffffffffu, in);
    if (FAST && (biased || sums) && a.kept < a.groups) {
      const V low = -warp_most(in ? -gs : NONE), high = warp_most(here && !in ? gs : NONE);
      doubt = !(low - high > eps) && high > NONE;
    }
  }
  K key[C], best = 0;
  int at = 0;
  {
    const int size = a.experts / a.groups;
    int g = lane * C / size, left = (g + 1) * size - lane * C;   // the expert's group, experts left in it
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const bool in = lane * C + i < a.experts && ((kept >> g) & 1u);
      if (--left == 0) {
        ++g;
        left = size;
      }
      key[i] = in ? (v[i] > NONE ? key_of(v[i]) : (K)1) : (K)0;
      if (key[i] > best) {
        best = key[i];
        at = i;
      }
    }
  }
  const int rounds = FAST && biased ? a.topk + 1 : a.topk;
  K got = 0;
  for (int j = 0; j < rounds; ++j) {
    const K top = warp_kmax(best);
    const int e = (int)__reduce_min_sync(0xffffffffu, best == top ? (uint32_t)(lane * C + at) : 0x7fffffffu);
    if (lane == j) {
      mine = e;
      got = top;
    }
    if (e / C == lane) {   // its owner drops it
      best = 0;
#pragma unroll
      for (int i = 0; i < C; ++i) {
        if (i == at) key[i] = 0;
      }
      int na = 0;
#pragma unroll
      for (int i = 0; i < C; ++i) {
        if (key[i] > best) {
          best = key[i];
          na = i;
        }
      }
      at = na;
    }
  }
  if (FAST && biased) {
    // neighbours in the ranking (lane j and j + 1, to the first one left out): far enough apart, or the
    // same logit and bias, whose order is that of their ids
    const K nk = __shfl_down_sync(0xffffffffu, got, 1);
    const int ne = __shfl_down_sync(0xffffffffu, mine, 1);
    bool near = false;
    if (lane < a.topk && got > 1 && nk > 1) {
      const auto val = [](uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); };
      near = !(val((uint32_t)got) - val((uint32_t)nk) > (float)eps);
      if (near && a.bias[mine] == a.bias[ne] && row[mine] == row[ne]) near = false;
    }
    doubt = doubt || __any_sync(0xffffffffu, near);
  }
  return doubt;
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

// a token's selection in 64 bits (out of line: rare, and its registers are not the others')
template <int C, typename T>
__device__ __noinline__ int select_exact(const TopkArgs& a, const T* row, int lane, float lowest) {
  float l[C];
  load_row<C, T>(a, row, lane, lowest, l);
  int mine = 0;
  select<double, C, T>(a, row, l, lane, row_max<C>(l), mine);
  return mine;
}

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
  const float mx = row_max<C>(l);
  int mine = 0;
  if (select<float, C, T>(a, row, l, lane, mx, mine)) mine = select_exact<C, T>(a, row, lane, lowest);
  // weights of the chosen ones, from their unbiased scores
  float sum = 1.f;
  if (a.score == SCORE_SOFTMAX) {
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < C; ++i) sum += l[i] > -INFINITY ? expf(l[i] - mx) : 0.f;
    sum = warp_sum(sum);
  }
  float w = 0.f;
  if (lane < a.topk) {
    const float x = clean(logit(row + mine), lowest);
    if (x > -INFINITY) w = score<float>(a.score, x, mx, sum);
  }
  if (a.renorm) {
    const float s = warp_sum(w);
    w = s > 0.f ? __fdiv_rn(w, s) : 0.f;
  }
  if (lane < a.topk) {
    a.weights[t * a.topk + lane] = w * a.scale;
    a.ids[t * a.topk + lane] = mine;
  }
}

// ── expert order ───────────────────────────────────────────────────────────────────────────────
constexpr int OW = 8;               // warps of a block
constexpr int OSEG = 256;           // consecutive pairs of a warp
constexpr int OBLOCK = OW * OSEG;

__device__ __forceinline__ int pair_expert(const OrderArgs& a, int64_t p) {
  if (p >= a.pairs) return -1;
  const int64_t e = a.ids[p];
  return e >= 0 && e < a.experts ? (int)e : -1;
}

// cnt[w][e]: pairs of expert e in warp w's segment
__device__ __forceinline__ void segment_counts(const OrderArgs& a, int* cnt, int64_t p0) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < OW * a.experts; i += OW * 32) cnt[i] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < OSEG; i += 32) {
    const int e = pair_expert(a, p0 + warp * OSEG + i + lane);
    if (e >= 0) atomicAdd(&cnt[warp * a.experts + e], 1);
  }
  __syncthreads();
}

__global__ void __launch_bounds__(OW * 32) order_count_kernel(OrderArgs a) {
  extern __shared__ int cnt[];
  pdl_wait();
  pdl_trigger();
  segment_counts(a, cnt, (int64_t)blockIdx.x * OBLOCK);
  for (int e = threadIdx.x; e < a.experts; e += OW * 32) {
    int s = 0;
#pragma unroll
    for (int w = 0; w < OW; ++w) s += cnt[w * a.experts + e];
    a.hist[(int64_t)blockIdx.x * a.experts + e] = s;
  }
}

__global__ void __launch_bounds__(OW * 32) order_kernel(OrderArgs a) {
  extern __shared__ int cnt[];
  __shared__ int wsum[OW];
  __shared__ int total;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t p0 = (int64_t)blockIdx.x * OBLOCK;
  pdl_wait();
  pdl_trigger();
  segment_counts(a, cnt, p0);
  // four experts a thread: all pairs of each, and those in earlier blocks
  int all[4], before[4], mine = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int e = threadIdx.x * 4 + j;
    all[j] = before[j] = 0;
    if (e < a.experts) {
      if (a.blocks == 1) {
#pragma unroll
        for (int w = 0; w < OW; ++w) all[j] += cnt[w * a.experts + e];
      } else {
#pragma unroll 8
        for (int b = 0; b < a.blocks; ++b) {
          const int v = a.hist[(int64_t)b * a.experts + e];
          all[j] += v;
          before[j] += b < (int)blockIdx.x ? v : 0;
        }
      }
    }
    mine += all[j];
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
  for (int j = 0; j < 4; ++j) {
    const int e = threadIdx.x * 4 + j;
    if (e < a.experts) {
      if (blockIdx.x == 0) a.offsets[e] = base;
      int at = base + before[j];
#pragma unroll
      for (int w = 0; w < OW; ++w) {   // counts become each segment's first place
        const int v = cnt[w * a.experts + e];
        cnt[w * a.experts + e] = at;
        at += v;
      }
    }
    base += all[j];
  }
  __syncthreads();
  if (blockIdx.x == 0 && threadIdx.x == 0) a.offsets[a.experts] = total;
  int* cursor = cnt + warp * a.experts;
  for (int i = 0; i < OSEG; i += 32) {
    const int64_t p = p0 + warp * OSEG + i + lane;
    const int e = pair_expert(a, p);
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const int rank = __popc(same & ((1u << lane) - 1u));
    int at = -1;
    if (e >= 0) at = cursor[e] + rank;
    __syncwarp();
    if (e >= 0 && rank == 0) cursor[e] += __popc(same);
    __syncwarp();
    if (p < a.pairs) {
      a.places[p] = at;
      if (at >= 0) a.tokens[at] = (int)(p / a.topk);
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
  if (dtype == SB_F32) return topk::launch_topk_t<float>(a, st);
  if (dtype == SB_F16) return topk::launch_topk_t<__half>(a, st);
  return topk::launch_topk_t<__nv_bfloat16>(a, st);
}

int64_t order_blocks(int64_t pairs) { return (pairs + topk::OBLOCK - 1) / topk::OBLOCK; }

cudaError_t launch_expert_order(const OrderArgs& a, cudaStream_t st) {
  const dim3 grid(a.blocks), block(topk::OW * 32);
  const size_t smem = (size_t)topk::OW * a.experts * sizeof(int);
  if (a.blocks > 1) {
    const cudaError_t e = launch_pdl(topk::order_count_kernel, grid, block, smem, st, a);
    if (e != cudaSuccess) return e;
  }
  return launch_pdl(topk::order_kernel, grid, block, smem, st, a);
}

}  // namespace sb
