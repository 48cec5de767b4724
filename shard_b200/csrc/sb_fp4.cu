// Microscaled 4-bit floating point: quantisation of activations, its inverse, and the scale layout
// of the fp4 x fp4 products (sb_fp4mm.cu).
//
//   MXFP4  per 32 values: s = 2^t, t the smallest integer with amax <= 6 2^t (t >= -126)
//   NVFP4  per 16 values: s = e4m3(min(448, amax / (6 ts))), ts the fp32 tensor scale: the caller's, or
//          one per row, max(2^-126, amax_row / 2688)
//   q = e2m1(x / (s ts)) to nearest, ties to the even code, saturating at 6
//
// Quotients are rounded as the real quotient is: a plain fp32 division may land on a border between
// two codes that the real number only comes near, so each value is rounded from both ends of an
// interval around its quotient, and where these differ the border is compared exactly. A block that
// holds a non-finite value gets a NaN scale and zero codes, and does not count for its row's scale.
//
// Operand layout. Codes are row-major, row r at r * kp / 2, kp = K rounded up to 32 (zero codes behind
// K). Scales lie in atoms of 128 rows x 4 scales, 512 bytes, the source form of the scale-factor copy
// into tensor memory: row r's word at 16 (r % 32) + 4 (r / 32 % 4); atoms along K, then row blocks.
// With expert groups, group e starts at row block offsets[e] / 128 + e, so that every group starts
// its own atoms and any row finds its place from the offsets alone.
//
// Both directions are bound by HBM at prompt sizes and by launch latency at one row.
#include <type_traits>

#include "sb_device.cuh"
#include "sb_fp4.h"
#include "sb_launch.h"

namespace sb {
namespace fp4 {

// eight floats -> eight e2m1 codes, value 0 in the low nibble
__device__ __forceinline__ uint32_t cvt8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n .reg .b8 b0, b1, b2, b3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
      " mov.b32 %0, {b0, b1, b2, b3};\n}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// (a x, b x): two fp32 products in one instruction
__device__ __forceinline__ void mul2(float a, float b, float x, float& ra, float& rb) {
  asm("{\n .reg .b64 u, v, w;\n mov.b64 u, {%2, %3};\n mov.b64 v, {%4, %4};\n mul.rn.f32x2 w, u, v;\n"
      " mov.b64 {%0, %1}, w;\n}"
      : "=f"(ra), "=f"(rb)
      : "f"(a), "f"(b), "f"(x));
}

// the border between e2m1 magnitudes c and c + 1
__device__ __forceinline__ float border(uint32_t c) {
  return c < 4 ? 0.25f + 0.5f * (float)c : (c == 4 ? 2.5f : (c == 5 ? 3.5f : 5.0f));
}

// Tensor scales for which fp32 arithmetic decides exactly: neither they nor their products with any block scale
// under- or overflow.
__device__ __forceinline__ bool mid_range(float ts) { return ts >= 7.9e-28f && ts <= 1.2e27f; }

// 1 / v within 2^-22, v in the middle of the range
__device__ __forceinline__ float rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// e4m3 code of min(448, a / (6 ts))
__device__ __noinline__ uint32_t scale_exact(float a, float ts) {
  const double v = (double)a / (6.0 * (double)ts);
  uint32_t lo = 0, hi = 126;   // largest code not above v (e4m3 codes ascend with their values)
  if (v >= 448.0) return 126;
  while (hi - lo > 1) {
    const uint32_t c = (lo + hi) >> 1;
    if ((double)e4m3_to_f32(c) <= v) lo = c; else hi = c;
  }
  const double mid = 0.5 * ((double)e4m3_to_f32(lo) + (double)e4m3_to_f32(lo + 1));
  return v > mid || (v == mid && (lo & 1u)) ? lo + 1 : lo;
}

__device__ __forceinline__ uint32_t scale_code(float a, float ts, float inv6ts, bool mid) {
  if (!mid) return scale_exact(a, ts);
  const float v = a * inv6ts;
  const uint32_t two = __nv_cvt_float2_to_fp8x2(make_float2(v * (1.f - 9.6e-7f), v * (1.f + 9.6e-7f)), __NV_SATFINITE, __NV_E4M3);
  const uint32_t lo = two & 0xFFu, hi = two >> 8;
  if (lo == hi) return lo;
  // a against 6 ts times the middle of the two: the product-sum rounds once, so its sign is exact
  const float r = fmaf(-3.f * (e4m3_to_f32(lo) + e4m3_to_f32(hi)), ts, a);
  return r > 0.f || (r == 0.f && (lo & 1u)) ? hi : lo;
}

// magnitude code of |x| / (s ts)
__device__ __noinline__ uint32_t code_exact(float x, float s, float ts) {
  const double d = (double)s * (double)ts, v = fabs((double)x);
  uint32_t c = 0;
#pragma unroll
  for (uint32_t i = 0; i < 7; ++i) {
    const double m = (double)border(i) * d;
    if (v > m || (v == m && (i & 1u))) c = i + 1;
  }
  return c;
}

template <typename T>
struct Traits;
template <>
struct Traits<__nv_bfloat16> {
  static constexpr uint32_t INF = 0x7F80u;
  static constexpr uint32_t BELOW = 0xFFFFu;   // fp32 bits below the type's last one
  static __device__ __forceinline__ float f(uint32_t h) { return __uint_as_float(h << 16); }
  // of two pairs, the larger magnitudes (their signs are of no account; NaN stays)
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
};
template <>
struct Traits<__half> {
  static constexpr uint32_t INF = 0x7C00u;
  static constexpr uint32_t BELOW = 0x1FFFu;
  static __device__ __forceinline__ float f(uint32_t h) { return __half2float(__ushort_as_half((unsigned short)h)); }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
};

// 16 consecutive values of a row
template <typename T>
struct Unit {
  uint32_t w[8];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ void load(const T* p) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(p)), b = __ldg(reinterpret_cast<const uint4*>(p) + 1);
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
  }
  __device__ __forceinline__ void load_tail(const T* p, int n) {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t a = 2 * i < n ? q[2 * i] : 0u, b = 2 * i + 1 < n ? q[2 * i + 1] : 0u;
      w[i] = a | (b << 16);
    }
  }
  // bits of the largest magnitude (INF and above: not finite)
  __device__ __forceinline__ uint32_t hmax() const {
    uint32_t m = w[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) m = Traits<T>::max2(m, w[i]);
    return max(m & 0x7FFFu, (m >> 16) & 0x7FFFu);
  }
  // and as fp32 (0x7F800000 and above: not finite)
  __device__ __forceinline__ uint32_t amax() const {
    const uint32_t h = hmax();
    return h >= Traits<T>::INF ? 0x7FC00000u : __float_as_uint(Traits<T>::f(h));
  }
  __device__ __forceinline__ float get(int i) const {
    return Traits<T>::f((i & 1) ? (w[i >> 1] >> 16) : (w[i >> 1] & 0xFFFFu));
  }
};
template <>
struct Unit<float> {
  float v[16];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = 0.f;
  }
  __device__ __forceinline__ void load(const float* p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(p) + i);
      v[4 * i] = a.x; v[4 * i + 1] = a.y; v[4 * i + 2] = a.z; v[4 * i + 3] = a.w;
    }
  }
  __device__ __forceinline__ void load_tail(const float* p, int n) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = i < n ? p[i] : 0.f;
  }
  __device__ __forceinline__ uint32_t amax() const {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    return m;
  }
  __device__ __forceinline__ float get(int i) const { return v[i]; }
};

constexpr uint32_t F32_INF = 0x7F800000u;

// How 1 / p has to be turned so that one rounding of x / p decides as the real quotient does, for 16-bit x. The borders
// between codes are p / 4 times 1, 3, 5, 7, 10, 14 and 20: four mantissas k p. The 16-bit values that come near a border
// (2^-19 of it) all have the mantissa of the one grid point next to k p, so that its exact side of k (p + e)
// decides for all of them; on the border itself the even code is the lower one for k = 1 and 5, the upper one for
// 3 and 7. Other values are further than 2^-20 away. Returns 0 (no value comes near), 1 (down), 2 (up), 3 (both: no
// one factor serves). With one scale per row such values are common: there 6 p is the row's largest value in
// its own block.
template <typename T>
__device__ __forceinline__ uint32_t lean(float p, float e, float first) {   // of the mantissas first (1 or 5) and first + 2
  uint32_t need = 0u;
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const float k = m ? first + 2.f : first;
    const uint32_t b = __float_as_uint(p * k);
    const float g = __uint_as_float((b + (Traits<T>::BELOW + 1u) / 2u) & ~Traits<T>::BELOW);
    const float r = fmaf(-k, e, fmaf(-k, p, g));
    const uint32_t side = r > 0.f || (r == 0.f && m) ? 2u : 1u;
    if (((b + 16u) & Traits<T>::BELOW) <= 32u) need |= side;
  }
  return need;
}

// What x is multiplied by for the scale s ts, turned as lean() says, but for s's exponent: for a row's ts, lane m < 8 holds
// it for the subnormal scale m / 8 2^-6, lane 8 + m for the mantissa 1 + m / 8 (times 2^-7). Below 0: no one factor
// serves. (Found once per row, each half warp two of lean()'s borders: as many as 66 instructions a unit otherwise.)
template <typename T>
__device__ __forceinline__ float factors(float ts, int lane) {
  const float s = (float)((lane & 7) + (lane & 8)) * ((lane & 8) ? 0.0009765625f : 0.001953125f);
  const float p = s * ts, inv = rcp(p), e = fmaf(s, ts, -p);
  uint32_t need = lean<T>(p, e, lane < 16 ? 1.f : 5.f);
  need |= __shfl_xor_sync(0xffffffffu, need, 16);
  const float f = need == 0u ? inv : need == 1u ? inv * (1.f - 4.8e-7f) : need == 2u ? inv * (1.f + 4.8e-7f) : -inv;
  return s == 0.f ? 0.f : f;
}

// the unit's 16 codes of x f
template <typename T>
__device__ __forceinline__ uint2 codes_by(const Unit<T>& u, float f) {
  uint32_t out[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float a[8];
#pragma unroll
    for (int i = 0; i < 8; i += 2) mul2(u.get(8 * h + i), u.get(8 * h + i + 1), f, a[i], a[i + 1]);
    out[h] = cvt8(a);
  }
  return make_uint2(out[0], out[1]);
}

// the unit's 16 codes for the scale s ts (NVFP4), from both ends of an interval around each quotient; mid: ts in mid_range
template <typename T>
__device__ __forceinline__ uint2 codes_nv(const Unit<T>& u, float s, float ts, bool mid) {
  if (s == 0.f) return make_uint2(0u, 0u);
  uint32_t out[2];
  if (mid) {
    const float p = s * ts, inv = rcp(p);
    const float e = fmaf(s, ts, -p);   // s ts = p + e exactly
    const float lo = inv * (1.f - 9.6e-7f), hi = inv * (1.f + 9.6e-7f);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float a[8], b[8];
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float x0 = u.get(8 * h + i), x1 = u.get(8 * h + i + 1);
        mul2(x0, x1, lo, a[i], a[i + 1]);
        mul2(x0, x1, hi, b[i], b[i + 1]);
      }
      out[h] = cvt8(a);
      const uint32_t diff = out[h] ^ cvt8(b);
      if (diff != 0u) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if ((diff >> (4 * i)) & 0xFu) {
            // |x| - m (p + e): the first difference is exact this near to the border m p
            const uint32_t c = (out[h] >> (4 * i)) & 7u;
            const float m = border(c), r = fmaf(-m, e, fmaf(-m, p, fabsf(u.get(8 * h + i))));
            if (r > 0.f || (r == 0.f && (c & 1u))) out[h] += 1u << (4 * i);
          }
        }
      }
    }
  } else {
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
      out[h] = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = h ? u.get(8 + i) : u.get(i);
        const uint32_t c = code_exact(x, s, ts) | (x < 0.f ? 8u : 0u);
        out[h] |= c << (4 * i);
      }
    }
  }
  return make_uint2(out[0], out[1]);
}
// Out of line, for the units whose scale lies next to a border or whose codes no one factor serves, and those that are not
// finite: codes, scale.
template <typename T>
__device__ __noinline__ uint3 unit_rare(Unit<T> u, uint32_t h, float ts, float inv6) {
  if (h >= Traits<T>::INF) return make_uint3(0u, 0u, 0x7Fu);
  const uint32_t sc = scale_code(Traits<T>::f(h), ts, inv6, true);
  const uint2 c = codes_nv<T>(u, e4m3_to_f32(sc), ts, true);
  return make_uint3(c.x, c.y, sc);
}

template <typename T>
__device__ __forceinline__ uint2 codes_mx(const Unit<T>& u, float inv) {
  float a[8], b[8];
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    mul2(u.get(i), u.get(i + 1), inv, a[i], a[i + 1]);
    mul2(u.get(8 + i), u.get(9 + i), inv, b[i], b[i + 1]);
  }
  return make_uint2(cvt8(a), cvt8(b));
}

// unit k of a row; VEC: rows of whole units at 16-byte addresses, where a unit behind the row's last is the last again
// (it adds nothing to the row's largest value, and nothing of it is stored)
template <typename T, bool VEC>
__device__ __forceinline__ void load_unit(Unit<T>& u, const T* row, int k, const QuantArgs& a, bool has) {
  if (VEC) {
    u.load(row + (int64_t)min(k, a.k / 16 - 1) * 16);
  } else {
    u.zero();
    if (has && k * 16 < a.k) u.load_tail(row + (int64_t)k * 16, a.k - k * 16);
  }
}

// The row's place among the scale atoms' rows, or -1 where it is none of the operand's (a whole warp's call).
__device__ __forceinline__ int64_t place(const QuantArgs& a, int64_t row, int lane) {
  if (row >= a.rows) return -1;
  if (a.offsets == nullptr) return row;
  int g = 0;   // the row's group: how many end at or before it
  for (int i = lane; i < a.groups; i += 32) g += a.offsets[i + 1] <= row ? 1 : 0;
  g = __reduce_add_sync(0xffffffffu, g);
  if (g >= a.groups) return -1;
  const int64_t o = a.offsets[g], pos = ((o >> 7) + g) * 128 + (row - o);
  return o < 0 || o > row || pos >= a.blocks * 128 ? -1 : pos;
}

// A row's warps take its units (16 values a thread) in turn, V at a time with their loads issued together. With
// one tensor scale per row the row is read twice, first for its largest value and each unit's, which are kept in shared
// memory, then, from L1 or L2, for its codes. 118 instructions a unit and 250 a warp and row bound it (NVFP4, 8192 x
// 7168: 37 us, 4.1 TB/s; with the caller's scale 29; MXFP4 25). (Blocks that take rows in turn: 45 against 41 at the time.)
constexpr int QUANT_WARPS = 8;    // warps of a row at most
constexpr int QUANT_FIRST = 4;    // units in flight while a row's largest value is found

template <typename T, bool NV, int V, bool VEC>
__global__ void __launch_bounds__(QUANT_WARPS * 32, 4) quant_kernel(QuantArgs a) {
  // 16-bit values with a scale per row: the units' largest magnitudes, of each thread's own
  constexpr bool HALF = NV && sizeof(T) == 2;
  constexpr int W = V == 1 ? 1 : QUANT_FIRST;
  __shared__ uint32_t red[QUANT_WARPS];
  extern __shared__ uint16_t stash[];
  const int lane = threadIdx.x & 31, rw = threadIdx.y, tr = threadIdx.x;   // a block: some rows' threads
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + rw;
  pdl_wait();
  pdl_trigger();
  int64_t src = row;
  const int64_t pos = place(a, row, lane);
  const bool live = pos >= 0;
  bool has = live;
  if (live && a.rows_in != nullptr) {
    src = a.rows_in[row];
    has = src >= 0 && src < a.src_rows;   // no such row: zeros
  }
  // (a row without a source reads row 0, and its values count as zeros)
  const T* xr = reinterpret_cast<const T*>(a.x) + (has ? src : 0) * a.stride;
  const int step = blockDim.x, whole = has ? (a.k + 15) / 16 : 0;   // units with values
  float ts = 1.f;
  bool empty = false;   // a row of zeros (and blocks that are not finite)
  if (NV) {
    if (a.ts != nullptr) {
      ts = *a.ts;
    } else {
      uint32_t m = 0u;
      if constexpr (HALF) {
        uint16_t* to = stash + rw * a.stash + tr;
        const T* p = xr + tr * 16;
        auto turn = [&](int k0, auto full) {
          Unit<T> u[W];
#pragma unroll
          for (int i = 0; i < W; ++i) {
            if (VEC && decltype(full)::value) u[i].load(p + i * step * 16);
            else load_unit<T, VEC>(u[i], xr, k0 + i * step, a, has);
          }
#pragma unroll
          for (int i = 0; i < W; ++i) {
            const uint32_t h = u[i].hmax();
            to[i * step] = (uint16_t)h;
            m = max(m, h < Traits<T>::INF ? h : 0u);
          }
          to += W * step;
          p += W * step * 16;
        };
        int k0 = tr;
        for (const int last = a.k / 16 - (W - 1) * step; k0 < last; k0 += W * step) turn(k0, std::true_type{});
        for (; k0 < a.units; k0 += W * step) turn(k0, std::false_type{});
        m = __float_as_uint(Traits<T>::f(m));
      } else {
        for (int k0 = tr; k0 < a.units; k0 += step * V) {
          Unit<T> u[V];
#pragma unroll
          for (int i = 0; i < V; ++i) load_unit<T, VEC>(u[i], xr, k0 + i * step, a, has);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const uint32_t am = u[i].amax();
            m = max(m, am < F32_INF ? am : 0u);
          }
        }
      }
      m = __reduce_max_sync(0xffffffffu, m);
      if (a.wpr > 1) {
        if (lane == 0) red[rw * a.wpr + (tr >> 5)] = m;
        __syncthreads();   // (all rows' warps: barriers of the rows' own, by number, cost the SM half of its blocks)
        m = lane < a.wpr ? red[rw * a.wpr + lane] : 0u;
        m = __reduce_max_sync(0xffffffffu, m);
      }
      empty = !has || m == 0u;
      ts = fmaxf(__fdiv_rn(has ? __uint_as_float(m) : 0.f, 2688.f), 1.17549435e-38f);
      if (live && tr == 0) a.row_ts[row] = ts;
    }
  }
  if (!live) return;   // whole warps: a row's warps share `live`
  const bool ts_ok = ts > 0.f && __float_as_uint(ts) < F32_INF;
  const bool ts_mid = mid_range(ts);
  const float inv6 = NV ? rcp(6.f * ts) : 0.f;
  uint8_t* cr = a.codes + row * a.row_bytes;
  uint8_t* sr = a.flat ? a.scales + row * a.atoms * 4
                       : a.scales + ((pos >> 7) * a.atoms) * 512 + (pos & 31) * 16 + ((pos >> 5) & 3) * 4;
  const int64_t atom = a.flat ? 4 : 512;
  if constexpr (HALF) {
    if (ts_mid || empty) {
      const float fs = empty ? 0.f : factors<T>(ts, lane);
      const uint16_t* from = stash + rw * a.stash + tr;
      const int end = (a.units + 3) & ~3;   // (the last scale word is written whole)
      uint8_t* st = sr + (tr >> 2) * atom + (tr & 3);
      const int64_t st_step = (step >> 2) * atom;
      uint2* ct = reinterpret_cast<uint2*>(cr) + tr;
      auto units = [&](int base, auto full, auto own) {   // own: the row's scale is its own, the largest values are at hand
        constexpr bool FULL = decltype(full)::value, OWN = decltype(own)::value;
        Unit<T> u[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if (FULL && VEC) u[i].load(xr + (base + tr + i * step) * 16);
          else load_unit<T, VEC>(u[i], xr, base + tr + i * step, a, has);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int k = base + tr + i * step;
          const bool in = FULL || k < whole;
          uint32_t h = OWN ? from[i * step] : u[i].hmax();
          if (!in) h = 0u;
          const float v = Traits<T>::f(h) * inv6;
          const uint32_t two =
              __nv_cvt_float2_to_fp8x2(make_float2(v * (1.f - 9.6e-7f), v * (1.f + 9.6e-7f)), __NV_SATFINITE, __NV_E4M3);
          uint32_t sc = two & 0xFFu;
          const float f0 = __shfl_sync(0xffffffffu, fs, (int)min(sc, (sc & 7u) | 8u));
          const float f = __uint_as_float(__float_as_uint(f0) - ((sc & 0x78u) << 20));
          uint2 c = codes_by<T>(u[i], f);
          if (two >> 8 != sc || f < 0.f || h >= Traits<T>::INF) {
            const uint3 r = unit_rare<T>(u[i], h, ts, inv6);
            c = make_uint2(r.x, r.y);
            sc = r.z;
          }
          if (!in) c = make_uint2(0u, 0u);
          if (FULL || k < end) st[i * st_step] = (uint8_t)sc;
          if (FULL || k < a.units) ct[i * step] = c;
        }
        from += V * step;
        st += V * st_step;
        ct += V * step;
      };
      auto row_units = [&](auto own) {
        int base = 0;
        for (; base + step * V <= whole; base += step * V) units(base, std::true_type{}, own);
        for (; base < a.units; base += step * V) units(base, std::false_type{}, own);
      };
      if (a.ts == nullptr) row_units(std::true_type{});
      else row_units(std::false_type{});
      return;
    }
  }
  for (int base = 0; base < a.units; base += step * V) {
    Unit<T> u[V];
#pragma unroll
    for (int i = 0; i < V; ++i) load_unit<T, VEC>(u[i], xr, base + tr + i * step, a, has);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int k = base + tr + i * step;
      const uint32_t am = k < whole ? u[i].amax() : 0u;
      uint32_t sc;
      uint2 c = make_uint2(0u, 0u);
      if (NV) {
        const bool fine = am < F32_INF && ts_ok;
        sc = fine ? scale_code(__uint_as_float(am), ts, inv6, ts_mid) : 0x7Fu;
        if (fine) c = codes_nv<T>(u[i], e4m3_to_f32(sc), ts, ts_mid);
        if (k >= a.units) sc = 0u;
        uint32_t w = sc << (8 * (k & 3));
        w |= __shfl_xor_sync(0xffffffffu, w, 1);
        w |= __shfl_xor_sync(0xffffffffu, w, 2);
        if (k < a.units && (k & 3) == 0) *reinterpret_cast<uint32_t*>(sr + (k >> 2) * atom) = w;
      } else {
        const uint32_t m = max(am, __shfl_xor_sync(0xffffffffu, am, 1));
        // amax = f 2^e: t = e - 2 for f <= 1.5, else e - 1; biased and floored at 2^-126
        sc = m < F32_INF ? (uint32_t)max((int)((m + 0x3FFFFFu) >> 23) - 2, 1) : 0xFFu;
        if (m < F32_INF && k < whole) c = codes_mx<T>(u[i], __uint_as_float((254u - sc) << 23));
        if (k >= a.units) sc = 0u;
        uint32_t w = sc << (8 * ((k >> 1) & 3));
        w |= __shfl_xor_sync(0xffffffffu, w, 2);
        w |= __shfl_xor_sync(0xffffffffu, w, 4);
        if (k < a.units && (k & 7) == 0) *reinterpret_cast<uint32_t*>(sr + (k >> 3) * atom) = w;
      }
      if (k < a.units) *reinterpret_cast<uint2*>(cr + (int64_t)k * 8) = c;
    }
  }
}

// Rows of an operand copied from the quantised source rows (codes, scale words row by row, tensor scales), a warp a row.
__global__ void __launch_bounds__(256) gather_kernel(QuantArgs a, const uint8_t* __restrict__ codes,
                                                     const uint32_t* __restrict__ words, const float* __restrict__ ts) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  pdl_wait();
  pdl_trigger();
  const int64_t pos = place(a, row, lane);
  if (pos < 0) return;
  const int64_t src = a.rows_in[row];
  const bool has = src >= 0 && src < a.src_rows;
  const uint4* from = reinterpret_cast<const uint4*>(codes + (has ? src : 0) * a.row_bytes);
  uint4* to = reinterpret_cast<uint4*>(a.codes + row * a.row_bytes);
  const int n = (int)(a.row_bytes / 16);
#pragma unroll 4
  for (int i = lane; i < n; i += 32) {
    const uint4 v = __ldg(from + i);
    to[i] = has ? v : make_uint4(0u, 0u, 0u, 0u);
  }
  const uint32_t* w = words + (has ? src : 0) * a.atoms;
  uint8_t* sr = a.scales + ((pos >> 7) * a.atoms) * 512 + (pos & 31) * 16 + ((pos >> 5) & 3) * 4;
  // (a missing row's scales are those of zeros: 0, or 2^-126; NaN where the caller's tensor scale is no scale)
  const int nb = a.nv ? a.units : a.units / 2;
  const float ts1 = a.ts != nullptr ? *a.ts : 1.f;
  const uint32_t zeros = !a.nv ? 0x01010101u : ts1 > 0.f && ts1 < INFINITY ? 0u : 0x7F7F7F7Fu;
#pragma unroll 4
  for (int i = lane; i < a.atoms; i += 32) {
    const uint32_t none = zeros >> (8 * max(0, 4 - (nb - 4 * i)));
    *reinterpret_cast<uint32_t*>(sr + (int64_t)i * 512) = has ? __ldg(w + i) : none;
  }
  if (a.row_ts != nullptr && lane == 0) a.row_ts[row] = has ? ts[src] : 1.17549435e-38f;
}

template <typename T>
__device__ __forceinline__ T to_out(float v);
template <>
__device__ __forceinline__ float to_out<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half to_out<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 to_out<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// y = code s ts: code s is exact in fp32 (6 significant bits), the product with ts rounds once. A thread
// takes 16 values at a time, the warps of a row as in quant_kernel.
template <typename T, bool NV>
__global__ void __launch_bounds__(1024) dequant_kernel(DequantArgs a) {
  const int warp = threadIdx.x >> 5;
  const int rpc = (blockDim.x >> 5) / a.wpr;
  const int rw = warp / a.wpr, tr = threadIdx.x - rw * a.wpr * 32;
  const int64_t row = (int64_t)blockIdx.x * rpc + rw;
  pdl_wait();
  pdl_trigger();
  if (row >= a.rows) return;
  const float ts = NV && a.ts != nullptr ? a.ts[a.ts_row ? row : 0] : 1.f;
  const uint8_t* cr = a.codes + row * a.row_bytes;
  const uint8_t* sr = a.scales + ((row >> 7) * a.atoms) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4;
  for (int k = tr; k < a.units; k += a.wpr * 32) {
    const uint2 c = *reinterpret_cast<const uint2*>(cr + (int64_t)k * 8);
    const int b = NV ? k : k >> 1;
    const uint32_t sb = sr[(int64_t)(b >> 2) * 512 + (b & 3)];
    const float s = NV ? e4m3_to_f32(sb) : (sb == 0xFFu ? __uint_as_float(0x7FC00000u) : e8m0_to_f32(sb));
    alignas(16) T o[16];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t h = e2m1x2_to_f16x2((j < 4 ? c.x : c.y) >> (8 * (j & 3)));
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      float v0, v1;
      mul2(f.x, f.y, s, v0, v1);
      if (NV) mul2(v0, v1, ts, v0, v1);
      o[2 * j] = to_out<T>(v0);
      o[2 * j + 1] = to_out<T>(v1);
    }
    T* y = reinterpret_cast<T*>(a.y) + row * a.k + (int64_t)k * 16;
    const int left = a.k - k * 16;
    if (a.vec && left >= 16) {
#pragma unroll
      for (int j = 0; j < (int)sizeof(T); ++j) reinterpret_cast<uint4*>(y)[j] = reinterpret_cast<const uint4*>(o)[j];
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (j < left) y[j] = o[j];
    }
  }
}

// canonical scales [mats][n][nb] bytes -> atoms, each matrix padded to whole row blocks (zero scales)
__global__ void __launch_bounds__(256) tile_scales_kernel(const uint8_t* __restrict__ src, uint8_t* __restrict__ dst,
                                                          int64_t mats, int64_t n, int64_t nb, int64_t atoms) {
  pdl_wait();
  const int64_t blocks = (n + 127) >> 7;
  const int64_t words = mats * blocks * atoms * 128;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < words; i += (int64_t)gridDim.x * blockDim.x) {
    const int in = (int)(i & 127);                // word of the atom: row 32 (in % 4) + in / 4
    const int64_t at = (i >> 7) % atoms, blk = (i >> 7) / atoms;
    const int64_t mat = blk / blocks, r = (blk % blocks) * 128 + 32 * (in & 3) + (in >> 2);
    uint32_t w = 0u;
    if (r < n) {
      const uint8_t* s = src + (mat * n + r) * nb + at * 4;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (at * 4 + j < nb) w |= (uint32_t)s[j] << (8 * j);
    }
    reinterpret_cast<uint32_t*>(dst)[i] = w;
  }
}

template <typename T, bool NV, bool VEC>
static cudaError_t launch_quant_v(QuantArgs q, int v, dim3 grid, dim3 block, cudaStream_t st) {
  // each thread's units, whole turns of them
  size_t smem = 0;
  if (NV && sizeof(T) == 2 && q.ts == nullptr) {
    const int w = v == 1 ? 1 : QUANT_FIRST, turns = (q.units + q.wpr * 32 * w - 1) / (q.wpr * 32 * w);
    q.stash = turns * w * (int)block.x;
    smem = (size_t)q.stash * block.y * sizeof(uint16_t);
  }
  if (v == 1) return launch_pdl(quant_kernel<T, NV, 1, VEC>, grid, block, smem, st, q);
  return launch_pdl(quant_kernel<T, NV, 2, VEC>, grid, block, smem, st, q);
}

template <typename T>
static cudaError_t launch_quant_t(const QuantArgs& q, int v, bool vec, dim3 grid, dim3 block, cudaStream_t st) {
  if (q.nv) return vec ? launch_quant_v<T, true, true>(q, v, grid, block, st) : launch_quant_v<T, true, false>(q, v, grid, block, st);
  return vec ? launch_quant_v<T, false, true>(q, v, grid, block, st) : launch_quant_v<T, false, false>(q, v, grid, block, st);
}

}  // namespace fp4

static cudaError_t launch_rows(const QuantArgs& args, int dtype, cudaStream_t st) {
  QuantArgs q = args;
  // Units per thread: one while the rows do not fill the GPU, up to four at large sizes, where what a warp does once per
  // row counts (8192 x 7168 NVFP4: two 47 us, four 37, eight, whose rows outgrow L1 between their two readings, 39).
  // Two are in flight. Blocks of four warps, or of a row's (of eight: 40 us).
  const int64_t per = q.rows * q.units / ((int64_t)num_sms() * 1536);
  const int each = per < 1 ? 1 : (per > 4 ? 4 : (int)per), v = each == 1 ? 1 : 2;
  q.wpr = (q.units + 32 * each - 1) / (32 * each);
  if (q.wpr > fp4::QUANT_WARPS) q.wpr = fp4::QUANT_WARPS;
  const int rpc = q.wpr < 4 ? 4 / q.wpr : 1;
  const dim3 grid((unsigned)((q.rows + rpc - 1) / rpc)), block(q.wpr * 32, rpc);
  const int es = dtype == SB_F32 ? 4 : 2;
  const bool vec = (reinterpret_cast<uintptr_t>(q.x) & 15u) == 0 && (q.stride * es) % 16 == 0 && q.k % 16 == 0 && q.src_rows > 0;
  if (dtype == SB_F32) return fp4::launch_quant_t<float>(q, v, vec, grid, block, st);
  if (dtype == SB_F16) return fp4::launch_quant_t<__half>(q, v, vec, grid, block, st);
  return fp4::launch_quant_t<__nv_bfloat16>(q, v, vec, grid, block, st);
}

// A gather that takes each source row twice or more quantises the source once and copies, from 4 M values on (2048 rows
// of 4096, each taken eight times, and their w13 product: 246 us without, 221 with; below, the second launch
// costs more than it saves).
size_t fp4_quant_workspace(int64_t src_rows, int64_t rows, int64_t row_bytes, int64_t atoms) {
  return rows >= 2 * src_rows && src_rows > 0 && rows * row_bytes >= (2 << 20)
             ? (size_t)(src_rows * (row_bytes + 4 * atoms + 4))
             : 0;
}

cudaError_t launch_fp4_quant(const QuantArgs& a, int dtype, void* workspace, cudaStream_t st) {
  if (a.rows_in == nullptr || workspace == nullptr) return launch_rows(a, dtype, st);
  QuantArgs q = a;
  q.rows = a.src_rows;
  q.rows_in = nullptr;
  q.offsets = nullptr;
  q.codes = (uint8_t*)workspace;
  q.scales = q.codes + a.src_rows * a.row_bytes;
  q.row_ts = reinterpret_cast<float*>(q.scales + a.src_rows * a.atoms * 4);
  q.flat = 1;
  const cudaError_t e = launch_rows(q, dtype, st);
  if (e != cudaSuccess) return e;
  return launch_pdl(fp4::gather_kernel, dim3((unsigned)((a.rows + 7) / 8)), dim3(256), 0, st, a, q.codes,
                    (const uint32_t*)q.scales, q.row_ts);
}

template <typename T>
static cudaError_t launch_dequant_t(const DequantArgs& a, dim3 grid, dim3 block, cudaStream_t st) {
  if (a.nv) return launch_pdl(fp4::dequant_kernel<T, true>, grid, block, 0, st, a);
  return launch_pdl(fp4::dequant_kernel<T, false>, grid, block, 0, st, a);
}

static unsigned grid_of(int64_t work, int64_t cap) {
  const int64_t g = (work + 255) / 256;
  return (unsigned)(g < 1 ? 1 : (g < cap ? g : cap));
}

cudaError_t launch_fp4_dequant(const DequantArgs& args, int dtype, cudaStream_t st) {
  DequantArgs a = args;
  const int es = dtype == SB_F32 ? 4 : 2;
  a.vec = (reinterpret_cast<uintptr_t>(a.y) & 15u) == 0 && (a.k * es) % 16 == 0;
  const int v = a.rows * a.units <= (int64_t)num_sms() * 1024 ? 1 : 4;
  a.wpr = (a.units + 32 * v - 1) / (32 * v);
  if (a.wpr > 32) a.wpr = 32;
  const int rpc = a.wpr >= 8 ? 1 : 8 / a.wpr;
  const dim3 grid((unsigned)((a.rows + rpc - 1) / rpc)), block(rpc * a.wpr * 32);
  if (dtype == SB_F32) return launch_dequant_t<float>(a, grid, block, st);
  if (dtype == SB_F16) return launch_dequant_t<__half>(a, grid, block, st);
  return launch_dequant_t<__nv_bfloat16>(a, grid, block, st);
}

cudaError_t launch_fp4_tile_scales(const uint8_t* src, uint8_t* dst, int64_t mats, int64_t n, int64_t nb,
                                   cudaStream_t st) {
  const int64_t atoms = (nb + 3) / 4, words = mats * ((n + 127) / 128) * atoms * 128;
  return launch_pdl(fp4::tile_scales_kernel, dim3(grid_of(words, (int64_t)num_sms() * 64)), dim3(256), 0, st, src, dst,
                    mats, n, nb, atoms);
}

}  // namespace sb
