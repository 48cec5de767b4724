// Products of two microscaled 4-bit operands on the tensor cores: y[token][n] = sum_k a[token][k] W[n][k],
// one weight matrix for all tokens, or one per expert with the tokens' rows sorted by expert.
//
// tcgen05.mma kind::mxf4nvf4 / kind::mxf4 multiplies e2m1 by e2m1 with a scale per 16 (e4m3) or per 32
// (e8m0) values of either side and sums in fp32, so the whole K accumulates in tensor memory and is
// read once; the fp32 tensor scales are applied there.
//
// The weights are the M operand, the tokens N: a token tile takes any multiple of 8 columns, so one
// decoded token costs an 8-column tile and ragged expert groups waste little. A CTA takes 128 weight
// rows; where there are tiles for all SMs, two CTAs form a pair (cta_group::2) that shares the token
// rows of a 256-row tile, each loading half of them, and one of them issues for both.
// Where one token tile's weight rows are too few for the SMs, a cluster of CTAs splits K between them and adds its
// sums through distributed shared memory, in the order of K.
// Stages hold 256 K: 128 weight rows and the token rows of 128 bytes each, landed by TMA in the 128-byte-
// swizzled K-major form, and their scale atoms. Roles (352 threads): warp 8 copies codes, warp 9 scales,
// warp 10 moves scale atoms to tensor memory and issues the MMAs, warps 0-7 read the accumulator (a
// thread: one weight row, every other 32 columns) and store. Two accumulators alternate, so that one tile's
// readback overlaps the next tile's products: of up to 192 columns each, or in pairs of 256, which share 64
// columns to leave room for the scales; the readback begins with those and releases them at once.
//
// Every wait is bounded: on timeout the CTA sets the device's error word and winds down. Offsets that descend set it, too.
#include <cudaTypedefs.h>
#include <string.h>

#include <atomic>
#include <type_traits>

#include "sb_fp4.h"
#include "sb_launch.h"
#include "sb_tcgen05.cuh"

namespace sb {
namespace fp4mm {

using namespace tc5;

constexpr int EPI_WARPS = 8;
constexpr int CODE_WARP = 8;         // copies codes,
constexpr int SCALE_WARP = 9;        // and their scales
constexpr int MMA_WARP = 10;
constexpr int NTHREADS = 352;
constexpr int NT_MAX = 256;          // token columns of a tile: 256 in a pair, elsewhere up to
constexpr int NT_APART = 192;        // so many, whose two accumulators lie side by side
constexpr int BOX = 32;              // token rows of one copy with expert groups
constexpr int A_BYTES = 128 * 128;   // a stage's weight rows
constexpr int MAX_STAGES = 10;
constexpr int MAX_MATS = 1024;
constexpr int RING = 16;             // tiles found ahead of their products and readback: more than MAX_STAGES + 3
constexpr int TMEM_COLS = 512;
constexpr int SFA_COL = NT_APART + NT_MAX;  // scale factors: 4 atoms x 4 columns of the weights,
constexpr int SFB_COL = SFA_COL + 16;  // 4 atoms x 8 columns of the tokens (two row blocks)
constexpr uint32_t WAIT_LIMIT = 1u << 16;
constexpr int SMEM_LIMIT = 232448;
constexpr int64_t L2_AHEAD = 32 << 20;

enum Form { SINGLE = 0, PAIRED = 1, SPLIT = 2 };

template <bool NV>
constexpr int SF_BLOCK = NV ? 2048 : 1024;   // a stage's scale atoms of 128 rows

__device__ int g_err;

struct Args {
  CUtensorMap map_w, map_a;     // codes
  CUtensorMap map_ws, map_as;   // scale atoms
  CUtensorMap map_n;            // token codes of a pair's narrower tiles
  Fp4MmArgs g;
  int nt;            // token columns of a full tile (a multiple of 64 when a matrix has several)
  int box;           // token rows of one copy
  int stages;
  int b_bytes;       // token rows of a stage (of one CTA)
  int sblk;          // row blocks of token scales that a copy brings
  int ksteps;        // MMAs along K (64 values each)
  int vec;           // 16-byte stores to y
  int split;         // CTAs that share a tile's K
  int ahead;         // stages of weights brought to L2 before the kernel before this one has ended
};

struct Ctl {
  uint64_t full[MAX_STAGES], empty[MAX_STAGES], accfull[2], accempty[2], shared, drain, told[RING];
  uint32_t tmem_base;
  int abort;
  alignas(128) uint8_t turn[EPI_WARPS][2048];       // 32 rows x 32 outputs of 16 bits, to be turned
  alignas(16) float scale[EPI_WARPS][NT_MAX / 2];   // of each warp's tokens: tensor scale,
  alignas(16) float weight[EPI_WARPS][NT_MAX / 2];  // row weight
  int4 tile[RING];           // of each tile: matrix, first weight row, first row of its tokens, tokens
  int tile_t0[RING];         // and its first token in the group
  int tiles[MAX_MATS + 1];   // tiles before each matrix
  int rows[MAX_MATS + 1];    // first token row of each matrix's group, and the end of the last
};

struct Tile {
  int mat, n0, t0, cnt, row0;   // matrix, first weight row, first token of the group, tokens, group's first row
  int blk;                      // the tokens' first scale row block
};

// instruction descriptor: e2m1 x e2m1, M = 128 (256 of a pair), N = n (bits 4 and 29 up: which scale bytes of either side's words)
template <bool NV, bool PAIR>
__device__ __forceinline__ uint32_t idesc(uint32_t n) {
  return (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((NV ? 0u : 1u) << 23) | (((PAIR ? 256u : 128u) >> 4) << 24);
}

#define SB_MMA(group, kind)                                                                                        \
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"                                                       \
               " tcgen05.mma.cta_group::" group ".kind::" kind " [%0], %1, %2, %3, [%5], [%6], p;\n}\n" ::"r"(d),  \
               "l"(ad), "l"(bd), "r"(id), "r"(acc), "r"(sfa), "r"(sfb))

template <bool NV, bool PAIR>
__device__ __forceinline__ void mma(uint32_t d, uint64_t ad, uint64_t bd, uint32_t id, uint32_t sfa, uint32_t sfb,
                                    uint32_t acc) {
  if constexpr (NV && PAIR) SB_MMA("2", "mxf4nvf4.block_scale.scale_vec::4X");
  else if constexpr (NV) SB_MMA("1", "mxf4nvf4.block_scale.scale_vec::4X");
  else if constexpr (PAIR) SB_MMA("2", "mxf4.block_scale.scale_vec::2X");
  else SB_MMA("1", "mxf4.block_scale.scale_vec::2X");
}
#undef SB_MMA

// a scale atom as the source of a copy: 32 rows of 16 bytes, no swizzle
__device__ __forceinline__ uint64_t sf_desc(uint32_t src) {
  uint64_t d = 0;
  d |= (uint64_t)((src >> 4) & 0x3FFFu);
  d |= (uint64_t)(128 >> 4) << 16;
  d |= (uint64_t)(128 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  return d;
}
// one scale atom into four tensor memory columns of every 32-lane quarter
template <bool PAIR>
__device__ __forceinline__ void cp_sf(uint32_t taddr, uint64_t desc) {
  if constexpr (PAIR)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n" ::"r"(taddr), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n" ::"r"(taddr), "l"(desc) : "memory");
}

// arrive, once all MMAs issued so far have finished, on `bar` (of both CTAs of a pair)
template <bool PAIR>
__device__ __forceinline__ void commit_to(uint32_t bar) {
  if constexpr (PAIR)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
  else
    commit(bar);
}

// a box of codes into L2
__device__ __forceinline__ void prefetch_2d(const CUtensorMap* map, int c0, int c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];\n" ::"l"(reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1)
               : "memory");
}

// tensor copies into this CTA's shared memory; a pair's complete on the first CTA's barrier
template <bool PAIR>
__device__ __forceinline__ void load_2d(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  if constexpr (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
        "[%4];\n" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
  else
    tma_load_2d(dst, map, c0, c1, bar);
}
template <bool PAIR>
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  if constexpr (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
        "[%1, {%2, %3, %4}], [%5];\n" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(
            dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
        : "memory");
}

// the address of this shared memory location in CTA 0 of the pair
__device__ __forceinline__ uint32_t in_first(uint32_t addr) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;\n" : "=r"(r) : "r"(addr));
  return r;
}
// Without release: what it follows are reads of tensor memory, complete at tcgen05.wait::ld in every lane (their values are in
// registers) and ordered before the arrival by fence::before_thread_sync and, between the lanes, __syncwarp. It hands over
// nothing else: a read or write of shared or global memory that the other CTA had to see or wait for would need a release
// here. (A release at cluster scope waits for the stores to y before it: 1000 cycles twice a tile, in the readback and
// in the products that wait for it.)
__device__ __forceinline__ void arrive_remote(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
// arrive on the accumulator's barrier where the MMAs are issued
template <bool PAIR>
__device__ __forceinline__ void release(uint32_t bar) {
  if constexpr (PAIR) arrive_remote(in_first(bar));
  else arrive(bar);
}
// a float of this CTA's shared memory as CTA `rank` of the cluster has it
__device__ __forceinline__ float peer_float(uint32_t addr, int rank) {
  uint32_t r;
  float v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(r) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;\n" ::: "memory");
}

// One stage: its scale atoms, then `steps` MMAs of 64 K (FULL: four). Descriptors are made once per kernel
// and only added to, and a full stage is unrolled: building each descriptor from its address made the issuing
// thread the bound (203 ns a stage without scales, 122 so, at N = 8; the tensor pipe takes 213 at N = 192).
template <bool NV, bool PAIR, int SBLK, bool FULL>
__device__ __forceinline__ void issue(uint32_t tbase, uint32_t acc, uint32_t sfb, uint64_t ad, uint64_t bd, uint64_t sd,
                                      uint32_t id, int steps, bool first) {
  constexpr int PER = NV ? 1 : 2;   // MMAs per scale atom
#pragma unroll
  for (int j = 0; j < 4 / PER; ++j) {
    if (FULL || j * PER < steps) {
      cp_sf<PAIR>(tbase + SFA_COL + 4 * j, sd + j * 32);
#pragma unroll
      for (int b = 0; b < SBLK; ++b) cp_sf<PAIR>(tbase + SFB_COL + 8 * j + 4 * b, sd + (SF_BLOCK<NV> >> 4) * (1 + b) + j * 32);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (FULL || j < steps) {
      const uint32_t h = NV ? 0u : (uint32_t)(j & 1) * 2u;
      mma<NV, PAIR>(acc, ad + 2 * j, bd + 2 * j, id | (h << 4) | (h << 29), (tbase + SFA_COL + 4 * (j / PER)) | (h << 30),
                    (sfb + 8 * (j / PER)) | (h << 30), j > 0 || !first ? 1u : 0u);
    }
  }
}

// the first token row of matrix mat's group (mat == mats: the end), inside [0, m] whatever the offsets hold
__device__ __forceinline__ int group_begin(const Fp4MmArgs& g, int mat) {
  return g.offsets ? min(max(g.offsets[mat], 0), g.m) : (mat == 0 ? 0 : g.m);
}

// The copying and issuing warps each run on one elected thread, whose waits need no vote of the warp (a vote and
// a re-election per stage cost the issuing warp 100 ns of 330). `probes` > 0 (a test's limit, on the consumers' waits):
// that many probes without suspension instead.
__device__ __forceinline__ bool wait(volatile int* abortf, uint32_t bar, uint32_t parity, uint32_t probes = 0u) {
  if (probes > 0u) return wait_bounded<true>(abortf, &g_err, bar, parity, probes);
  return mbar_try_wait(bar, parity) || wait_bounded(abortf, &g_err, bar, parity, WAIT_LIMIT);
}
// one answer for the whole warp, whose next instructions need all of its lanes
__device__ __forceinline__ bool warp_wait(volatile int* abortf, uint32_t bar, uint32_t parity, uint32_t probes) {
  return __all_sync(0xffffffffu, wait(abortf, bar, parity, probes));
}

// Tiles of one matrix run in bands of 12 weight blocks by all token tiles, so that the tiles in flight
// share both operands in L2.
template <bool PAIR>
__device__ __forceinline__ Tile tile_at(const Args& a, const Ctl& c, int i) {
  constexpr int MT = PAIR ? 256 : 128;
  int lo = 0, hi = a.g.mats;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (c.tiles[mid] <= i) lo = mid; else hi = mid;
  }
  const int r = i - c.tiles[lo], nb = (a.g.n + MT - 1) / MT, tiles = c.tiles[lo + 1] - c.tiles[lo];
  Tile t;
  t.mat = lo;
  t.row0 = c.rows[lo];
  const int all = c.rows[lo + 1] - t.row0;
  if (tiles == nb) {   // one token tile (the divisions below cost small products 0.5 us)
    t.n0 = r * MT;
    t.t0 = 0;
    t.cnt = min(all, a.nt);
  } else {
    const int tb = tiles / nb, band = r / (12 * tb), left = r - band * 12 * tb, wide = min(12, nb - band * 12);
    // a group's tokens in tiles alike, of whole 64-row steps of the scale atoms
    const int each = ((all + tb - 1) / tb + 63) & ~63;
    t.n0 = (band * 12 + left % wide) * MT;
    t.t0 = left / wide * each;
    t.cnt = min(all - t.t0, each);
  }
  t.blk = (a.g.offsets ? (t.row0 >> 7) + lo : 0) + (t.t0 >> 7);
  return t;
}

// clamps that let NaN through
__device__ __forceinline__ float clamp_hi(float v, float lim) { return v > lim ? lim : v; }
__device__ __forceinline__ float clamp_lo(float v, float lim) { return v < lim ? lim : v; }

template <typename T>
__device__ __forceinline__ T to_out(float v);
template <>
__device__ __forceinline__ float to_out<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half to_out<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 to_out<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 r = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 r = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ void st_shared16(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// four 8 x 8 tiles of 16-bit values, read turned: lane l gets rows 2 (l % 4), + 1 of column l / 4 of each
__device__ __forceinline__ uint4 read_turned(uint32_t addr) {
  uint4 v;
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// silu(gate) * up of one pair of rows: the even lane holds gate, the odd lane up, of two tokens; each lane
// gets one of the tokens' results. The fast exponential and division are off by |gate| 2^-23 + 2^-20 of the result (less
// than a rounding to 16 bits); for gates below -87, where silu is below 1e-35, the division may give 0.
__device__ __forceinline__ float gated(float v0, float v1, int lane, float lim) {
  const float o = __shfl_xor_sync(0xffffffffu, (lane & 1) ? v0 : v1, 1);
  const float gate = clamp_hi((lane & 1) ? o : v0, lim), up = clamp_lo(clamp_hi((lane & 1) ? v1 : o, lim), -lim);
  return __fdividef(gate, 1.f + __expf(-gate)) * up;
}

// Outputs are (d w) s, d the accumulator, w the weight row's scale, s the token's: with w between 2^-50 and 2^50, d w is a plain
// number for any sum of products and s scales it with one rounding. (s w by itself is subnormal or inf where the
// output is not: off by 1.4e-3 at rows of 1e-35 and weight scales of 4e-5.) Whether w is none of these:
__device__ __forceinline__ bool odd_row(float w) {
  return (__float_as_uint(w) & 0x7FFFFFFFu) - ((127u - 50u) << 23) > (100u << 23);
}
// s times a row weight that left fp32's range (or is 0)
__device__ __forceinline__ bool odd_col(float s) { return !(fabsf(s) >= 1.17549435e-38f && fabsf(s) < INFINITY); }

// 32 accumulator columns (tokens tok ..) of this thread's weight row to y; sc, wt: the tokens' scales and weights in
// shared memory. 16-bit outputs go through the warp's `turn` in shared memory, rows of 32 tokens in, tokens of up to
// 8 neighbouring rows out, the 16-byte pieces of a row placed so that neither side meets a bank conflict. This
// readback bounds tiles of K <= 1024 (690 cycles a chunk, gated 1330; a stage takes 520): 8192 x 4096 x 2048 took 62 us
// turned by shuffles (32 of them a chunk, against 8 accesses so), 46 at the time, now 34; with a 2-byte store per row and
// column a tile of 192 columns took 8.5 us. FULL: a whole chunk, without a branch per group of columns, which would
// keep the groups from overlapping.
template <bool SWIGLU, bool FULL, typename T>
__device__ __forceinline__ void store_chunk(const Args& a, const uint32_t (&d)[32], int64_t tok, int row, int lane, int left,
                                            bool vec, float wts, const float* sc, const float* wt, uint32_t turn) {
  const Fp4MmArgs& g = a.g;
  T* y = reinterpret_cast<T*>(g.y);
  const int64_t ld = g.ldy;
  const float lim = g.limit > 0.f ? g.limit : INFINITY;
  if constexpr (sizeof(T) == 2) {
    if (vec) {
      const int e = lane & 7, i = lane >> 3;   // this lane's part of an address list: row e of tile i
      if constexpr (SWIGLU) {
        // rows of 16 results: tokens 0, 2, .. 30 (even lanes), then 1, 3, .. 31
        const int hr = lane >> 1;
        const uint32_t to = turn + hr * 64;
        const uint32_t gw = (uint32_t)((hr >> 2) ^ ((hr >> 1) & 1)) & 3u;
#pragma unroll
        for (int j = 0; j < 32; j += 16) {
          float h[8];
#pragma unroll
          for (int m = 0; m < 8; ++m) {
            const float2 s = *reinterpret_cast<const float2*>(sc + j + 2 * m);
            h[m] = gated(__uint_as_float(d[j + 2 * m]) * wts * s.x, __uint_as_float(d[j + 2 * m + 1]) * wts * s.y, lane, lim) *
                   wt[j + 2 * m + (lane & 1)];
          }
          st_shared16(to + ((((lane & 1) * 2 + (j >> 4)) ^ gw) << 4), pack2<T>(h[0], h[1]), pack2<T>(h[2], h[3]),
                      pack2<T>(h[4], h[5]), pack2<T>(h[6], h[7]));
        }
        __syncwarp();
        const int r = 4 * (e >> 1) + 2 * (i & 1) + (e & 1), q = lane & 3;
        const uint32_t from = turn + r * 64, gr = (uint32_t)((r >> 2) ^ ((r >> 1) & 1)) & 3u;
        const int base = ((row - lane) >> 1) + 4 * q;
        T* yp = y + tok * ld + base;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint4 o = read_turned(from + (((2 * u + (i >> 1)) ^ gr) << 4));
          const int t0 = 2 * (lane >> 2) + u, t1 = t0 + 16;
          if ((FULL || t0 < left) && 2 * base < g.n) *reinterpret_cast<uint2*>(yp + (int64_t)t0 * ld) = make_uint2(o.x, o.y);
          if ((FULL || t1 < left) && 2 * base < g.n) *reinterpret_cast<uint2*>(yp + (int64_t)t1 * ld) = make_uint2(o.z, o.w);
        }
      } else {
        const uint32_t to = turn + lane * 64, gw = (uint32_t)((lane >> 3) + (lane >> 1)) & 3u;
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          const float4 s0 = *reinterpret_cast<const float4*>(sc + j), s1 = *reinterpret_cast<const float4*>(sc + j + 4);
          const float s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
          float v[8];
#pragma unroll
          for (int m = 0; m < 8; ++m) v[m] = __uint_as_float(d[j + m]) * wts * s[m];
          st_shared16(to + (((j >> 3) ^ gw) << 4), pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]),
                      pack2<T>(v[6], v[7]));
        }
        __syncwarp();
        const int r = 8 * (e >> 1) + 2 * i + (e & 1);
        const uint32_t from = turn + r * 64, gr = (uint32_t)((r >> 3) + (r >> 1)) & 3u;
        const int base = row - lane + 8 * (lane & 3);
        T* yp = y + (tok + (lane >> 2)) * ld + base;
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          const uint4 o = read_turned(from + (((j >> 3) ^ gr) << 4));
          if ((FULL || j + (lane >> 2) < left) && base < g.n) *reinterpret_cast<uint4*>(yp + (int64_t)j * ld) = o;
        }
      }
      __syncwarp();
      return;
    }
  }
  const bool in = row < g.n;
  if constexpr (SWIGLU) {
    T* yp = y + (tok + (lane & 1)) * ld + (row >> 1);
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
      if (FULL || j < left) {
        const float2 s = *reinterpret_cast<const float2*>(sc + j);
        const float h = gated(__uint_as_float(d[j]) * wts * s.x, __uint_as_float(d[j + 1]) * wts * s.y, lane, lim) *
                        wt[j + (lane & 1)];
        if (in && (FULL || j + (lane & 1) < left)) yp[(int64_t)j * ld] = to_out<T>(h);
      }
    }
  } else {
    T* yp = y + tok * ld + row;
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      if (FULL || j < left) {
        const float4 s = *reinterpret_cast<const float4*>(sc + j);
        const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int m = 0; m < 4; ++m)
          if (in && (FULL || j + m < left)) yp[(int64_t)(j + m) * ld] = to_out<T>(__uint_as_float(d[j + m]) * wts * v[m]);
      }
    }
  }
  __syncwarp();   // the warp's next read of tensor memory needs all of its lanes
}

// The same for an odd_row or odd_cols, in 64 bits, where s w is exact and the result rounds once. False, and nothing is done,
// where all that such scales multiply is zero and they are small (weight rows of zeros have the smallest scale), or a
// token's weight is zero. s: what store_chunk would take; weight: the lane's token's; odd: 32 floats of the warp's. Rare,
// out of line: within the loop it cost products of K 512 6%.
struct Chunk {
  uint32_t d[32];
};
template <bool SWIGLU, typename T>
__device__ __noinline__ bool store_wide(const Args& a, Chunk v, int64_t tok, int row, int lane, int left, float wts, float s,
                                        float weight, float* odd) {
  const Fp4MmArgs& g = a.g;
  const bool in = row < g.n, col_odd = !SWIGLU && weight != 0.f && odd_col(s), row_odd = wts != 0.f && odd_row(wts);
  odd[lane] = col_odd ? 1.f : 0.f;
  __syncwarp();
  float sum = (col_odd && !(fabsf(s) < 1.f)) || (row_odd && !(fabsf(wts) < 1.f)) ? 1.f : 0.f;
#pragma unroll
  for (int j = 0; j < 32; j += 4) {
    const float4 f = *reinterpret_cast<const float4*>(odd + j);
    const float w[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
    for (int m = 0; m < 4; ++m) sum = fmaf(fabsf(__uint_as_float(v.d[j + m])), row_odd ? 1.f : w[m], sum);
  }
  __syncwarp();
  if (!__any_sync(0xffffffffu, sum != 0.f)) return false;
  s = weight = 1.f;
  if (lane < left) {
    if (g.a_ts != nullptr) s = g.a_ts[g.a_ts_row ? tok + lane : 0];
    if (g.row_weight != nullptr) weight = g.row_weight[tok + lane];
  }
  T* yp = reinterpret_cast<T*>(g.y) + tok * g.ldy;
  const float lim = g.limit > 0.f ? g.limit : INFINITY;
#pragma unroll
  for (int j = 0; j < 32; j += 2) {
    float h[2], w[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      w[m] = __shfl_sync(0xffffffffu, weight, j + m);
      const double f = (double)__shfl_sync(0xffffffffu, s, j + m) * (double)wts;
      h[m] = (float)((double)__uint_as_float(v.d[j + m]) * f * (SWIGLU ? 1.0 : (double)w[m]));
    }
    if constexpr (SWIGLU) {
      const float o = gated(h[0], h[1], lane, lim) * w[lane & 1];
      if (in && j + (lane & 1) < left) yp[(j + (lane & 1)) * g.ldy + (row >> 1)] = to_out<T>(o);
    } else {
#pragma unroll
      for (int m = 0; m < 2; ++m)
        if (in && j + m < left) yp[(j + m) * g.ldy + row] = to_out<T>(h[m]);
    }
  }
  __syncwarp();
  return true;
}

template <bool NV, bool SWIGLU, Form FORM, typename T>
__global__ void __launch_bounds__(NTHREADS, 1) fp4_mm_kernel(const __grid_constant__ Args a) {
  constexpr bool PAIR = FORM == PAIRED;
  extern __shared__ uint8_t raw[];
  // (both CTAs of a pair round the same address up, so that their stages lie at the same places)
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  const int s_bytes = SF_BLOCK<NV> * (1 + a.sblk);
  uint8_t* sA = base;
  uint8_t* sB = sA + a.stages * A_BYTES;
  uint8_t* sS = sB + a.stages * a.b_bytes;
  Ctl& c = *reinterpret_cast<Ctl*>(sS + a.stages * s_bytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const int rank = PAIR ? (int)(blockIdx.x & 1) : 0;
  const int piece = FORM == SPLIT ? (int)blockIdx.x % a.split : 0;
  const int first = PAIR ? (int)(blockIdx.x >> 1) : FORM == SPLIT ? (int)blockIdx.x / a.split : (int)blockIdx.x;
  const int stride = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;   // (SPLIT: one tile a cluster)
  const Fp4MmArgs& g = a.g;

  if (warp == 0) {
    if (lane < a.stages) {
      mbar_init(smem_addr(&c.full[lane]), 2);
      mbar_init(smem_addr(&c.empty[lane]), 1);
    }
    if (lane < RING) mbar_init(smem_addr(&c.told[lane]), 1);
    if (lane < 2) {
      mbar_init(smem_addr(&c.accfull[lane]), 1);
      mbar_init(smem_addr(&c.accempty[lane]), PAIR ? 2 * EPI_WARPS : EPI_WARPS);
    }
    if (lane == 0) {
      mbar_init(smem_addr(&c.shared), 2 * EPI_WARPS);
      mbar_init(smem_addr(&c.drain), 1);
      c.abort = 0;
    }
    mbar_init_fence();
  }
  if (warp == MMA_WARP) {
    if constexpr (PAIR)
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_addr(&c.tmem_base)),
                   "n"(TMEM_COLS)
                   : "memory");
    else
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_addr(&c.tmem_base)),
                   "n"(TMEM_COLS)
                   : "memory");
  }
  if (warp == CODE_WARP && lane == 0) {
    prefetch_map(&a.map_w);
    prefetch_map(&a.map_a);
    prefetch_map(&a.map_ws);
    prefetch_map(&a.map_as);
    // The first weights on their way to L2 while the kernel before this one ends. Nothing is read yet: what it
    // writes, were it these weights, is still seen by the copies behind the wait.
    if (FORM != PAIRED && g.offsets == nullptr && a.ahead > 0) {
      const int nb = (g.n + 127) >> 7, tile = FORM == SPLIT ? (int)blockIdx.x / a.split : (int)blockIdx.x;
      const int all = (a.ksteps + 3) >> 2, k0 = FORM == SPLIT ? all * ((int)blockIdx.x % a.split) / a.split : 0;
      for (int k = k0; k < min(all, k0 + a.ahead); ++k) prefetch_2d(&a.map_w, k * 128, (tile % nb) * 128);
    }
  }
  pdl_wait();
  pdl_trigger();
  if (warp == 0) {
    // tiles before each matrix
    const int nb = (g.n + (PAIR ? 255 : 127)) / (PAIR ? 256 : 128);
    int run = 0;
    bool down = false;
    for (int m0 = 0; m0 < g.mats; m0 += 32) {
      const int m = m0 + lane;
      const int r0 = m < g.mats ? group_begin(g, m) : 0, cnt = m < g.mats ? group_begin(g, m + 1) - r0 : 0;
      down |= cnt < 0;
      const int v = (cnt + a.nt - 1) / a.nt * nb;
      int inc = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
      }
      if (m < g.mats) {
        c.tiles[m] = run + inc - v;
        c.rows[m] = r0;
        if (m == g.mats - 1) c.rows[g.mats] = r0 + cnt;
      }
      run += __shfl_sync(0xffffffffu, inc, 31);
    }
    // Offsets that descend name rows more than once, in all perhaps more than the tiles can be counted: no tile is made.
    down = __any_sync(0xffffffffu, down);
    if (lane == 0) c.tiles[g.mats] = down ? 0 : run;
    if (lane == 0 && down) atomicExch(&g_err, 1);
  }
  fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();
  fence_after();
  const uint32_t tbase = c.tmem_base;
  const int total = c.tiles[g.mats];
  const int kall = (a.ksteps + 3) >> 2;
  const int kbegin = FORM == SPLIT ? kall * piece / a.split : 0, kend = FORM == SPLIT ? kall * (piece + 1) / a.split : kall;
  volatile int* abortf = &c.abort;

  if (warp == CODE_WARP || warp == SCALE_WARP) {
    if (elect_one()) {
      uint32_t it = 0, s = 0, ph = 1, n = 0;
      bool ok = true;
      const bool codes = warp == CODE_WARP;
      const uint32_t own0 = smem_addr(&c.full[0]), full0 = PAIR ? in_first(own0) : own0, empty0 = smem_addr(&c.empty[0]);
      const uint32_t a0 = smem_addr(sA), b0 = smem_addr(sB), s0 = smem_addr(sS);
      for (int i = first; ok && i < total; i += stride, ++n) {
        const Tile t = tile_at<PAIR>(a, c, i);
        if (!codes) {
          // For the products and the readback, which would find it in 700 to 1100 cycles a tile. The place is free: the last
          // stage of the tile before was, so that a tile at most MAX_STAGES before that one was begun, and the readback
          // of the second before it is over.
          c.tile[n % RING] = make_int4(t.mat, t.n0, t.row0 + t.t0, t.cnt);
          c.tile_t0[n % RING] = t.t0;
          arrive(smem_addr(&c.told[n % RING]));
        }
        // token rows that this CTA brings: all, or its half of the pair's columns
        const int half = PAIR ? ((t.cnt + 15) >> 4) << 3 : t.cnt;
        const bool narrow = PAIR && half <= NT_APART / 2;
        const int box = narrow ? NT_APART / 2 : a.box, nbox = (half + box - 1) / box;
        const CUtensorMap* map_a = narrow ? &a.map_n : &a.map_a;
        const int wrow = t.mat * g.n + t.n0 + rank * 128, arow = t.row0 + t.t0 + rank * half;
        const int wblk = t.mat * ((g.n + 127) >> 7) + (t.n0 >> 7) + rank;
        const uint32_t bytes = (PAIR ? 2u : 1u) * (codes ? A_BYTES + nbox * box * 128 : s_bytes);
        for (int k = kbegin; k < kend; ++k, ++it) {
          if (!wait(abortf, empty0 + 8 * s, ph)) {
            ok = false;
            break;
          }
          const uint32_t full = full0 + 8 * s;
          if (rank == 0) mbar_expect_tx(own0 + 8 * s, bytes);
          if (codes) {
            load_2d<PAIR>(a0 + s * A_BYTES, &a.map_w, k * 128, wrow, full);
            const uint32_t dst = b0 + s * a.b_bytes;
            for (int b = 0; b < nbox; ++b) load_2d<PAIR>(dst + b * box * 128, map_a, k * 128, arow + b * box, full);
          } else {
            const uint32_t dst = s0 + s * s_bytes;
            const int at = k * (NV ? 4 : 2);
            load_3d<PAIR>(dst, &a.map_ws, 0, at, wblk, full);
            load_3d<PAIR>(dst + SF_BLOCK<NV>, &a.map_as, 0, at, t.blk, full);
          }
          if (++s == (uint32_t)a.stages) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      // The copies in flight land before the CTA's shared memory goes (a stage that only one of the warps filled
      // never completes: its wait ends by its limit).
      if (!ok && rank == 0) {
        const uint32_t n = it < (uint32_t)a.stages ? it : (uint32_t)a.stages;
        for (uint32_t j = it - n; j < it; ++j)
          for (uint32_t p = 0; p < WAIT_LIMIT / 16; ++p)
            if (mbar_try_wait_sleep(own0 + 8 * (j % a.stages), (j / a.stages) & 1u, 1000u)) break;
      }
    }
    __syncwarp();
  } else if (warp == MMA_WARP) {
    if (rank == 0 && elect_one()) {
      uint32_t s = 0, ph = 0, n = 0;
      bool ok = true;
      const uint64_t ad0 = sdesc(smem_addr(sA)), bd0 = sdesc(smem_addr(sB)), sd0 = sf_desc(smem_addr(sS));
      const uint32_t b_step = (uint32_t)(a.b_bytes >> 4), s_step = (uint32_t)(s_bytes >> 4);
      const uint32_t full0 = smem_addr(&c.full[0]), empty0 = smem_addr(&c.empty[0]);
      const int kfull = a.ksteps >> 2, ktail = a.ksteps & 3;
      for (int i = first; ok && i < total; i += stride, ++n) {
        if (!wait(abortf, smem_addr(&c.told[n % RING]), (n / RING) & 1u)) break;
        const int cnt = c.tile[n % RING].w, t0 = c.tile_t0[n % RING];
        const uint32_t q = n & 1u, acc = tbase + q * NT_APART;
        const uint32_t sfb = tbase + SFB_COL + ((t0 & 127) >> 5);
        const uint32_t id = idesc<NV, PAIR>(PAIR ? (uint32_t)(cnt + 15) & ~15u : (uint32_t)(cnt + 7) & ~7u);
        if (!wait(abortf, smem_addr(&c.accempty[q]), ((n >> 1) & 1u) ^ 1u)) break;
        if (PAIR && a.nt > NT_APART && n > 0 && !wait(abortf, smem_addr(&c.shared), (n - 1) & 1u)) break;
        fence_after();
        auto stage = [&](auto blocks, auto whole, int k) {
          if (!wait(abortf, full0 + 8 * s, ph, g.probes)) {
            ok = false;
            return;
          }
          fence_after();
          issue<NV, PAIR, decltype(blocks)::value, decltype(whole)::value>(tbase, acc, sfb, ad0 + s * (A_BYTES >> 4),
                                                                           bd0 + s * b_step, sd0 + s * s_step, id, ktail, k == kbegin);
          commit_to<PAIR>(empty0 + 8 * s);
          if (++s == (uint32_t)a.stages) {
            s = 0;
            ph ^= 1u;
          }
        };
        auto tile = [&](auto blocks) {
          for (int k = kbegin; ok && k < min(kend, kfull); ++k) stage(blocks, std::true_type{}, k);
          if (ok && kfull < kend) stage(blocks, std::false_type{}, kfull);
        };
        if ((t0 & 127) + cnt > 128) tile(std::integral_constant<int, 2>{});
        else tile(std::integral_constant<int, 1>{});
        if (ok) commit_to<PAIR>(smem_addr(&c.accfull[q]));
      }
      // every MMA issued has completed once `drain` fires
      commit_to<PAIR>(smem_addr(&c.drain));
      for (uint32_t p = 0; p < WAIT_LIMIT; ++p)
        if (mbar_try_wait_sleep(smem_addr(&c.drain), 0, 1000u)) break;
    }
    __syncwarp();
  } else {
    constexpr int CHUNKS = NT_MAX / 64;
    uint32_t n = 0;
    const int half = warp >> 2;   // this warp's 32-column chunks: half, half + 2, ...
    const uint32_t quarter = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t turn = smem_addr(c.turn[warp]);
    float* sc = c.scale[warp];
    float* wt = c.weight[warp];
    // a tile's place, scales and weights are fetched while the one before it is stored (1900 cycles a tile otherwise)
    int4 next = make_int4(0, 0, 0, 0);
    float s_next[CHUNKS], w_next[CHUNKS], wts_next = 1.f;
    auto look_ahead = [&](int i, uint32_t n) {
      if (i >= total) return true;
      if (!warp_wait(abortf, smem_addr(&c.told[n % RING]), (n / RING) & 1u, 0u)) return false;
      next = c.tile[n % RING];
      const int row = next.y + rank * 128 + (warp & 3) * 32 + lane;
      wts_next = 1.f;
      if (g.w_ts != nullptr && row < g.n)
        wts_next = g.w_ts[g.w_ts_n == 0 ? row : next.x * g.w_ts_n + (g.w_ts_n == 2 ? (row & 1) : 0)];
#pragma unroll
      for (int j = 0; j < CHUNKS; ++j) {
        const int col = 32 * (half + 2 * j) + lane;
        const int64_t tok = (int64_t)next.z + col;
        s_next[j] = w_next[j] = 1.f;
        if (col < next.w) {
          if (g.a_ts != nullptr) s_next[j] = g.a_ts[g.a_ts_row ? tok : 0];
          if (g.row_weight != nullptr) w_next[j] = g.row_weight[tok];
        }
      }
      return true;
    };
    bool ok = look_ahead(first, 0u);
    for (int i = first; ok && i < total; i += stride, ++n) {
      const int n0 = next.y + rank * 128, cnt = next.w;
      const int64_t tok0 = next.z;
      const float wts = wts_next;
#pragma unroll
      for (int j = 0; j < CHUNKS; ++j) {
        sc[32 * j + lane] = SWIGLU ? s_next[j] : s_next[j] * w_next[j];
        if (SWIGLU) wt[32 * j + lane] = w_next[j];
      }
      bool odd = odd_row(wts);   // or, with weights, a column
      if (!SWIGLU && g.row_weight != nullptr) {
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j) {
          wt[32 * j + lane] = w_next[j];
          odd |= odd_col(s_next[j] * w_next[j]);
        }
      }
      const bool wide = __any_sync(0xffffffffu, odd);
      __syncwarp();
      if constexpr (FORM != SPLIT) ok = look_ahead(i + stride, n + 1);
      const uint32_t q = n & 1u;
      const uint32_t acc = tbase + q * NT_APART + quarter;
      const int row = n0 + (warp & 3) * 32 + lane;
      const bool vec = a.vec && (n0 + 128 <= g.n || (SWIGLU ? g.n % 16 : g.n % 8) == 0);
      if (!ok || !warp_wait(abortf, smem_addr(&c.accfull[q]), (n >> 1) & 1u, g.probes)) break;
      fence_after();
      if constexpr (FORM == SPLIT) {
        // the products have read all stages: their place takes this piece's sums, [token][row]
        float* part = reinterpret_cast<float*>(base);
        for (int ch = half; ch * 32 < cnt; ch += 2) {
          uint32_t d[32];
          ld32(acc + ch * 32, d);
          ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) part[(ch * 32 + j) * 128 + (warp & 3) * 32 + lane] = __uint_as_float(d[j]);
        }
        break;
      }
      // This warp's chunks, those in the columns that the next tile's accumulator shares first: the last ones of the lower
      // accumulator, the first ones of the upper.
      const int mine = ((cnt + 31) / 32 - half + 1) >> 1;
      const bool overlaps = PAIR && a.nt > NT_APART;
      for (int u = 0; u < mine; ++u) {
        const int j = overlaps && q == 0 ? mine - 1 - u : u, ch = half + 2 * j;
        uint32_t d[32];
        ld32(acc + ch * 32, d);
        ld_wait();
        if (u == mine - 1 || (overlaps && u == 0)) {
          fence_before();
          __syncwarp();
          if (lane == 0 && overlaps && u == 0) release<PAIR>(smem_addr(&c.shared));
          if (lane == 0 && u == mine - 1) release<PAIR>(smem_addr(&c.accempty[q]));
        }
        const int left = cnt - ch * 32;
        if (wide) {
          Chunk v;
#pragma unroll
          for (int m = 0; m < 32; ++m) v.d[m] = d[m];
          if (store_wide<SWIGLU, T>(a, v, tok0 + ch * 32, row, lane, min(left, 32), wts, sc[32 * j + lane],
                                    g.row_weight != nullptr ? wt[32 * j + lane] : 1.f, reinterpret_cast<float*>(c.turn[warp])))
            continue;
        }
        if (left >= 32)
          store_chunk<SWIGLU, true, T>(a, d, tok0 + ch * 32, row, lane, 32, vec, wts, sc + 32 * j, wt + 32 * j, turn);
        else
          store_chunk<SWIGLU, false, T>(a, d, tok0 + ch * 32, row, lane, left, vec, wts, sc + 32 * j, wt + 32 * j, turn);
      }
      if (mine <= 0) {
        fence_before();
        __syncwarp();
        if (lane == 0 && overlaps) release<PAIR>(smem_addr(&c.shared));
        if (lane == 0) release<PAIR>(smem_addr(&c.accempty[q]));
      }
      __syncwarp();
    }
  }
  fence_before();
  __syncthreads();
  if constexpr (FORM == SPLIT) {
    // each CTA adds and stores its share of the tokens
    cluster_sync();
    if (first < total) {
      const Tile t = tile_at<false>(a, c, first);
      const uint32_t part = smem_addr(base);
      const int mine = (t.cnt - piece + a.split - 1) / a.split * 128;
      for (int i = tid; i < mine; i += NTHREADS) {
        const int col = piece + (i >> 7) * a.split, r = i & 127, row = t.n0 + r;
        float v = 0.f;
        for (int p = 0; p < a.split; ++p) v += peer_float(part + (col * 128 + r) * 4, p);
        if (row < g.n) {
          const float s = g.a_ts ? g.a_ts[g.a_ts_row ? t.t0 + col : 0] : 1.f;
          const float w = g.w_ts ? g.w_ts[g.w_ts_n == 0 ? row : 0] : 1.f;
          v = !odd_row(w) ? v * w * s : (float)((double)v * ((double)s * (double)w));
          reinterpret_cast<T*>(g.y)[(int64_t)(t.t0 + col) * g.ldy + row] = to_out<T>(v);
        }
      }
    }
    cluster_sync();   // the others have read this CTA's sums
  }
  if constexpr (PAIR) cluster_sync();   // the other CTA's products read this one's shared memory to the end
  if (warp == MMA_WARP) {
    fence_after();
    if constexpr (PAIR) {
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n");
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tbase), "n"(TMEM_COLS));
    } else {
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n");
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tbase), "n"(TMEM_COLS));
    }
  }
}

}  // namespace fp4mm

static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}

// codes [rows][row_bytes] in boxes of `box` rows x 128 bytes
static cudaError_t code_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t row_bytes, uint32_t box) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = encode_fn();
  if (enc == nullptr) return cudaErrorNotSupported;
  const cuuint64_t dims[2] = {row_bytes, rows};
  const cuuint64_t strides[1] = {row_bytes};
  const cuuint32_t boxes[2] = {128, box};
  const cuuint32_t es[2] = {1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, boxes, es,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

// scale atoms [blocks][atoms][512 bytes] in boxes of `row_blocks` blocks x `along` atoms
static cudaError_t scale_map(CUtensorMap* map, const void* base, uint64_t blocks, uint64_t atoms, uint32_t row_blocks,
                             uint32_t along) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = encode_fn();
  if (enc == nullptr) return cudaErrorNotSupported;
  const cuuint64_t dims[3] = {128, atoms, blocks};
  const cuuint64_t strides[2] = {512, atoms * 512};
  const cuuint32_t boxes[3] = {128, along, row_blocks};
  const cuuint32_t es[3] = {1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<void*>(base), dims, strides, boxes, es,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <bool NV, bool SWIGLU, fp4mm::Form FORM, typename T>
static cudaError_t launch_mm(const fp4mm::Args& a, int grid, size_t smem, cudaStream_t st) {
  const auto kernel = fp4mm::fp4_mm_kernel<NV, SWIGLU, FORM, T>;
  // the limit belongs to the kernel on one device: set once for each
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (!(done.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, fp4mm::SMEM_LIMIT);
    if (e != cudaSuccess) return e;
    done.fetch_or(bit, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(fp4mm::NTHREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = FORM == fp4mm::PAIRED ? 2 : a.split;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = FORM == fp4mm::SINGLE ? 1 : 2;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <fp4mm::Form FORM, typename T>
static cudaError_t launch_mm_t(const fp4mm::Args& a, int grid, size_t smem, cudaStream_t st) {
  if constexpr (FORM != fp4mm::SPLIT) {
    if (a.g.swiglu) return a.g.nv ? launch_mm<true, true, FORM, T>(a, grid, smem, st) : launch_mm<false, true, FORM, T>(a, grid, smem, st);
  }
  return a.g.nv ? launch_mm<true, false, FORM, T>(a, grid, smem, st) : launch_mm<false, false, FORM, T>(a, grid, smem, st);
}

template <fp4mm::Form FORM>
static cudaError_t launch_mm_f(const fp4mm::Args& a, int dtype, int grid, size_t smem, cudaStream_t st) {
  if (dtype == SB_F32) return launch_mm_t<FORM, float>(a, grid, smem, st);
  if (dtype == SB_F16) return launch_mm_t<FORM, __half>(a, grid, smem, st);
  return launch_mm_t<FORM, __nv_bfloat16>(a, grid, smem, st);
}

cudaError_t launch_fp4_mm(const Fp4MmArgs& g, int dtype, cudaStream_t st) {
  using namespace fp4mm;
  Args a;
  memset(&a, 0, sizeof a);
  a.g = g;
  a.ksteps = (g.kp + 63) / 64;
  const int atoms = g.nv ? a.ksteps : (a.ksteps + 1) / 2, sms = num_sms();
  // Token columns of a tile: all of them when they fit one, else 128 or 192 (whole 64-row steps of the
  // scale atoms), whichever leaves fewer columns unused. With groups the counts are on the device: the
  // average decides.
  if (g.offsets != nullptr) {
    const int avg = (g.m + g.mats - 1) / g.mats;
    a.nt = avg > 128 ? 192 : 128;
  } else if (g.m <= NT_APART) {
    a.nt = (g.m + 15) & ~15;
  } else {
    const int c128 = (g.m + 127) / 128 * 128, c192 = (g.m + 191) / 192 * 192;
    a.nt = c128 < c192 - c192 / 8 ? 128 : 192;
  }
  // tiles of 128 rows, or with groups the most there can be
  const int64_t nb = (g.n + 127) / 128;
  const int64_t tt = g.offsets ? (int64_t)g.m / a.nt + (g.mats < g.m ? g.mats : g.m) : (g.m + a.nt - 1) / a.nt;
  const int64_t tiles = tt * nb;
  // Pairs where tiles of full width need more than one round of the SMs: they halve the token bytes that each SM copies and
  // reads per product (1024 x 4096 x 8192: 18.0 us, 26.3 without; 2048 x 2048 x 4096: 12.7 and 16.0). With fewer tiles single
  // CTAs use more SMs (256 x 8192 x 8192: 15.0, pairs 17.8), and narrow tiles are bound by the weights, which pairs do not
  // share.
  const bool pair = a.nt >= 128 && g.m >= 128 * (int64_t)g.mats && tiles > sms;
  // A pair's tiles have 256 tokens: fewer bytes of shared memory per product than 192, which have both accumulators to
  // themselves (when this was chosen, 8192 x 4096 x 8192: 104 us and 124; x 2048: 45 and 54; x 512 and 32 groups of 512
  // tokens: even; now 98, 34).
  if (pair) a.nt = 256;
  // K is split, for one token tile, as far as the SMs go and every piece keeps two stages (one token against 4096 x 8192:
  // 12.0 us whole, 9.3 in four pieces, 8.6 with the weights ahead in L2).
  a.split = 1;
  if (g.offsets == nullptr && tt == 1)
    while (a.split < 8 && tiles * a.split * 2 <= sms && (a.ksteps + 3) / 4 >= a.split * 4) a.split *= 2;
  // (one token tile: a CTA's first tile is its own row block, whose stages it all reads; no more than a quarter of L2 in all,
  // or the first ones leave it before they are copied: 1 x 18944 x 32768 took 88 us without this limit, 76 with it)
  if (g.offsets == nullptr && tt == 1) {
    const int64_t ctas = tiles * a.split < sms ? tiles * a.split : sms, most = L2_AHEAD / (ctas * A_BYTES);
    a.ahead = ((a.ksteps + 3) / 4 + a.split - 1) / a.split;
    if (a.ahead > most) a.ahead = (int)most;
  }
  // Token rows of a copy: a whole tile's (of a pair's half), but with narrow groups 32 at a time, as many as the group has.
  // (Three copies of 32 rows in place of one of 96 made the copying thread the bound: 0.33 us a stage, one copy 0.26.)
  a.box = pair ? a.nt / 2 : g.offsets ? BOX : a.nt;
  a.b_bytes = (pair ? a.nt / 2 : a.nt) * 128;
  a.sblk = a.nt > 128 ? 2 : 1;
  a.vec = (reinterpret_cast<uintptr_t>(g.y) & 15u) == 0 && g.ldy % 8 == 0;
  const int sf = g.nv ? SF_BLOCK<true> : SF_BLOCK<false>;
  const int stage = A_BYTES + a.b_bytes + sf * (1 + a.sblk);
  const int room = SMEM_LIMIT - 1024 - (int)sizeof(Ctl);
  a.stages = room / stage < MAX_STAGES ? room / stage : MAX_STAGES;
  const size_t smem = 1024 + (size_t)a.stages * stage + sizeof(Ctl);
  const uint64_t row_bytes = (uint64_t)g.kp / 2;
  const uint64_t a_blocks = g.offsets ? (uint64_t)g.m / 128 + g.mats : ((uint64_t)g.m + 127) / 128;
  const uint32_t along = g.nv ? 4 : 2;
  cudaError_t e = code_map(&a.map_w, g.w, (uint64_t)g.mats * g.n, row_bytes, 128);
  if (e == cudaSuccess) e = code_map(&a.map_a, g.a, (uint64_t)g.m, row_bytes, (uint32_t)a.box);
  if (e == cudaSuccess && pair) e = code_map(&a.map_n, g.a, (uint64_t)g.m, row_bytes, NT_APART / 2);
  if (e == cudaSuccess) e = scale_map(&a.map_ws, g.w_s, (uint64_t)g.mats * nb, (uint64_t)atoms, 1, along);
  if (e == cudaSuccess) e = scale_map(&a.map_as, g.a_s, a_blocks, (uint64_t)atoms, (uint32_t)a.sblk, along);
  if (e != cudaSuccess) return e;
  if (pair) return launch_mm_f<PAIRED>(a, dtype, sms & ~1, smem, st);
  if (a.split > 1) return launch_mm_f<SPLIT>(a, dtype, (int)tiles * a.split, smem, st);
  return launch_mm_f<SINGLE>(a, dtype, (int)(tiles < sms ? tiles : sms), smem, st);
}

cudaError_t fp4_mm_error(int* host_out, cudaStream_t st) {
  void* p = nullptr;
  cudaError_t e = cudaGetSymbolAddress(&p, fp4mm::g_err);
  if (e == cudaSuccess) e = cudaMemcpyAsync(host_out, p, sizeof(int), cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaMemsetAsync(p, 0, sizeof(int), st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  return e;
}

}  // namespace sb
