// Products of two microscaled 4-bit operands on the tensor cores: y[token][n] = sum_k a[token][k] W[n][k],
// one weight matrix for all tokens, or one per expert with the tokens' rows sorted by expert.
//
// tcgen05.mma kind::mxf4nvf4 / kind::mxf4 multiplies e2m1 by e2m1 with a scale per 16 (e4m3) or per 32
// (e8m0) values of either side and sums in fp32, so the whole K accumulates in tensor memory and is
// read once; the fp32 tensor scales are applied there.
//
// The weights are the M operand (128 rows a tile), the tokens N: a token tile takes any multiple of 8
// columns, so one decoded token costs an 8-column tile and ragged expert groups waste at most 7.
// Stages hold 256 K: 128 weight rows and the tile's token rows of 128 bytes each, landed by TMA in the
// 128-byte-swizzled K-major form, and their scale atoms by bulk copies. Roles (192 threads): warp 4
// copies, warp 5 moves scale atoms to tensor memory and issues the MMAs, warps 0-3 read the
// accumulator (thread = weight row) and store 32 consecutive outputs of one token per instruction.
// Two accumulators of up to 192 columns alternate, so that one tile's readback overlaps the next
// tile's products; 192 and not 256 leaves room for the scales beside two of them.
//
// Every wait is bounded: on timeout the CTA sets the device's error word and winds down.
#include <cudaTypedefs.h>
#include <string.h>

#include <atomic>

#include "sb_fp4.h"
#include "sb_launch.h"
#include "sb_tcgen05.cuh"

namespace sb {
namespace fp4mm {

using namespace tc5;

constexpr int NTHREADS = 192;
constexpr int PRODUCER_WARP = 4;
constexpr int MMA_WARP = 5;
constexpr int NT_MAX = 192;          // token columns of a tile
constexpr int BOX = 32;              // token rows of one copy with expert groups
constexpr int A_BYTES = 128 * 128;   // a stage's weight rows
constexpr int SF_BLOCK = 4 * 512;    // a stage's scale atoms of 128 rows
constexpr int MAX_STAGES = 10;
constexpr int MAX_MATS = 1024;
constexpr int TMEM_COLS = 512;
constexpr int SFA_COL = 2 * NT_MAX;  // scale factors: 4 atoms x 4 columns of the weights,
constexpr int SFB_COL = SFA_COL + 16;  // 4 atoms x 8 columns of the tokens (two row blocks)
constexpr uint32_t WAIT_LIMIT = 1u << 16;
constexpr int SMEM_LIMIT = 232448;

__device__ int g_err;

struct Args {
  CUtensorMap map_w, map_a;
  Fp4MmArgs g;
  int nt;            // token columns of a full tile (a multiple of 64 when a matrix has several)
  int box;           // token rows of one copy
  int stages;
  int b_bytes;       // token rows of a stage
  int sfb_bytes;     // their scale atoms
  int atoms;         // scale atoms along K
  int ksteps;        // MMAs along K (64 values each)
};

struct Ctl {
  uint64_t full[MAX_STAGES], empty[MAX_STAGES], accfull[2], accempty[2], drain;
  uint32_t tmem_base;
  int abort;
  int tiles[MAX_MATS + 1];   // tiles before each matrix
  int rows[MAX_MATS + 1];    // first token row of each matrix's group, and the end of the last
};

struct Tile {
  int mat, n0, t0, cnt, row0;   // matrix, first weight row, first token of the group, tokens, group's first row
  int64_t blk;                  // group's first scale row block
};

// instruction descriptor: e2m1 x e2m1, M = 128, N = n, scale byte pair `id` of both sides' words
template <bool NV>
__device__ __forceinline__ uint32_t idesc(uint32_t n, uint32_t id) {
  return (id << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((NV ? 0u : 1u) << 23) | ((128u >> 4) << 24) | (id << 29);
}

template <bool NV>
__device__ __forceinline__ void mma(uint32_t d, uint64_t ad, uint64_t bd, uint32_t id, uint32_t sfa, uint32_t sfb,
                                    uint32_t acc) {
  if constexpr (NV) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%5], [%6], p;\n}\n" ::"r"(d),
        "l"(ad), "l"(bd), "r"(id), "r"(acc), "r"(sfa), "r"(sfb));
  } else {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n}\n" ::"r"(d),
        "l"(ad), "l"(bd), "r"(id), "r"(acc), "r"(sfa), "r"(sfb));
  }
}

// one scale atom into four tensor memory columns of every 32-lane quarter
__device__ __forceinline__ void cp_sf(uint32_t taddr, uint32_t src) {
  uint64_t d = 0;
  d |= (uint64_t)((src >> 4) & 0x3FFFu);
  d |= (uint64_t)(128 >> 4) << 16;
  d |= (uint64_t)(128 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n" ::"r"(taddr), "l"(d) : "memory");
}

// the first token row of matrix mat's group (mat == mats: the end), inside [0, m] whatever the offsets hold
__device__ __forceinline__ int group_begin(const Fp4MmArgs& g, int mat) {
  return g.offsets ? min(max(g.offsets[mat], 0), g.m) : (mat == 0 ? 0 : g.m);
}

// one answer for the whole warp, whose next instructions need all of its lanes
__device__ __forceinline__ bool warp_wait(volatile int* abortf, uint32_t bar, uint32_t parity) {
  return __all_sync(0xffffffffu, wait_bounded(abortf, &g_err, bar, parity, WAIT_LIMIT));
}

// Tiles of one matrix run in bands of 12 weight blocks by all token tiles, so that the tiles in flight
// share both operands in L2.
__device__ __forceinline__ Tile tile_at(const Args& a, const Ctl& c, int i) {
  int lo = 0, hi = a.g.mats;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (c.tiles[mid] <= i) lo = mid; else hi = mid;
  }
  const int r = i - c.tiles[lo], nb = (a.g.n + 127) >> 7;
  const int tb = (c.tiles[lo + 1] - c.tiles[lo]) / nb;
  const int band = r / (12 * tb), left = r - band * 12 * tb, wide = min(12, nb - band * 12);
  Tile t;
  t.mat = lo;
  t.n0 = (band * 12 + left % wide) * 128;
  t.row0 = c.rows[lo];
  t.t0 = left / wide * a.nt;
  t.cnt = min(c.rows[lo + 1] - t.row0 - t.t0, a.nt);
  t.blk = a.g.offsets ? (t.row0 >> 7) + lo : 0;
  return t;
}

template <typename T>
__device__ __forceinline__ T to_out(float v);
template <>
__device__ __forceinline__ float to_out<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half to_out<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 to_out<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <bool NV, bool SWIGLU, typename T>
__global__ void __launch_bounds__(NTHREADS, 1) fp4_mm_kernel(const __grid_constant__ Args a) {
  extern __shared__ uint8_t raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* sA = base;
  uint8_t* sB = sA + a.stages * A_BYTES;
  uint8_t* sS = sB + a.stages * a.b_bytes;
  const int s_bytes = SF_BLOCK + a.sfb_bytes;
  Ctl& c = *reinterpret_cast<Ctl*>(sS + a.stages * s_bytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const Fp4MmArgs& g = a.g;

  if (tid == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(smem_addr(&c.full[s]), 1);
      mbar_init(smem_addr(&c.empty[s]), 1);
    }
    for (int q = 0; q < 2; ++q) {
      mbar_init(smem_addr(&c.accfull[q]), 1);
      mbar_init(smem_addr(&c.accempty[q]), 4);
    }
    mbar_init(smem_addr(&c.drain), 1);
    c.abort = 0;
    mbar_init_fence();
  }
  if (warp == MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_addr(&c.tmem_base)),
                 "n"(TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n");
  }
  if (warp == PRODUCER_WARP && lane == 0) {
    prefetch_map(&a.map_w);
    prefetch_map(&a.map_a);
  }
  pdl_wait();
  pdl_trigger();
  if (warp == 0) {
    // tiles before each matrix
    const int nb = (g.n + 127) >> 7;
    int run = 0;
    for (int m0 = 0; m0 < g.mats; m0 += 32) {
      const int m = m0 + lane;
      const int r0 = m < g.mats ? group_begin(g, m) : 0, cnt = m < g.mats ? max(group_begin(g, m + 1) - r0, 0) : 0;
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
    if (lane == 0) c.tiles[g.mats] = run;
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tbase = c.tmem_base;
  const int total = c.tiles[g.mats];
  const int kstages = (a.ksteps + 3) >> 2;
  constexpr int STEPS_PER_ATOM = NV ? 1 : 2;
  volatile int* abortf = &c.abort;

  if (warp == PRODUCER_WARP) {
    uint32_t it = 0, s = 0, ph = 0;
    bool ok = true;
    for (int i = blockIdx.x; ok && i < total; i += gridDim.x) {
      const Tile t = tile_at(a, c, i);
      const int nbox = (t.cnt + a.box - 1) / a.box;
      const int sblk = ((t.t0 & 127) + t.cnt + 127) >> 7;
      const int wrow = t.mat * g.n + t.n0, arow = t.row0 + t.t0;
      const uint8_t* ws = g.w_s + ((int64_t)t.mat * ((g.n + 127) >> 7) + (t.n0 >> 7)) * a.atoms * 512;
      const uint8_t* as = g.a_s + (t.blk + (t.t0 >> 7)) * a.atoms * 512;
      for (int k = 0; k < kstages; ++k, ++it) {
        if (!warp_wait(abortf, smem_addr(&c.empty[s]), ph ^ 1u)) {
          ok = false;
          break;
        }
        const int at0 = k * 4 / STEPS_PER_ATOM, nat = min(4 / STEPS_PER_ATOM, a.atoms - at0);
        if (elect_one()) {
          const uint32_t full = smem_addr(&c.full[s]);
          const uint32_t sf = smem_addr(sS + s * s_bytes);
          mbar_expect_tx(full, A_BYTES + nbox * a.box * 128 + (1 + sblk) * nat * 512);
          tma_load_2d(smem_addr(sA + s * A_BYTES), &a.map_w, k * 128, wrow, full);
          for (int b = 0; b < nbox; ++b)
            tma_load_2d(smem_addr(sB + s * a.b_bytes) + b * a.box * 128, &a.map_a, k * 128, arow + b * a.box, full);
          bulk_g2s(sf, ws + (int64_t)at0 * 512, nat * 512, full);
          for (int b = 0; b < sblk; ++b)
            bulk_g2s(sf + SF_BLOCK * (1 + b), as + ((int64_t)b * a.atoms + at0) * 512, nat * 512, full);
        }
        __syncwarp();
        if (++s == (uint32_t)a.stages) {
          s = 0;
          ph ^= 1u;
        }
      }
    }
    // the copies in flight land before the CTA's shared memory goes
    if (!ok) {
      const uint32_t n = it < (uint32_t)a.stages ? it : (uint32_t)a.stages;
      for (uint32_t j = it - n; j < it; ++j)
        for (uint32_t p = 0; p < WAIT_LIMIT; ++p)
          if (mbar_try_wait_sleep(smem_addr(&c.full[j % a.stages]), (j / a.stages) & 1u, 1000u)) break;
    }
  } else if (warp == MMA_WARP) {
    uint32_t s = 0, ph = 0, n = 0;
    bool ok = true;
    for (int i = blockIdx.x; ok && i < total; i += gridDim.x, ++n) {
      const Tile t = tile_at(a, c, i);
      const int sblk = ((t.t0 & 127) + t.cnt + 127) >> 7;
      const uint32_t cols = (uint32_t)(t.cnt + 7) & ~7u;
      const uint32_t q = n & 1u, acc = tbase + q * NT_MAX;
      const uint32_t sfb = tbase + SFB_COL + ((t.t0 & 127) >> 5);
      if (!warp_wait(abortf, smem_addr(&c.accempty[q]), ((n >> 1) & 1u) ^ 1u)) break;
      fence_after();
      for (int k = 0; k < kstages; ++k) {
        if (!warp_wait(abortf, smem_addr(&c.full[s]), ph)) {
          ok = false;
          break;
        }
        fence_after();
        if (elect_one()) {
          const uint32_t sa = smem_addr(sA + s * A_BYTES), sb = smem_addr(sB + s * a.b_bytes);
          const uint32_t sf = smem_addr(sS + s * s_bytes);
          const int steps = min(4, a.ksteps - 4 * k), nat = (steps + STEPS_PER_ATOM - 1) / STEPS_PER_ATOM;
          for (int j = 0; j < nat; ++j) {
            cp_sf(tbase + SFA_COL + 4 * j, sf + j * 512);
            for (int b = 0; b < sblk; ++b) cp_sf(tbase + SFB_COL + 8 * j + 4 * b, sf + SF_BLOCK * (1 + b) + j * 512);
          }
          for (int j = 0; j < steps; ++j) {
            const uint32_t id = NV ? 0u : (uint32_t)(j & 1) * 2u, at = (uint32_t)(j / STEPS_PER_ATOM);
            mma<NV>(acc, sdesc(sa + j * 32), sdesc(sb + j * 32), idesc<NV>(cols, id),
                    (tbase + SFA_COL + 4 * at) | (id << 30), (sfb + 8 * at) | (id << 30), (k | j) != 0 ? 1u : 0u);
          }
          commit(smem_addr(&c.empty[s]));
        }
        __syncwarp();
        if (++s == (uint32_t)a.stages) {
          s = 0;
          ph ^= 1u;
        }
      }
      if (!ok) break;
      if (elect_one()) commit(smem_addr(&c.accfull[q]));
      __syncwarp();
    }
    // every MMA issued has completed once `drain` fires
    if (elect_one()) commit(smem_addr(&c.drain));
    __syncwarp();
    for (uint32_t p = 0; p < WAIT_LIMIT; ++p)
      if (mbar_try_wait_sleep(smem_addr(&c.drain), 0, 1000u)) break;
  } else {
    uint32_t n = 0;
    T* y = reinterpret_cast<T*>(g.y);
    for (int i = blockIdx.x; i < total; i += gridDim.x, ++n) {
      const Tile t = tile_at(a, c, i);
      const uint32_t q = n & 1u;
      const uint32_t acc = tbase + q * NT_MAX + ((uint32_t)(warp * 32) << 16);
      const int row = t.n0 + tid;
      const bool in = row < g.n;
      float wts = 1.f;
      if (g.w_ts != nullptr) wts = g.w_ts_n == 0 ? (in ? g.w_ts[row] : 0.f) : g.w_ts[t.mat * g.w_ts_n + (g.w_ts_n == 2 ? (row & 1) : 0)];
      if (!warp_wait(abortf, smem_addr(&c.accfull[q]), (n >> 1) & 1u)) break;
      fence_after();
      for (int c0 = 0; c0 < t.cnt; c0 += 32) {
        uint32_t d[32];
        ld32(acc + c0, d);
        const int64_t tok = (int64_t)t.row0 + t.t0 + c0;
        const int left = min(32, t.cnt - c0);
        float ats = 1.f, rw = 1.f;
        if (lane < left) {
          if (g.a_ts != nullptr) ats = g.a_ts[g.a_ts_row ? tok + lane : 0];
          if (g.row_weight != nullptr) rw = g.row_weight[tok + lane];
        }
        ld_wait();
        if (SWIGLU) {
          T* yp = y + (tok + (lane & 1)) * g.ldy + (row >> 1);
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            if (j < left) {
              const float s0 = __shfl_sync(0xffffffffu, ats, j), s1 = __shfl_sync(0xffffffffu, ats, j + 1);
              const float w = __shfl_sync(0xffffffffu, rw, j + (lane & 1));
              const float v0 = __uint_as_float(d[j]) * (s0 * wts), v1 = __uint_as_float(d[j + 1]) * (s1 * wts);
              // the even lane holds gate, the odd lane up: each takes one of the two tokens
              const float o = __shfl_xor_sync(0xffffffffu, (lane & 1) ? v0 : v1, 1);
              float gate = (lane & 1) ? o : v0, up = (lane & 1) ? v1 : o;
              if (g.limit > 0.f) {
                gate = fminf(gate, g.limit);
                up = fminf(fmaxf(up, -g.limit), g.limit);
              }
              const float h = __fdividef(gate, 1.f + __expf(-gate)) * up * w;
              if (in && j + (lane & 1) < left) yp[(int64_t)j * g.ldy] = to_out<T>(h);
            }
          }
        } else {
          T* yp = y + tok * g.ldy + row;
          ats *= rw;
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            if (j < left) {
              const float s = __shfl_sync(0xffffffffu, ats, j);
              if (in) yp[(int64_t)j * g.ldy] = to_out<T>(__uint_as_float(d[j]) * (s * wts));
            }
          }
        }
      }
      fence_before();
      __syncwarp();
      if (lane == 0) arrive(smem_addr(&c.accempty[q]));
    }
  }
  fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tbase), "n"(TMEM_COLS));
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
  memset(map, 0, sizeof *map);
  const cuuint64_t dims[2] = {row_bytes, rows};
  const cuuint64_t strides[1] = {row_bytes};
  const cuuint32_t boxes[2] = {128, box};
  const cuuint32_t es[2] = {1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, boxes, es,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <bool NV, bool SWIGLU, typename T>
static cudaError_t launch_mm(const fp4mm::Args& a, int grid, size_t smem, cudaStream_t st) {
  // the limit belongs to the kernel on one device: set once for each
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (!(done.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(fp4mm::fp4_mm_kernel<NV, SWIGLU, T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             fp4mm::SMEM_LIMIT);
    if (e != cudaSuccess) return e;
    done.fetch_or(bit, std::memory_order_relaxed);
  }
  return launch_pdl(fp4mm::fp4_mm_kernel<NV, SWIGLU, T>, dim3(grid), dim3(fp4mm::NTHREADS), smem, st, a);
}

template <typename T>
static cudaError_t launch_mm_t(const fp4mm::Args& a, int grid, size_t smem, cudaStream_t st) {
  if (a.g.nv) return a.g.swiglu ? launch_mm<true, true, T>(a, grid, smem, st) : launch_mm<true, false, T>(a, grid, smem, st);
  return a.g.swiglu ? launch_mm<false, true, T>(a, grid, smem, st) : launch_mm<false, false, T>(a, grid, smem, st);
}

cudaError_t launch_fp4_mm(const Fp4MmArgs& g, int dtype, cudaStream_t st) {
  using namespace fp4mm;
  Args a;
  a.g = g;
  a.ksteps = (g.kp + 63) / 64;
  a.atoms = g.nv ? a.ksteps : (a.ksteps + 1) / 2;
  // Token columns of a tile: all of them when they fit one, else 128 or 192 (whole 64-row steps of the
  // scale atoms), whichever leaves fewer columns unused. With groups the counts are on the device: the
  // average decides.
  if (g.offsets != nullptr) {
    const int avg = (g.m + g.mats - 1) / g.mats;
    a.nt = avg > 256 ? 192 : 128;
    a.box = BOX;
  } else if (g.m <= NT_MAX) {
    a.nt = (g.m + 7) & ~7;
    a.box = a.nt;
  } else {
    const int c128 = (g.m + 127) / 128 * 128, c192 = (g.m + 191) / 192 * 192;
    a.nt = c128 < c192 - c192 / 8 ? 128 : 192;
    a.box = a.nt;
  }
  a.b_bytes = a.nt * 128;
  a.sfb_bytes = (a.nt > 64 ? 2 : 1) * SF_BLOCK;
  const int stage = A_BYTES + a.b_bytes + SF_BLOCK + a.sfb_bytes;
  const int room = SMEM_LIMIT - 1024 - (int)sizeof(Ctl);
  a.stages = room / stage < MAX_STAGES ? room / stage : MAX_STAGES;
  const size_t smem = 1024 + (size_t)a.stages * stage + sizeof(Ctl);
  const uint64_t row_bytes = (uint64_t)g.kp / 2;
  cudaError_t e = code_map(&a.map_w, g.w, (uint64_t)g.mats * g.n, row_bytes, 128);
  if (e == cudaSuccess) e = code_map(&a.map_a, g.a, (uint64_t)g.m, row_bytes, (uint32_t)a.box);
  if (e != cudaSuccess) return e;
  const int64_t nb = (g.n + 127) / 128;
  // tiles, or with groups the most there can be
  const int64_t tiles = g.offsets ? ((int64_t)g.m / a.nt + (g.mats < g.m ? g.mats : g.m)) * nb : (g.m + a.nt - 1) / a.nt * nb;
  const int grid = (int)(tiles < num_sms() ? tiles : num_sms());
  if (dtype == SB_F32) return launch_mm_t<float>(a, grid, smem, st);
  if (dtype == SB_F16) return launch_mm_t<__half>(a, grid, smem, st);
  return launch_mm_t<__nv_bfloat16>(a, grid, smem, st);
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
