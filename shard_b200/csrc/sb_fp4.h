// Arguments of the fp4 x fp4 operators' kernels (sb_fp4.cu, sb_fp4mm.cu) and of the stand-alone router
// (sb_topk.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/shard_b200.h"

namespace sb {

struct QuantArgs {
  const void* x;
  int64_t stride;            // elements between rows of x
  int64_t rows, src_rows;    // rows written; rows of x
  int k, units;              // values per row; 16-value units of the padded row
  int nv;                    // NVFP4 (else MXFP4)
  const int32_t* rows_in;    // row of x for each row written, or null
  const int32_t* offsets;    // [groups + 1] row ranges of the expert groups, or null
  int groups;
  int64_t blocks;            // row blocks that the scale buffer holds
  const float* ts;           // NVFP4: the caller's tensor scale, or null: one per row
  float* row_ts;
  uint8_t* codes;
  int64_t row_bytes;
  uint8_t* scales;
  int64_t atoms;
  int flat;                  // scale words row by row, not in atoms
  int wpr, stash;            // warps per row, shared halfwords per row (set by the launch)
};

struct DequantArgs {
  const uint8_t* codes;
  const uint8_t* scales;
  const float* ts;
  int ts_row;                // 1: one tensor scale per row
  int64_t rows;
  int k, units, nv;
  int64_t row_bytes, atoms;
  void* y;
  int vec, wpr;              // set by the launch: y can be written 16 bytes at a time; warps per row
};

struct Fp4MmArgs {
  const uint8_t* w;          // codes [mats * n][row_bytes]
  const uint8_t* w_s;
  const float* w_ts;         // fp32 [mats][w_ts_n], or null
  int w_ts_n;                // 2: one for the even rows (w1), one for the odd rows (w3); 0: [n], one per row
  const uint8_t* a;          // codes [m][row_bytes]
  const uint8_t* a_s;
  const float* a_ts;         // fp32 [m] or [1], or null
  int a_ts_row;
  const float* row_weight;   // fp32 [m] or null
  const int32_t* offsets;    // [mats + 1] or null (one matrix, all rows)
  int nv, mats, n, m;
  int kp;                    // K, padded to 32
  void* y;
  int64_t ldy;
  int swiglu;                // rows 2i / 2i + 1 of W are gate / up
  float limit;               // swiglu: clamp, 0 for none
  uint32_t probes;           // > 0: the consumers' waits give up after so many probes (for tests)
};

struct TopkArgs {
  const void* logits;
  int64_t stride, tokens;    // elements between rows
  const float* bias;         // fp32 [experts] or null
  int experts, topk, score;
  int groups, kept, group_two;   // group_two: a group's score is the sum of its two best, else its best
  int renorm;
  float scale;
  float* weights;
  int64_t* ids;
  int vec;                   // set by the launch: rows can be read 16 bytes at a time
  float lowest;              // set by the launch: the lowest finite value of 16-bit logits
  int size, span, span_log;  // set by the launch: experts and lanes of a group (span 0: groups share lanes)
  int vec_bias;
};

struct OrderArgs {
  const int64_t* ids;        // [pairs]
  int64_t pairs;
  int topk, experts;
  int blocks, scanned;       // set by the launch
  int32_t* hist;             // [order_counts][experts]
  int32_t* offsets;          // [experts + 1]
  int32_t* tokens;           // [pairs]
  int32_t* places;           // [pairs]
};

int64_t order_counts(int64_t pairs);   // rows of counts that go through memory, 0: none
cudaError_t launch_topk(const TopkArgs& a, int dtype, cudaStream_t st);
cudaError_t launch_expert_order(const OrderArgs& a, cudaStream_t st);
// bytes of the copy of a gather's quantised source rows, 0 where none is made
size_t fp4_quant_workspace(int64_t src_rows, int64_t rows, int64_t row_bytes, int64_t atoms);
cudaError_t launch_fp4_quant(const QuantArgs& a, int dtype, void* workspace, cudaStream_t st);
cudaError_t launch_fp4_dequant(const DequantArgs& a, int dtype, cudaStream_t st);
cudaError_t launch_fp4_tile_scales(const uint8_t* src, uint8_t* dst, int64_t mats, int64_t n, int64_t nb, cudaStream_t st);
cudaError_t launch_fp4_mm(const Fp4MmArgs& a, int dtype, cudaStream_t st);
cudaError_t fp4_mm_error(int* host_out, cudaStream_t st);

}  // namespace sb
