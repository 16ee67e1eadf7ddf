// Products of microscaled 4-bit operands of prompt-sized batches (entry: mxfp4_gemm.cu).
#pragma once
#include "tma_desc.cuh"

namespace mx4 {

struct PairCall {
  void* y; int64_t ldy;                // [T, N] 16-bit, or the codes of the gated unit (bytes)
  void* y_scales;
  const void* bias;                    // [N] in the output's type, or null
  const void *x, *x_scales, *w, *w_scales;
  int64_t T, N, K, ldx, ldw;           // row strides of codes in bytes
  bool gated;
  bool early;                          // weights may be requested before the previous kernel has ended
};

// whether the pair kernel takes the call and is the faster one (mxfp4_gemm_pair.cu)
bool pair_wanted(const PairCall& g);
int pair_gemm(const PairCall& g, int dtype, cudaStream_t st);

// the same for routed experts (T: tiles of 128 or 256 rows, N: rows of one expert's weights)
int rows_gemm(const PairCall& g, const void* table, int tile_rows, int experts, cudaStream_t st);

}  // namespace mx4
