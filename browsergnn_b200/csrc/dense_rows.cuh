// The products for a few rows of x (dense_rows.cu).
#pragma once

#include "act.cuh"

// Up to eight rows always run there: the warps stream the weights in less time
// than the tensor-core kernel's pipeline takes to fill (1 x 1,024 -> 2 x 4,096:
// 3.6 us against 10.8; 8 x 4,096 -> 4,096: 20 against 27).  So do small products
// of more rows: at 64 x 512 -> 512 it is 5.8 us against 6.8, at 16 x 2,048 ->
// 512 6.3 against 13; twice the outputs (512 x 128 -> 128) take 6.8 against 5.2.
constexpr uint32_t FEW_ROWS = 8;
constexpr uint64_t SMALL_OUT = 1ull << 15, SMALL_MACS = 1ull << 24;
inline bool few_rows(uint64_t m, uint64_t k, uint64_t n, bool two) {
  return m <= FEW_ROWS || (m * n <= SMALL_OUT && m * n * k * (two ? 2 : 1) <= SMALL_MACS);
}

struct RowsArgs {
  const void* x;
  uint64_t ld_x;
  const float* x_scale;
  int two;  // gated: two weights (their addresses are NULL when k is 0)
  const void* w[2];
  uint64_t ld_w[2];
  const float* w_scale[2];
  uint32_t m, k, n;
  const void* bias[2];
  int bias_type;
  int act;
  float act_p;
  const void* other;  // residual, not gated
  int other_type;
  uint64_t ld_other;
  int out_type;
  void* out;
  uint64_t ld_out;
};
// where few_rows says so; m, n >= 1
int bgnn_run_dense_rows(bgnn_ctx* ctx, int type, const RowsArgs& a);
