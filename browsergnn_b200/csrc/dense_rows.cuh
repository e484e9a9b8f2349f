// The products for a few rows of x (dense_rows.cu).
#pragma once

#include "act.cuh"

// Rows up to which they run there: the warps stream the weights in less than
// the tensor-core kernel's pipeline takes to fill.
constexpr uint32_t FEW_ROWS = 8;

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
// 1 <= m <= FEW_ROWS, n >= 1
int bgnn_run_dense_rows(bgnn_ctx* ctx, int type, const RowsArgs& a);
