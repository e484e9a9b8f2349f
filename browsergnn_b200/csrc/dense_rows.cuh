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

// The gradients of so few rows that dz can stay in f32 (bf16, with an activation
// and a bias, against the tensor cores, which take dz rounded): 1 x 1,024 -> 512
// 18 us against 40, 4 x 4,096 -> 4,096 57 against 79, 8 x 256 -> 32,000 79
// against 208; but 8 x 4,096 -> 4,096 107 against 79, 8 x 16,384 -> 256 118
// against 108.
constexpr uint32_t FEW_BACKWARD = 4, NARROW = 512;
inline bool few_rows_backward(uint64_t m, uint64_t k) {
  return m <= FEW_BACKWARD || (m <= FEW_ROWS && k <= NARROW);
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
  const void* grad;  // backward: the upstream gradient [m, n]
  uint64_t ld_grad;
  float* dz[2];      // backward: dz, or dg and du, [m, n] each
};
// where few_rows says so; m, n >= 1
int bgnn_run_dense_rows(bgnn_ctx* ctx, int type, const RowsArgs& a);

// where few_rows_backward says so: the gradients (m, n >= 1) of a product with an
// activation, or of a gated one; a.out, a.other and the scales are not used.
// Any of the results may be NULL.
struct RowsGrads {
  void* x;       // [m, k]
  void* w[2];    // [n, k]
  void* bias[2]; // [n], a.bias_type
};
int bgnn_run_dense_rows_backward(bgnn_ctx* ctx, int type, RowsArgs a, const RowsGrads& out);
