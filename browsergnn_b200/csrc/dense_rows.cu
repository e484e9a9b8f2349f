// The products of dense16.cu for a few rows of x (one token or node served, or
// a handful): out = act(x w^T + b) + residual and
// out = act(x wg^T + bg) * (x wu^T + bu).
//
// Bound by the weights' bytes: each weight is read once and used m times, far
// below what would feed the tensor cores.  A warp owns one output column: its
// lanes stream the weight's row (rows) in 16-byte pieces, several in flight,
// multiply with the rows of x (which stay in L1), and add up in f32: one chain
// a lane, then a tree of shuffles.  Rows that do not start on 16 bytes are read
// an element a lane.  Small products of more rows run here too, eight rows a
// block: no tensor maps, no copies of rows that TMA cannot take.
//
// The gradients of few rows stay here as well, because dz (dg, du) then needs no
// rounding to 16 bits: it is kept in f32 between the kernel that computes it and
//   dx = dz w (+ ..)  a column (or eight) a thread over a range of w's rows, the
//                     ranges' sums added in their order,
//   dw = dz^T x       the rows of x in registers, w's rows one by one.
// With so few elements the rounding's share of dx would vary: 1.4 times the
// result's own rounding on average, up to twice for a row.
#include "lowp.cuh"

#include "dense_rows.cuh"

namespace {

constexpr int WARPS = 8;

// the elements of one 16-byte piece, or one element
template <int DT, int VEC>
__device__ __forceinline__ void piece(const void* row, uint32_t c, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    if constexpr (DT == BGNN_E4M3)
      v[0] = __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<const uint8_t*>(row)[c],
                                                         __NV_E4M3)));
    else
      v[0] = Elt<DT>::get(static_cast<const elt_t<DT>*>(row)[c]);
  } else if constexpr (DT == BGNN_E4M3) {
    const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(row) + c);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
          (__nv_fp8x2_storage_t)(w[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
      const float2 f = __half22float2(__half2(h));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  } else {
    load8<DT>(static_cast<const elt_t<DT>*>(row) + c, v);
  }
}

template <int DT, int M, bool TWO, int VEC, bool BWD>
__global__ void __launch_bounds__(WARPS * 32) k_dense_rows(const RowsArgs a) {
  const int lane = threadIdx.x & 31;
  const uint32_t col = blockIdx.x * WARPS + (threadIdx.x >> 5);
  if (col >= a.n) return;
  constexpr uint32_t ES = DT == BGNN_E4M3 ? 1 : 2;
  const char* w[2];
  w[0] = static_cast<const char*>(a.w[0]) + (uint64_t)col * a.ld_w[0] * ES;
  w[1] = TWO ? static_cast<const char*>(a.w[1]) + (uint64_t)col * a.ld_w[1] * ES : nullptr;
  const char* x[M];
  const uint32_t row0 = blockIdx.y * M, rows = a.m - row0 < M ? a.m - row0 : M;
#pragma unroll
  for (int i = 0; i < M; i++)  // a row that is not there repeats the last
    x[i] = static_cast<const char*>(a.x) +
           (uint64_t)(row0 + ((uint32_t)i < rows ? i : rows - 1)) * a.ld_x * ES;
  float s[TWO ? 2 : 1][M];
#pragma unroll
  for (int t = 0; t < (TWO ? 2 : 1); t++)
#pragma unroll
    for (int i = 0; i < M; i++) s[t][i] = 0.0f;
  auto add = [&](const float (&u)[VEC], const float (&g)[VEC], uint32_t c) {
#pragma unroll
    for (int i = 0; i < M; i++) {
      float v[VEC];
      piece<DT, VEC>(x[i], c, v);
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        s[0][i] = fmaf(u[j], v[j], s[0][i]);
        if (TWO) s[TWO][i] = fmaf(g[j], v[j], s[TWO][i]);
      }
    }
  };
  constexpr uint32_t STEP = 32 * VEC;
  constexpr int DEEP = VEC == 1 ? 8 : 4;  // pieces in flight
  uint32_t c = lane * VEC;
  for (; c + (DEEP - 1) * STEP + VEC <= a.k; c += DEEP * STEP) {
    float u[DEEP][VEC], g[DEEP][VEC];
#pragma unroll
    for (int d = 0; d < DEEP; d++) {
      piece<DT, VEC>(w[0], c + d * STEP, u[d]);
      if (TWO) piece<DT, VEC>(w[1], c + d * STEP, g[d]);
    }
#pragma unroll
    for (int d = 0; d < DEEP; d++) add(u[d], g[d], c + d * STEP);
  }
  for (; c + VEC <= a.k; c += STEP) {
    float u[VEC], g[VEC];
    piece<DT, VEC>(w[0], c, u);
    if (TWO) piece<DT, VEC>(w[1], c, g);
    add(u, g, c);
  }
  if (VEC > 1) {  // the last columns, fewer than a piece: an element a lane
    const uint32_t e = a.k / VEC * VEC + lane;
    if (e < a.k) {
      float u[1], g[1] = {0.0f}, v[1];
      piece<DT, 1>(w[0], e, u);
      if (TWO) piece<DT, 1>(w[1], e, g);
#pragma unroll
      for (int i = 0; i < M; i++) {
        piece<DT, 1>(x[i], e, v);
        s[0][i] = fmaf(u[0], v[0], s[0][i]);
        if (TWO) s[TWO][i] = fmaf(g[0], v[0], s[TWO][i]);
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int t = 0; t < (TWO ? 2 : 1); t++)
#pragma unroll
      for (int i = 0; i < M; i++) s[t][i] += __shfl_xor_sync(0xffffffffu, s[t][i], o);
  // lane i finishes row i
  float z0 = 0.0f, z1 = 0.0f;
#pragma unroll
  for (int i = 0; i < M; i++)
    if (lane == i) {
      z0 = s[0][i];
      if (TWO) z1 = s[TWO][i];
    }
  if ((uint32_t)lane >= rows) return;
  const uint64_t row = row0 + lane;
  if (DT == BGNN_E4M3) {
    z0 *= a.x_scale[row] * a.w_scale[0][col];
    if (TWO) z1 *= a.x_scale[row] * a.w_scale[1][col];
  }
  if (a.bias[0]) z0 += load_any(a.bias[0], a.bias_type, col);
  if (TWO && a.bias[1]) z1 += load_any(a.bias[1], a.bias_type, col);
  if constexpr (BWD) {
    float2 f = make_float2(0.0f, 0.0f);  // act(z0), act'(z0)
    with_act(a.act, [&](auto act) {
      float2 unused;
      act_grad_two<decltype(act)::value>(make_float2(z0, 0.0f), a.act_p, f, unused);
    });
    const float g = load_any(a.grad, DT, row * a.ld_grad + col);
    a.dz[0][row * a.n + col] = (TWO ? z1 * f.y : f.y) * g;
    if (TWO) a.dz[1][row * a.n + col] = f.x * g;
    return;
  }
  float o = z0;
  with_act(a.act, [&](auto act) {
    o = act_two<decltype(act)::value>(make_float2(z0, 0.0f), a.act_p).x;
  });
  if (TWO) o *= z1;
  else if (a.other) o += load_any(a.other, a.other_type, row * a.ld_other + col);
  store_any(a.out, a.out_type, row * a.ld_out + col, o);
}

template <int DT, int M, bool TWO, int VEC>
int launch_rows(bgnn_ctx* ctx, const RowsArgs& a) {
  const dim3 grid((a.n + WARPS - 1) / WARPS, (a.m + M - 1) / M);
  if constexpr (DT != BGNN_E4M3) {
    if (a.grad) {
      k_dense_rows<DT, M, TWO, VEC, true><<<grid, WARPS * 32, 0, ctx->stream>>>(a);
      BGNN_LAUNCHED(ctx);
      return BGNN_OK;
    }
  }
  k_dense_rows<DT, M, TWO, VEC, false><<<grid, WARPS * 32, 0, ctx->stream>>>(a);
  BGNN_LAUNCHED(ctx);
  return BGNN_OK;
}
// Single elements go four rows at a time at most: with eight, 8 x 3,501 -> 3,901
// takes 109 us against 35, and 100 x 301 -> 271 takes 11.3 against 5.6.
template <int DT, bool TWO, int VEC>
int launch_m(bgnn_ctx* ctx, const RowsArgs& a) {
  if (a.m == 1) return launch_rows<DT, 1, TWO, VEC>(ctx, a);
  if (a.m == 2) return launch_rows<DT, 2, TWO, VEC>(ctx, a);
  if (a.m <= 4 || VEC == 1) return launch_rows<DT, 4, TWO, VEC>(ctx, a);
  return launch_rows<DT, VEC == 1 ? 4 : 8, TWO, VEC>(ctx, a);
}
template <int DT, bool TWO>
int launch_vec(bgnn_ctx* ctx, const RowsArgs& a, bool vec) {
  constexpr int VEC = DT == BGNN_E4M3 ? 16 : 8;
  return vec ? launch_m<DT, TWO, VEC>(ctx, a) : launch_m<DT, TWO, 1>(ctx, a);
}
template <int DT>
int launch_two(bgnn_ctx* ctx, const RowsArgs& a, bool vec) {
  return a.two ? launch_vec<DT, true>(ctx, a, vec) : launch_vec<DT, false>(ctx, a, vec);
}

// ---- gradients ---------------------------------------------------------------------
// part[range][i][c] = sum over the range's rows r of w, of both weights, of
// dz[i][r] w[r][c]: the block's warps take the rows in turn
template <int DT, int M, int VEC>
__global__ void __launch_bounds__(WARPS * 32) k_rows_dx(const RowsArgs a, uint32_t per,
                                                        float* __restrict__ part) {
  __shared__ float sm[WARPS][32 * VEC];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t c = (blockIdx.x * 32 + lane) * VEC, first = blockIdx.y * per;
  const uint32_t end = a.n - first < per ? a.n : first + per;
  float s[M][VEC];
#pragma unroll
  for (int i = 0; i < M; i++)
#pragma unroll
    for (int j = 0; j < VEC; j++) s[i][j] = 0.0f;
  if (c < a.k)  // VEC > 1: k is whole vectors
    for (int t = 0; t < (a.two ? 2 : 1); t++) {
      const elt_t<DT>* w = static_cast<const elt_t<DT>*>(a.w[t]);
#pragma unroll 4
      for (uint32_t r = first + warp; r < end; r += WARPS) {
        float v[VEC];
        piece<DT, VEC>(w + r * a.ld_w[t], c, v);
#pragma unroll
        for (int i = 0; i < M; i++) {
          const float d = a.dz[t][(uint64_t)((uint32_t)i < a.m ? i : a.m - 1) * a.n + r];
#pragma unroll
          for (int j = 0; j < VEC; j++) s[i][j] = fmaf(d, v[j], s[i][j]);
        }
      }
    }
#pragma unroll
  for (int i = 0; i < M; i++) {
    if ((uint32_t)i >= a.m) break;
#pragma unroll
    for (int j = 0; j < VEC; j++) sm[warp][lane * VEC + j] = s[i][j];
    __syncthreads();
    const uint32_t col = blockIdx.x * 32 * VEC + threadIdx.x;
    if (threadIdx.x < 32 * VEC && col < a.k) {
      float v = sm[0][threadIdx.x];
      for (int q = 1; q < WARPS; q++) v += sm[q][threadIdx.x];
      part[((uint64_t)blockIdx.y * a.m + i) * a.k + col] = v;
    }
    __syncthreads();
  }
}

// dw[t][r][c] = sum over i of dz[t][i][r] x[i][c]
template <int DT, int M, int VEC>
__global__ void __launch_bounds__(WARPS * 32) k_rows_dw(const RowsArgs a, elt_t<DT>* dw0,
                                                        elt_t<DT>* dw1) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t c = (blockIdx.x * 32 + lane) * VEC;
  if (c >= a.k) return;
  float x[M][VEC];
#pragma unroll
  for (int i = 0; i < M; i++) {
    if ((uint32_t)i < a.m) {
      piece<DT, VEC>(static_cast<const elt_t<DT>*>(a.x) + i * a.ld_x, c, x[i]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; j++) x[i][j] = 0.0f;
    }
  }
  for (int t = 0; t < (a.two ? 2 : 1); t++) {
    elt_t<DT>* out = t ? dw1 : dw0;
    for (uint32_t r = blockIdx.y * WARPS + warp; r < a.n; r += gridDim.y * WARPS) {
      float v[VEC];
#pragma unroll
      for (int j = 0; j < VEC; j++) v[j] = 0.0f;
#pragma unroll
      for (int i = 0; i < M; i++) {
        if ((uint32_t)i >= a.m) break;
        const float d = a.dz[t][(uint64_t)i * a.n + r];
#pragma unroll
        for (int j = 0; j < VEC; j++) v[j] = fmaf(d, x[i][j], v[j]);
      }
      elt_t<DT>* p = out + (uint64_t)r * a.k + c;
      if constexpr (VEC == 8) store8<DT>(p, v);
      else p[0] = Elt<DT>::put(v[0]);
    }
  }
}

// f(the smallest compiled number of rows that holds m)
template <class F>
int with_rows(uint32_t m, F&& f) {
  if (m == 1) return f(std::integral_constant<int, 1>{});
  if (m == 2) return f(std::integral_constant<int, 2>{});
  if (m <= 4) return f(std::integral_constant<int, 4>{});
  return f(std::integral_constant<int, 8>{});
}

template <int DT, int VEC>
int run_dx(bgnn_ctx* ctx, const RowsArgs& a, void* dx, int type) {
  // ranges of at least 64 rows, two blocks an SM
  const uint32_t cb = (a.k + 32 * VEC - 1) / (32 * VEC);
  uint32_t ranges = (uint32_t)ctx->num_sms * 2 / cb, most = (a.n + 63) / 64;
  if (ranges > most) ranges = most;
  if (ranges < 1) ranges = 1;
  const uint32_t per = (a.n + ranges - 1) / ranges;
  ranges = (a.n + per - 1) / per;
  DevTmp part;
  const uint64_t size = (uint64_t)a.m * a.k;
  BGNN_TRY(bgnn_tmp_alloc(ctx, part, ranges * size * sizeof(float)));
  BGNN_TRY(with_rows(a.m, [&](auto rows) -> int {
    k_rows_dx<DT, decltype(rows)::value, VEC>
        <<<dim3(cb, ranges), WARPS * 32, 0, ctx->stream>>>(a, per, part.as<float>());
    BGNN_LAUNCHED(ctx);
    return BGNN_OK;
  }));
  return bgnn_run_sum_parts(ctx, part.as<float>(), ranges, size, dx, type);
}

template <int DT, int VEC>
int run_dw(bgnn_ctx* ctx, const RowsArgs& a, void* dw0, void* dw1) {
  const uint32_t cb = (a.k + 32 * VEC - 1) / (32 * VEC);
  uint32_t rows = (uint32_t)ctx->num_sms * 4 / cb, most = (a.n + WARPS - 1) / WARPS;
  if (rows > most) rows = most;
  if (rows < 1) rows = 1;
  return with_rows(a.m, [&](auto m) -> int {
    k_rows_dw<DT, decltype(m)::value, VEC><<<dim3(cb, rows), WARPS * 32, 0, ctx->stream>>>(
        a, static_cast<elt_t<DT>*>(dw0), static_cast<elt_t<DT>*>(dw1));
    BGNN_LAUNCHED(ctx);
    return BGNN_OK;
  });
}

// every row starts on 16 bytes
bool whole_rows(const void* p, uint64_t ld, uint32_t es) {
  return ((uintptr_t)p & 15u) == 0 && ld * es % 16 == 0;
}

template <int DT>
int run_backward(bgnn_ctx* ctx, int type, const RowsArgs& a, const RowsGrads& out) {
  if (out.x && a.k) {
    const bool vec = a.k % 8 == 0 && whole_rows(a.w[0], a.ld_w[0], 2) &&
                     (!a.two || whole_rows(a.w[1], a.ld_w[1], 2));
    BGNN_TRY((vec ? run_dx<DT, 8>(ctx, a, out.x, type) : run_dx<DT, 1>(ctx, a, out.x, type)));
  }
  if (out.w[0] && a.k) {
    const bool vec = a.k % 8 == 0 && whole_rows(a.x, a.ld_x, 2) && whole_rows(out.w[0], a.k, 2) &&
                     (!a.two || whole_rows(out.w[1], a.k, 2));
    BGNN_TRY((vec ? run_dw<DT, 8>(ctx, a, out.w[0], out.w[1])
                  : run_dw<DT, 1>(ctx, a, out.w[0], out.w[1])));
  }
  for (int t = 0; t < (a.two ? 2 : 1); t++)
    if (out.bias[t])
      BGNN_TRY(bgnn_run_sum_parts(ctx, a.dz[t], a.m, a.n, out.bias[t], a.bias_type));
  return BGNN_OK;
}

}  // namespace

int bgnn_run_dense_rows_backward(bgnn_ctx* ctx, int type, RowsArgs a, const RowsGrads& out) {
  DevTmp dz;
  const uint64_t size = (uint64_t)a.m * a.n;
  BGNN_TRY(bgnn_tmp_alloc(ctx, dz, (a.two ? 2 : 1) * size * sizeof(float)));
  a.dz[0] = dz.as<float>();
  a.dz[1] = a.two ? a.dz[0] + size : nullptr;
  BGNN_TRY(bgnn_run_dense_rows(ctx, type, a));
  return type == BGNN_BF16 ? run_backward<BGNN_BF16>(ctx, type, a, out)
                           : run_backward<BGNN_F16>(ctx, type, a, out);
}

int bgnn_run_dense_rows(bgnn_ctx* ctx, int type, const RowsArgs& a) {
  const uint32_t es = (uint32_t)dtype_size(type);
  auto whole = [&](const void* p, uint64_t ld) {
    return ((uintptr_t)p & 15u) == 0 && ld * es % 16 == 0;
  };
  const bool vec = whole(a.x, a.ld_x) && whole(a.w[0], a.ld_w[0]) &&
                   (!a.two || whole(a.w[1], a.ld_w[1]));
  switch (type) {
    case BGNN_BF16: return launch_two<BGNN_BF16>(ctx, a, vec);
    case BGNN_F16: return launch_two<BGNN_F16>(ctx, a, vec);
    default: return launch_two<BGNN_E4M3>(ctx, a, vec);
  }
}
