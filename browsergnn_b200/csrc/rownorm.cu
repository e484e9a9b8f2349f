// Root-mean-square norm of rows with the residual's addition, and its
// backward.
//
//   t = x + r, rounded to the residual's type (t is what the next layer adds to);
//   s = (mean_j t_j^2 + eps)^(-1/2);   y_j = w_j (t_j s);
//   out = y in f32 / bf16 / f16, or q = e4m3(y * 448 / amax) with the row's
//   scale = amax / 448, amax = max_j |y_j|.
//
// Backward, xh_j = t_j s, for an upstream gradient gy and the gradient gt
// that reaches t along the residual stream:
//   gt_j + s (gy_j w_j - xh_j mean_i(gy_i w_i xh_i))  is the gradient of x and of r,
//   gw_j = sum over the rows of gy_j xh_j.
// s is computed from the rounded t that the forward wrote, so forward and
// backward see the same row and nothing but t has to be kept.
//
// Memory bound: each row is read once into registers (all statistics are f32
// there) and written once.  A row belongs to `tpr` threads, each holding NV
// vectors of VEC elements; up to 32 threads the sums are shuffles, above that
// one row fills a block.  Rows longer than the registers hold (RowShape) take
// the k_*_long kernels, which read the row again from L2.
#include "lowp.cuh"

namespace {

struct RmsArgs {
  const void* x;
  uint64_t ld_x;
  const void* res;  // may be NULL
  uint64_t ld_res;
  const void* w;
  int w_type;
  uint64_t rows;
  uint32_t cols;
  float eps;
  void* total;
  void* out;
  float* scale;
};

// Sum (or maximum) over the tpr threads of a row; every thread gets it.
// tpr <= 32: the row's threads are consecutive lanes.  tpr > 32: the block.
// `red` has a slot a warp; `flip` alternates its two halves, so that one
// barrier a call is enough.
template <bool MAX>
__device__ __forceinline__ float row_reduce(float v, int tpr, float* red, int& flip) {
  const int lim = tpr < 32 ? tpr : 32;
  for (int o = 1; o < lim; o <<= 1) {
    const float u = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? fmaxf(v, u) : v + u;
  }
  if (tpr > 32) {
    float* slot = red + flip * 32;
    flip ^= 1;
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
    __syncthreads();
    const int warps = tpr >> 5;
    v = slot[0];
    for (int i = 1; i < warps; i++) v = MAX ? fmaxf(v, slot[i]) : v + slot[i];
  }
  return v;
}


constexpr float E4M3_MAX = 448.0f;

// (scale, 1/scale) of a row whose largest magnitude is amax.  An all-zero
// row has scale 1; a scale below the smallest normal is held there.
__device__ __forceinline__ float2 e4m3_scale(float amax) {
  if (amax == 0.0f) return make_float2(1.0f, 1.0f);
  const float s = fmaxf(__fdiv_rn(amax, E4M3_MAX), 1.17549435e-38f);
  const float sc = amax != amax ? amax : s;
  return make_float2(sc, __fdiv_rn(1.0f, sc));
}

template <int VEC, int DT>
__device__ __forceinline__ void load_v(const elt_t<DT>* p, float (&v)[VEC]) {
  if constexpr (VEC == 8) load8<DT>(p, v);
  else v[0] = Elt<DT>::get(*p);
}
template <int VEC, int DT>
__device__ __forceinline__ void store_v(elt_t<DT>* p, const float (&v)[VEC]) {
  if constexpr (VEC == 8) store8<DT>(p, v);
  else *p = Elt<DT>::put(v[0]);
}

// threads a block may have: the row's registers decide
template <int VEC, int NV>
constexpr int row_threads = VEC * NV > 8 ? 512 : 1024;

template <int TX, int TR, int TO, int VEC, int NV>
__global__ void __launch_bounds__(row_threads<VEC, NV>) k_rms(const RmsArgs a, int tpr) {
  __shared__ float red[64];
  int flip = 0;
  const int sub = threadIdx.x / tpr, lane = threadIdx.x % tpr, rpb = blockDim.x / tpr;
  const uint32_t nvec = a.cols / VEC;
  float w[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const uint32_t c = (uint32_t)(i * tpr + lane);
#pragma unroll
    for (int j = 0; j < VEC; j++)
      w[i][j] = c < nvec ? load_any(a.w, a.w_type, (uint64_t)c * VEC + j) : 0.0f;
  }
  const float inv_n = __fdiv_rn(1.0f, (float)a.cols);
  for (uint64_t base = (uint64_t)blockIdx.x * rpb; base < a.rows;
       base += (uint64_t)gridDim.x * rpb) {
    const uint64_t row = base + sub;
    const bool on = row < a.rows;
    const elt_t<TX>* xr = static_cast<const elt_t<TX>*>(a.x) + row * a.ld_x;
    float t[NV][VEC];
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const uint32_t c = (uint32_t)(i * tpr + lane);
      if (on && c < nvec) {
        load_v<VEC, TX>(xr + (uint64_t)c * VEC, t[i]);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; j++) t[i][j] = 0.0f;
      }
    }
    if (a.res) {
      const elt_t<TR>* rr = static_cast<const elt_t<TR>*>(a.res) + row * a.ld_res;
      elt_t<TR>* tr = static_cast<elt_t<TR>*>(a.total) + row * a.cols;
#pragma unroll
      for (int i = 0; i < NV; i++) {
        const uint32_t c = (uint32_t)(i * tpr + lane);
        if (on && c < nvec) {
          float r[VEC];
          load_v<VEC, TR>(rr + (uint64_t)c * VEC, r);
#pragma unroll
          for (int j = 0; j < VEC; j++) t[i][j] = rounded<TR>(t[i][j] + r[j]);
          store_v<VEC, TR>(tr + (uint64_t)c * VEC, t[i]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int j = 0; j < VEC; j++) ss = fmaf(t[i][j], t[i][j], ss);
    ss = row_reduce<false>(ss, tpr, red, flip);
    const float s = __frsqrt_rn(fmaf(ss, inv_n, a.eps));
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int j = 0; j < VEC; j++) t[i][j] = w[i][j] * (t[i][j] * s);
    if constexpr (TO == BGNN_E4M3) {
      float m = 0.0f;
      float nan = 0.0f;  // +0, or NaN once an element is
#pragma unroll
      for (int i = 0; i < NV; i++)
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          m = fmaxf(m, fabsf(t[i][j]));
          nan = t[i][j] != t[i][j] ? t[i][j] : nan;
        }
      m = row_reduce<true>(m, tpr, red, flip);
      nan = row_reduce<false>(nan, tpr, red, flip);
      const float2 sc = e4m3_scale(m + nan);
#pragma unroll
      for (int i = 0; i < NV; i++)
#pragma unroll
        for (int j = 0; j < VEC; j++) t[i][j] *= sc.y;
      if (on && lane == 0) a.scale[row] = sc.x;
    }
    elt_t<TO>* orow = static_cast<elt_t<TO>*>(a.out) + row * a.cols;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const uint32_t c = (uint32_t)(i * tpr + lane);
      if (on && c < nvec) store_v<VEC, TO>(orow + (uint64_t)c * VEC, t[i]);
    }
  }
}

// a row longer than the registers of a block: read again from L2
template <int TX, int TR, int TO>
__global__ void __launch_bounds__(1024) k_rms_long(const RmsArgs a) {
  __shared__ float red[64];
  int flip = 0;
  const int nt = blockDim.x;
  for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const elt_t<TX>* xr = static_cast<const elt_t<TX>*>(a.x) + row * a.ld_x;
    const elt_t<TR>* rr = static_cast<const elt_t<TR>*>(a.res) + row * a.ld_res;
    elt_t<TR>* tr = static_cast<elt_t<TR>*>(a.total) + row * a.cols;
    elt_t<TO>* orow = static_cast<elt_t<TO>*>(a.out) + row * a.cols;
    auto at = [&](uint32_t c) {  // after the first pass: a thread reads back its own stores
      return a.res ? Elt<TR>::get(tr[c]) : Elt<TX>::get(xr[c]);
    };
    float ss = 0.0f;
    for (uint32_t c = threadIdx.x; c < a.cols; c += nt) {
      float t = Elt<TX>::get(xr[c]);
      if (a.res) {
        const elt_t<TR> q = Elt<TR>::put(t + Elt<TR>::get(rr[c]));
        tr[c] = q;
        t = Elt<TR>::get(q);
      }
      ss = fmaf(t, t, ss);
    }
    ss = row_reduce<false>(ss, nt, red, flip);
    const float s = __frsqrt_rn(fmaf(ss, __fdiv_rn(1.0f, (float)a.cols), a.eps));
    float2 sc = make_float2(1.0f, 1.0f);
    if constexpr (TO == BGNN_E4M3) {
      float m = 0.0f, nan = 0.0f;
      for (uint32_t c = threadIdx.x; c < a.cols; c += nt) {
        const float y = load_any(a.w, a.w_type, c) * (at(c) * s);
        m = fmaxf(m, fabsf(y));
        nan = y != y ? y : nan;
      }
      m = row_reduce<true>(m, nt, red, flip);
      nan = row_reduce<false>(nan, nt, red, flip);
      sc = e4m3_scale(m + nan);
      if (threadIdx.x == 0) a.scale[row] = sc.x;
    }
    for (uint32_t c = threadIdx.x; c < a.cols; c += nt) {
      float y = load_any(a.w, a.w_type, c) * (at(c) * s);
      if constexpr (TO == BGNN_E4M3) y *= sc.y;
      orow[c] = Elt<TO>::put(y);
    }
  }
}

struct RmsBwdArgs {
  const void* gy;
  uint64_t ld_gy;
  const void* t;
  uint64_t ld_t;
  const void* gt;  // may be NULL
  uint64_t ld_gt;
  const void* w;
  int w_type;
  uint64_t rows;
  uint32_t cols;
  float eps;
  void* gx;
  float* part;  // [grid, cols] sums of gy * xh over each block's rows
};

template <int TG, int TT, int VEC, int NV>
__global__ void __launch_bounds__(512) k_rms_bwd(const RmsBwdArgs a, int tpr) {
  extern __shared__ float fold[];  // [cols] when a block holds several rows
  __shared__ float red[64];
  int flip = 0;
  const int sub = threadIdx.x / tpr, lane = threadIdx.x % tpr, rpb = blockDim.x / tpr;
  const uint32_t nvec = a.cols / VEC;
  float w[NV][VEC], gw[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const uint32_t c = (uint32_t)(i * tpr + lane);
#pragma unroll
    for (int j = 0; j < VEC; j++) {
      w[i][j] = c < nvec ? load_any(a.w, a.w_type, (uint64_t)c * VEC + j) : 0.0f;
      gw[i][j] = 0.0f;
    }
  }
  const float inv_n = __fdiv_rn(1.0f, (float)a.cols);
  for (uint64_t base = (uint64_t)blockIdx.x * rpb; base < a.rows;
       base += (uint64_t)gridDim.x * rpb) {
    const uint64_t row = base + sub;
    const bool on = row < a.rows;
    const elt_t<TT>* tr = static_cast<const elt_t<TT>*>(a.t) + row * a.ld_t;
    const elt_t<TG>* gr = static_cast<const elt_t<TG>*>(a.gy) + row * a.ld_gy;
    float t[NV][VEC], g[NV][VEC];
    float ss = 0.0f, dot = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const uint32_t c = (uint32_t)(i * tpr + lane);
      if (on && c < nvec) {
        load_v<VEC, TT>(tr + (uint64_t)c * VEC, t[i]);
        load_v<VEC, TG>(gr + (uint64_t)c * VEC, g[i]);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; j++) t[i][j] = g[i][j] = 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        ss = fmaf(t[i][j], t[i][j], ss);
        dot = fmaf(g[i][j] * w[i][j], t[i][j], dot);
      }
    ss = row_reduce<false>(ss, tpr, red, flip);
    dot = row_reduce<false>(dot, tpr, red, flip);
    const float s = __frsqrt_rn(fmaf(ss, inv_n, a.eps));
    const float c1 = dot * s * inv_n;  // mean(gy w xh)
    const elt_t<TT>* sr = static_cast<const elt_t<TT>*>(a.gt) + row * a.ld_gt;
    elt_t<TT>* xr = static_cast<elt_t<TT>*>(a.gx) + row * a.cols;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const uint32_t c = (uint32_t)(i * tpr + lane);
      if (on && c < nvec) {
        float o[VEC];
        if (a.gt) {
          load_v<VEC, TT>(sr + (uint64_t)c * VEC, o);
        } else {
#pragma unroll
          for (int j = 0; j < VEC; j++) o[j] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          const float xh = t[i][j] * s;
          o[j] = fmaf(s, fmaf(-xh, c1, g[i][j] * w[i][j]), o[j]);
          gw[i][j] = fmaf(g[i][j], xh, gw[i][j]);
        }
        store_v<VEC, TT>(xr + (uint64_t)c * VEC, o);
      }
    }
  }
  // the block's sums, in a fixed order: row group 0 first
  if (!a.part) return;
  float* prow = a.part + (uint64_t)blockIdx.x * a.cols;
  for (int r = 0; r < rpb; r++) {
    if (sub == r) {
#pragma unroll
      for (int i = 0; i < NV; i++) {
        const uint32_t c = (uint32_t)(i * tpr + lane);
        if (c < nvec) {
#pragma unroll
          for (int j = 0; j < VEC; j++) {
            const uint32_t e = c * VEC + j;
            const float v = r ? fold[e] + gw[i][j] : gw[i][j];
            if (r + 1 < rpb) fold[e] = v;
            else prow[e] = v;
          }
        }
      }
    }
    if (r + 1 < rpb) __syncthreads();
  }
}

// long rows: per row (s, mean(gy w xh))
template <int TG, int TT>
__global__ void __launch_bounds__(1024) k_rms_bwd_stats(const RmsBwdArgs a, float2* stats) {
  __shared__ float red[64];
  int flip = 0;
  for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const elt_t<TT>* tr = static_cast<const elt_t<TT>*>(a.t) + row * a.ld_t;
    const elt_t<TG>* gr = static_cast<const elt_t<TG>*>(a.gy) + row * a.ld_gy;
    float ss = 0.0f, dot = 0.0f;
    for (uint32_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
      const float t = Elt<TT>::get(tr[c]);
      ss = fmaf(t, t, ss);
      dot = fmaf(Elt<TG>::get(gr[c]) * load_any(a.w, a.w_type, c), t, dot);
    }
    ss = row_reduce<false>(ss, blockDim.x, red, flip);
    dot = row_reduce<false>(dot, blockDim.x, red, flip);
    const float inv_n = __fdiv_rn(1.0f, (float)a.cols);
    const float s = __frsqrt_rn(fmaf(ss, inv_n, a.eps));
    if (threadIdx.x == 0) stats[row] = make_float2(s, dot * s * inv_n);
  }
}
// long rows: a column a thread over a slab of rows (blockIdx.y)
template <int TG, int TT>
__global__ void __launch_bounds__(256) k_rms_bwd_apply(const RmsBwdArgs a, const float2* stats) {
  const uint32_t c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= a.cols) return;
  const float w = load_any(a.w, a.w_type, c);
  float gw = 0.0f;
  for (uint64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float2 st = stats[row];
    const float xh = Elt<TT>::get(static_cast<const elt_t<TT>*>(a.t)[row * a.ld_t + c]) * st.x;
    const float g = Elt<TG>::get(static_cast<const elt_t<TG>*>(a.gy)[row * a.ld_gy + c]);
    const float o = a.gt ? Elt<TT>::get(static_cast<const elt_t<TT>*>(a.gt)[row * a.ld_gt + c])
                         : 0.0f;
    static_cast<elt_t<TT>*>(a.gx)[row * a.cols + c] =
        Elt<TT>::put(fmaf(st.x, fmaf(-xh, st.y, g * w), o));
    gw = fmaf(g, xh, gw);
  }
  if (a.part) a.part[(uint64_t)blockIdx.y * a.cols + c] = gw;
}

// out[c] = sum over the parts, part 0 first within each of 8 interleaved
// chains: 32 columns a block, 8 chains a column
__global__ void __launch_bounds__(256) k_sum_parts(const float* __restrict__ part, uint32_t parts,
                                                   uint64_t cols, void* out, int out_type) {
  __shared__ float s[8][33];
  const int lane = threadIdx.x & 31, ch = threadIdx.x >> 5;
  const uint64_t c = (uint64_t)blockIdx.x * 32 + lane;
  float v = 0.0f;
  if (c < cols)
    for (uint32_t p = ch; p < parts; p += 8) v += part[(uint64_t)p * cols + c];
  s[ch][lane] = v;
  __syncthreads();
  if (ch == 0 && c < cols) {
#pragma unroll
    for (int i = 1; i < 8; i++) v += s[i][lane];
    store_any(out, out_type, c, v);
  }
}

// How a row of `cols` elements is held: vectors of 8 when every row of every
// array starts on a vector, else single elements; threads a row so that each
// holds at most NV vectors.
struct RowShape {
  int vec, nv, tpr, block;
  bool fits;
};
RowShape row_shape(uint32_t cols, bool vec_ok, int nv_wide, bool backward) {
  RowShape r;
  r.vec = vec_ok ? 8 : 1;
  const uint32_t nvec = cols / r.vec;
  // a warp a row while one vector a thread is enough; beyond, several
  // vectors a thread before several warps a row (no block barrier)
  r.nv = r.vec == 1 ? 8 : (nvec <= 32 ? 1 : nv_wide);
  uint32_t t = (nvec + r.nv - 1) / r.nv;
  if (t <= 32) {
    r.tpr = 1;
    while ((uint32_t)r.tpr < t) r.tpr *= 2;
  } else {
    r.tpr = (int)((t + 31) / 32) * 32;
  }
  r.fits = t <= (backward || r.vec * r.nv > 8 ? 512u : 1024u);
  r.block = !r.fits ? 1024 : r.tpr <= 32 ? 256 : r.tpr;
  if (!r.fits) r.tpr = 1024;
  return r;
}

bool vec_rows(const void* p, uint64_t ld) { return ((uintptr_t)p & 15u) == 0 && ld % 8 == 0; }

// resident blocks fill the GPU once; each loops over its share of the rows
unsigned row_grid(const bgnn_ctx* ctx, uint64_t rows, const RowShape& r) {
  const uint64_t rpb = (uint64_t)(r.block / r.tpr);
  const uint64_t want = (rows + rpb - 1) / rpb;
  const uint64_t cap = (uint64_t)ctx->num_sms * (2048 / r.block);
  return (unsigned)(want < cap ? want : cap);
}

template <int TX, int TR, int TO>
int launch_rms(bgnn_ctx* ctx, const RmsArgs& a, const RowShape& r) {
  const unsigned grid = row_grid(ctx, a.rows, r);
  if (!r.fits) {
    k_rms_long<TX, TR, TO><<<grid, 1024, 0, ctx->stream>>>(a);
  } else if (r.vec == 1) {
    k_rms<TX, TR, TO, 1, 8><<<grid, r.block, 0, ctx->stream>>>(a, r.tpr);
  } else if (r.nv == 1) {
    k_rms<TX, TR, TO, 8, 1><<<grid, r.block, 0, ctx->stream>>>(a, r.tpr);
  } else {
    k_rms<TX, TR, TO, 8, 4><<<grid, r.block, 0, ctx->stream>>>(a, r.tpr);
  }
  BGNN_LAUNCHED(ctx);
  return BGNN_OK;
}
template <int TX, int TR>
int rms_out(bgnn_ctx* ctx, const RmsArgs& a, const RowShape& r, int out_type) {
  switch (out_type) {
    case BGNN_F32: return launch_rms<TX, TR, BGNN_F32>(ctx, a, r);
    case BGNN_BF16: return launch_rms<TX, TR, BGNN_BF16>(ctx, a, r);
    case BGNN_F16: return launch_rms<TX, TR, BGNN_F16>(ctx, a, r);
    default: return launch_rms<TX, TR, BGNN_E4M3>(ctx, a, r);
  }
}

template <int TG, int TT>
int launch_rms_bwd(bgnn_ctx* ctx, RmsBwdArgs a, const RowShape& r, void* gw, int w_type) {
  DevTmp part, stats;
  uint32_t parts;
  if (r.fits) {
    parts = row_grid(ctx, a.rows, r);
    if (gw) BGNN_TRY(bgnn_tmp_alloc(ctx, part, (size_t)parts * a.cols * sizeof(float)));
    a.part = part.as<float>();
    const size_t dyn = r.block > r.tpr ? (size_t)a.cols * sizeof(float) : 0;
    if (r.vec == 1)
      k_rms_bwd<TG, TT, 1, 8><<<parts, r.block, dyn, ctx->stream>>>(a, r.tpr);
    else if (r.nv == 1)
      k_rms_bwd<TG, TT, 8, 1><<<parts, r.block, dyn, ctx->stream>>>(a, r.tpr);
    else
      k_rms_bwd<TG, TT, 8, 2><<<parts, r.block, dyn, ctx->stream>>>(a, r.tpr);
    BGNN_LAUNCHED(ctx);
  } else {
    const unsigned grid = row_grid(ctx, a.rows, r);
    BGNN_TRY(bgnn_tmp_alloc(ctx, stats, (size_t)a.rows * sizeof(float2)));
    k_rms_bwd_stats<TG, TT><<<grid, 1024, 0, ctx->stream>>>(a, stats.as<float2>());
    BGNN_LAUNCHED(ctx);
    parts = (uint32_t)(a.rows < 64 ? a.rows : 64);
    if (gw) BGNN_TRY(bgnn_tmp_alloc(ctx, part, (size_t)parts * a.cols * sizeof(float)));
    a.part = part.as<float>();
    k_rms_bwd_apply<TG, TT><<<dim3((a.cols + 255) / 256, parts), 256, 0, ctx->stream>>>(
        a, stats.as<float2>());
    BGNN_LAUNCHED(ctx);
  }
  if (gw) {
    k_sum_parts<<<(unsigned)(((uint64_t)a.cols + 31) / 32), 256, 0, ctx->stream>>>(
        part.as<float>(), parts, a.cols, gw, w_type);
    BGNN_LAUNCHED(ctx);
  }
  return BGNN_OK;
}

}  // namespace

int bgnn_run_sum_parts(bgnn_ctx* ctx, const float* part, uint32_t parts, uint64_t cols, void* out,
                       int out_type) {
  if (cols == 0) return BGNN_OK;
  k_sum_parts<<<(unsigned)((cols + 31) / 32), 256, 0, ctx->stream>>>(part, parts, cols, out,
                                                                     out_type);
  BGNN_LAUNCHED(ctx);
  return BGNN_OK;
}

extern "C" int bgnn_rms_norm(bgnn_ctx* ctx, int x_type, const void* x, uint64_t ld_x, int res_type,
                             const void* residual, uint64_t ld_res, int w_type, const void* weight,
                             uint64_t rows, uint32_t cols, double eps, void* total, int out_type,
                             void* out, float* scale) {
  BGNN_ON_DEVICE(ctx);
  BGNN_REQUIRE(ctx, dtype_float(x_type) && dtype_float(w_type), "rms_norm: unknown element type");
  BGNN_REQUIRE(ctx, dtype_float(out_type) || out_type == BGNN_E4M3,
               "rms_norm: unknown output type %d", out_type);
  BGNN_REQUIRE(ctx, !residual || res_type == x_type || res_type == BGNN_F32,
               "rms_norm: the residual has the input's type or f32");
  BGNN_REQUIRE(ctx, eps >= 0.0, "rms_norm: negative or NaN eps");
  if (rows == 0 || cols == 0) return BGNN_OK;
  BGNN_REQUIRE(ctx, x && weight && out, "rms_norm: NULL argument");
  BGNN_REQUIRE(ctx, !residual || total, "rms_norm: a residual needs a buffer for the sum");
  BGNN_REQUIRE(ctx, out_type != BGNN_E4M3 || scale, "rms_norm: an e4m3 output needs scales");
  BGNN_REQUIRE(ctx, ld_x >= cols && (!residual || ld_res >= cols),
               "rms_norm: row stride below the row length");
  RmsArgs a;
  a.x = x;
  a.ld_x = ld_x;
  a.res = residual;
  a.ld_res = ld_res;
  a.w = weight;
  a.w_type = w_type;
  a.rows = rows;
  a.cols = cols;
  a.eps = (float)eps;
  a.total = total;
  a.out = out;
  a.scale = scale;
  const bool vec = cols % 8 == 0 && vec_rows(x, ld_x) && vec_rows(out, cols) &&
                   (!residual || (vec_rows(residual, ld_res) && vec_rows(total, cols)));
  const RowShape r = row_shape(cols, vec, 4, false);
  const bool wide = residual && res_type == BGNN_F32;  // f32 stream under a 16-bit input
  switch (x_type) {
    case BGNN_F32: return rms_out<BGNN_F32, BGNN_F32>(ctx, a, r, out_type);
    case BGNN_BF16:
      return wide ? rms_out<BGNN_BF16, BGNN_F32>(ctx, a, r, out_type)
                  : rms_out<BGNN_BF16, BGNN_BF16>(ctx, a, r, out_type);
    default:
      return wide ? rms_out<BGNN_F16, BGNN_F32>(ctx, a, r, out_type)
                  : rms_out<BGNN_F16, BGNN_F16>(ctx, a, r, out_type);
  }
}

extern "C" int bgnn_rms_norm_backward(bgnn_ctx* ctx, int grad_type, const void* grad,
                                      uint64_t ld_grad, int total_type, const void* total,
                                      uint64_t ld_total, const void* grad_total,
                                      uint64_t ld_grad_total, int w_type, const void* weight,
                                      uint64_t rows, uint32_t cols, double eps, void* grad_x,
                                      void* grad_weight) {
  BGNN_ON_DEVICE(ctx);
  BGNN_REQUIRE(ctx, dtype_float(grad_type) && dtype_float(total_type) && dtype_float(w_type),
               "rms_norm_backward: unknown element type");
  BGNN_REQUIRE(ctx, grad_type == total_type || total_type == BGNN_F32,
               "rms_norm_backward: the gradient has the row's type, or the row is f32");
  BGNN_REQUIRE(ctx, eps >= 0.0, "rms_norm_backward: negative or NaN eps");
  if (cols == 0) return BGNN_OK;
  if (rows == 0) {
    if (grad_weight)
      BGNN_CUDA(ctx, cudaMemsetAsync(grad_weight, 0, cols * dtype_size(w_type), ctx->stream));
    return BGNN_OK;
  }
  BGNN_REQUIRE(ctx, grad && total && weight && grad_x, "rms_norm_backward: NULL argument");
  BGNN_REQUIRE(ctx, ld_grad >= cols && ld_total >= cols && (!grad_total || ld_grad_total >= cols),
               "rms_norm_backward: row stride below the row length");
  RmsBwdArgs a;
  a.gy = grad;
  a.ld_gy = ld_grad;
  a.t = total;
  a.ld_t = ld_total;
  a.gt = grad_total;
  a.ld_gt = ld_grad_total;
  a.w = weight;
  a.w_type = w_type;
  a.rows = rows;
  a.cols = cols;
  a.eps = (float)eps;
  a.gx = grad_x;
  a.part = nullptr;
  const bool vec = cols % 8 == 0 && vec_rows(grad, ld_grad) && vec_rows(total, ld_total) &&
                   vec_rows(grad_x, cols) && (!grad_total || vec_rows(grad_total, ld_grad_total));
  const RowShape r = row_shape(cols, vec, 2, true);
  if (total_type == BGNN_F32) {
    switch (grad_type) {
      case BGNN_F32: return launch_rms_bwd<BGNN_F32, BGNN_F32>(ctx, a, r, grad_weight, w_type);
      case BGNN_BF16: return launch_rms_bwd<BGNN_BF16, BGNN_F32>(ctx, a, r, grad_weight, w_type);
      default: return launch_rms_bwd<BGNN_F16, BGNN_F32>(ctx, a, r, grad_weight, w_type);
    }
  }
  if (total_type == BGNN_BF16)
    return launch_rms_bwd<BGNN_BF16, BGNN_BF16>(ctx, a, r, grad_weight, w_type);
  return launch_rms_bwd<BGNN_F16, BGNN_F16>(ctx, a, r, grad_weight, w_type);
}
