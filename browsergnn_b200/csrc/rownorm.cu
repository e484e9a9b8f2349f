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
// there) and written once.  A row belongs to up to 32 threads, each holding NV
// vectors of eight columns, so that its sums are shuffles; longer rows to
// several warps and one barrier a sum.  Rows that do not start on 16 bytes (an
// odd width) are read as aligned 16-byte words shifted into place, and leave
// through shared memory the same way: 2.4 TB/s at 20,000 x 1,433 f16 backward
// (4.3 aligned, at 1,432 columns); element by element 0.56.  2.45M x 256 f32 with
// an f32 residual: 6.0 TB/s, 92 % of what a copy reaches.  Rows longer than the
// registers of a block hold (RowShape) take the k_*_long kernels, which read
// the row again from L2.
#include "lowp.cuh"
#include "row_words.cuh"

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
  uint32_t edge;  // edge_rows of the operands
  void* total;
  void* out;
  float* scale;
};

// Sum (or, on float bits, maximum) over the tpr threads of a row; every thread
// gets it.  tpr <= 32: the row's threads are consecutive lanes.  tpr > 32: the
// block.  `red` has two halves of 16 slots, used in turn, so that one barrier a
// call is enough.
__device__ __forceinline__ float2 row_sums(float2 v, int tpr, float2* red, int& flip) {
  const int lim = tpr < 32 ? tpr : 32;
  for (int o = 1; o < lim; o <<= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if (tpr > 32) {
    float2* slot = red + flip * 32;
    flip ^= 1;
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
    __syncthreads();
    v = slot[0];
    for (int i = 1; i < tpr >> 5; i++) v.x += slot[i].x, v.y += slot[i].y;
  }
  return v;
}
// the largest magnitude, as bits: NaN (0x7f800001 and up) above all others
__device__ __forceinline__ uint32_t row_amax(uint32_t v, int tpr, float2* red, int& flip) {
  const int lim = tpr < 32 ? tpr : 32;
  for (int o = 1; o < lim; o <<= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (tpr > 32) {
    uint32_t* slot = reinterpret_cast<uint32_t*>(red + flip * 32);
    flip ^= 1;
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
    __syncthreads();
    v = slot[0];
    for (int i = 1; i < tpr >> 5; i++) v = max(v, slot[i]);
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

// bytes [sh, sh + 16) of the 32 bytes a, b; WORDS: sh is a multiple of 4
template <bool WORDS>
__device__ __forceinline__ uint4 window(const uint4 a, const uint4 b, uint32_t sh) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  uint32_t y[6], z[5];
#pragma unroll
  for (int i = 0; i < 6; i++) y[i] = (sh & 8u) ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; i++) z[i] = (sh & 4u) ? y[i + 1] : y[i];
  if (WORDS) return make_uint4(z[0], z[1], z[2], z[3]);
  const uint32_t r = (sh & 3u) * 8;
  return make_uint4(__funnelshift_r(z[0], z[1], r), __funnelshift_r(z[1], z[2], r),
                    __funnelshift_r(z[2], z[3], r), __funnelshift_r(z[3], z[4], r));
}

// the memory of a matrix, [lo, hi): a 16-byte word is only read whole inside it
struct Span {
  const char *lo, *hi;
};
template <class T>
__device__ __forceinline__ Span span_of(const void* p, uint64_t rows, uint64_t ld, uint32_t cols) {
  const char* c = static_cast<const char*>(p);
  return {c, c + ((rows - 1) * ld + cols) * sizeof(T)};
}
__device__ __forceinline__ uint4 word_at(const char* p, const Span& m) {
  if (p >= m.lo && p + 16 <= m.hi) return *reinterpret_cast<const uint4*>(p);
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; i++)
    if (p + 2 * i >= m.lo && p + 2 * i + 2 <= m.hi)
      w[i >> 1] |= (uint32_t)*reinterpret_cast<const uint16_t*>(p + 2 * i) << (16 * (i & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// eight columns as they are stored
template <int DT>
struct Raw {
  uint4 w[DT == BGNN_F32 ? 2 : 1];
};
// The 16-byte words that hold a thread's vectors of a row, on their way in.
// MIS: one more a vector, since the row starts anywhere in the first.  All of a
// row's loads are issued before the first is looked at.
template <int DT, int NV, bool MIS>
struct Words {
  static constexpr int PER = 16 / sizeof(elt_t<DT>);  // columns of a word
  static constexpr int W = 8 / PER;
  uint4 w[NV][W + MIS];
  uint32_t sh;
  // vector i is columns [c0 + i * step, + 8); none from cols on.  Its words are
  // read whole: of inner rows only, or with !MIS, where they are the vector's.
  __device__ __forceinline__ void fetch(const elt_t<DT>* row, uint32_t c0, uint32_t step,
                                        uint32_t cols) {
    const char* p = reinterpret_cast<const char*>(row + c0);
    sh = MIS ? (uint32_t)(uintptr_t)p & 15u : 0u;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const uint4* q = reinterpret_cast<const uint4*>(p - sh + (uint64_t)i * step * sizeof(elt_t<DT>));
#pragma unroll
      for (int k = 0; k < W + MIS; k++)
        w[i][k] = c0 + i * step < cols ? q[k] : make_uint4(0, 0, 0, 0);
    }
  }
  // the first and the last rows (edge_rows): no word reaches out of the matrix
  __device__ __forceinline__ void fetch_edge(const elt_t<DT>* row, uint32_t c0, uint32_t step,
                                             uint32_t cols, const Span& m) {
    const char* p = reinterpret_cast<const char*>(row + c0);
    sh = (uint32_t)(uintptr_t)p & 15u;
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int k = 0; k < W + MIS; k++)
        w[i][k] = c0 + i * step < cols
                      ? word_at(p - sh + (uint64_t)i * step * sizeof(elt_t<DT>) + 16 * k, m)
                      : make_uint4(0, 0, 0, 0);
  }
  // vector i as stored, columns from cols on zero
  __device__ __forceinline__ Raw<DT> get(int i, uint32_t c, uint32_t cols) const {
    Raw<DT> r;
#pragma unroll
    for (int k = 0; k < W; k++) {
      uint4 v = MIS ? window<DT == BGNN_F32>(w[i][k], w[i][k + MIS], sh) : w[i][k];
      if (MIS && c + (k + 1) * PER > cols) {  // what is behind the row's end is another row's
        const uint32_t n = c + k * PER < cols ? (cols - c - k * PER) * (uint32_t)sizeof(elt_t<DT>) : 0u;
        v.x = n >= 4 ? v.x : n ? v.x & 0xffffu : 0u;
        v.y = n >= 8 ? v.y : n > 4 ? v.y & 0xffffu : 0u;
        v.z = n >= 12 ? v.z : n > 8 ? v.z & 0xffffu : 0u;
        v.w = n >= 16 ? v.w : n > 12 ? v.w & 0xffffu : 0u;
      }
      r.w[k] = v;
    }
    return r;
  }
};
template <int DT>
__device__ __forceinline__ void unpack(const Raw<DT>& r, float (&v)[8]) {
  const uint4* q = r.w;
  if constexpr (DT == BGNN_F32) {
    v[0] = __uint_as_float(q[0].x), v[1] = __uint_as_float(q[0].y);
    v[2] = __uint_as_float(q[0].z), v[3] = __uint_as_float(q[0].w);
    v[4] = __uint_as_float(q[1].x), v[5] = __uint_as_float(q[1].y);
    v[6] = __uint_as_float(q[1].z), v[7] = __uint_as_float(q[1].w);
  } else {
    load8<DT>(reinterpret_cast<const elt_t<DT>*>(q), v);
  }
}

// A row on its way out, eight columns at a time (put), then, MIS, from the
// group's own shared memory to the row (flush): `lanes` lanes hold NV * lanes
// vectors from column `first` on.
template <int DT, bool MIS>
struct RowOut {
  elt_t<DT>* row;
  uint32_t first, lane, lanes, cols;  // cols 0: no such row
  char* stage;
  __device__ __forceinline__ void begin() const {
    if (MIS) __syncwarp();  // the last row's readers
  }
  __device__ __forceinline__ void put(int i, const float (&v)[8]) const {
    const uint32_t c = (i * lanes + lane) * 8;
    if (MIS) store8<DT>(reinterpret_cast<elt_t<DT>*>(stage) + c, v);
    else if (first + c < cols) store8<DT>(row + first + c, v);
  }
  template <int NV>
  __device__ __forceinline__ void flush() const {
    if (!MIS) return;
    constexpr uint32_t ES = sizeof(elt_t<DT>);
    __syncwarp();
    if (first < cols) {
      const uint32_t len = NV * lanes * 8 < cols - first ? NV * lanes * 8 : cols - first;
      const uint32_t bytes = len * ES;
      char* out = reinterpret_cast<char*>(row + first);
      uint32_t head = (16u - ((uint32_t)(uintptr_t)out & 15u)) & 15u;
      if (head > bytes) head = bytes;
      const uint32_t words = (bytes - head) / 16;
      for (uint32_t k = lane; k < words; k += lanes) {
        const uint32_t at = head + 16 * k, sh = at & 15u;
        const uint4* q = reinterpret_cast<const uint4*>(stage + at - sh);
        *reinterpret_cast<uint4*>(out + at) = window<DT == BGNN_F32>(q[0], q[1], sh);
      }
      const uint32_t tail = head + 16 * words;
      for (uint32_t e = lane; e < head / ES; e += lanes)
        row[first + e] = reinterpret_cast<const elt_t<DT>*>(stage)[e];
      for (uint32_t e = tail / ES + lane; e < len; e += lanes)
        row[first + e] = reinterpret_cast<const elt_t<DT>*>(stage)[e];
    }
  }
};

// weights of eight columns
__device__ __forceinline__ void load_w(const void* w, int type, bool vec, uint32_t c, uint32_t cols,
                                       float (&o)[8]) {
  if (vec && c + 8 <= cols) {
    load8<BGNN_F32>(static_cast<const float*>(w) + c, o);
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) o[j] = c + j < cols ? load_any(w, type, c + j) : 0.0f;
  }
}

// where a thread's columns are: tpr threads a row; up to 32 share a warp with
// other rows, more are whole warps with a run of columns each
struct RowPlace {
  int sub, rpb;
  uint32_t lane, lanes, first;
  char* stage;
};
template <int NV>
__device__ __forceinline__ RowPlace row_place(int tpr, uint32_t stage_bytes, char* smem) {
  RowPlace r;
  r.sub = threadIdx.x / tpr;
  r.rpb = blockDim.x / tpr;
  r.lanes = tpr < 32 ? tpr : 32;
  r.lane = threadIdx.x % r.lanes;
  r.first = tpr > 32 ? (threadIdx.x >> 5) * (32 * NV * 8) : 0;
  r.stage = smem + (threadIdx.x / r.lanes) * stage_bytes;
  return r;
}

template <int TX, int TR, int TO, int NV, bool MIS>
__global__ void __launch_bounds__(NV == 1 ? 256 : 512, NV > 1 ? 1 : MIS ? 4 : 5) k_rms(const RmsArgs a, int tpr,
                                               uint32_t stage_bytes) {
  extern __shared__ __align__(16) char stages[];
  __shared__ float2 red[64];
  int flip = 0;
  const RowPlace at = row_place<NV>(tpr, stage_bytes, stages);
  const bool wvec = a.w_type == BGNN_F32 && ((uintptr_t)a.w & 15u) == 0;
  const Span mx = span_of<elt_t<TX>>(a.x, a.rows, a.ld_x, a.cols);
  const Span mr = span_of<elt_t<TR>>(a.res, a.rows, a.ld_res, a.cols);
  float w1[8];
  if (NV == 1) load_w(a.w, a.w_type, wvec, at.first + at.lane * 8, a.cols, w1);
  const float inv_n = __fdiv_rn(1.0f, (float)a.cols);
  for (uint64_t base = (uint64_t)blockIdx.x * at.rpb; base < a.rows;
       base += (uint64_t)gridDim.x * at.rpb) {
    const uint64_t row = base + at.sub;
    const bool on = row < a.rows, inner = inner_row(row, a.rows, a.edge);
    const uint32_t cols = on ? a.cols : 0;
    const uint32_t c0 = at.first + at.lane * 8, step = at.lanes * 8;
    float t[NV][8];
    const elt_t<TX>* xr = static_cast<const elt_t<TX>*>(a.x) + row * a.ld_x;
    Words<TX, NV, MIS> x;
    if (a.res) {
      const elt_t<TR>* rr = static_cast<const elt_t<TR>*>(a.res) + row * a.ld_res;
      Words<TR, NV, MIS> r;
      if (!MIS || inner) {
        x.fetch(xr, c0, step, cols);
        r.fetch(rr, c0, step, cols);
      } else {
        x.fetch_edge(xr, c0, step, cols, mx);
        r.fetch_edge(rr, c0, step, cols, mr);
      }
      const RowOut<TR, MIS> to = {static_cast<elt_t<TR>*>(a.total) + row * a.cols, at.first,
                                  at.lane, at.lanes, cols, at.stage};
      to.begin();
#pragma unroll
      for (int i = 0; i < NV; i++) {
        float u[8];
        unpack<TX>(x.get(i, c0 + i * step, cols), t[i]);
        unpack<TR>(r.get(i, c0 + i * step, cols), u);
#pragma unroll
        for (int j = 0; j < 8; j++) t[i][j] = rounded<TR>(t[i][j] + u[j]);
        to.put(i, t[i]);
      }
      to.template flush<NV>();
    } else {
      if (!MIS || inner) x.fetch(xr, c0, step, cols);
      else x.fetch_edge(xr, c0, step, cols, mx);
#pragma unroll
      for (int i = 0; i < NV; i++) unpack<TX>(x.get(i, c0 + i * step, cols), t[i]);
    }
    float2 ss = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        ss.x = fmaf(t[i][j], t[i][j], ss.x);
        ss.y = fmaf(t[i][j + 1], t[i][j + 1], ss.y);
      }
    ss = row_sums(make_float2(ss.x + ss.y, 0.0f), tpr, red, flip);
    const float s = __frsqrt_rn(fmaf(ss.x, inv_n, a.eps));
    uint32_t am = 0;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      float w[8];
      if (NV == 1) {
#pragma unroll
        for (int j = 0; j < 8; j++) w[j] = w1[j];
      } else {
        load_w(a.w, a.w_type, wvec, at.first + (i * at.lanes + at.lane) * 8, a.cols, w);
      }
#pragma unroll
      for (int j = 0; j < 8; j++) {
        // what is behind the row's end stays 0: 0 * s may be NaN
        const bool in = at.first + (i * at.lanes + at.lane) * 8 + j < a.cols;
        t[i][j] = in ? w[j] * (t[i][j] * s) : 0.0f;
        if (TO == BGNN_E4M3) am = max(am, __float_as_uint(t[i][j]) & 0x7fffffffu);
      }
    }
    if constexpr (TO == BGNN_E4M3) {
      const float2 sc = e4m3_scale(__uint_as_float(row_amax(am, tpr, red, flip)));
#pragma unroll
      for (int i = 0; i < NV; i++)
#pragma unroll
        for (int j = 0; j < 8; j++) t[i][j] *= sc.y;
      if (on && threadIdx.x % tpr == 0) a.scale[row] = sc.x;
    }
    const RowOut<TO, MIS> out = {static_cast<elt_t<TO>*>(a.out) + row * a.cols, at.first, at.lane,
                                 at.lanes, cols, at.stage};
    out.begin();
#pragma unroll
    for (int i = 0; i < NV; i++) out.put(i, t[i]);
    out.template flush<NV>();
  }
}

// a row longer than the registers of a block: read again from L2
template <int TX, int TR, int TO>
__global__ void __launch_bounds__(1024) k_rms_long(const RmsArgs a) {
  __shared__ float2 red[64];
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
    ss = row_sums(make_float2(ss, 0.0f), nt, red, flip).x;
    const float s = __frsqrt_rn(fmaf(ss, __fdiv_rn(1.0f, (float)a.cols), a.eps));
    float2 sc = make_float2(1.0f, 1.0f);
    if constexpr (TO == BGNN_E4M3) {
      uint32_t am = 0;
      for (uint32_t c = threadIdx.x; c < a.cols; c += nt)
        am = max(am, __float_as_uint(load_any(a.w, a.w_type, c) * (at(c) * s)) & 0x7fffffffu);
      sc = e4m3_scale(__uint_as_float(row_amax(am, nt, red, flip)));
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
  uint32_t edge;  // edge_rows of the operands
  void* gx;
  float* part;  // [grid, cols] sums of gy * xh over each block's rows
};

template <int TG, int TT, int NV, bool MIS>
__global__ void __launch_bounds__(512) k_rms_bwd(const RmsBwdArgs a, int tpr,
                                                   uint32_t stage_bytes) {
  extern __shared__ __align__(16) char stages[];  // then [cols] f32 when a block has several rows
  __shared__ float2 red[64];
  int flip = 0;
  const RowPlace at = row_place<NV>(tpr, stage_bytes, stages);
  const bool wvec = a.w_type == BGNN_F32 && ((uintptr_t)a.w & 15u) == 0;
  const Span mt = span_of<elt_t<TT>>(a.t, a.rows, a.ld_t, a.cols);
  const Span mg = span_of<elt_t<TG>>(a.gy, a.rows, a.ld_gy, a.cols);
  const Span ms = span_of<elt_t<TT>>(a.gt, a.rows, a.ld_gt, a.cols);
  auto col = [&](int i) { return at.first + (i * at.lanes + at.lane) * 8; };
  float w1[8], gw[NV][8];
  if (NV == 1) load_w(a.w, a.w_type, wvec, col(0), a.cols, w1);
#pragma unroll
  for (int i = 0; i < NV; i++)
#pragma unroll
    for (int j = 0; j < 8; j++) gw[i][j] = 0.0f;
  auto weights = [&](int i, float (&w)[8]) {
    if (NV == 1) {
#pragma unroll
      for (int j = 0; j < 8; j++) w[j] = w1[j];
    } else {
      load_w(a.w, a.w_type, wvec, col(i), a.cols, w);
    }
  };
  const float inv_n = __fdiv_rn(1.0f, (float)a.cols);
  for (uint64_t base = (uint64_t)blockIdx.x * at.rpb; base < a.rows;
       base += (uint64_t)gridDim.x * at.rpb) {
    const uint64_t row = base + at.sub;
    const bool on = row < a.rows, inner = inner_row(row, a.rows, a.edge);
    const uint32_t cols = on ? a.cols : 0;
    const elt_t<TT>* sr = static_cast<const elt_t<TT>*>(a.gt) + row * a.ld_gt;
    // the row stays as stored (16-bit: half the registers) and is unpacked twice
    const uint32_t c0 = at.first + at.lane * 8, step = at.lanes * 8;
    const elt_t<TT>* tr = static_cast<const elt_t<TT>*>(a.t) + row * a.ld_t;
    const elt_t<TG>* gr = static_cast<const elt_t<TG>*>(a.gy) + row * a.ld_gy;
    Raw<TT> t[NV], st[NV];
    Raw<TG> g[NV];
    {
      Words<TT, NV, MIS> tw, sw;
      Words<TG, NV, MIS> gw_;
      if (!MIS || inner) {
        tw.fetch(tr, c0, step, cols);
        gw_.fetch(gr, c0, step, cols);
        if (a.gt) sw.fetch(sr, c0, step, cols);
      } else {
        tw.fetch_edge(tr, c0, step, cols, mt);
        gw_.fetch_edge(gr, c0, step, cols, mg);
        if (a.gt) sw.fetch_edge(sr, c0, step, cols, ms);
      }
#pragma unroll
      for (int i = 0; i < NV; i++) {
        t[i] = tw.get(i, c0 + i * step, cols);
        g[i] = gw_.get(i, c0 + i * step, cols);
        if (a.gt) st[i] = sw.get(i, c0 + i * step, cols);
      }
    }
    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < NV; i++) {
      float u[8], q[8], w[8];
      unpack<TT>(t[i], u);
      unpack<TG>(g[i], q);
      weights(i, w);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        sum.x = fmaf(u[j], u[j], sum.x);
        sum.y = fmaf(q[j] * w[j], u[j], sum.y);
      }
    }
    sum = row_sums(sum, tpr, red, flip);
    const float s = __frsqrt_rn(fmaf(sum.x, inv_n, a.eps));
    const float c1 = sum.y * s * inv_n;  // mean(gy w xh)
    const RowOut<TT, MIS> out = {static_cast<elt_t<TT>*>(a.gx) + row * a.cols, at.first, at.lane,
                                 at.lanes, cols, at.stage};
    out.begin();
#pragma unroll
    for (int i = 0; i < NV; i++) {
      float u[8], q[8], w[8], o[8];
      unpack<TT>(t[i], u);
      unpack<TG>(g[i], q);
      weights(i, w);
      if (a.gt) {
        unpack<TT>(st[i], o);
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) o[j] = 0.0f;
      }
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float xh = u[j] * s;
        o[j] = fmaf(s, fmaf(-xh, c1, q[j] * w[j]), o[j]);
        // a row that is not there: 0 * s may be NaN
        if (on) gw[i][j] = fmaf(q[j], xh, gw[i][j]);
      }
      out.put(i, o);
    }
    out.template flush<NV>();
  }
  if (!a.part) return;
  // the block's sums: its row groups' side by side, added in their order
  float* prow = a.part + (uint64_t)blockIdx.x * a.cols;
  float* fold = reinterpret_cast<float*>(stages + (blockDim.x / at.lanes) * stage_bytes);
  const bool several = at.rpb > 1;
#pragma unroll
  for (int i = 0; i < NV; i++)
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (col(i) + j < a.cols)
        (several ? fold + (uint64_t)at.sub * a.cols : prow)[col(i) + j] = gw[i][j];
  if (!several) return;
  __syncthreads();
  for (uint32_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
    float v = fold[c];
    for (int r = 1; r < at.rpb; r++) v += fold[(uint64_t)r * a.cols + c];
    prow[c] = v;
  }
}

// long rows: per row (s, mean(gy w xh))
template <int TG, int TT>
__global__ void __launch_bounds__(1024) k_rms_bwd_stats(const RmsBwdArgs a, float2* stats) {
  __shared__ float2 red[64];
  int flip = 0;
  for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const elt_t<TT>* tr = static_cast<const elt_t<TT>*>(a.t) + row * a.ld_t;
    const elt_t<TG>* gr = static_cast<const elt_t<TG>*>(a.gy) + row * a.ld_gy;
    float2 sum = make_float2(0.0f, 0.0f);
    for (uint32_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
      const float t = Elt<TT>::get(tr[c]);
      sum.x = fmaf(t, t, sum.x);
      sum.y = fmaf(Elt<TG>::get(gr[c]) * load_any(a.w, a.w_type, c), t, sum.y);
    }
    sum = row_sums(sum, blockDim.x, red, flip);
    const float inv_n = __fdiv_rn(1.0f, (float)a.cols);
    const float s = __frsqrt_rn(fmaf(sum.x, inv_n, a.eps));
    if (threadIdx.x == 0) stats[row] = make_float2(s, sum.y * s * inv_n);
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

// out[c] = sum over the parts: 32 columns a block, 32 chains a column (each in
// ascending order), then the chains in order.  Few columns have few blocks, so
// a chain keeps four loads in flight.
__global__ void __launch_bounds__(1024) k_sum_parts(const float* __restrict__ part, uint32_t parts,
                                                    uint64_t cols, void* out, int out_type) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, ch = threadIdx.x >> 5;
  const uint64_t c = (uint64_t)blockIdx.x * 32 + lane;
  float v = 0.0f;
  if (c < cols) {
    uint32_t p = ch;
    for (; p + 96 < parts; p += 128) {
      const float a0 = part[(uint64_t)p * cols + c], a1 = part[(uint64_t)(p + 32) * cols + c];
      const float a2 = part[(uint64_t)(p + 64) * cols + c], a3 = part[(uint64_t)(p + 96) * cols + c];
      v = v + a0 + a1 + a2 + a3;
    }
    for (; p < parts; p += 32) v += part[(uint64_t)p * cols + c];
  }
  s[ch][lane] = v;
  __syncthreads();
  if (ch == 0 && c < cols) {
#pragma unroll
    for (int i = 1; i < 32; i++) v += s[i][lane];
    store_any(out, out_type, c, v);
  }
}

// How a row of `cols` elements is held.
struct RowShape {
  int nv, tpr, block, per_sm;  // vectors and threads of a row; blocks an SM
  bool fits, mis;
  uint32_t stage, shared;  // bytes a group of lanes stages, and a block's shared memory
};
// A warp a row while `most` vectors a thread are enough (four; two where f32
// rows are shifted into place or kept for the backward, whose words would not
// fit the registers); then several warps, up to 512 threads, with three or four
// vectors each (two), whichever leaves fewer idle.  es: bytes of the widest
// output element; backward: the block's column sums need shared memory.
RowShape row_shape(uint32_t cols, bool mis, bool f32, uint32_t es, bool backward) {
  RowShape r = {};
  r.mis = mis;
  const uint32_t nvec = (cols + 7) / 8;
  const uint32_t most = f32 && (mis || backward) ? 2 : 4;
  if (nvec <= 32 * most) {
    r.nv = nvec <= 32 ? 1 : nvec <= 64 ? 2 : 4;
    r.tpr = 1;
    while ((uint32_t)r.tpr * r.nv < nvec) r.tpr *= 2;
    r.block = 256;
    r.fits = true;
  } else {
    const uint32_t t3 = (nvec + 95) / 96 * 32, tm = (nvec + 32 * most - 1) / (32 * most) * 32;
    r.nv = most == 4 && 3 * t3 < 4 * tm && t3 <= 512 ? 3 : (int)most;
    r.tpr = r.block = (int)(r.nv == 3 ? t3 : tm);
    r.fits = r.block <= 512;
    if (!r.fits) r.tpr = r.block = 1024;
  }
  // registers: three or four vectors a thread take about 128 in the backward
  r.per_sm = (backward && r.nv > 2 ? 512 : r.nv > 1 ? 1536 : 2048) / r.block;
  if (r.per_sm < 1) r.per_sm = 1;
  const uint32_t lanes = r.tpr < 32 ? r.tpr : 32;
  r.stage = mis ? (lanes * r.nv * 8 * es + 15) / 16 * 16 + 16 : 0;
  r.shared = r.stage * (r.block / lanes);
  if (backward && r.block > r.tpr) r.shared += cols * 4 * (r.block / r.tpr);
  return r;
}

// every row starts on 16 bytes and is whole vectors
bool vec_rows(const void* p, uint64_t ld) { return ((uintptr_t)p & 15u) == 0 && ld % 8 == 0; }

// resident blocks fill the GPU; each loops over its share of the rows
unsigned row_grid(const bgnn_ctx* ctx, uint64_t rows, const RowShape& r) {
  const uint64_t rpb = (uint64_t)(r.block / r.tpr);
  const uint64_t want = (rows + rpb - 1) / rpb, cap = (uint64_t)ctx->num_sms * r.per_sm;
  return (unsigned)(want < cap ? want : cap);
}

constexpr uint32_t STATIC_SHARED = 64 * sizeof(float2);  // the kernels' `red`
template <class K, class... A>
int launch_rows(bgnn_ctx* ctx, K kernel, unsigned grid, const RowShape& r, A... args) {
  if (r.shared + STATIC_SHARED > 48 * 1024)  // what a launch may take without being asked for
    BGNN_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)r.shared));
  kernel<<<grid, r.block, r.shared, ctx->stream>>>(args...);
  BGNN_LAUNCHED(ctx);
  return BGNN_OK;
}

template <int TX, int TR, int TO, bool MIS>
int launch_rms(bgnn_ctx* ctx, const RmsArgs& a, const RowShape& r) {
  const unsigned grid = row_grid(ctx, a.rows, r);
  if (r.nv == 1) return launch_rows(ctx, k_rms<TX, TR, TO, 1, MIS>, grid, r, a, r.tpr, r.stage);
  if constexpr (!MIS || (TX != BGNN_F32 && TR != BGNN_F32)) {  // as row_shape chooses
    if (r.nv == 3) return launch_rows(ctx, k_rms<TX, TR, TO, 3, MIS>, grid, r, a, r.tpr, r.stage);
    if (r.nv == 4) return launch_rows(ctx, k_rms<TX, TR, TO, 4, MIS>, grid, r, a, r.tpr, r.stage);
  }
  return launch_rows(ctx, k_rms<TX, TR, TO, 2, MIS>, grid, r, a, r.tpr, r.stage);
}
template <int TX, int TR, int TO>
int rms_mis(bgnn_ctx* ctx, const RmsArgs& a, const RowShape& r) {
  if (!r.fits) return launch_rows(ctx, k_rms_long<TX, TR, TO>, row_grid(ctx, a.rows, r), r, a);
  return r.mis ? launch_rms<TX, TR, TO, true>(ctx, a, r) : launch_rms<TX, TR, TO, false>(ctx, a, r);
}
template <int TX, int TR>
int rms_out(bgnn_ctx* ctx, const RmsArgs& a, const RowShape& r, int out_type) {
  switch (out_type) {
    case BGNN_F32: return rms_mis<TX, TR, BGNN_F32>(ctx, a, r);
    case BGNN_BF16: return rms_mis<TX, TR, BGNN_BF16>(ctx, a, r);
    case BGNN_F16: return rms_mis<TX, TR, BGNN_F16>(ctx, a, r);
    default: return rms_mis<TX, TR, BGNN_E4M3>(ctx, a, r);
  }
}

template <int TG, int TT, bool MIS>
int launch_rms_bwd(bgnn_ctx* ctx, const RmsBwdArgs& a, const RowShape& r, unsigned grid) {
  if (r.nv == 1) return launch_rows(ctx, k_rms_bwd<TG, TT, 1, MIS>, grid, r, a, r.tpr, r.stage);
  if constexpr (TT != BGNN_F32) {
    if (r.nv == 3) return launch_rows(ctx, k_rms_bwd<TG, TT, 3, MIS>, grid, r, a, r.tpr, r.stage);
    if (r.nv == 4) return launch_rows(ctx, k_rms_bwd<TG, TT, 4, MIS>, grid, r, a, r.tpr, r.stage);
  }
  return launch_rows(ctx, k_rms_bwd<TG, TT, 2, MIS>, grid, r, a, r.tpr, r.stage);
}
template <int TG, int TT>
int rms_bwd(bgnn_ctx* ctx, RmsBwdArgs a, const RowShape& r, void* gw, int w_type) {
  DevTmp part, stats;
  uint32_t parts = row_grid(ctx, a.rows, r);
  if (r.fits) {
    if (gw) BGNN_TRY(bgnn_tmp_alloc(ctx, part, (size_t)parts * a.cols * sizeof(float)));
    a.part = part.as<float>();
    if (r.mis) BGNN_TRY((launch_rms_bwd<TG, TT, true>(ctx, a, r, parts)));
    else BGNN_TRY((launch_rms_bwd<TG, TT, false>(ctx, a, r, parts)));
  } else {
    BGNN_TRY(bgnn_tmp_alloc(ctx, stats, (size_t)a.rows * sizeof(float2)));
    k_rms_bwd_stats<TG, TT><<<parts, 1024, 0, ctx->stream>>>(a, stats.as<float2>());
    BGNN_LAUNCHED(ctx);
    parts = (uint32_t)(a.rows < 64 ? a.rows : 64);
    if (gw) BGNN_TRY(bgnn_tmp_alloc(ctx, part, (size_t)parts * a.cols * sizeof(float)));
    a.part = part.as<float>();
    k_rms_bwd_apply<TG, TT><<<dim3((a.cols + 255) / 256, parts), 256, 0, ctx->stream>>>(
        a, stats.as<float2>());
    BGNN_LAUNCHED(ctx);
  }
  return gw ? bgnn_run_sum_parts(ctx, a.part, parts, a.cols, gw, w_type) : BGNN_OK;
}

}  // namespace

int bgnn_run_sum_parts(bgnn_ctx* ctx, const float* part, uint32_t parts, uint64_t cols, void* out,
                       int out_type) {
  if (cols == 0) return BGNN_OK;
  k_sum_parts<<<(unsigned)((cols + 31) / 32), 1024, 0, ctx->stream>>>(part, parts, cols, out,
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
  BGNN_REQUIRE_COLS(ctx, "rms_norm", cols);
  BGNN_REQUIRE(ctx, eps >= 0.0, "rms_norm: negative or NaN eps");
  if (rows == 0 || cols == 0) {
    if (rows && scale && out_type == BGNN_E4M3)
      BGNN_CUDA(ctx, cudaMemsetAsync(scale, 0, rows * sizeof(float), ctx->stream));
    return BGNN_OK;
  }
  BGNN_REQUIRE(ctx, x && weight && out, "rms_norm: NULL argument");
  BGNN_REQUIRE(ctx, !residual || total, "rms_norm: a residual needs a buffer for the sum");
  BGNN_REQUIRE(ctx, !residual || total != residual || rows == 1 || ld_res == cols,
               "rms_norm: the sum in the residual's buffer needs its row stride, the row length");
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
  a.edge = edge_rows(residual && ld_res < ld_x ? ld_res : ld_x);
  a.total = total;
  a.out = out;
  a.scale = scale;
  const bool vec = cols % 8 == 0 && vec_rows(x, ld_x) && vec_rows(out, cols) &&
                   (!residual || (vec_rows(residual, ld_res) && vec_rows(total, cols)));
  const uint32_t es = residual && res_type == BGNN_F32 ? 4u
                      : residual && dtype_size(out_type) < 2 ? 2u : (uint32_t)dtype_size(out_type);
  const RowShape r = row_shape(
      cols, !vec, x_type == BGNN_F32 || (residual && res_type == BGNN_F32), es, false);
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
  BGNN_REQUIRE_COLS(ctx, "rms_norm_backward", cols);
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
  uint64_t ld = ld_grad < ld_total ? ld_grad : ld_total;
  if (grad_total && ld_grad_total < ld) ld = ld_grad_total;
  a.edge = edge_rows(ld);
  a.gx = grad_x;
  a.part = nullptr;
  const bool vec = cols % 8 == 0 && vec_rows(grad, ld_grad) && vec_rows(total, ld_total) &&
                   vec_rows(grad_x, cols) && (!grad_total || vec_rows(grad_total, ld_grad_total));
  const RowShape r = row_shape(cols, !vec, total_type == BGNN_F32, (uint32_t)dtype_size(total_type), true);
  if (total_type == BGNN_F32) {
    switch (grad_type) {
      case BGNN_F32: return rms_bwd<BGNN_F32, BGNN_F32>(ctx, a, r, grad_weight, w_type);
      case BGNN_BF16: return rms_bwd<BGNN_BF16, BGNN_F32>(ctx, a, r, grad_weight, w_type);
      default: return rms_bwd<BGNN_F16, BGNN_F32>(ctx, a, r, grad_weight, w_type);
    }
  }
  if (total_type == BGNN_BF16)
    return rms_bwd<BGNN_BF16, BGNN_BF16>(ctx, a, r, grad_weight, w_type);
  return rms_bwd<BGNN_F16, BGNN_F16>(ctx, a, r, grad_weight, w_type);
}
