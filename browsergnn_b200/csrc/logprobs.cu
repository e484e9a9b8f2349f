// Log probabilities of each row's given choice, with the entropy, the
// log-sum-exp and the top alternatives; and their gradient.
//
// Over the choices that are left in a row (not masked, logit above -inf):
//   lse = m + log S,  S = sum_j exp(x_j - m),  m = max_j x_j
//   logp_t = (x_t - m) - log S
//   H = -sum_j p_j log p_j = log S - (1/S) sum_j (x_j - m) exp(x_j - m)
// and, for the gradients g_l of logp_t and g_h of H,
//   dx_j = p_j (-g_l - g_h (log p_j + H)) + g_l [j = t],   p_j = exp(x_j - lse).
//
// One pass: every thread keeps a running (m, S, W = sum a 2^a), a = (x - m)
// log2(e), in f32 and rescales it when its maximum moves (W' = 2^d (W + d S));
// pairs merge the same way.  The k-th largest of a block's 256 thread maxima is
// at most the row's k-th largest logit, so the top list is among the elements
// that reach it: about k of them, in the vectors of the threads whose maximum
// does, which are read once more (from L2) and ranked by counting: 157 us for
// 8,192 x 32,000 bf16, k = 20 (3.3 TB/s), 117 us without a list.  (Keeping the
// list sorted in a warp's lanes while reading took 565 us; it is what a row with
// hundreds of equal logits at the border falls back to.)  A long row is split
// over blocks and joined by k_logp_join; short rows take a warp each.  The logits
// (and masks) are read once; about seven instructions an element, one of them
// 2^x, bound it before memory does.
#include <atomic>

#include "lowp.cuh"

namespace {

constexpr uint32_t NO_CHOICE = 0xffffffffu;
constexpr int TOP_MAX = 32;
constexpr int LP_WARPS = 8;  // of a block in the split kernel

struct LogpArgs {
  const void* x;
  uint64_t ld;
  uint32_t rows, cols;
  const uint8_t* mask;  // may be NULL
  uint64_t ld_mask;     // 0: one mask for all rows
  const uint32_t* targets;
  int top;
  uint32_t splits, seg;  // a row is cut into `splits` segments of `seg` elements
  float* logp;
  float* entropy;
  float* lse;
  uint32_t* top_ids;
  float* top_logp;
  float4* part;       // [rows, splits] (m, S, W, -)
  float* part_v;      // [rows, splits, top]
  uint32_t* part_id;  // [rows, splits, top]
  int* err;
};

constexpr float LN2 = 0.6931471805599453f;
// An exponent on its way into 2^a and a 2^a: not below -150, where 2^a is 0, so
// that a 2^a is never -inf * 0 (x - m may be -inf beside a mask of the type's
// lowest value).  NaN stays NaN.
__device__ __forceinline__ float not_below(float a, float least) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(least));
  return r;
}
__device__ __forceinline__ float floored(float a) { return not_below(a, -150.0f); }
__device__ __forceinline__ float exponent(float d) { return floored(d * LOG2E); }

struct Stat {
  float m, s, w;
};

__device__ __forceinline__ Stat stat_merge(Stat a, Stat b) {
  const float m = fmaxf(a.m, b.m);
  const float ms = m == -INFINITY ? 0.0f : m;
  // the side with nothing in it contributes S = W = 0 whatever its m
  const float da = a.m == -INFINITY ? 0.0f : exponent(a.m - ms);
  const float db = b.m == -INFINITY ? 0.0f : exponent(b.m - ms);
  const float ea = ex2(da), eb = ex2(db);
  Stat r;
  r.m = m;
  r.s = a.s * ea + b.s * eb;
  r.w = (a.w + da * a.s) * ea + (b.w + db * b.s) * eb;
  return r;
}

__device__ __forceinline__ Stat warp_stat(Stat t) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stat u;
    u.m = __shfl_xor_sync(0xffffffffu, t.m, o);
    u.s = __shfl_xor_sync(0xffffffffu, t.s, o);
    u.w = __shfl_xor_sync(0xffffffffu, t.w, o);
    t = stat_merge(t, u);
  }
  return t;
}

// a before b in the list: greater value, then lower index
__device__ __forceinline__ bool before(float av, uint32_t ai, float bv, uint32_t bi) {
  return av > bv || (av == bv && ai < bi);
}

// a warp's sorted list of the best `top` elements, lane i holding the i-th
struct TopList {
  float v = -INFINITY;
  uint32_t id = NO_CHOICE;
  float last_v = -INFINITY;  // the last that is still in the list
  uint32_t last_id = NO_CHOICE;

  // offers one element a lane; all lanes call
  __device__ __forceinline__ void offer(float cv, uint32_t ci, int top, int lane) {
    if (cv == -INFINITY) ci = NO_CHOICE;  // not an alternative
    uint32_t in = __ballot_sync(0xffffffffu, before(cv, ci, last_v, last_id));
    while (in) {
      const int src = __ffs((int)in) - 1;
      const float nv = __shfl_sync(0xffffffffu, cv, src);
      const uint32_t ni = __shfl_sync(0xffffffffu, ci, src);
      const int pos = __popc(__ballot_sync(0xffffffffu, before(v, id, nv, ni)));
      const float uv = __shfl_up_sync(0xffffffffu, v, 1);
      const uint32_t ui = __shfl_up_sync(0xffffffffu, id, 1);
      if (lane > pos) v = uv, id = ui;
      if (lane == pos) v = nv, id = ni;
      last_v = __shfl_sync(0xffffffffu, v, top - 1);
      last_id = __shfl_sync(0xffffffffu, id, top - 1);
      in &= in - 1;
      in &= __ballot_sync(0xffffffffu, before(cv, ci, last_v, last_id));
    }
  }
};

// the eight elements [e, e + 8) of a row, -inf outside [lo, hi) and where masked
template <int DT>
__device__ __forceinline__ void load_left(const elt_t<DT>* xr, const uint8_t* mr, bool mask_vec,
                                          int64_t e, int64_t lo, int64_t hi, float (&v)[8]) {
  if (e >= lo && e + 8 <= hi) {
    load8<DT>(xr + e, v);
    if (mr) {
      if (mask_vec) {
        const uint2 mm = *reinterpret_cast<const uint2*>(mr + e);
#pragma unroll
        for (int j = 0; j < 8; j++)
          if (((j < 4 ? mm.x >> (8 * j) : mm.y >> (8 * (j - 4))) & 0xffu) != 0) v[j] = -INFINITY;
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
          if (mr[e + j]) v[j] = -INFINITY;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int64_t i = e + j;
      v[j] = (i >= lo && i < hi && !(mr && mr[i])) ? Elt<DT>::get(xr[i]) : -INFINITY;
    }
  }
}

// eight elements as they are stored
template <int DT>
struct Vec {
  uint4 w[DT == BGNN_F32 ? 2 : 1];
};
template <int DT>
__device__ __forceinline__ Vec<DT> load_vec(const elt_t<DT>* p) {
  Vec<DT> r;
#pragma unroll
  for (int i = 0; i < (DT == BGNN_F32 ? 2 : 1); i++) r.w[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}

// elements before the row's first that share its 8-element vector
template <int DT>
__device__ __forceinline__ int row_lead(const elt_t<DT>* xr) {
  return (int)(((uintptr_t)xr / sizeof(elt_t<DT>)) & 7u);
}

__device__ __forceinline__ void stat_add(Stat& t, const float (&v)[8]) {
  float cm = v[0];
#pragma unroll
  for (int j = 1; j < 8; j++) cm = fmaxf(cm, v[j]);
  if (cm > t.m) {
    const float d = t.m == -INFINITY ? 0.0f : exponent(t.m - cm);
    const float e = ex2(d);
    t.w = (t.w + d * t.s) * e;
    t.s *= e;
    t.m = cm;
  }
  const float m = t.m == -INFINITY ? 0.0f : t.m;
  float2 s = make_float2(0.0f, 0.0f), w = make_float2(0.0f, t.w);
  const float2 mm = make_float2(-m, -m);
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const float2 d = mul2(add2(make_float2(v[j], v[j + 1]), mm), make_float2(LOG2E, LOG2E));
    const float2 a = make_float2(floored(d.x), floored(d.y));
    const float2 e = make_float2(ex2(a.x), ex2(a.y));
    s = add2(s, e);
    w = fma2(a, e, w);
  }
  t.s += s.x + s.y;
  t.w = w.x + w.y;
}

// a row's log-sum-exp, entropy and log probability from its statistics
template <int DT>
__device__ __forceinline__ void finish_row(const LogpArgs& a, uint64_t row, Stat t) {
  const bool empty = t.m == -INFINITY && t.s == 0.0f;
  // a +inf logit leaves no finite difference: all figures NaN, as for a NaN
  // logit.  x - m first: m + log S alone drops log S beside a large m.
  const float ls = logf(t.s);
  if (a.lse) a.lse[row] = empty ? -INFINITY : t.m + ls;
  if (a.entropy) a.entropy[row] = empty ? 0.0f : fmaf(-t.w * LN2, __fdiv_rn(1.0f, t.s), ls);
  if (a.logp) {
    const uint32_t c = a.targets[row];
    float lp = 0.0f;  // no choice given
    if (c != NO_CHOICE) {
      if (c >= a.cols) {
        dev_raise(a.err, DEVERR_INDEX, c, 60);
        lp = __int_as_float(0x7fc00000);
      } else {
        const bool out = a.mask && a.mask[row * a.ld_mask + c];
        const float x = Elt<DT>::get(static_cast<const elt_t<DT>*>(a.x)[row * a.ld + c]);
        lp = (empty || out) ? -INFINITY : (x - t.m) - ls;
      }
    }
    a.logp[row] = lp;
  }
}
// entry i of a row's list
__device__ __forceinline__ void put_top(const LogpArgs& a, uint64_t row, Stat t, int i, float v,
                                        uint32_t id) {
  const bool some = v > -INFINITY;
  a.top_ids[row * a.top + i] = some ? id : NO_CHOICE;
  a.top_logp[row * a.top + i] = some ? (v - t.m) - logf(t.s) : -INFINITY;
}

// ---- the top list of a block ---------------------------------------------------
constexpr int CANDS = 256;  // candidates that are ranked by counting
struct TopShared {
  float m[LP_WARPS], s[LP_WARPS], w[LP_WARPS];
  float v[CANDS];
  uint32_t id[CANDS];
  uint32_t key[LP_WARPS * 32], low;
  int n, reach;  // candidates; threads that reach the border
};
// a whole number that orders as the float does; 0: nothing
__device__ __forceinline__ uint32_t order_key(float v) {
  if (!(v > -INFINITY)) return 0u;
  const uint32_t b = __float_as_uint(v + 0.0f);  // -0 as +0
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
// A border that at least k of the block's keys reach, and not many more: the
// k-th largest, or its leading bits.  0 when fewer than k keys are not 0.  One
// warp searches (a barrier a bit took three times as long); all threads get it.
__device__ __forceinline__ uint32_t border(TopShared& sm, uint32_t key, int k, int warp, int lane) {
  sm.key[threadIdx.x] = key;
  __syncthreads();
  if (warp == 0) {
    uint32_t q[LP_WARPS];
#pragma unroll
    for (int i = 0; i < LP_WARPS; i++) q[i] = sm.key[i * 32 + lane];
    uint32_t p = 0;
    for (int bit = 31; bit >= 0; bit--) {
      const uint32_t t = p | (1u << bit);
      int c = 0;
#pragma unroll
      for (int i = 0; i < LP_WARPS; i++) c += q[i] >= t;
      c = __reduce_add_sync(0xffffffffu, c);
      if (c >= k) {
        p = t;
        if (c <= k + 8) break;
      }
    }
    if (lane == 0) sm.low = p;
  }
  __syncthreads();
  return sm.low;
}
// appends a candidate a lane; all lanes of the warp call.  (Their order is not
// kept: candidates are ranked.)
__device__ __forceinline__ void add_cands(float* vs, uint32_t* ids, int* count, int most, bool in,
                                          float v, uint32_t id, int lane) {
  const uint32_t b = __ballot_sync(0xffffffffu, in);
  if (b == 0) return;
  int at = 0;
  if (lane == 0) at = atomicAdd(count, __popc(b));
  at = __shfl_sync(0xffffffffu, at, 0) + __popc(b & ((1u << lane) - 1));
  if (in && at < most) vs[at] = v, ids[at] = id;
}
__device__ __forceinline__ void add_cand(TopShared& sm, float v, uint32_t id) {
  const int at = atomicAdd(&sm.n, 1);
  if (at < CANDS) sm.v[at] = v, sm.id[at] = id;
}
// the block's statistics, in every thread
__device__ __forceinline__ Stat block_stat(TopShared& sm, Stat t, int warp, int lane) {
  t = warp_stat(t);
  if (lane == 0) sm.m[warp] = t.m, sm.s[warp] = t.s, sm.w[warp] = t.w;
  __syncthreads();
  t = {sm.m[0], sm.s[0], sm.w[0]};
#pragma unroll
  for (int i = 1; i < LP_WARPS; i++) t = stat_merge(t, {sm.m[i], sm.s[i], sm.w[i]});
  return t;
}
// put(i, v, id) for the list's entries, i ascending over the block's threads
template <class F>
__device__ __forceinline__ void rank_cands(const TopShared& sm, int top, F put) {
  const int n = sm.n;
  for (int i = threadIdx.x; i < n; i += LP_WARPS * 32) {
    const float v = sm.v[i];
    const uint32_t id = sm.id[i];
    int r = 0;
    for (int j = 0; j < n; j++) r += before(sm.v[j], sm.id[j], v, id);
    if (r < top) put(r, v, id);
  }
  for (int i = n + threadIdx.x; i < top; i += LP_WARPS * 32) put(i, -INFINITY, NO_CHOICE);
}
// the warps' sorted lists as one; warp 0 gets it.  Uses sm.v and sm.id.
__device__ __forceinline__ void join_lists(TopShared& sm, TopList& best, int top, int warp,
                                           int lane) {
  static_assert(CANDS == LP_WARPS * TOP_MAX, "a list a warp");
  __syncthreads();
  sm.v[warp * TOP_MAX + lane] = best.v;
  sm.id[warp * TOP_MAX + lane] = best.id;
  __syncthreads();
  if (warp == 0)
    for (int w = 1; w < LP_WARPS; w++)
      best.offer(lane < top ? sm.v[w * TOP_MAX + lane] : -INFINITY,
                 lane < top ? sm.id[w * TOP_MAX + lane] : NO_CHOICE, top, lane);
}

// rows of one segment: block = (row, segment); its warps interleave vectors
template <int DT>
__global__ void __launch_bounds__(LP_WARPS * 32) k_logp(const LogpArgs a) {
  __shared__ TopShared sm;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint64_t row = blockIdx.x / a.splits;
  const uint32_t split = blockIdx.x % a.splits;
  const elt_t<DT>* xr = static_cast<const elt_t<DT>*>(a.x) + row * a.ld;
  const uint8_t* mr = a.mask ? a.mask + row * a.ld_mask : nullptr;
  const int64_t lead = row_lead<DT>(xr);
  const bool mask_vec = mr && (((uintptr_t)mr - (uintptr_t)lead) & 7u) == 0;
  // segments are cut at whole vectors: [lo, hi) in elements of the row
  const int64_t first = (int64_t)split * a.seg - lead;
  const int64_t lo = first > 0 ? first : 0;
  const int64_t end = first + a.seg;
  const int64_t hi = end < (int64_t)a.cols ? end : (int64_t)a.cols;
  constexpr int STEP = LP_WARPS * 256;
  const int64_t mine = first + warp * 256 + lane * 8;  // this thread's vectors: mine + i * STEP
  if (threadIdx.x == 0) sm.n = sm.reach = 0;
  Stat t = {-INFINITY, 0.0f, 0.0f};
  {
    int64_t e = mine;
    if (e < lo) {  // the row starts inside this vector
      float v[8];
      load_left<DT>(xr, mr, mask_vec, e, lo, hi, v);
      stat_add(t, v);
      e += STEP;
    }
    if (!mr) {
      // whole vectors, four loads in flight
      const elt_t<DT>* q = xr + e;
      int64_t left = hi - e;
      for (; left >= 3 * STEP + 8; left -= 4 * STEP, q += 4 * STEP) {
        Vec<DT> r[4];
#pragma unroll
        for (int i = 0; i < 4; i++) r[i] = load_vec<DT>(q + i * STEP);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          float v[8];
          load8<DT>(reinterpret_cast<const elt_t<DT>*>(r[i].w), v);
          stat_add(t, v);
        }
      }
      e = hi - left;
    }
    for (; e < hi; e += STEP) {
      float v[8];
      load_left<DT>(xr, mr, mask_vec, e, lo, hi, v);
      stat_add(t, v);
    }
  }
  const uint32_t key = order_key(t.m);
  t = block_stat(sm, t, warp, lane);
  const uint64_t p = row * a.splits + split;
  auto put = [&](int i, float v, uint32_t id) {
    if (a.splits == 1) {
      put_top(a, row, t, i, v, id);
    } else {
      a.part_v[p * a.top + i] = v;
      a.part_id[p * a.top + i] = id;
    }
  };
  if (a.top) {
    const uint32_t low = border(sm, key, a.top, warp, lane);
    // The threads that reach the border, one a half-warp: its lanes read sixteen
    // of the thread's vectors, and the few elements that reach it are taken.
    if (key >= low && key != 0) sm.key[atomicAdd(&sm.reach, 1)] = threadIdx.x;
    __syncthreads();
    const int reach = sm.reach;
    for (int f = threadIdx.x >> 4; f < reach; f += 2 * LP_WARPS) {
      int64_t e = first + (int64_t)sm.key[f] * 8 + (lane & 15) * STEP;
      for (; e < hi; e += 16 * STEP) {
        float v[8];
        load_left<DT>(xr, mr, mask_vec, e, lo, hi, v);
        float cm = v[0];
#pragma unroll
        for (int j = 1; j < 8; j++) cm = fmaxf(cm, v[j]);
        if (order_key(cm) < low) continue;
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const uint32_t k = order_key(v[j]);
          if (k >= low && k != 0) add_cand(sm, v[j], (uint32_t)(e + j));
        }
      }
    }
    __syncthreads();
    if (sm.n <= CANDS) {
      rank_cands(sm, a.top, put);
    } else {  // hundreds of equal logits: the lists kept while reading
      TopList best;
      for (int64_t b = first + warp * 256; b < hi; b += STEP) {
        const int64_t e = b + lane * 8;
        float v[8];
        load_left<DT>(xr, mr, mask_vec, e, lo, hi, v);
        float cm = v[0];
#pragma unroll
        for (int j = 1; j < 8; j++) cm = fmaxf(cm, v[j]);
        // strictly above: a warp sees its elements in ascending order, so an
        // equal one comes after the one that is listed
        if (__any_sync(0xffffffffu, cm > best.last_v)) {
#pragma unroll
          for (int j = 0; j < 8; j++) best.offer(v[j], (uint32_t)(e + j), a.top, lane);
        }
      }
      join_lists(sm, best, a.top, warp, lane);
      if (warp == 0 && lane < a.top) put(lane, best.v, best.id);
    }
  }
  if (threadIdx.x == 0) {
    if (a.splits == 1) finish_row<DT>(a, row, t);
    else a.part[p] = make_float4(t.m, t.s, t.w, 0.0f);
  }
}

// joins a row's segments: one block a row
template <int DT>
__global__ void __launch_bounds__(LP_WARPS * 32) k_logp_join(const LogpArgs a) {
  __shared__ TopShared sm;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint64_t row = blockIdx.x;
  if (threadIdx.x == 0) sm.n = sm.reach = 0;
  Stat t = {-INFINITY, 0.0f, 0.0f};
  for (uint32_t s = threadIdx.x; s < a.splits; s += LP_WARPS * 32) {
    const float4 p = a.part[row * a.splits + s];
    t = stat_merge(t, {p.x, p.y, p.z});
  }
  t = block_stat(sm, t, warp, lane);
  if (a.top) {
    const uint32_t n = a.splits * (uint32_t)a.top;
    const float* pv = a.part_v + row * n;
    const uint32_t* pi = a.part_id + row * n;
    float m = -INFINITY;
#pragma unroll 8
    for (uint32_t i = threadIdx.x; i < n; i += LP_WARPS * 32) m = fmaxf(m, pv[i]);
    const uint32_t low = border(sm, order_key(m), a.top, warp, lane);
#pragma unroll 8
    for (uint32_t i = threadIdx.x; i < n; i += LP_WARPS * 32) {
      const float v = pv[i];
      const uint32_t k = order_key(v);
      if (k >= low && k != 0) add_cand(sm, v, pi[i]);
    }
    __syncthreads();
    if (sm.n <= CANDS) {
      rank_cands(sm, a.top, [&](int i, float v, uint32_t id) { put_top(a, row, t, i, v, id); });
    } else {
      TopList best;
      for (uint32_t b = warp * 32; b < n; b += LP_WARPS * 32) {
        const bool on = b + lane < n;
        best.offer(on ? pv[b + lane] : -INFINITY, on ? pi[b + lane] : NO_CHOICE, a.top, lane);
      }
      join_lists(sm, best, a.top, warp, lane);
      if (warp == 0 && lane < a.top) put_top(a, row, t, lane, best.v, best.id);
    }
  }
  if (threadIdx.x == 0) finish_row<DT>(a, row, t);
}

// Short rows: a warp a row, the whole row in its registers (E elements a lane,
// element i of lane l being i * 32 + l), so the maximum comes first and nothing
// is rescaled.  The list as in k_logp.  Its border comes from the 32 lane maxima
// for up to FEW_TOP entries; a longer list would take all of them and the border
// let half the row through (8,192 x 1,000 f32, 32 entries: 77 us, 26 with the
// maxima of GROUPS parts of a lane's elements), so that it takes those.
constexpr int SHORT_CANDS = 64;
constexpr int FEW_TOP = 16, GROUPS = 4;
template <int DT, int E>
__global__ void __launch_bounds__(LP_WARPS * 32) k_logp_short(const LogpArgs a) {
  __shared__ float sm_v[LP_WARPS][SHORT_CANDS];
  __shared__ uint32_t sm_id[LP_WARPS][SHORT_CANDS];
  __shared__ int sm_n[LP_WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint64_t step = (uint64_t)gridDim.x * LP_WARPS;
  for (uint64_t row = (uint64_t)blockIdx.x * LP_WARPS + warp; row < a.rows; row += step) {
    const elt_t<DT>* xr = static_cast<const elt_t<DT>*>(a.x) + row * a.ld;
    const uint8_t* mr = a.mask ? a.mask + row * a.ld_mask : nullptr;
    float v[E];
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < E; i++) {
      const uint32_t c = i * 32 + lane;
      v[i] = c < a.cols && !(mr && mr[c]) ? Elt<DT>::get(xr[c]) : -INFINITY;
      m = fmaxf(m, v[i]);
    }
    const uint32_t key = order_key(m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float ms = m == -INFINITY ? 0.0f : m;
    Stat t = {m, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < E; i++) {
      const float q = exponent(v[i] - ms), e = ex2(q);
      t.s += e;
      t.w = fmaf(q, e, t.w);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      t.s += __shfl_xor_sync(0xffffffffu, t.s, o);
      t.w += __shfl_xor_sync(0xffffffffu, t.w, o);
    }
    if (lane == 0) finish_row<DT>(a, row, t);
    if (a.top) {
      uint32_t low = 0;
      auto search = [&](auto reach) {  // reach(q): how many maxima reach q
        for (int bit = 31; bit >= 0; bit--) {
          const uint32_t q = low | (1u << bit);
          const int c = reach(q);
          if (c >= a.top) {
            low = q;
            if (c <= a.top + 4) break;
          }
        }
      };
      if (a.top <= FEW_TOP) {
        search([&](uint32_t q) { return __popc(__ballot_sync(0xffffffffu, key >= q)); });
      } else {
        constexpr int G = E < GROUPS ? E : GROUPS;
        uint32_t keys[G];
#pragma unroll
        for (int g = 0; g < G; g++) {
          float gm = v[g];
#pragma unroll
          for (int i = g + G; i < E; i += G) gm = fmaxf(gm, v[i]);
          keys[g] = order_key(gm);
        }
        search([&](uint32_t q) {
          int c = 0;
#pragma unroll
          for (int i = 0; i < G; i++) c += __popc(__ballot_sync(0xffffffffu, keys[i] >= q));
          return c;
        });
      }
      if (lane == 0) sm_n[warp] = 0;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < E; i++) {
        const uint32_t k = order_key(v[i]);
        add_cands(sm_v[warp], sm_id[warp], &sm_n[warp], SHORT_CANDS, k >= low && k != 0, v[i],
                  i * 32 + lane, lane);
      }
      __syncwarp();
      const int n = sm_n[warp];
      if (n <= SHORT_CANDS) {
        for (int i = lane; i < n; i += 32) {
          const float cv = sm_v[warp][i];
          const uint32_t ci = sm_id[warp][i];
          int r = 0;
          for (int j = 0; j < n; j++) r += before(sm_v[warp][j], sm_id[warp][j], cv, ci);
          if (r < a.top) put_top(a, row, t, r, cv, ci);
        }
        if (lane >= n && lane < a.top) put_top(a, row, t, lane, -INFINITY, NO_CHOICE);
      } else {
        TopList best;
#pragma unroll
        for (int i = 0; i < E; i++) best.offer(v[i], i * 32 + lane, a.top, lane);
        if (lane < a.top) put_top(a, row, t, lane, best.v, best.id);
      }
      __syncwarp();
    }
  }
}

struct LogpBwdArgs {
  const void* x;
  uint64_t ld;
  uint32_t rows, cols;
  const uint8_t* mask;
  uint64_t ld_mask;
  const uint32_t* targets;
  const float* lse;
  const float* entropy;
  const float* g_logp;
  const float* g_ent;  // either may be NULL
  void* dx;            // [rows, cols]
  uint32_t splits, seg;
  int* err;
};

// From |lse| = 128 on, its last bit is worth 2^-17 and more of a probability:
// such a row is summed again.
constexpr float LSE_EXACT = 128.0f;
__device__ __forceinline__ bool far_row(float lse) {
  return fabsf(lse) >= LSE_EXACT && fabsf(lse) < INFINITY;
}
// Every block of a far row needs the sum, and a launch that makes it before costs
// every call 5 to 7 us of the host's time.  So each block sums the row, and where
// a row has many blocks, clusters of this many share that work: 1 x 2.45M f32
// 45 us (each block alone 595), a near row 5.5 (4.8 without clusters; eight
// blocks: 80 and 5.3).
constexpr uint32_t FAR_CLUSTER = 16;
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
// *p of the cluster's block `rank`
__device__ __forceinline__ float cluster_load(const float* p, uint32_t rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(a)
               : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

// two elements' gradients; x -inf: not left, and all of an empty row: none.  log p
// not below -104, where p is 0: gh times a log p near the type's lowest value is
// infinite, and p times that NaN.
__device__ __forceinline__ float2 grad_two(float2 x, float m, float ls, float k0, float gl, float gh,
                                           bool hit0, bool hit1) {
  const float2 d = add2(add2(x, make_float2(-m, -m)), make_float2(-ls, -ls));
  const float2 lp = make_float2(not_below(d.x, -104.0f), not_below(d.y, -104.0f));
  const float2 t = mul2(lp, make_float2(LOG2E, LOG2E));
  const float2 g = mul2(make_float2(ex2(t.x), ex2(t.y)),
                        fma2(make_float2(-gh, -gh), lp, make_float2(k0, k0)));
  return make_float2(x.x == -INFINITY ? 0.0f : hit0 ? g.x + gl : g.x,
                     x.y == -INFINITY ? 0.0f : hit1 ? g.y + gl : g.y);
}
__device__ __forceinline__ float grad_of(float x, float m, float ls, float k0, float gl, float gh,
                                         bool hit) {
  return grad_two(make_float2(x, -INFINITY), m, ls, k0, gl, gh, hit, false).x;
}

// short rows: a warp a row, an element a lane at a time
template <int DT>
__global__ void __launch_bounds__(256) k_logp_bwd_short(const LogpBwdArgs a) {
  const int lane = threadIdx.x & 31;
  const uint64_t step = (uint64_t)gridDim.x * 8;
  for (uint64_t row = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5); row < a.rows; row += step) {
    const elt_t<DT>* xr = static_cast<const elt_t<DT>*>(a.x) + row * a.ld;
    elt_t<DT>* dr = static_cast<elt_t<DT>*>(a.dx) + row * a.cols;
    const uint8_t* mr = a.mask ? a.mask + row * a.ld_mask : nullptr;
    const uint32_t c = a.targets[row];
    if (c != NO_CHOICE && c >= a.cols && lane == 0) dev_raise(a.err, DEVERR_INDEX, c, 61);
    const float gl = a.g_logp && c != NO_CHOICE ? a.g_logp[row] : 0.0f;
    const float gh = a.g_ent ? a.g_ent[row] : 0.0f;
    const float k0 = fmaf(-gh, a.g_ent ? a.entropy[row] : 0.0f, -gl);
    float m = 0.0f, ls = a.lse[row];
    auto at = [&](uint32_t e) {
      return mr && mr[e] ? -INFINITY : Elt<DT>::get(xr[e]);
    };
    if (far_row(ls)) {
      Stat t = {-INFINITY, 0.0f, 0.0f};
      for (uint32_t e = lane; e < a.cols; e += 32) {
        const float x = at(e);
        if (x > -INFINITY) t = stat_merge(t, {x, 1.0f, 0.0f});
      }
      t = warp_stat(t);
      m = t.m;
      ls = logf(t.s);
    }
#pragma unroll 4
    for (uint32_t e = lane; e < a.cols; e += 32)
      dr[e] = Elt<DT>::put(grad_of(at(e), m, ls, k0, gl, gh, e == c));
  }
}

// sum exp(x - lse) over a far row, in every thread of every block of the cluster
// (or of the block, launched without one): the blocks take its vectors in turn,
// and their sums are added in the order of their ranks.
template <int DT>
__device__ __forceinline__ float far_sum(const elt_t<DT>* xr, const uint8_t* mr, bool mask_vec,
                                         int64_t lead, int64_t cols, float lse, float (&sm)[9]) {
  const uint32_t rank = cluster_rank(), size = cluster_size();
  float2 s = make_float2(0.0f, 0.0f);
  const float2 minus = make_float2(-lse, -lse), log2e = make_float2(LOG2E, LOG2E);
  for (int64_t e = (int64_t)(rank * 256 + threadIdx.x) * 8 - lead; e < cols; e += size * 256 * 8) {
    float v[8];
    load_left<DT>(xr, mr, mask_vec, e, 0, cols, v);
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const float2 t = mul2(add2(make_float2(v[j], v[j + 1]), minus), log2e);
      s = add2(s, make_float2(ex2(t.x), ex2(t.y)));
    }
  }
  float t = s.x + s.y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  __syncthreads();  // the last far row's readers
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = t;
  __syncthreads();
  t = sm[0];
  for (int i = 1; i < 8; i++) t += sm[i];
  if (size > 1) {  // far rows are the same for all blocks of a cluster
    if (threadIdx.x == 0) sm[8] = t;
    cluster_sync();
    t = 0.0f;
    for (uint32_t i = 0; i < size; i++) t += cluster_load(&sm[8], i);
    cluster_sync();  // no block goes on to write sm, or leaves, before all have read
  }
  return t;
}

template <int DT>
__global__ void __launch_bounds__(256, 8) k_logp_bwd(const LogpBwdArgs a) {
  __shared__ float sm[9];
  const uint64_t units = (uint64_t)a.rows * a.splits;
  for (uint64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const uint64_t row = u / a.splits;
    const uint32_t split = (uint32_t)(u % a.splits);
    const elt_t<DT>* xr = static_cast<const elt_t<DT>*>(a.x) + row * a.ld;
    elt_t<DT>* dr = static_cast<elt_t<DT>*>(a.dx) + row * a.cols;
    const uint8_t* mr = a.mask ? a.mask + row * a.ld_mask : nullptr;
    const int64_t lead = row_lead<DT>(xr);
    const bool mask_vec = mr && (((uintptr_t)mr - (uintptr_t)lead) & 7u) == 0;
    const bool out_vec = (((uintptr_t)dr - (uintptr_t)lead * sizeof(elt_t<DT>)) & 15u) == 0;
    const int64_t first = (int64_t)split * a.seg - lead;
    const int64_t lo = first > 0 ? first : 0;
    const int64_t end = first + a.seg;
    const int64_t hi = end < (int64_t)a.cols ? end : (int64_t)a.cols;
    const uint32_t c = a.targets[row];
    const float lse = a.lse[row];
    const float gl = a.g_logp && c != NO_CHOICE ? a.g_logp[row] : 0.0f;
    const float gh = a.g_ent ? a.g_ent[row] : 0.0f;
    const float h = a.g_ent ? a.entropy[row] : 0.0f;
    if (c != NO_CHOICE && c >= a.cols && split == 0 && threadIdx.x == 0)
      dev_raise(a.err, DEVERR_INDEX, c, 61);
    const float k0 = fmaf(-gh, h, -gl);
    float m = 0.0f, ls = lse;  // log p = (x - m) - ls
    if (far_row(lse)) {  // log p = (x - lse) - log sum exp(x - lse)
      m = lse;
      ls = logf(far_sum<DT>(xr, mr, mask_vec, lead, a.cols, lse, sm));
    }
    for (int64_t e = first + (int64_t)threadIdx.x * 8; e < hi; e += 256 * 8) {
      float v[8];
      load_left<DT>(xr, mr, mask_vec, e, lo, hi, v);
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float2 d = grad_two(make_float2(v[j], v[j + 1]), m, ls, k0, gl, gh,
                                  e + j == (int64_t)c, e + j + 1 == (int64_t)c);
        v[j] = d.x;
        v[j + 1] = d.y;
      }
      if (out_vec && e >= lo && e + 8 <= hi) {
        store8<DT>(dr + e, v);
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
          if (e + j >= lo && e + j < hi) dr[e + j] = Elt<DT>::put(v[j]);
      }
    }
  }
}

// Segments of a row so that rows * segments fill the GPU's resident blocks;
// a segment keeps at least `least` elements and is whole vectors.
void cut_rows(const bgnn_ctx* ctx, uint32_t rows, uint32_t cols, uint32_t blocks_per_sm,
              uint32_t least, uint32_t* splits, uint32_t* seg) {
  const uint64_t want = (uint64_t)ctx->num_sms * blocks_per_sm;
  uint64_t s = rows >= want ? 1 : want / rows;
  const uint64_t most = ((uint64_t)cols + least - 1) / least;
  if (s > most) s = most;
  if (s < 1) s = 1;
  // + 7: the first vector may start before the row
  uint64_t n = (((uint64_t)cols + 7 + s - 1) / s + 2047) / 2048 * 2048;
  if (s == 1) n = ((uint64_t)cols + 7 + 7) / 8 * 8;
  *seg = (uint32_t)n;
  *splits = (uint32_t)(((uint64_t)cols + 7 + n - 1) / n);
}

constexpr uint32_t LP_SHORT = 1024;  // columns up to which a row takes a warp

template <int DT>
int run_logp(bgnn_ctx* ctx, LogpArgs a) {
  if (a.cols <= LP_SHORT) {
    const uint64_t want = ((uint64_t)a.rows + LP_WARPS - 1) / LP_WARPS;
    const uint64_t cap = (uint64_t)ctx->num_sms * 8;
    const unsigned grid = (unsigned)(want < cap ? want : cap);
    if (a.cols <= 64) k_logp_short<DT, 2><<<grid, LP_WARPS * 32, 0, ctx->stream>>>(a);
    else if (a.cols <= 256) k_logp_short<DT, 8><<<grid, LP_WARPS * 32, 0, ctx->stream>>>(a);
    else if (a.cols <= 512) k_logp_short<DT, 16><<<grid, LP_WARPS * 32, 0, ctx->stream>>>(a);
    else k_logp_short<DT, 32><<<grid, LP_WARPS * 32, 0, ctx->stream>>>(a);
    BGNN_LAUNCHED(ctx);
    return BGNN_OK;
  }
  cut_rows(ctx, a.rows, a.cols, 2, 4096, &a.splits, &a.seg);
  DevTmp ws;
  const uint64_t parts = (uint64_t)a.rows * a.splits;
  if (a.splits > 1) {
    BGNN_TRY(bgnn_tmp_alloc(ctx, ws, parts * (sizeof(float4) + 8 * (uint64_t)a.top)));
    a.part = ws.as<float4>();
    a.part_v = reinterpret_cast<float*>(a.part + parts);
    a.part_id = reinterpret_cast<uint32_t*>(a.part_v + parts * a.top);
  }
  k_logp<DT><<<(unsigned)parts, LP_WARPS * 32, 0, ctx->stream>>>(a);
  BGNN_LAUNCHED(ctx);
  if (a.splits > 1) {
    k_logp_join<DT><<<a.rows, LP_WARPS * 32, 0, ctx->stream>>>(a);
    BGNN_LAUNCHED(ctx);
  }
  return BGNN_OK;
}

template <int DT>
int run_logp_bwd(bgnn_ctx* ctx, LogpBwdArgs a) {
  if (a.cols <= LP_SHORT) {
    const uint64_t want = ((uint64_t)a.rows + 7) / 8, cap = (uint64_t)ctx->num_sms * 16;
    k_logp_bwd_short<DT><<<(unsigned)(want < cap ? want : cap), 256, 0, ctx->stream>>>(a);
    BGNN_LAUNCHED(ctx);
    return BGNN_OK;
  }
  cut_rows(ctx, a.rows, a.cols, 8, 2048, &a.splits, &a.seg);
  const bool clusters = a.splits >= FAR_CLUSTER;
  if (clusters)  // a cluster's blocks work on one row: whole clusters of them (some with nothing)
    a.splits = (a.splits + FAR_CLUSTER - 1) / FAR_CLUSTER * FAR_CLUSTER;
  const uint64_t units = (uint64_t)a.rows * a.splits, cap = (uint64_t)ctx->num_sms * 64;
  if (clusters) {
    static std::atomic<uint64_t> ready{0};  // devices (below 64) where 16 blocks are allowed
    const uint64_t bit = ctx->device < 64 ? 1ull << ctx->device : 0;
    if (!(ready.load(std::memory_order_relaxed) & bit)) {
      BGNN_CUDA(ctx, cudaFuncSetAttribute(k_logp_bwd<DT>,
                                          cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
      ready.fetch_or(bit, std::memory_order_relaxed);
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units < cap ? units : cap));
  cfg.blockDim = dim3(256);
  cfg.stream = ctx->stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = FAR_CLUSTER;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = clusters ? 1 : 0;
  BGNN_CUDA(ctx, cudaLaunchKernelEx(&cfg, k_logp_bwd<DT>, a));
  BGNN_LAUNCHED(ctx);
  return BGNN_OK;
}

}  // namespace

extern "C" int bgnn_log_probs(bgnn_ctx* ctx, int type, const void* logits, uint64_t ld,
                              uint32_t rows, uint32_t cols, const uint8_t* mask, uint64_t ld_mask,
                              const uint32_t* targets, uint32_t top_k, float* logp, float* entropy,
                              float* lse, uint32_t* top_ids, float* top_logp) {
  BGNN_ON_DEVICE(ctx);
  BGNN_REQUIRE(ctx, dtype_float(type), "log_probs: unknown element type %d", type);
  BGNN_REQUIRE_COLS(ctx, "log_probs", cols);
  BGNN_REQUIRE(ctx, top_k <= TOP_MAX, "log_probs: top_k %u above %d", top_k, TOP_MAX);
  if (rows == 0) return BGNN_OK;
  BGNN_REQUIRE(ctx, logits || cols == 0, "log_probs: NULL logits");
  BGNN_REQUIRE(ctx, ld >= cols && (!mask || ld_mask == 0 || ld_mask >= cols),
               "log_probs: row stride below the row length");
  BGNN_REQUIRE(ctx, !logp || targets, "log_probs: logp needs targets");
  BGNN_REQUIRE(ctx, top_k == 0 || (top_ids && top_logp), "log_probs: NULL top list");
  LogpArgs a = {};
  a.x = logits;
  a.ld = ld;
  a.rows = rows;
  a.cols = cols;
  a.mask = cols ? mask : nullptr;
  a.ld_mask = ld_mask;
  a.targets = targets;
  a.top = (int)top_k;
  a.logp = logp;
  a.entropy = entropy;
  a.lse = lse;
  a.top_ids = top_ids;
  a.top_logp = top_logp;
  a.err = ctx->d_err;
  switch (type) {
    case BGNN_F32: return run_logp<BGNN_F32>(ctx, a);
    case BGNN_BF16: return run_logp<BGNN_BF16>(ctx, a);
    default: return run_logp<BGNN_F16>(ctx, a);
  }
}

extern "C" int bgnn_log_probs_backward(bgnn_ctx* ctx, int type, const void* logits, uint64_t ld,
                                       uint32_t rows, uint32_t cols, const uint8_t* mask,
                                       uint64_t ld_mask, const uint32_t* targets, const float* lse,
                                       const float* entropy, const float* grad_logp,
                                       const float* grad_entropy, void* grad_logits) {
  BGNN_ON_DEVICE(ctx);
  BGNN_REQUIRE(ctx, dtype_float(type), "log_probs_backward: unknown element type %d", type);
  BGNN_REQUIRE_COLS(ctx, "log_probs_backward", cols);
  if (rows == 0 || cols == 0) return BGNN_OK;
  BGNN_REQUIRE(ctx, logits && targets && lse && grad_logits, "log_probs_backward: NULL argument");
  BGNN_REQUIRE(ctx, !grad_entropy || entropy, "log_probs_backward: grad_entropy needs the entropy");
  BGNN_REQUIRE(ctx, ld >= cols && (!mask || ld_mask == 0 || ld_mask >= cols),
               "log_probs_backward: row stride below the row length");
  LogpBwdArgs a = {};
  a.x = logits;
  a.ld = ld;
  a.rows = rows;
  a.cols = cols;
  a.mask = mask;
  a.ld_mask = ld_mask;
  a.targets = targets;
  a.lse = lse;
  a.entropy = entropy;
  a.g_logp = grad_logp;
  a.g_ent = grad_entropy;
  a.dx = grad_logits;
  a.err = ctx->d_err;
  switch (type) {
    case BGNN_F32: return run_logp_bwd<BGNN_F32>(ctx, a);
    case BGNN_BF16: return run_logp_bwd<BGNN_BF16>(ctx, a);
    default: return run_logp_bwd<BGNN_F16>(ctx, a);
  }
}
