// Dense products of 16-bit and 8-bit operands on the 5th-generation tensor
// cores, each with its epilogue in the same kernel:
//
//   linear   out = act(x w^T + b) + residual
//   gated    out = act(x wg^T + bg) * (x wu^T + bu)
//   and their backward passes, which keep nothing of the forward:
//     dz = g act'(z)                     z = x w^T + b, once more
//     dg = g u act'(zg), du = g act(zg)  zg, u once more, one kernel
//     dx = dz w (dg wg + du wu as one product over both),  dw = dz^T x,
//     db = column sums of dz
//
// Operands are bf16 or f16, or e4m3 with one f32 scale a row of x and of w
// (then z = xs_i ws_j sum_k x_ik w_jk).  Products accumulate in f32 in tensor
// memory; bias, activation, product and residual are f32 and the result is
// rounded once.  dz (dg, du) is rounded to the operands' type once, because
// the two products that follow take it as an operand.
//
// Kernel: persistent, one CTA an SM, 128 x BN output tiles, warp-specialised:
//   warp 8    TMA producer: per k block (128 bytes of k) the A tile and the B
//             tile into a ring of shared-memory stages, 128-byte swizzle;
//   warp 9    MMA issuer (one thread): tcgen05.mma, M = 128, N = BN, into one
//             of two tensor-memory accumulators;
//   warps 0-7 epilogue: warp w takes the accumulator lanes (rows) of its
//             quadrant w % 4 and every other 32-column chunk, and turns them
//             round through shared memory so that global reads and writes
//             run along rows.
// An operand whose contraction runs down its rows (w in dx, both in dw) is
// read as it lies ("MN-major": boxes of 64 columns x 64 rows), never
// transposed in memory.  The gated kernels load BN/2 rows of each weight side
// by side into the B tile, so one accumulator holds both halves.
// dw sums over all rows of x: a long axis with few output tiles.  It is cut
// into `splits` ranges whose f32 partial tiles are added in a fixed order.
//
// Every mbarrier wait is bounded: one that gives up raises the context's
// error word (BGNN_ERR_TIMEOUT at the next synchronisation) and tells the
// other roles; copies and products still in flight are waited for (bounded)
// before tensor memory is freed.  TMA loads use no multicast and read only
// this GPU's memory.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "lowp.cuh"

namespace {

constexpr int BM = 128;
constexpr int EPI_WARPS = 8;
constexpr int THREADS = (EPI_WARPS + 2) * 32;
constexpr int MAX_STAGES = 8;
constexpr int A_BYTES = BM * 128;
constexpr int TURN_BYTES = 32 * 32 * 4;  // an epilogue warp's turning buffer
constexpr int RING_BYTES = 192 * 1024;
constexpr int SMEM_BYTES = 1024 + RING_BYTES + EPI_WARPS * TURN_BYTES + 512;
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory of one SM");
constexpr uint32_t SPIN_LIMIT = 1u << 24;     // polls before a wait gives up,
constexpr uint64_t SPIN_NS = 2000000000ull;  // or this long

enum Epi : int { EPI_LINEAR, EPI_GATED, EPI_LINEAR_BWD, EPI_GATED_BWD, EPI_PARTIAL };

// One contraction segment: A [m, k] and B [n, k] tiles of one or two tensors.
// Where `b1` is used (gated), B's tile is rows of b0 above rows of b1.
struct Maps {
  CUtensorMap a[2], b[2];
};

struct GemmArgs {
  uint32_t m, n;          // output size (gated: n columns of h, 2n of the product)
  uint32_t bn;            // columns of a tile in tensor memory: 32, 64, 128, 256
  uint32_t stages, stage_bytes;
  uint32_t nkb[2];        // k blocks of each segment (0: no second segment)
  uint32_t batches;       // dw: products that share B (dg^T x, du^T x)
  uint32_t splits, per;   // dw: ranges of the contraction, k blocks in each
  uint32_t idesc;
  int fp8;
  int a_mn, b_mn;         // MN-major operands
  int in_type;
  // epilogue
  const float* x_scale;   // [m] or NULL
  const float* w_scale[2];  // [n] or NULL
  const void* bias[2];    // [n] or NULL
  int bias_type;
  int act;
  float act_p;
  const void* other;      // residual (linear) or the upstream gradient (backward)
  int other_type;
  uint64_t ld_other;
  int out_type;
  void* out[2];           // gated backward: dg and du; dw: one a batch
  uint64_t ld_out;
  float* part;            // EPI_PARTIAL: [splits, batches, m, n]
  int* err;
};

// ---- PTX ---------------------------------------------------------------------
__device__ __forceinline__ uint32_t s_addr(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void mbar_init(uint32_t a, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(a), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t a, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(a), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t a) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(a) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t a, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(a), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ uint64_t now_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
// bounded wait; false when it gave up or another role already did
__device__ __forceinline__ bool mbar_wait(uint32_t a, uint32_t parity, volatile uint32_t* abort_flag,
                                          int* err, int where) {
  if (mbar_try(a, parity)) return true;
  const uint64_t t0 = now_ns();
  for (uint32_t i = 0; i < SPIN_LIMIT; i++) {
    if (mbar_try(a, parity)) return true;
    if (*abort_flag) return false;
    if ((i & 63u) == 63u && now_ns() - t0 > SPIN_NS) break;
  }
  *abort_flag = 1u;
  dev_raise(err, DEVERR_TIMEOUT, (uint64_t)blockIdx.x, where);
  return false;
}
// for what is in flight when a role has given up
__device__ __forceinline__ void mbar_drain(uint32_t a, uint32_t parity) {
  const uint64_t t0 = now_ns();
  for (uint32_t i = 0; i < SPIN_LIMIT; i++)
    if (mbar_try(a, parity) || now_ns() - t0 > SPIN_NS / 4) return;
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y,
                                            uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// Shared-memory matrix descriptor, 128-byte swizzle, version 1.  Eight-row
// groups (K-major: 8 rows of m or n; MN-major: 8 rows of k) are 1024 bytes
// apart; in an MN-major tile the next 64 columns start after all 64 rows.
__device__ __forceinline__ uint64_t smem_desc(uint32_t a, int mn_major) {
  return (uint64_t)((a & 0x3FFFFu) >> 4) | ((uint64_t)(mn_major ? 8192 >> 4 : 1) << 16) |
         ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   bar)
               : "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
// 32 columns of this warp's 32 lanes
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int j = 0; j < 32; j++) v[j] = __uint_as_float(r[j]);
}

// ---- activations, f32 ----------------------------------------------------------
__device__ __forceinline__ float sigmoid_f(float z) { return __fdividef(1.0f, 1.0f + __expf(-z)); }
constexpr float GELU_C = 0.7978845608028654f;  // sqrt(2/pi)
__device__ __forceinline__ float gelu_arg(float z) {
  return GELU_C * z * fmaf(0.044715f * z, z, 1.0f);
}
__device__ __forceinline__ float act_f(float z, int act, float p) {
  switch (act) {
    case BGNN_ACT_RELU: return z > 0.0f ? z : 0.0f;
    case BGNN_ACT_RELU_MAX: return z != z ? z : (z > 0.0f ? z : 0.0f);
    case BGNN_ACT_ELU: return z > 0.0f ? z : p * expm1f(z);
    case BGNN_ACT_LEAKY_RELU: return z > 0.0f ? z : p * z;
    case BGNN_ACT_SIGMOID: return sigmoid_f(z);
    case BGNN_ACT_TANH: return tanhf(z);
    case BGNN_ACT_GELU: return z * sigmoid_f(2.0f * gelu_arg(z));  // 0.5 (1 + tanh v)
    case BGNN_ACT_SILU: return z * sigmoid_f(z);
    default: return z;
  }
}
// act(z) and act'(z)
__device__ __forceinline__ float2 act_both(float z, int act, float p) {
  switch (act) {
    case BGNN_ACT_RELU: return z > 0.0f ? make_float2(z, 1.0f) : make_float2(0.0f, 0.0f);
    case BGNN_ACT_RELU_MAX:
      return z != z ? make_float2(z, z) : z > 0.0f ? make_float2(z, 1.0f) : make_float2(0.0f, 0.0f);
    case BGNN_ACT_ELU: {
      const float e = p * expm1f(z);
      return z > 0.0f ? make_float2(z, 1.0f) : make_float2(e, e + p);
    }
    case BGNN_ACT_LEAKY_RELU: return z > 0.0f ? make_float2(z, 1.0f) : make_float2(p * z, p);
    case BGNN_ACT_SIGMOID: {
      const float s = sigmoid_f(z);
      return make_float2(s, s * sigmoid_f(-z));
    }
    case BGNN_ACT_TANH: {
      const float t = tanhf(z);
      return make_float2(t, (1.0f - t) * (1.0f + t));
    }
    case BGNN_ACT_GELU: {
      const float s = sigmoid_f(2.0f * gelu_arg(z));
      const float dv = 2.0f * GELU_C * fmaf(3.0f * 0.044715f * z, z, 1.0f);
      // far out s is 0 or 1 and z (1 - s) 0, whatever dv is
      const float q = s * (1.0f - s);
      return make_float2(z * s, q == 0.0f ? s : fmaf(z * q, dv, s));
    }
    case BGNN_ACT_SILU: {
      const float s = sigmoid_f(z);
      return make_float2(z * s, s * fmaf(z, 1.0f - s, 1.0f));
    }
    default: return make_float2(z, 1.0f);
  }
}

// ---- the turning buffer: 32 rows x 32 f32, 16-byte units swizzled by row --------
__device__ __forceinline__ float4* turn_unit(float* t, int row, int unit) {
  return reinterpret_cast<float4*>(t + row * 32 + ((unit ^ (row & 7)) << 2));
}
__device__ __forceinline__ void turn_put_row(float* t, int row, const float (&v)[32]) {
#pragma unroll
  for (int u = 0; u < 8; u++)
    *turn_unit(t, row, u) = make_float4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
}

// four consecutive elements along a row, or those of them that exist
__device__ __forceinline__ float4 load4_row(const void* p, int dt, uint64_t i, uint32_t left,
                                            bool vec) {
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (vec && left >= 4) {
    if (dt == BGNN_F32) return *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
    if (dt == BGNN_BF16)
      return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u),
                         __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    return make_float4(a.x, a.y, b.x, b.y);
  }
  if (left > 0) v.x = load_any(p, dt, i);
  if (left > 1) v.y = load_any(p, dt, i + 1);
  if (left > 2) v.z = load_any(p, dt, i + 2);
  if (left > 3) v.w = load_any(p, dt, i + 3);
  return v;
}
__device__ __forceinline__ void store4_row(void* p, int dt, uint64_t i, uint32_t left, bool vec,
                                           float4 v) {
  if (vec && left >= 4) {
    if (dt == BGNN_F32) {
      *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = v;
    } else {
      const uint2 w = dt == BGNN_BF16
                          ? make_uint2(pack2<BGNN_BF16>(v.x, v.y), pack2<BGNN_BF16>(v.z, v.w))
                          : make_uint2(pack2<BGNN_F16>(v.x, v.y), pack2<BGNN_F16>(v.z, v.w));
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) = w;
    }
    return;
  }
  if (left > 0) store_any(p, dt, i, v.x);
  if (left > 1) store_any(p, dt, i + 1, v.y);
  if (left > 2) store_any(p, dt, i + 2, v.z);
  if (left > 3) store_any(p, dt, i + 3, v.w);
}
// whether four elements at (row stride ld, column a multiple of 4) are one access
__device__ __forceinline__ bool vec4_ok(const void* p, int dt, uint64_t ld) {
  const uint32_t b = dt == BGNN_F32 ? 16u : 8u;
  return ((uintptr_t)p & (b - 1)) == 0 && ld % 4 == 0;
}

// what a tile index stands for
struct Tile {
  uint32_t m0, n0, batch, split;
};
template <int EPI>
__device__ __forceinline__ Tile tile_at(const GemmArgs& g, uint64_t t, uint32_t n_tiles,
                                        uint32_t m_tiles, uint32_t wn) {
  Tile r;
  const uint64_t q = t / n_tiles;
  r.n0 = (uint32_t)(t % n_tiles) * wn;
  r.m0 = (uint32_t)(q % m_tiles) * BM;
  const uint32_t z = (uint32_t)(q / m_tiles);
  r.batch = EPI == EPI_PARTIAL ? z % g.batches : 0;
  r.split = EPI == EPI_PARTIAL ? z / g.batches : 0;
  return r;
}

template <int EPI>
__global__ void __launch_bounds__(THREADS, 1)
    k_dense16(const __grid_constant__ Maps maps, const GemmArgs g) {
  constexpr bool TWO = EPI == EPI_GATED || EPI == EPI_GATED_BWD;  // B tile of two weights
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = s_addr(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;  // swizzle atoms start on 1024 bytes
  uint8_t* gbase = smem_raw + (base - raw);
  float* turns = reinterpret_cast<float*>(gbase + RING_BYTES);
  uint64_t* bars = reinterpret_cast<uint64_t*>(gbase + RING_BYTES + EPI_WARPS * TURN_BYTES);
  const uint32_t b_full = s_addr(bars), b_empty = b_full + 8 * MAX_STAGES;
  const uint32_t b_accf = b_empty + 8 * MAX_STAGES, b_acce = b_accf + 16, b_last = b_acce + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * MAX_STAGES + 5);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t S = g.stages;
  const uint32_t tmem_cols = 2 * g.bn < 32 ? 32 : 2 * g.bn;

  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < S; s++) {
      mbar_init(b_full + 8 * s, 1);
      mbar_init(b_empty + 8 * s, 1);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(b_accf + 8 * b, 1);
      mbar_init(b_acce + 8 * b, EPI_WARPS * 32);
    }
    mbar_init(b_last, 1);
    *abort_flag = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == EPI_WARPS) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     s_addr(tmem_slot)),
                 "r"(tmem_cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const uint32_t wn = TWO ? g.bn / 2 : g.bn;  // output columns of a tile
  const uint32_t m_tiles = (g.m + BM - 1) / BM, n_tiles = (g.n + wn - 1) / wn;
  const uint64_t tiles = (uint64_t)m_tiles * n_tiles *
                         (EPI == EPI_PARTIAL ? (uint64_t)g.batches * g.splits : 1ull);
  const uint32_t nkb = g.nkb[0] + g.nkb[1];
  // k blocks [first, last) of a tile
  auto kb_first = [&](const Tile& t) { return EPI == EPI_PARTIAL ? t.split * g.per : 0u; };
  auto kb_last = [&](const Tile& t) {
    if (EPI != EPI_PARTIAL) return nkb;
    const uint32_t e = (t.split + 1) * g.per;
    return e < nkb ? e : nkb;
  };

  if (warp == EPI_WARPS) {
    // ---- TMA producer ----
    if (lane == 0) {
      uint32_t s = 0, ph = 0;
      uint64_t filled = 0;
      const uint32_t tx = A_BYTES + g.bn * 128;
      const int kw = g.fp8 ? 128 : 64;  // elements of a k block
      for (uint64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const Tile ti = tile_at<EPI>(g, t, n_tiles, m_tiles, wn);
        const uint32_t e = kb_last(ti);
        for (uint32_t kb = kb_first(ti); kb < e; kb++) {
          if (!mbar_wait(b_empty + 8 * s, ph ^ 1u, abort_flag, g.err, 70)) goto drain;
          mbar_expect_tx(b_full + 8 * s, tx);
          const int seg = EPI == EPI_PARTIAL ? (int)ti.batch : (kb >= g.nkb[0] ? 1 : 0);
          const int k0 = (int)((EPI != EPI_PARTIAL && seg ? kb - g.nkb[0] : kb)) * kw;
          const uint32_t st = base + s * g.stage_bytes, bar = b_full + 8 * s;
          if (g.a_mn) {
            for (int i = 0; i < BM / 64; i++)
              tma_load_2d(st + i * 8192, &maps.a[seg], (int)ti.m0 + i * 64, k0, bar);
          } else {
            tma_load_2d(st, &maps.a[seg], k0, (int)ti.m0, bar);
          }
          if (TWO) {
            tma_load_2d(st + A_BYTES, &maps.b[0], k0, (int)ti.n0, bar);
            tma_load_2d(st + A_BYTES + wn * 128, &maps.b[1], k0, (int)ti.n0, bar);
          } else if (g.b_mn) {
            const CUtensorMap* mb = EPI == EPI_PARTIAL ? &maps.b[0] : &maps.b[seg];
            for (uint32_t i = 0; i < g.bn / 64; i++)
              tma_load_2d(st + A_BYTES + i * 8192, mb, (int)(ti.n0 + i * 64), k0, bar);
          } else {
            tma_load_2d(st + A_BYTES, &maps.b[seg], k0, (int)ti.n0, bar);
          }
          filled++;
          if (++s == S) s = 0, ph ^= 1u;
        }
      }
    drain:
      if (*abort_flag)  // the last fill of every stage lands before the CTA ends
        for (uint64_t f = filled > S ? filled - S : 0; f < filled; f++)
          mbar_drain(b_full + 8 * (uint32_t)(f % S), (uint32_t)((f / S) & 1u));
    }
  } else if (warp == EPI_WARPS + 1) {
    // ---- MMA issuer ----
    if (lane == 0) {
      uint32_t s = 0, ph = 0, buf = 0, aph = 0;
      const uint32_t step_a = g.a_mn ? 2048u : 32u, step_b = g.b_mn ? 2048u : 32u;
      for (uint64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const Tile ti = tile_at<EPI>(g, t, n_tiles, m_tiles, wn);
        const uint32_t f = kb_first(ti), e = kb_last(ti);
        if (!mbar_wait(b_acce + 8 * buf, aph ^ 1u, abort_flag, g.err, 71)) break;
        tc_fence_after();
        const uint32_t d = tmem + buf * g.bn;
        bool gave_up = false;
        for (uint32_t kb = f; kb < e; kb++) {
          if (!mbar_wait(b_full + 8 * s, ph, abort_flag, g.err, 72)) {
            gave_up = true;
            break;
          }
          tc_fence_after();
          const uint32_t st = base + s * g.stage_bytes;
#pragma unroll
          for (uint32_t kk = 0; kk < 4; kk++) {
            const uint64_t da = smem_desc(st + kk * step_a, g.a_mn);
            const uint64_t db = smem_desc(st + A_BYTES + kk * step_b, g.b_mn);
            const uint32_t acc = (kb != f || kk != 0) ? 1u : 0u;
            if (g.fp8) mma_f8(d, da, db, g.idesc, acc);
            else mma_f16(d, da, db, g.idesc, acc);
          }
          mma_commit(b_empty + 8 * s);
          if (++s == S) s = 0, ph ^= 1u;
        }
        if (gave_up) break;
        mma_commit(b_accf + 8 * buf);
        if (++buf == 2) buf = 0, aph ^= 1u;
      }
      // every product issued is done before tensor memory is freed
      mma_commit(b_last);
      mbar_drain(b_last, 0);
    }
  } else {
    // ---- epilogue ----
    const int quad = warp & 3, half = warp >> 2;
    float* turn = turns + warp * (TURN_BYTES / 4);
    uint32_t buf = 0, aph = 0;
    const bool vec_out = EPI == EPI_PARTIAL ? g.n % 4 == 0
                                            : vec4_ok(g.out[0], g.out_type, g.ld_out) &&
                                                  (EPI != EPI_GATED_BWD ||
                                                   vec4_ok(g.out[1], g.out_type, g.ld_out));
    const bool vec_other = g.other && vec4_ok(g.other, g.other_type, g.ld_other);
    for (uint64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
      const Tile ti = tile_at<EPI>(g, t, n_tiles, m_tiles, wn);
      const bool any_k = kb_first(ti) < kb_last(ti);
      if (!mbar_wait(b_accf + 8 * buf, aph, abort_flag, g.err, 73)) break;
      tc_fence_after();
      const uint32_t acc = tmem + ((uint32_t)(quad * 32) << 16) + buf * g.bn;
      const uint32_t row0 = ti.m0 + quad * 32;  // this warp's rows
      const float xs = g.x_scale && row0 + lane < g.m ? g.x_scale[row0 + lane] : 1.0f;
      for (uint32_t c = half * 32; c < wn; c += 64) {
        const uint32_t col0 = ti.n0 + c;
        if (col0 >= g.n) break;  // uniform: the chunk is past the last column
        float v[32];
        tmem_ld32(acc + c, v);
        if (!any_k) {
#pragma unroll
          for (int j = 0; j < 32; j++) v[j] = 0.0f;
        }
        if constexpr (EPI != EPI_PARTIAL) {
          if (g.x_scale) {
#pragma unroll
            for (int j = 0; j < 32; j++)
              v[j] *= xs * (col0 + j < g.n ? g.w_scale[0][col0 + j] : 0.0f);
          }
          if (g.bias[0]) {
#pragma unroll
            for (int j = 0; j < 32; j++)
              if (col0 + j < g.n) v[j] += load_any(g.bias[0], g.bias_type, col0 + j);
          }
        }
        // the upstream gradient of this chunk, read along rows
        auto other_rows = [&](float (&o)[32]) {
          __syncwarp();
          for (int i = 0; i < 8; i++) {
            const int r = i * 4 + (lane >> 3), u = lane & 7;
            const uint32_t row = row0 + r, col = col0 + u * 4;
            float4 w = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (row < g.m && col < g.n)
              w = load4_row(g.other, g.other_type, (uint64_t)row * g.ld_other + col, g.n - col,
                            vec_other);
            *turn_unit(turn, r, u) = w;
          }
          __syncwarp();
#pragma unroll
          for (int u = 0; u < 8; u++) {
            const float4 w = *turn_unit(turn, lane, u);
            o[4 * u] = w.x, o[4 * u + 1] = w.y, o[4 * u + 2] = w.z, o[4 * u + 3] = w.w;
          }
        };
        // v (a row a lane) out along rows; with_other: add the residual on the way
        auto rows_out = [&](void* out, int out_type, uint64_t ld, bool with_other) {
          __syncwarp();
          turn_put_row(turn, lane, v);
          __syncwarp();
          for (int i = 0; i < 8; i++) {
            const int r = i * 4 + (lane >> 3), u = lane & 7;
            const uint32_t row = row0 + r, col = col0 + u * 4;
            if (row < g.m && col < g.n) {
              float4 w = *turn_unit(turn, r, u);
              if (with_other) {
                const float4 q = load4_row(g.other, g.other_type,
                                           (uint64_t)row * g.ld_other + col, g.n - col, vec_other);
                w.x += q.x, w.y += q.y, w.z += q.z, w.w += q.w;
              }
              store4_row(out, out_type, (uint64_t)row * ld + col, g.n - col, vec_out, w);
            }
          }
        };
        if constexpr (EPI == EPI_LINEAR) {
          if (g.act != BGNN_ACT_NONE) {
#pragma unroll
            for (int j = 0; j < 32; j++) v[j] = act_f(v[j], g.act, g.act_p);
          }
          rows_out(g.out[0], g.out_type, g.ld_out, g.other != nullptr);
        } else if constexpr (EPI == EPI_PARTIAL) {
          rows_out(g.part + ((uint64_t)ti.split * g.batches + ti.batch) * g.m * g.n, BGNN_F32, g.n,
                   false);
        } else if constexpr (EPI == EPI_LINEAR_BWD) {
          float o[32];
          other_rows(o);
#pragma unroll
          for (int j = 0; j < 32; j++) v[j] = o[j] * act_both(v[j], g.act, g.act_p).y;
          rows_out(g.out[0], g.out_type, g.ld_out, false);
        } else {
          float u[32];
          tmem_ld32(acc + wn + c, u);
          if (!any_k) {
#pragma unroll
            for (int j = 0; j < 32; j++) u[j] = 0.0f;
          }
          if (g.x_scale) {
#pragma unroll
            for (int j = 0; j < 32; j++)
              u[j] *= xs * (col0 + j < g.n ? g.w_scale[1][col0 + j] : 0.0f);
          }
          if (g.bias[1]) {
#pragma unroll
            for (int j = 0; j < 32; j++)
              if (col0 + j < g.n) u[j] += load_any(g.bias[1], g.bias_type, col0 + j);
          }
          if constexpr (EPI == EPI_GATED) {
#pragma unroll
            for (int j = 0; j < 32; j++) v[j] = act_f(v[j], g.act, g.act_p) * u[j];
            rows_out(g.out[0], g.out_type, g.ld_out, false);
          } else {
            float o[32];
            other_rows(o);
#pragma unroll
            for (int j = 0; j < 32; j++) {
              const float2 f = act_both(v[j], g.act, g.act_p);
              v[j] = o[j] * u[j] * f.y;  // dg
              u[j] = o[j] * f.x;         // du
            }
            rows_out(g.out[0], g.out_type, g.ld_out, false);
#pragma unroll
            for (int j = 0; j < 32; j++) v[j] = u[j];
            rows_out(g.out[1], g.out_type, g.ld_out, false);
          }
        }
      }
      tc_fence_before();
      mbar_arrive(b_acce + 8 * buf);
      if (++buf == 2) buf = 0, aph ^= 1u;
    }
  }
  __syncthreads();
  if (warp == EPI_WARPS) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_cols)
                 : "memory");
  }
}

// dw: the splits' partial tiles added in order
__global__ void __launch_bounds__(256) k_add_splits(const float* __restrict__ part,
                                                    uint32_t splits, uint32_t batches, uint64_t mn,
                                                    void* out0, void* out1, int out_type) {
  const uint64_t total = mn * batches;
  for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (uint64_t)gridDim.x * blockDim.x) {
    float v = part[i];
    for (uint32_t s = 1; s < splits; s++) v += part[(uint64_t)s * total + i];
    store_any(i < mn ? out0 : out1, out_type, i < mn ? i : i - mn, v);
  }
}

// column sums of a [rows, cols] matrix over blockIdx.y's share of the rows
__global__ void __launch_bounds__(256) k_col_sums(const void* __restrict__ x, int dt, uint64_t ld,
                                                  uint64_t rows, uint32_t cols,
                                                  float* __restrict__ part) {
  __shared__ float s[8][33];
  const int lane = threadIdx.x & 31, ch = threadIdx.x >> 5;
  const uint32_t c = blockIdx.x * 32 + lane;
  float v = 0.0f;
  if (c < cols)
    for (uint64_t r = (uint64_t)blockIdx.y * 8 + ch; r < rows; r += (uint64_t)gridDim.y * 8)
      v += load_any(x, dt, r * ld + c);
  s[ch][lane] = v;
  __syncthreads();
  if (ch == 0 && c < cols) {
#pragma unroll
    for (int i = 1; i < 8; i++) v += s[i][lane];
    part[(uint64_t)blockIdx.y * cols + c] = v;
  }
}

// rows copied to a row stride that TMA takes (a multiple of 16 bytes)
template <class T>
__global__ void __launch_bounds__(256) k_repack(const T* __restrict__ x, uint64_t ld, uint64_t rows,
                                                uint32_t cols, uint32_t ldp, T* __restrict__ out) {
  const uint64_t total = rows * ldp;
  for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (uint64_t)gridDim.x * blockDim.x) {
    const uint64_t r = i / ldp;
    const uint32_t c = (uint32_t)(i - r * ldp);
    out[i] = c < cols ? x[r * ld + c] : T(0);
  }
}

// ---- host side -------------------------------------------------------------------
PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// a [rows, cols] matrix of 16- or 8-bit elements, rows ld apart
struct Mat {
  const void* p;
  uint64_t rows;
  uint32_t cols;
  uint64_t ld;
};

// boxes of 128 bytes x box_rows, 128-byte swizzle, zeros outside the matrix
int make_map(bgnn_ctx* ctx, CUtensorMap* map, int type, const Mat& x, uint32_t box_rows) {
  auto enc = encode_fn();
  if (!enc) return bgnn_set_error(ctx, BGNN_ERR_UNSUPPORTED, "cuTensorMapEncodeTiled unavailable");
  const uint32_t es = (uint32_t)dtype_size(type);
  cuuint64_t dims[2] = {x.cols, x.rows};
  cuuint64_t strides[1] = {x.ld * es};
  cuuint32_t box[2] = {128 / es, box_rows};
  cuuint32_t el[2] = {1, 1};
  const CUtensorMapDataType dt = type == BGNN_BF16  ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                 : type == BGNN_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                    : CU_TENSOR_MAP_DATA_TYPE_UINT8;
  const CUresult r = enc(map, dt, 2, const_cast<void*>(x.p), dims, strides, box, el,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return bgnn_set_error(ctx, BGNN_ERR_UNSUPPORTED, "tensor map encode failed (%d)", (int)r);
  return BGNN_OK;
}

// x as TMA can read it: itself, or a copy whose rows start on 16 bytes
int tma_ready(bgnn_ctx* ctx, int type, Mat* x, DevTmp& tmp) {
  const uint32_t es = (uint32_t)dtype_size(type);
  if (((uintptr_t)x->p & 15u) == 0 && (x->ld * es) % 16 == 0 && x->ld * es < (1ull << 40))
    return BGNN_OK;
  const uint32_t per = 16 / es;
  const uint32_t ldp = (x->cols + per - 1) / per * per;
  BGNN_TRY(bgnn_tmp_alloc(ctx, tmp, x->rows * (uint64_t)ldp * es));
  const uint64_t total = x->rows * (uint64_t)ldp, cap = (uint64_t)ctx->num_sms * 16;
  const uint64_t want = (total + 255) / 256;
  const unsigned grid = (unsigned)(want < cap ? want : cap);
  if (es == 2)
    k_repack<uint16_t><<<grid, 256, 0, ctx->stream>>>(static_cast<const uint16_t*>(x->p), x->ld,
                                                       x->rows, x->cols, ldp, tmp.as<uint16_t>());
  else
    k_repack<uint8_t><<<grid, 256, 0, ctx->stream>>>(static_cast<const uint8_t*>(x->p), x->ld,
                                                      x->rows, x->cols, ldp, tmp.as<uint8_t>());
  BGNN_LAUNCHED(ctx);
  x->p = tmp.p;
  x->ld = ldp;
  return BGNN_OK;
}

uint32_t blocks_of(uint64_t len, uint32_t per) { return (uint32_t)((len + per - 1) / per); }

// Tile width: the widest that still gives every SM a tile, since a wide tile
// reads A fewer times; a narrow output takes the narrowest that covers it.
uint32_t pick_bn(const bgnn_ctx* ctx, uint64_t m, uint64_t n, uint64_t z, bool two, uint32_t least) {
  uint32_t bn = 256;
  while (bn > least) {
    const uint64_t wn = two ? bn / 2 : bn;
    const uint64_t tiles = ((m + BM - 1) / BM) * ((n + wn - 1) / wn) * z;
    if (tiles >= (uint64_t)ctx->num_sms && n > wn / 2) break;
    bn /= 2;
  }
  return bn;
}

void set_tile(GemmArgs* g, uint32_t bn) {
  g->bn = bn;
  g->stage_bytes = A_BYTES + bn * 128;
  g->stages = RING_BYTES / g->stage_bytes;
  if (g->stages > MAX_STAGES) g->stages = MAX_STAGES;
}

// instruction descriptor: D f32, A and B of one type, majorness, N, M = 128
uint32_t make_idesc(int type, int a_mn, int b_mn, uint32_t bn) {
  const uint32_t f = type == BGNN_BF16 ? 1u : 0u;  // kind::f16: 0 f16, 1 bf16; f8f6f4: 0 e4m3
  return (1u << 4) | (f << 7) | (f << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         ((bn >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
}

template <int EPI>
int launch(bgnn_ctx* ctx, const Maps& maps, GemmArgs& g) {
  constexpr bool TWO = EPI == EPI_GATED || EPI == EPI_GATED_BWD;
  BGNN_CUDA(ctx, cudaFuncSetAttribute(k_dense16<EPI>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      SMEM_BYTES));
  g.idesc = make_idesc(g.in_type, g.a_mn, g.b_mn, g.bn);
  g.fp8 = g.in_type == BGNN_E4M3;
  g.err = ctx->d_err;
  const uint32_t wn = TWO ? g.bn / 2 : g.bn;
  const uint64_t tiles = (uint64_t)blocks_of(g.m, BM) * blocks_of(g.n, wn) *
                         (EPI == EPI_PARTIAL ? (uint64_t)g.batches * g.splits : 1ull);
  const int sms = ctx->grid_sms > 0 && ctx->grid_sms < ctx->num_sms ? ctx->grid_sms : ctx->num_sms;
  const unsigned grid = (unsigned)(tiles < (uint64_t)sms ? tiles : sms);
  k_dense16<EPI><<<grid, THREADS, SMEM_BYTES, ctx->stream>>>(maps, g);
  BGNN_LAUNCHED(ctx);
  return BGNN_OK;
}

// z = x w^T (one weight or two) with the epilogue of `EPI`
template <int EPI>
int run_nt(bgnn_ctx* ctx, GemmArgs& g, Mat x, const Mat (&w)[2], uint32_t k) {
  constexpr bool TWO = EPI == EPI_GATED || EPI == EPI_GATED_BWD;
  DevTmp tx, tw[2];
  Maps maps;
  g.a_mn = g.b_mn = 0;
  set_tile(&g, pick_bn(ctx, g.m, g.n, 1, TWO, TWO ? 64 : 32));
  g.nkb[0] = blocks_of(k, g.in_type == BGNN_E4M3 ? 128 : 64);
  g.nkb[1] = 0;
  if (k) {
    BGNN_TRY(tma_ready(ctx, g.in_type, &x, tx));
    BGNN_TRY(make_map(ctx, &maps.a[0], g.in_type, x, BM));
    for (int i = 0; i < (TWO ? 2 : 1); i++) {
      Mat wi = w[i];
      BGNN_TRY(tma_ready(ctx, g.in_type, &wi, tw[i]));
      BGNN_TRY(make_map(ctx, &maps.b[i], g.in_type, wi, TWO ? g.bn / 2 : g.bn));
    }
  }
  return launch<EPI>(ctx, maps, g);
}

// dx = dz0 w0 (+ dz1 w1): contraction over the rows of w
int run_dx(bgnn_ctx* ctx, int type, uint32_t m, uint32_t n, uint32_t k, const Mat (&dz)[2],
           const Mat (&w)[2], int terms, void* dx) {
  GemmArgs g = {};
  DevTmp tz[2], tw[2];
  Maps maps;
  g.m = m;
  g.n = k;
  g.in_type = type;
  g.a_mn = 0;
  g.b_mn = 1;
  set_tile(&g, pick_bn(ctx, m, k, 1, false, 64));
  for (int i = 0; i < terms; i++) {
    Mat a = dz[i], b = w[i];
    g.nkb[i] = blocks_of(n, 64);
    if (n == 0) continue;
    BGNN_TRY(tma_ready(ctx, type, &a, tz[i]));
    BGNN_TRY(tma_ready(ctx, type, &b, tw[i]));
    BGNN_TRY(make_map(ctx, &maps.a[i], type, a, BM));
    BGNN_TRY(make_map(ctx, &maps.b[i], type, b, 64));
  }
  g.out_type = type;
  g.out[0] = dx;
  g.ld_out = k;
  return launch<EPI_LINEAR>(ctx, maps, g);
}

// dw_i = dz_i^T x: contraction over the m rows of both
int run_dw(bgnn_ctx* ctx, int type, uint32_t m, uint32_t n, uint32_t k, const Mat (&dz)[2], Mat x,
           int terms, void* const (&dw)[2]) {
  GemmArgs g = {};
  DevTmp tz[2], tx, part;
  Maps maps;
  g.m = n;
  g.n = k;
  g.in_type = type;
  g.a_mn = g.b_mn = 1;
  g.batches = (uint32_t)terms;
  set_tile(&g, k <= 64 ? 64 : k <= 128 ? 128 : 256);
  g.nkb[0] = blocks_of(m, 64);
  // ranges so that every SM has a tile, each of at least 8 k blocks
  const uint64_t tiles = (uint64_t)blocks_of(n, BM) * blocks_of(k, g.bn) * terms;
  uint64_t s = tiles >= (uint64_t)ctx->num_sms ? 1 : (uint64_t)ctx->num_sms / tiles;
  if (s > (g.nkb[0] + 7) / 8) s = (g.nkb[0] + 7) / 8;
  if (s < 1) s = 1;
  g.per = blocks_of(g.nkb[0], (uint32_t)s);
  if (g.per < 1) g.per = 1;
  g.splits = blocks_of(g.nkb[0], g.per);
  if (g.splits < 1) g.splits = 1;
  if (m) {
    BGNN_TRY(tma_ready(ctx, type, &x, tx));
    BGNN_TRY(make_map(ctx, &maps.b[0], type, x, 64));
    for (int i = 0; i < terms; i++) {
      Mat a = dz[i];
      BGNN_TRY(tma_ready(ctx, type, &a, tz[i]));
      BGNN_TRY(make_map(ctx, &maps.a[i], type, a, 64));
    }
  }
  const uint64_t mn = (uint64_t)n * k;
  BGNN_TRY(bgnn_tmp_alloc(ctx, part, mn * terms * g.splits * sizeof(float)));
  g.part = part.as<float>();
  g.out_type = BGNN_F32;
  BGNN_TRY(launch<EPI_PARTIAL>(ctx, maps, g));
  const uint64_t want = (mn * terms + 255) / 256, cap = (uint64_t)ctx->num_sms * 16;
  k_add_splits<<<(unsigned)(want < cap ? want : cap), 256, 0, ctx->stream>>>(
      g.part, g.splits, (uint32_t)terms, mn, dw[0], dw[1], type);
  BGNN_LAUNCHED(ctx);
  return BGNN_OK;
}

int run_db(bgnn_ctx* ctx, int type, const Mat& dz, void* db, int db_type) {
  if (dz.rows == 0) {
    BGNN_CUDA(ctx, cudaMemsetAsync(db, 0, dz.cols * dtype_size(db_type), ctx->stream));
    return BGNN_OK;
  }
  const uint32_t cb = blocks_of(dz.cols, 32);
  uint64_t parts = ((uint64_t)ctx->num_sms * 8 + cb - 1) / cb;
  const uint64_t most = (dz.rows + 63) / 64;
  if (parts > most) parts = most;
  if (parts > 65535) parts = 65535;
  DevTmp part;
  BGNN_TRY(bgnn_tmp_alloc(ctx, part, parts * dz.cols * sizeof(float)));
  k_col_sums<<<dim3(cb, (unsigned)parts), 256, 0, ctx->stream>>>(dz.p, type, dz.ld, dz.rows,
                                                                  dz.cols, part.as<float>());
  BGNN_LAUNCHED(ctx);
  return bgnn_run_sum_parts(ctx, part.as<float>(), (uint32_t)parts, dz.cols, db, db_type);
}

int check_act16(bgnn_ctx* ctx, int act) {
  BGNN_REQUIRE(ctx, act >= BGNN_ACT_NONE && act <= BGNN_ACT_SILU, "unknown activation %d", act);
  return BGNN_OK;
}

// the checks that the four entry points share
int check_product(bgnn_ctx* ctx, const char* name, int type, bool scales, const void* x,
                  uint64_t ld_x, const void* w0, uint64_t ld_w0, const void* w1, uint64_t ld_w1,
                  uint64_t m, uint32_t k, uint32_t n, int act) {
  BGNN_TRY(check_act16(ctx, act));
  BGNN_REQUIRE(ctx, m <= 0x7fffff00ull && k <= 0x7fffff00u && n <= 0x7fffff00u,
               "%s: a size above 2^31", name);
  BGNN_REQUIRE(ctx, dtype_half(type) || (type == BGNN_E4M3 && scales),
               "%s: operands are bf16, f16, or e4m3 with scales (f32: bgnn_dense)", name);
  BGNN_REQUIRE(ctx, (x && w0 && w1) || (uint64_t)k * n == 0 || m == 0, "%s: NULL operand", name);
  BGNN_REQUIRE(ctx, ld_x >= k && ld_w0 >= k && ld_w1 >= k, "%s: row stride below the row length",
               name);
  return BGNN_OK;
}

}  // namespace

extern "C" int bgnn_linear_fused(bgnn_ctx* ctx, int type, const void* x, uint64_t ld_x,
                                 const float* x_scale, const void* w, uint64_t ld_w,
                                 const float* w_scale, uint64_t m, uint32_t k, uint32_t n,
                                 int bias_type, const void* bias, int act, double act_param,
                                 int res_type, const void* residual, uint64_t ld_res, int out_type,
                                 void* out, uint64_t ld_out) {
  BGNN_ON_DEVICE(ctx);
  BGNN_TRY(check_product(ctx, "linear_fused", type, true, x, ld_x, w, ld_w, w, ld_w, m, k, n, act));
  BGNN_REQUIRE(ctx, dtype_float(out_type), "linear_fused: unknown output type %d", out_type);
  BGNN_REQUIRE(ctx, !bias || dtype_float(bias_type), "linear_fused: unknown bias type");
  BGNN_REQUIRE(ctx, !residual || (dtype_float(res_type) && ld_res >= n),
               "linear_fused: residual type or row stride");
  if (m == 0 || n == 0) return BGNN_OK;
  BGNN_REQUIRE(ctx, out && ld_out >= n, "linear_fused: NULL out or its row stride below n");
  BGNN_REQUIRE(ctx, type != BGNN_E4M3 || (x_scale && w_scale),
               "linear_fused: e4m3 operands need a scale a row");
  GemmArgs g = {};
  g.m = (uint32_t)m;
  g.n = n;
  g.in_type = type;
  if (type == BGNN_E4M3) {
    g.x_scale = x_scale;
    g.w_scale[0] = w_scale;
  }
  g.bias[0] = bias;
  g.bias_type = bias_type;
  g.act = act;
  g.act_p = (float)act_param;
  g.other = residual;
  g.other_type = res_type;
  g.ld_other = ld_res;
  g.out_type = out_type;
  g.out[0] = out;
  g.ld_out = ld_out;
  const Mat ws[2] = {{w, n, k, ld_w}, {w, n, k, ld_w}};
  return run_nt<EPI_LINEAR>(ctx, g, {x, m, k, ld_x}, ws, k);
}

extern "C" int bgnn_gated_linear(bgnn_ctx* ctx, int type, const void* x, uint64_t ld_x,
                                 const float* x_scale, const void* w_gate, uint64_t ld_gate,
                                 const float* gate_scale, const void* w_up, uint64_t ld_up,
                                 const float* up_scale, uint64_t m, uint32_t k, uint32_t n,
                                 int bias_type, const void* bias_gate, const void* bias_up, int act,
                                 double act_param, int out_type, void* out, uint64_t ld_out) {
  BGNN_ON_DEVICE(ctx);
  BGNN_TRY(check_product(ctx, "gated_linear", type, true, x, ld_x, w_gate, ld_gate, w_up, ld_up, m,
                         k, n, act));
  BGNN_REQUIRE(ctx, dtype_float(out_type), "gated_linear: unknown output type %d", out_type);
  BGNN_REQUIRE(ctx, !(bias_gate || bias_up) || dtype_float(bias_type),
               "gated_linear: unknown bias type");
  if (m == 0 || n == 0) return BGNN_OK;
  BGNN_REQUIRE(ctx, out && ld_out >= n, "gated_linear: NULL out or its row stride below n");
  BGNN_REQUIRE(ctx, type != BGNN_E4M3 || (x_scale && gate_scale && up_scale),
               "gated_linear: e4m3 operands need a scale a row");
  GemmArgs g = {};
  g.m = (uint32_t)m;
  g.n = n;
  g.in_type = type;
  if (type == BGNN_E4M3) {
    g.x_scale = x_scale;
    g.w_scale[0] = gate_scale;
    g.w_scale[1] = up_scale;
  }
  g.bias[0] = bias_gate;
  g.bias[1] = bias_up;
  g.bias_type = bias_type;
  g.act = act;
  g.act_p = (float)act_param;
  g.out_type = out_type;
  g.out[0] = out;
  g.ld_out = ld_out;
  const Mat ws[2] = {{w_gate, n, k, ld_gate}, {w_up, n, k, ld_up}};
  return run_nt<EPI_GATED>(ctx, g, {x, m, k, ld_x}, ws, k);
}

extern "C" int bgnn_linear_fused_backward(bgnn_ctx* ctx, int type, const void* grad,
                                          uint64_t ld_grad, const void* x, uint64_t ld_x,
                                          const void* w, uint64_t ld_w, uint64_t m, uint32_t k,
                                          uint32_t n, int bias_type, const void* bias, int act,
                                          double act_param, void* grad_x, void* grad_w,
                                          void* grad_bias) {
  BGNN_ON_DEVICE(ctx);
  BGNN_TRY(check_product(ctx, "linear_fused_backward", type, false, x, ld_x, w, ld_w, w, ld_w, m, k,
                         n, act));
  BGNN_REQUIRE(ctx, !(bias || grad_bias) || dtype_float(bias_type),
               "linear_fused_backward: unknown bias type");
  BGNN_REQUIRE(ctx, (grad || (uint64_t)m * n == 0) && ld_grad >= n,
               "linear_fused_backward: NULL gradient or its row stride below n");
  if (n == 0) {
    if (grad_x && m && k) BGNN_CUDA(ctx, cudaMemsetAsync(grad_x, 0, m * k * 2, ctx->stream));
    return BGNN_OK;
  }
  const uint32_t ldz = (n + 7) / 8 * 8;
  Mat dz[2] = {{grad, m, n, ld_grad}, {}};
  DevTmp tz, tg;
  if (act != BGNN_ACT_NONE && m) {
    BGNN_TRY(bgnn_tmp_alloc(ctx, tz, m * ldz * 2));
    GemmArgs g = {};
    g.m = (uint32_t)m;
    g.n = n;
    g.in_type = type;
    g.bias[0] = bias;
    g.bias_type = bias_type;
    g.act = act;
    g.act_p = (float)act_param;
    g.other = grad;
    g.other_type = type;
    g.ld_other = ld_grad;
    g.out_type = type;
    g.out[0] = tz.p;
    g.ld_out = ldz;
    const Mat ws[2] = {{w, n, k, ld_w}, {w, n, k, ld_w}};
    BGNN_TRY(run_nt<EPI_LINEAR_BWD>(ctx, g, {x, m, k, ld_x}, ws, k));
    dz[0] = {tz.p, m, n, ldz};
  } else if (m && k && grad_x && grad_w) {
    BGNN_TRY(tma_ready(ctx, type, &dz[0], tg));  // once for both products
  }
  const Mat ws[2] = {{w, n, k, ld_w}, {}};
  if (grad_x && m && k) BGNN_TRY(run_dx(ctx, type, (uint32_t)m, n, k, dz, ws, 1, grad_x));
  if (grad_w && k) {
    void* const dw[2] = {grad_w, nullptr};
    BGNN_TRY(run_dw(ctx, type, (uint32_t)m, n, k, dz, {x, m, k, ld_x}, 1, dw));
  }
  if (grad_bias) BGNN_TRY(run_db(ctx, type, dz[0], grad_bias, bias_type));
  return BGNN_OK;
}

extern "C" int bgnn_gated_linear_backward(bgnn_ctx* ctx, int type, const void* grad,
                                          uint64_t ld_grad, const void* x, uint64_t ld_x,
                                          const void* w_gate, uint64_t ld_gate, const void* w_up,
                                          uint64_t ld_up, uint64_t m, uint32_t k, uint32_t n,
                                          int bias_type, const void* bias_gate,
                                          const void* bias_up, int act, double act_param,
                                          void* grad_x, void* grad_w_gate, void* grad_w_up,
                                          void* grad_bias_gate, void* grad_bias_up) {
  BGNN_ON_DEVICE(ctx);
  BGNN_TRY(check_product(ctx, "gated_linear_backward", type, false, x, ld_x, w_gate, ld_gate, w_up,
                         ld_up, m, k, n, act));
  BGNN_REQUIRE(ctx, !(bias_gate || bias_up || grad_bias_gate || grad_bias_up) ||
                        dtype_float(bias_type),
               "gated_linear_backward: unknown bias type");
  BGNN_REQUIRE(ctx, (grad || (uint64_t)m * n == 0) && ld_grad >= n,
               "gated_linear_backward: NULL gradient or its row stride below n");
  BGNN_REQUIRE(ctx, (grad_w_gate == nullptr) == (grad_w_up == nullptr),
               "gated_linear_backward: both weight gradients or neither");
  if (n == 0) {
    if (grad_x && m && k) BGNN_CUDA(ctx, cudaMemsetAsync(grad_x, 0, m * k * 2, ctx->stream));
    return BGNN_OK;
  }
  const uint32_t ldz = (n + 7) / 8 * 8;
  DevTmp tz;
  BGNN_TRY(bgnn_tmp_alloc(ctx, tz, 2 * m * ldz * 2));
  uint16_t* z0 = tz.as<uint16_t>();
  uint16_t* z1 = z0 + m * ldz;
  const Mat ws[2] = {{w_gate, n, k, ld_gate}, {w_up, n, k, ld_up}};
  if (m) {
    GemmArgs g = {};
    g.m = (uint32_t)m;
    g.n = n;
    g.in_type = type;
    g.bias[0] = bias_gate;
    g.bias[1] = bias_up;
    g.bias_type = bias_type;
    g.act = act;
    g.act_p = (float)act_param;
    g.other = grad;
    g.other_type = type;
    g.ld_other = ld_grad;
    g.out_type = type;
    g.out[0] = z0;
    g.out[1] = z1;
    g.ld_out = ldz;
    BGNN_TRY(run_nt<EPI_GATED_BWD>(ctx, g, {x, m, k, ld_x}, ws, k));
  }
  const Mat dz[2] = {{z0, m, n, ldz}, {z1, m, n, ldz}};
  if (grad_x && m && k) BGNN_TRY(run_dx(ctx, type, (uint32_t)m, n, k, dz, ws, 2, grad_x));
  if (grad_w_gate && k) {
    void* const dw[2] = {grad_w_gate, grad_w_up};
    BGNN_TRY(run_dw(ctx, type, (uint32_t)m, n, k, dz, {x, m, k, ld_x}, 2, dw));
  }
  if (grad_bias_gate) BGNN_TRY(run_db(ctx, type, dz[0], grad_bias_gate, bias_type));
  if (grad_bias_up) BGNN_TRY(run_db(ctx, type, dz[1], grad_bias_up, bias_type));
  return BGNN_OK;
}
