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
// memory, f32 results in pieces (PIECE); bias, activation, product and residual
// are f32 and the result is rounded once.  dz (dg, du) is rounded to the
// operands' type once (not for a few rows, dense_rows.cu), because the two products that follow take it as an
// operand and kind::f16 has no wider one: against 64 bits the gradients of a
// gated product are off by 0.0023 norm-wise in bf16, where the results' own
// rounding is 0.0017.
//
// Kernel: persistent, one CTA an SM, warp-specialised.  A tile is 256 rows by 256
// columns on a pair of CTAs (cta_group::2: each holds 128 rows of A and half of
// B), or 512 columns for long contractions; where those are too few for the GPU,
// 128 rows by 32 to 256 columns on one CTA (pick_shape):
//   warp 16   TMA producer: per k block (128 bytes of k) its CTA's A tile and
//             share of the B tile into a ring of shared-memory stages, 128-byte
//             swizzle;
//   warp 17   MMA issuer (one thread of the pair): tcgen05.mma, M = 256 or 128,
//             N up to 256, into one of two tensor-memory accumulators (512
//             columns fill it with one);
//   warps 0-15 epilogue: warp w takes the accumulator lanes (rows) of its
//             quadrant w % 4 and every fourth 32-column chunk; a chunk of the
//             residual comes by TMA into one shared-memory slot, the result
//             goes out through the other, turned round to run along rows.
//             Sixteen warps, four a scheduler: with eight the activations of a
//             short contraction ran at a third of the issue rate and bound the
//             kernel.
// An operand whose contraction runs down its rows (w in dx, both in dw) is
// read as it lies ("MN-major": boxes of 64 columns x 64 rows), never
// transposed in memory.  The gated kernels load BN/2 rows of each weight side
// by side into the B tile, so one accumulator holds both halves.
// Measured: 16,384 x 4,096 -> 4,096 bf16 1,594 TFLOP/s (93 % of what the library's
// product reaches), gated 1,534; a short contraction (2.45M x 256 -> 512 gated,
// 990 TFLOP/s) is bound by its epilogue and the shared memory that it shares
// with the loads and the products.
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

#include <atomic>
#include <cstring>
#include <mutex>

#include "act.cuh"
#include "dense_rows.cuh"

namespace {

constexpr int BM = 128;
constexpr int EPI_WARPS = 16;
constexpr int THREADS = (EPI_WARPS + 4) * 32;  // five warpgroups; warps 18 and 19 idle
// Registers a thread: at most 96 at launch (65,536 / 640), then split unevenly:
// 4 * 104 + 64 = 5 * 96.
constexpr int EPI_REGS = 104, ISSUE_REGS = 64;
constexpr int MAX_STAGES = 8;
constexpr int A_BYTES = BM * 128;
constexpr int SLOT_BYTES = 32 * 64;         // 32 rows x 32 16-bit or 16 f32 columns
constexpr int WARP_BYTES = 2 * SLOT_BYTES;  // an epilogue warp's two slots
constexpr int RING_BYTES = 160 * 1024;
constexpr int SMEM_BYTES = 1024 + RING_BYTES + EPI_WARPS * WARP_BYTES + 512;
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory of one SM");
constexpr uint32_t SPIN_LIMIT = 1u << 24;     // polls before a wait gives up,
constexpr long long SPIN_CLOCKS = 4000000000ll;  // or clocks (about two seconds)

enum Epi : int {
  EPI_LINEAR,
  EPI_LINEAR_F32,
  EPI_GATED,
  EPI_GATED_F32,
  EPI_LINEAR_BWD,
  EPI_GATED_BWD,
  EPI_PARTIAL
};
// the B tile holds two weights
template <int EPI>
constexpr bool TWO_WEIGHTS = EPI == EPI_GATED || EPI == EPI_GATED_F32 || EPI == EPI_GATED_BWD;
// The result stays f32: an accumulator takes the products of PIECE k blocks, and
// these pieces are added in f32 registers.  (The tensor cores cut their additions,
// of 16 products each, short by up to 2^-23 of the sum so far: 8,192 positive
// terms lose 3e-5 in one accumulator and 4e-7 in pieces.  Gated 16,384 x 4,096 ->
// 4,096 takes 836 us in pieces, 769 without.)
template <int EPI>
constexpr bool PIECES = EPI == EPI_LINEAR_F32 || EPI == EPI_GATED_F32;
constexpr uint32_t PIECE = 8;
// k blocks of a dw range: 32,768 products, whose additions lose at most 2.4e-4 of
// their sum, half of what the result's rounding to f16 may
constexpr uint32_t MAX_PER = 512;

// a, b: the operands of each contraction segment (dx), of each batch (dw: a), or
// the two weights of a gated product (b).
// in: the residual or upstream gradient in boxes of a slot.
struct Maps {
  CUtensorMap a[2], b[2], in;
};

struct GemmArgs {
  uint32_t m, n;          // output size (gated: n columns of h, 2n of the product)
  uint32_t bn;            // columns of a tile in tensor memory: 32, 64, 128, 256, 512
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
  float* bsum[2];         // backward: column sums of 32 rows each, [rows / 32, n], or NULL
  float* part;            // EPI_PARTIAL: [splits, batches, m, ld_out]; NULL: dw whole, no parts
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
// bounded wait of one thread; false when it gave up or another role already did
__device__ __forceinline__ bool mbar_wait(uint32_t a, uint32_t parity, volatile uint32_t* abort_flag,
                                          int* err, int where) {
  long long t0 = 0;
  for (uint32_t i = 0; i < SPIN_LIMIT; i++) {
    if (mbar_try(a, parity)) return true;
    if ((i & 31u) == 31u) {
      if (*abort_flag) return false;
      if (t0 == 0) t0 = clock64();
      else if (clock64() - t0 > SPIN_CLOCKS) break;
    }
  }
  *abort_flag = 1u;
  dev_raise(err, DEVERR_TIMEOUT, (uint64_t)blockIdx.x, where);
  return false;
}
// The same for a whole warp.  Each lane polls (what it reads next is ordered
// after its own wait), and one that gave up takes the others along: the warp's
// next instructions need all of its lanes, and lanes that left alone would keep
// the rest waiting there without a limit.
__device__ __forceinline__ bool warp_wait(uint32_t a, uint32_t parity, volatile uint32_t* abort_flag,
                                          int* err, int where) {
  return __all_sync(0xffffffffu, mbar_wait(a, parity, abort_flag, err, where)) != 0;
}
// for what is in flight when a role has given up
__device__ __forceinline__ void mbar_drain(uint32_t a, uint32_t parity) {
  const long long t0 = clock64();
  for (uint32_t i = 0; i < SPIN_LIMIT; i++)
    if (mbar_try(a, parity) || clock64() - t0 > SPIN_CLOCKS / 4) return;
}
// CG: CTAs that share one product (cta_group), 1 or a pair
template <int CG>
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y,
                                            uint32_t bar) {
  if constexpr (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2"
        " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
// the cluster address of this CTA's shared address `a` in the CTA `rank`
__device__ __forceinline__ uint32_t peer_addr(uint32_t a, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
// arrives on the issuing CTA's barrier.  It hands over tensor memory only, which
// tcgen05.fence::before_thread_sync orders: no release of other memory.
template <int CG>
__device__ __forceinline__ void mbar_arrive_at(uint32_t a) {
  if constexpr (CG == 2)
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                     peer_addr(a, 0))
                 : "memory");
  else
    asm volatile("mbarrier.arrive.relaxed.cta.shared::cta.b64 _, [%0];" ::"r"(a) : "memory");
}
// all threads of the CTA, or of the pair
template <int CG>
__device__ __forceinline__ void pair_sync() {
  __syncthreads();
  if constexpr (CG == 2) {
    __syncwarp();  // one lane of a warp may have come another way
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}
template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t cols) {
  if constexpr (CG == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot),
                 "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot),
                 "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t t, uint32_t cols) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(t), "r"(cols)
                 : "memory");
  else
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(t), "r"(cols)
                 : "memory");
}
// Shared-memory matrix descriptor, 128-byte swizzle, version 1.  Eight-row
// groups (K-major: 8 rows of m or n; MN-major: 8 rows of k) are 1024 bytes
// apart; in an MN-major tile the next 64 columns start after all 64 rows.
__device__ __forceinline__ uint64_t smem_desc(uint32_t a, int mn_major) {
  return (uint64_t)((a & 0x3FFFFu) >> 4) | ((uint64_t)(mn_major ? 8192 >> 4 : 1) << 16) |
         ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
template <int CG>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t acc) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
template <int CG>
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t acc) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
// arrives on this CTA's barrier when the products issued so far are done
template <int CG>
__device__ __forceinline__ void mma_commit_here(uint32_t bar) {
  if constexpr (CG == 2)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
        : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
        : "memory");
}
// ... and on the same barrier of the other CTA of a pair
template <int CG>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  if constexpr (CG == 2)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        " [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
  else
    mma_commit_here<CG>(bar);
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
// 32 columns of this warp's 32 lanes; the values are there after tmem_wait_ld
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]),
        "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]),
        "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]),
        "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]),
        "=f"(v[30]), "=f"(v[31])
      : "r"(taddr));
}
// the registers pass through, so that no use of them moves before the wait
__device__ __forceinline__ void tmem_wait_ld(float (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
      : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]),
        "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]),
        "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]),
        "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]),
        "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]),
        "+f"(v[30]), "+f"(v[31])
      :
      : "memory");
}

// ---- slots: 32 rows of 64 bytes, 16-byte units swizzled as TMA's 64-byte mode
// does, so that a row a lane has no bank conflicts ------------------------------
__device__ __forceinline__ uint4* slot_unit(void* slot, int row, int unit) {
  return reinterpret_cast<uint4*>(static_cast<char*>(slot) + row * 64 +
                                  ((unit ^ ((row >> 1) & 3)) << 4));
}
template <int DT>
__device__ __forceinline__ void put_row16(void* slot, int row, const float (&v)[32]) {
#pragma unroll
  for (int u = 0; u < 4; u++)
    *slot_unit(slot, row, u) =
        make_uint4(pack2<DT>(v[8 * u], v[8 * u + 1]), pack2<DT>(v[8 * u + 2], v[8 * u + 3]),
                   pack2<DT>(v[8 * u + 4], v[8 * u + 5]), pack2<DT>(v[8 * u + 6], v[8 * u + 7]));
}
// eight 16-bit elements of a slot's unit
__device__ __forceinline__ void unit16(const uint4 q, int dt, float (&o)[8]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if (dt == BGNN_BF16) {
      o[2 * i] = __uint_as_float(w[i] << 16);
      o[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      o[2 * i] = f.x;
      o[2 * i + 1] = f.y;
    }
  }
}
// `rows` rows of `cols` elements from a slot to rows `pitch` bytes apart, element
// by element, a row's side by side
template <class T>
__device__ __forceinline__ void give_elements(void* slot, char* out, uint64_t pitch, uint32_t lane,
                                              uint32_t cols, uint32_t rows) {
  constexpr uint32_t ES = sizeof(T), WIDTH = 64 / ES, STEP = 32 / WIDTH;
  const uint32_t e = lane % WIDTH;
  if (e >= cols) return;
  out += (lane / WIDTH) * pitch + e * ES;
#pragma unroll 8
  for (uint32_t r = lane / WIDTH; r < rows; r += STEP, out += STEP * pitch)
    *reinterpret_cast<T*>(out) = reinterpret_cast<const T*>(
        slot_unit(slot, (int)r, (int)(e * ES / 16)))[e % (16 / ES)];
}
__device__ __forceinline__ void fence_async() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// whether 16 bytes of a row, from a multiple of as many, are one access
__device__ __forceinline__ bool vec16_ok(const void* p, int dt, uint64_t ld) {
  return ((uintptr_t)p & 15u) == 0 && ld % (dt == BGNN_F32 ? 4 : 8) == 0;
}

// Lane j gets the sum over the warp's lanes of v[j]: halves of the columns are
// handed over at distances 16, 8, .. 1.  v is used up.
__device__ __forceinline__ float column_sum(float (&v)[32], int lane) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < o; i++) {
      const float give = up ? v[i] : v[i + o];
      v[i] = (up ? v[i + o] : v[i]) + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
  return v[0];
}

// the tiles of a CTA (pair), columns fastest
struct Tile {
  uint32_t m0, n0, batch, split;
};
template <int EPI, int CG>
struct Tiles {
  const GemmArgs& g;
  uint32_t n_tiles, m_tiles, wn, left, q, nt, step_q, step_n;
  __device__ __forceinline__ Tiles(const GemmArgs& args, uint32_t width) : g(args), wn(width) {
    n_tiles = (g.n + wn - 1) / wn;
    m_tiles = (g.m + BM * CG - 1) / (BM * CG);
    const uint32_t tiles = m_tiles * n_tiles * (EPI == EPI_PARTIAL ? g.batches * g.splits : 1u);
    const uint32_t first = blockIdx.x / CG, step = gridDim.x / CG;
    left = (tiles - first + step - 1) / step;  // the grid has at most `tiles` CTAs (pairs)
    q = first / n_tiles;
    nt = first - q * n_tiles;
    step_q = step / n_tiles;
    step_n = step - step_q * n_tiles;
  }
  __device__ __forceinline__ bool more() const { return left != 0; }
  __device__ __forceinline__ void next() {
    left--;
    q += step_q;
    nt += step_n;
    if (nt >= n_tiles) nt -= n_tiles, q++;
  }
  __device__ __forceinline__ Tile at() const {
    Tile r;
    r.n0 = nt * wn;
    if (EPI == EPI_PARTIAL) {
      const uint32_t z = q / m_tiles;
      r.m0 = (q - z * m_tiles) * (BM * CG);
      r.split = z / g.batches;
      r.batch = z - r.split * g.batches;
    } else {
      r.m0 = q * (BM * CG);
      r.split = r.batch = 0;
    }
    return r;
  }
};

template <int EPI, int CG>
__global__ void __launch_bounds__(THREADS, 1)
    k_dense16(const __grid_constant__ Maps maps, const GemmArgs g) {
  constexpr bool TWO = TWO_WEIGHTS<EPI>;  // B tile of two weights
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = s_addr(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;  // swizzle atoms start on 1024 bytes
  uint8_t* gbase = smem_raw + (base - raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(gbase + RING_BYTES + EPI_WARPS * WARP_BYTES);
  const uint32_t b_full = s_addr(bars), b_empty = b_full + 8 * MAX_STAGES;
  const uint32_t b_accf = b_empty + 8 * MAX_STAGES, b_acce = b_accf + 16, b_in = b_acce + 16;
  const uint32_t b_last = b_in + 8 * EPI_WARPS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * MAX_STAGES + 4 + EPI_WARPS + 1);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cta_rank() : 0u;  // of the pair; rank 0 issues the products
  const uint32_t S = g.stages;
  const uint32_t bufs = g.bn > 256 ? 1u : 2u;  // accumulators that tensor memory holds
  const uint32_t tmem_cols = bufs * g.bn;

  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < S; s++) {
      mbar_init(b_full + 8 * s, 1);
      mbar_init(b_empty + 8 * s, 1);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(b_accf + 8 * b, 1);
      mbar_init(b_acce + 8 * b, EPI_WARPS * CG);
    }
    for (int w = 0; w < EPI_WARPS; w++) mbar_init(b_in + 8 * w, 1);
    mbar_init(b_last, 1);
    *abort_flag = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == EPI_WARPS) {
    tmem_alloc<CG>(s_addr(tmem_slot), tmem_cols);
    tc_fence_before();
  }
  pair_sync<CG>();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const uint32_t wn = TWO ? g.bn / 2 : g.bn;  // output columns of a tile
  const uint32_t bl = g.bn / CG;              // rows of the B tile that this CTA loads
  const uint32_t nkb = g.nkb[0] + g.nkb[1];
  // k blocks [first, last) of a tile
  auto kb_first = [&](const Tile& t) { return EPI == EPI_PARTIAL ? t.split * g.per : 0u; };
  auto kb_last = [&](const Tile& t) {
    if (EPI != EPI_PARTIAL) return nkb;
    const uint32_t e = (t.split + 1) * g.per;
    return e < nkb ? e : nkb;
  };

  if (warp >= EPI_WARPS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(ISSUE_REGS));
    if (warp == EPI_WARPS) {
      // ---- TMA producer ----
      if (lane == 0) {
        uint32_t s = 0, ph = 0, st = base;
        uint64_t filled = 0;
        const uint32_t tx = CG * (A_BYTES + bl * 128);
        const int kw = g.fp8 ? 128 : 64;  // elements of a k block
        // both CTAs' loads count on the issuing CTA's barriers
        const uint32_t b_land = CG == 2 ? peer_addr(b_full, 0) : b_full;
        const bool a_mn = g.a_mn, b_mn = g.b_mn;
        const uint32_t nkb0 = g.nkb[0], stage_bytes = g.stage_bytes;
        for (Tiles<EPI, CG> ts(g, wn); ts.more(); ts.next()) {
          const Tile ti = ts.at();
          const int am = (int)(ti.m0 + rank * BM);
          // a 512-column tile is two products of 256: this CTA's half of each
          const uint32_t half_b = g.bn > 256 ? 128u : bl;
          const int bn0 = (int)(TWO && g.bn <= 256 ? ti.n0 : ti.n0 + rank * half_b);
          const uint32_t e = kb_last(ti);
          uint32_t kb = kb_first(ti);
          // dw: the batch's A; else the segment's A and B
          const CUtensorMap* ma = &maps.a[EPI == EPI_PARTIAL ? ti.batch : 0];
          const CUtensorMap* mb = &maps.b[TWO && CG == 2 && g.bn <= 256 ? rank : 0];  // a weight a CTA
          int k0 = (int)kb * kw;
          for (; kb < e; kb++, k0 += kw) {
            if (EPI != EPI_PARTIAL && !TWO && kb == nkb0) {  // the second segment
              ma = &maps.a[1];
              mb = &maps.b[1];
              k0 = 0;
            }
            if (!mbar_wait(b_empty + 8 * s, ph ^ 1u, abort_flag, g.err, 70)) goto drain;
            if (rank == 0) mbar_expect_tx(b_full + 8 * s, tx);
            const uint32_t bar = b_land + 8 * s;
            if (a_mn) {
#pragma unroll
              for (int i = 0; i < BM / 64; i++)
                tma_load_2d<CG>(st + i * 8192, ma, am + i * 64, k0, bar);
            } else {
              tma_load_2d<CG>(st, ma, k0, am, bar);
            }
            if (b_mn) {
              for (uint32_t i = 0; i < bl; i += 64)
                tma_load_2d<CG>(st + A_BYTES + i * 128, mb,
                                bn0 + (int)(i < half_b ? i : i + 128), k0, bar);
            } else if (g.bn > 256) {
              tma_load_2d<CG>(st + A_BYTES, mb, k0, bn0, bar);
              tma_load_2d<CG>(st + A_BYTES + 128 * 128, TWO ? &maps.b[1] : mb, k0,
                              TWO ? bn0 : bn0 + 256, bar);
            } else {
              tma_load_2d<CG>(st + A_BYTES, mb, k0, bn0, bar);
              if (TWO && CG == 1)
                tma_load_2d<CG>(st + A_BYTES + wn * 128, &maps.b[1], k0, bn0, bar);
            }
            filled++;
            st += stage_bytes;
            if (++s == S) s = 0, ph ^= 1u, st = base;
          }
        }
      drain:
        if (*abort_flag && rank == 0)  // the last fill of every stage lands before the CTA ends
          for (uint64_t f = filled > S ? filled - S : 0; f < filled; f++)
            mbar_drain(b_full + 8 * (uint32_t)(f % S), (uint32_t)((f / S) & 1u));
      }
    } else if (warp == EPI_WARPS + 1) {
      // ---- MMA issuer ----
      if (lane == 0 && rank == 0) {
        uint32_t s = 0, ph = 0, buf = 0, aph = 0;
        // The issuing thread's own instructions bound a stage once (about 1000
        // clocks against 512 of products): the descriptors are one addition each.
        const uint64_t desc_a = smem_desc(base, g.a_mn), desc_b = smem_desc(base + A_BYTES, g.b_mn);
        const uint32_t step_a = (g.a_mn ? 2048u : 32u) >> 4, step_b = (g.b_mn ? 2048u : 32u) >> 4;
        const uint32_t stage16 = g.stage_bytes >> 4, idesc = g.idesc, bn = g.bn;
        auto issue = [&](auto fp8, auto wide) -> bool {
          for (Tiles<EPI, CG> ts(g, wn); ts.more(); ts.next()) {
            const Tile ti = ts.at();
            const uint32_t last = kb_last(ti);
            uint32_t kb = kb_first(ti);
            do {  // a piece of the contraction into one accumulator
              const uint32_t e = PIECES<EPI> && last - kb > PIECE ? kb + PIECE : last;
              if (!mbar_wait(b_acce + 8 * buf, aph ^ 1u, abort_flag, g.err, 71)) return false;
              tc_fence_after();
              const uint32_t d = tmem + buf * bn;
              uint32_t acc = 0u;
              for (; kb < e; kb++) {
                if (!mbar_wait(b_full + 8 * s, ph, abort_flag, g.err, 72)) return false;
                tc_fence_after();
                const uint64_t da = desc_a + s * stage16, db = desc_b + s * stage16;
#pragma unroll
                for (uint32_t kk = 0; kk < 4; kk++) {
                  if (decltype(fp8)::value) mma_f8<CG>(d, da + kk * step_a, db + kk * step_b, idesc, acc);
                  else mma_f16<CG>(d, da + kk * step_a, db + kk * step_b, idesc, acc);
                  if (decltype(wide)::value) {  // the second 256 columns; A stays where it is
                    const uint64_t d2 = db + (128 * 128 >> 4) + kk * step_b;
                    if (decltype(fp8)::value) mma_f8<CG>(d + 256, da + kk * step_a, d2, idesc, acc);
                    else mma_f16<CG>(d + 256, da + kk * step_a, d2, idesc, acc);
                  }
                  acc = 1u;
                }
                mma_commit<CG>(b_empty + 8 * s);
                if (++s == S) s = 0, ph ^= 1u;
              }
              mma_commit<CG>(b_accf + 8 * buf);
              if (++buf == bufs) buf = 0, aph ^= 1u;
            } while (kb < last);
          }
          return true;
        };
        if (CG == 2 && bufs == 1) {
          if (g.fp8) issue(std::true_type{}, std::true_type{});
          else issue(std::false_type{}, std::true_type{});
        } else {
          if (g.fp8) issue(std::true_type{}, std::false_type{});
          else issue(std::false_type{}, std::false_type{});
        }
        // every product issued is done before tensor memory is freed
        mma_commit_here<CG>(b_last);
        mbar_drain(b_last, 0);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(EPI_REGS));
    // ---- epilogue ----
    const int quad = warp & 3, group = warp >> 2;  // rows; every fourth 32-column chunk
    uint8_t* slots = gbase + RING_BYTES + warp * WARP_BYTES;
    const uint32_t in_bar = b_in + 8 * warp;
    uint32_t buf = 0, aph = 0, in_ph = 0;
    const bool vec_out = EPI == EPI_PARTIAL && g.part
                             ? g.ld_out % 4 == 0
                             : vec16_ok(g.out[0], g.out_type, g.ld_out) &&
                                   (!g.out[1] || vec16_ok(g.out[1], g.out_type, g.ld_out));
    // hands the accumulator back once every lane has read it
    auto release = [&]() {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_at<CG>(b_acce + 8 * buf);
      if (++buf == bufs) buf = 0, aph ^= 1u;
    };
    bool gave_up = false, pending = false;  // pending: a slot was asked for
    for (Tiles<EPI, CG> ts(g, wn); ts.more() && !gave_up; ts.next()) {
      const Tile ti = ts.at();
      const uint32_t k_first = kb_first(ti), k_last = kb_last(ti);
      const bool any_k = k_first < k_last;
      const uint32_t row0 = ti.m0 + rank * BM + quad * 32;  // this warp's rows
      const uint32_t lanes = (uint32_t)(quad * 32) << 16;
      // Asks for 32 columns (f32: 16) of the residual / upstream gradient into
      // slot 0, with which every lane is done.
      auto ask = [&](uint32_t col) {
        if (!g.other || col >= g.n) return;
        pending = true;
        if (lane == 0) {
          fence_async();
          mbar_expect_tx(in_bar, SLOT_BYTES);
          tma_load_2d<1>(s_addr(slots), &maps.in, (int)col, (int)row0, in_bar);
        }
      };
      auto asked = [&]() {
        if (!warp_wait(in_bar, in_ph, abort_flag, g.err, 74)) {
          gave_up = true;
          mbar_drain(in_bar, in_ph);
        }
        pending = false;
        in_ph ^= 1u;
      };
      // f(first column, 8 values) for this lane's row of the chunk at col0, eight
      // columns at a time; the first of it was asked for
      auto take = [&](uint32_t col0, auto f) {
        if (g.other_type != BGNN_F32) {
          asked();
#pragma unroll
          for (int u = 0; u < 4; u++) {
            float o[8];
            unit16(*slot_unit(slots, lane, u), g.other_type, o);
            f(8 * u, o);
          }
          __syncwarp();
        } else {
#pragma unroll
          for (int h = 0; h < 2; h++) {
            if (h == 0 || col0 + 16 < g.n) {
              if (h == 1) ask(col0 + 16);
              asked();
#pragma unroll
              for (int u = 0; u < 2; u++) {
                const uint4 a = *slot_unit(slots, lane, 2 * u), b = *slot_unit(slots, lane, 2 * u + 1);
                const float o[8] = {__uint_as_float(a.x), __uint_as_float(a.y), __uint_as_float(a.z),
                                    __uint_as_float(a.w), __uint_as_float(b.x), __uint_as_float(b.y),
                                    __uint_as_float(b.z), __uint_as_float(b.w)};
                f(16 * h + 8 * u, o);
              }
              __syncwarp();
            }
          }
        }
      };
      // Out, a row a lane: through slot 1, turned round, so that four lanes
      // write the 64 bytes of a row, or, where rows are not made of 16-byte
      // units, its elements side by side.  (TMA stores of a slot took turns with
      // the ring's loads: gated backward 669 us against 645.)
      auto give_slot = [&](void* out, uint64_t ld, int type, uint32_t col) {
        __syncwarp();
        const uint32_t es = type == BGNN_F32 ? 4u : 2u, width = 64u / es;
        char* at = static_cast<char*>(out) + ((uint64_t)row0 * ld + col) * es;
        const uint64_t pitch = ld * es;
        if (vec_out && col + width <= g.n) {
          const uint4* q = slot_unit(slots + SLOT_BYTES, lane >> 2, lane & 3);
          at += (lane >> 2) * pitch + (lane & 3) * 16;
          uint4 v[4];
#pragma unroll
          for (int i = 0; i < 4; i++) v[i] = q[i * 32];  // 8 rows on: the same swizzle
#pragma unroll
          for (int i = 0; i < 4; i++, at += 8 * pitch)
            if (row0 + (lane >> 2) + i * 8 < g.m) *reinterpret_cast<uint4*>(at) = v[i];
        } else {
          const uint32_t cols = g.n - col < width ? g.n - col : width;
          const uint32_t rows = g.m > row0 ? (g.m - row0 < 32 ? g.m - row0 : 32u) : 0u;
          if (es == 4) give_elements<uint32_t>(slots + SLOT_BYTES, at, pitch, lane, cols, rows);
          else give_elements<uint16_t>(slots + SLOT_BYTES, at, pitch, lane, cols, rows);
        }
        __syncwarp();
      };
      auto give = [&](const float (&v)[32], uint32_t col0, void* out, uint64_t ld, int type) {
        if (type == BGNN_F32) {
#pragma unroll
          for (int h = 0; h < 2; h++) {
            if (col0 + 16 * h >= g.n) break;
#pragma unroll
            for (int u = 0; u < 4; u++)
              *slot_unit(slots + SLOT_BYTES, lane, u) = make_uint4(
                  __float_as_uint(v[16 * h + 4 * u]), __float_as_uint(v[16 * h + 4 * u + 1]),
                  __float_as_uint(v[16 * h + 4 * u + 2]), __float_as_uint(v[16 * h + 4 * u + 3]));
            give_slot(out, ld, type, col0 + 16 * h);
          }
        } else {
          if (type == BGNN_BF16) put_row16<BGNN_BF16>(slots + SLOT_BYTES, lane, v);
          else put_row16<BGNN_F16>(slots + SLOT_BYTES, lane, v);
          give_slot(out, ld, type, col0);
        }
      };
      // scales and bias of a chunk: lane j holds column j's
      auto scaled = [&](float (&v)[32], uint32_t col0, int i) {
        const bool in = col0 + lane < g.n;
        if (g.x_scale) {
          const float xs = row0 + lane < g.m ? g.x_scale[row0 + lane] : 1.0f;
          const float ws = in ? g.w_scale[i][col0 + lane] : 0.0f;
#pragma unroll
          for (int j = 0; j < 32; j++) v[j] *= xs * __shfl_sync(0xffffffffu, ws, j);
        }
        if (g.bias[i]) {
          const float bv = in ? load_any(g.bias[i], g.bias_type, col0 + lane) : 0.0f;
#pragma unroll
          for (int j = 0; j < 32; j++) v[j] += __shfl_sync(0xffffffffu, bv, j);
        }
      };
      // the bias gradient's share of a chunk, before dz is rounded
      auto bias_sums = [&](float (&v)[32], uint32_t col0, float* bsum) {
        if (!bsum) return;
        const float t = column_sum(v, lane);
        if (col0 + lane < g.n && row0 < g.m)
          bsum[(uint64_t)(row0 / 32) * g.n + col0 + lane] = t;
      };
      auto linear_out = [&](float (&v)[32], uint32_t col0) {
        scaled(v, col0, 0);
        if (g.act != BGNN_ACT_NONE)
          with_act(g.act, [&](auto act) {
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const float2 f = act_two<decltype(act)::value>(make_float2(v[j], v[j + 1]), g.act_p);
              v[j] = f.x;
              v[j + 1] = f.y;
            }
          });
        if (g.other)
          take(col0, [&](int j0, const float (&o)[8]) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j0 + j] += o[j];
          });
        give(v, col0, g.out[0], g.ld_out, g.out_type);
      };

      if (group * 32 < wn) ask(ti.n0 + group * 32);
      auto gated_out = [&](float (&v)[32], float (&u)[32], uint32_t col0) {
        scaled(v, col0, 0);
        scaled(u, col0, 1);
        with_act(g.act, [&](auto act) {
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float2 f = mul2(act_two<decltype(act)::value>(make_float2(v[j], v[j + 1]), g.act_p),
                                  make_float2(u[j], u[j + 1]));
            v[j] = f.x;
            v[j + 1] = f.y;
          }
        });
        give(v, col0, g.out[0], g.ld_out, g.out_type);
      };
      if constexpr (PIECES<EPI>) {
        // pieces of the contraction added in f32 registers, rounded to nearest:
        // this warp's two chunks of columns, or both products of its one chunk
        const uint32_t step = TWO ? wn : 128u;
        auto mine = [&](int i) { return TWO ? group * 32 < wn : group * 32 + i * 128 < wn; };
        float sum[2][32];
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (int j = 0; j < 32; j++) sum[i][j] = 0.0f;
        uint32_t kb = k_first;
        do {
          if (!warp_wait(b_accf + 8 * buf, aph, abort_flag, g.err, 73)) {
            gave_up = true;
            break;
          }
          tc_fence_after();
          const uint32_t acc = tmem + lanes + buf * g.bn;
#pragma unroll
          for (int i = 0; i < 2; i++) {
            if (mine(i) && any_k) {
              float v[32];
              tmem_ld32(acc + group * 32 + i * step, v);
              tmem_wait_ld(v);
#pragma unroll
              for (int j = 0; j < 32; j++) sum[i][j] += v[j];
            }
          }
          release();
          kb += PIECE;
        } while (kb < k_last);
        if (gave_up) break;
        if constexpr (TWO) {
          const uint32_t c = group * 32;
          if (c < wn && ti.n0 + c < g.n) gated_out(sum[0], sum[1], ti.n0 + c);
        } else {
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const uint32_t c = group * 32 + i * 128;
            if (c < wn && ti.n0 + c < g.n) {
              if (i) ask(ti.n0 + c);
              linear_out(sum[i], ti.n0 + c);
            }
          }
        }
      } else {
        if (!warp_wait(b_accf + 8 * buf, aph, abort_flag, g.err, 73)) break;
        tc_fence_after();
        const uint32_t acc = tmem + lanes + buf * g.bn;
        for (uint32_t c = group * 32; c < wn; c += 128) {
          const uint32_t col0 = ti.n0 + c;
          if (col0 >= g.n) break;  // uniform: the chunk is past the last column
          if (c >= 128) ask(col0);
          float v[32], u[32];      // u: the second product's
          tmem_ld32(acc + c, v);
          if constexpr (TWO) tmem_ld32(acc + wn + c, u);
          tmem_wait_ld(v);
          if constexpr (TWO) tmem_wait_ld(u);
          if (!any_k) {
#pragma unroll
            for (int j = 0; j < 32; j++) {
              v[j] = 0.0f;
              if constexpr (TWO) u[j] = 0.0f;
            }
          }
          if constexpr (EPI == EPI_LINEAR) {
            linear_out(v, col0);
          } else if constexpr (EPI == EPI_PARTIAL) {
            if (g.part)
              give(v, col0,
                   g.part + ((uint64_t)ti.split * g.batches + ti.batch) * g.m * g.ld_out, g.ld_out,
                   BGNN_F32);
            else
              give(v, col0, ti.batch ? g.out[1] : g.out[0], g.ld_out, g.out_type);
          } else if constexpr (EPI == EPI_LINEAR_BWD) {
            scaled(v, col0, 0);
            // act' first, the gradient on top
            with_act(g.act, [&](auto act) {
#pragma unroll
              for (int j = 0; j < 32; j += 2) {
                float2 f0, f1;
                act_grad_two<decltype(act)::value>(make_float2(v[j], v[j + 1]), g.act_p, f0, f1);
                v[j] = f0.y;
                v[j + 1] = f1.y;
              }
            });
            take(col0, [&](int j0, const float (&o)[8]) {
#pragma unroll
              for (int j = 0; j < 8; j++) v[j0 + j] *= o[j];
            });
            give(v, col0, g.out[0], g.ld_out, g.out_type);
            bias_sums(v, col0, g.bsum[0]);
          } else if constexpr (EPI == EPI_GATED) {
            gated_out(v, u, col0);
          } else {
            scaled(v, col0, 0);
            scaled(u, col0, 1);
            with_act(g.act, [&](auto act) {
#pragma unroll
              for (int j = 0; j < 32; j += 2) {
                float2 f0, f1;
                act_grad_two<decltype(act)::value>(make_float2(v[j], v[j + 1]), g.act_p, f0, f1);
                v[j] = u[j] * f0.y;  // dg / grad
                v[j + 1] = u[j + 1] * f1.y;
                u[j] = f0.x;  // du / grad
                u[j + 1] = f1.x;
              }
            });
            take(col0, [&](int j0, const float (&o)[8]) {
#pragma unroll
              for (int j = 0; j < 8; j++) {
                v[j0 + j] *= o[j];
                u[j0 + j] *= o[j];
              }
            });
            give(v, col0, g.out[0], g.ld_out, g.out_type);
            give(u, col0, g.out[1], g.ld_out, g.out_type);
            bias_sums(v, col0, g.bsum[0]);
            bias_sums(u, col0, g.bsum[1]);
          }
        }
        release();
      }
    }
    if (pending) mbar_drain(in_bar, in_ph);  // gave up: the copy lands before the CTA ends
  }
  pair_sync<CG>();
  if (warp == EPI_WARPS) {
    __syncwarp();
    tc_fence_after();
    tmem_free<CG>(tmem, tmem_cols);
  }
}

// dw: the splits' partial matrices (rows ld f32 apart) added in order: CH chains
// an element, each in ascending order, then the chains in order.  One chain
// where elements are many; eight where splits are (47 x 256 over 143 splits:
// one chain took 14 us, all of it waiting).
template <int CH>
__global__ void __launch_bounds__(256) k_add_splits(const float* __restrict__ part, uint32_t splits,
                                                    uint32_t batches, uint32_t ld, uint32_t rows,
                                                    uint32_t cols, void* out0, void* out1,
                                                    int out_type) {
  constexpr int EL = 256 / CH;
  __shared__ float sm[CH][EL + 1];
  const uint64_t mn = (uint64_t)rows * cols, total = mn * batches;
  const uint64_t step = (uint64_t)rows * ld * batches;
  const int el = threadIdx.x % EL, ch = threadIdx.x / EL;
  for (uint64_t base = (uint64_t)blockIdx.x * EL; base < total; base += (uint64_t)gridDim.x * EL) {
    const uint64_t i = base + el;
    const uint32_t b = i >= mn;
    const uint64_t e = b ? i - mn : i;
    float v = 0.0f;
    if (i < total) {
      const uint32_t r = (uint32_t)(e / cols), c = (uint32_t)(e - (uint64_t)r * cols);
      const float* p = part + ((uint64_t)b * rows + r) * ld + c;
#pragma unroll 4
      for (uint32_t s = ch; s < splits; s += CH) v += p[s * step];
    }
    if (CH > 1) {
      sm[ch][el] = v;
      __syncthreads();
      if (ch == 0)
        for (int k = 1; k < CH; k++) v += sm[k][el];
      __syncthreads();
    }
    if (ch == 0 && i < total) store_any(b ? out1 : out0, out_type, e, v);
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

// rows copied to a row stride that TMA takes (a multiple of 16 bytes), 16 bytes
// a thread
template <class T>
__global__ void __launch_bounds__(256) k_repack(const T* __restrict__ x, uint64_t ld, uint64_t rows,
                                                uint32_t cols, uint32_t ldp, T* __restrict__ out) {
  constexpr uint32_t PER = 16 / sizeof(T);
  const uint32_t words = ldp / PER;  // of a row
  const uint64_t total = rows * words;
  for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (uint64_t)gridDim.x * blockDim.x) {
    const uint64_t r = total < (1ull << 32) ? (uint32_t)i / words : i / words;
    const uint32_t c = (uint32_t)(i - r * words) * PER;
    const T* p = x + r * ld + c;
    T v[PER];
#pragma unroll
    for (uint32_t j = 0; j < PER; j++) v[j] = c + j < cols ? p[j] : T(0);
    uint4 q;
    memcpy(&q, v, 16);
    reinterpret_cast<uint4*>(out)[i] = q;
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

// whether TMA can take a matrix as it lies
bool tma_takes(int type, const Mat& x) {
  const uint64_t pitch = x.ld * dtype_size(type);
  return ((uintptr_t)x.p & 15u) == 0 && pitch % 16 == 0 && pitch < (1ull << 40) &&
         x.rows < (1ull << 31);
}

// boxes of 64 bytes x 32 rows, 64-byte swizzle: the epilogue's slots
int make_chunk_map(bgnn_ctx* ctx, CUtensorMap* map, int type, const Mat& x) {
  auto enc = encode_fn();
  if (!enc) return bgnn_set_error(ctx, BGNN_ERR_UNSUPPORTED, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[2] = {x.cols, x.rows};
  cuuint64_t strides[1] = {x.ld * dtype_size(type)};
  cuuint32_t box[2] = {type == BGNN_F32 ? 16u : 32u, 32};
  cuuint32_t el[2] = {1, 1};
  const CUtensorMapDataType dt = type == BGNN_BF16  ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                 : type == BGNN_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                    : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  const CUresult r =
      enc(map, dt, 2, const_cast<void*>(x.p), dims, strides, box, el,
          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
          CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return bgnn_set_error(ctx, BGNN_ERR_UNSUPPORTED, "tensor map encode failed (%d)", (int)r);
  return BGNN_OK;
}
// x as TMA can read it: itself, or a copy whose rows start on 16 bytes
int tma_ready(bgnn_ctx* ctx, int type, Mat* x, DevTmp& tmp) {
  if (tma_takes(type, *x)) return BGNN_OK;
  const uint32_t es = (uint32_t)dtype_size(type);
  const uint32_t per = 16 / es;
  const uint32_t ldp = (x->cols + per - 1) / per * per;
  BGNN_TRY(bgnn_tmp_alloc(ctx, tmp, x->rows * (uint64_t)ldp * es));
  const uint64_t total = x->rows * (uint64_t)(ldp / per), cap = (uint64_t)ctx->num_sms * 32;
  const uint64_t want = (total + 255) / 256;
  const unsigned grid = (unsigned)(want < cap ? want : cap);
  auto pack = [&](auto zero) {
    using T = decltype(zero);
    k_repack<T><<<grid, 256, 0, ctx->stream>>>(static_cast<const T*>(x->p), x->ld, x->rows, x->cols,
                                               ldp, tmp.as<T>());
  };
  if (es == 4) pack(uint32_t(0));
  else if (es == 2) pack(uint16_t(0));
  else pack(uint8_t(0));
  BGNN_LAUNCHED(ctx);
  x->p = tmp.p;
  x->ld = ldp;
  return BGNN_OK;
}

uint32_t blocks_of(uint64_t len, uint32_t per) { return (uint32_t)((len + per - 1) / per); }

// The tile of a product: its columns in tensor memory (bn) and whether a pair
// of CTAs shares it (256 rows, each CTA loading half of B).
struct Shape {
  uint32_t bn;
  int cg;
};
// 256 columns for a pair while every pair has a tile, since a wide tile reads A
// fewer times and a pair reads B once for both; below that the widest of one
// CTA that gives every SM one; a narrow output takes the narrowest that covers
// it.  512 columns (where may_512) for a long contraction: a k block loads 48 KB a CTA
// for the products that two 32 KB ones take in 256 columns, and loads bound it (about
// 48 bytes a clock and SM), but the accumulator fills tensor memory, so that
// the epilogue does not overlap the next tile.  A 512-column tile takes about
// WIDE / 100 times a 256-column one.
constexpr uint64_t WIDE = 160;
Shape pick_shape(const bgnn_ctx* ctx, uint64_t m, uint64_t n, uint64_t z, bool two, uint32_t least,
                 uint32_t nkb, bool may_512) {
  const uint64_t sms = (uint64_t)ctx->num_sms, pairs = sms / 2;
  Shape s = {256, 2};
  auto tiles = [&](uint64_t rows, uint64_t cols) {
    return ((m + rows - 1) / rows) * ((n + cols - 1) / cols) * z;
  };
  const uint64_t wn = two ? 128 : 256, t256 = tiles(2 * BM, wn), t512 = tiles(2 * BM, 2 * wn);
  if (t256 >= pairs && n > wn / 2) {
    if (may_512 && nkb >= 64 &&
        (t512 + pairs - 1) / pairs * WIDE < (t256 + pairs - 1) / pairs * 100)
      s.bn = 512;
    return s;
  }
  s.cg = 1;
  while (s.bn > least) {
    const uint64_t w = two ? s.bn / 2 : s.bn;
    if (tiles(BM, w) >= sms && n > w / 2) break;
    s.bn /= 2;
  }
  return s;
}

void set_tile(GemmArgs* g, const Shape& s) {
  g->bn = s.bn;
  g->stage_bytes = A_BYTES + s.bn / s.cg * 128;
  g->stages = RING_BYTES / g->stage_bytes;
  if (g->stages > MAX_STAGES) g->stages = MAX_STAGES;
}

// instruction descriptor: D f32, A and B of one type, majorness, N, M
uint32_t make_idesc(int type, int a_mn, int b_mn, const Shape& s) {
  const uint32_t f = type == BGNN_BF16 ? 1u : 0u;  // kind::f16: 0 f16, 1 bf16; f8f6f4: 0 e4m3
  return (1u << 4) | (f << 7) | (f << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         (((s.bn > 256 ? 256 : s.bn) >> 3) << 17) | ((uint32_t)(BM * s.cg >> 4) << 24);
}

// Registers a thread that an instance was compiled to (the same on every
// device); setmaxnreg waits for good unless the launch holds what the epilogue
// and the issuing warps are given.
template <int EPI, int CG>
int compiled_regs() {
  static const int regs = [] {
    cudaFuncAttributes at;
    return cudaFuncGetAttributes(&at, k_dense16<EPI, CG>) == cudaSuccess ? at.numRegs : 0;
  }();
  return regs;
}
template <int EPI, int CG>
int launch_cg(bgnn_ctx* ctx, const Maps& maps, const GemmArgs& g, uint64_t tiles) {
  if (compiled_regs<EPI, CG>() * THREADS < (EPI_WARPS * EPI_REGS + 4 * ISSUE_REGS) * 32)
    return bgnn_set_error(ctx, BGNN_ERR_UNSUPPORTED, "product kernel compiled to %d registers",
                          compiled_regs<EPI, CG>());
  static std::atomic<uint64_t> ready{0};  // devices (below 64) whose limit is set
  const uint64_t bit = ctx->device < 64 ? 1ull << ctx->device : 0;
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    BGNN_CUDA(ctx, cudaFuncSetAttribute(k_dense16<EPI, CG>,
                                        cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  const int sms = ctx->grid_sms > 0 && ctx->grid_sms < ctx->num_sms ? ctx->grid_sms : ctx->num_sms;
  const uint64_t most = sms / CG > 0 ? sms / CG : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles < most ? tiles : most) * CG);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM_BYTES;
  cfg.stream = ctx->stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CG;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = CG == 2 ? 1 : 0;
  BGNN_CUDA(ctx, cudaLaunchKernelEx(&cfg, k_dense16<EPI, CG>, maps, g));
  BGNN_LAUNCHED(ctx);
  return BGNN_OK;
}

template <int EPI>
int launch(bgnn_ctx* ctx, const Maps& maps, GemmArgs& g, const Shape& s) {
  constexpr bool TWO = TWO_WEIGHTS<EPI>;
  g.idesc = make_idesc(g.in_type, g.a_mn, g.b_mn, s);
  g.fp8 = g.in_type == BGNN_E4M3;
  g.err = ctx->d_err;
  const uint32_t wn = TWO ? s.bn / 2 : s.bn;
  const uint64_t tiles = (uint64_t)blocks_of(g.m, BM * s.cg) * blocks_of(g.n, wn) *
                         (EPI == EPI_PARTIAL ? (uint64_t)g.batches * g.splits : 1ull);
  BGNN_REQUIRE(ctx, tiles < (1ull << 31), "product of %u x %u: too many tiles", g.m, g.n);
  return s.cg == 2 ? launch_cg<EPI, 2>(ctx, maps, g, tiles) : launch_cg<EPI, 1>(ctx, maps, g, tiles);
}

// z = x w^T (one weight or two) with the epilogue of `EPI`
template <int EPI>
int run_nt(bgnn_ctx* ctx, GemmArgs& g, Mat x, const Mat (&w)[2], uint32_t k) {
  constexpr bool TWO = TWO_WEIGHTS<EPI>;
  if constexpr (EPI == EPI_LINEAR || EPI == EPI_GATED)
    if (few_rows(g.m, k, g.n, TWO)) {
      RowsArgs r = {};
      r.x = x.p;
      r.ld_x = x.ld;
      r.x_scale = g.x_scale;
      r.two = TWO;
      for (int i = 0; i < (TWO ? 2 : 1); i++) {
        r.w[i] = w[i].p;
        r.ld_w[i] = w[i].ld;
        r.w_scale[i] = g.w_scale[i];
        r.bias[i] = g.bias[i];
      }
      r.m = g.m;
      r.k = k;
      r.n = g.n;
      r.bias_type = g.bias_type;
      r.act = g.act;
      r.act_p = g.act_p;
      r.other = g.other;
      r.other_type = g.other_type;
      r.ld_other = g.ld_other;
      r.out_type = g.out_type;
      r.out = g.out[0];
      r.ld_out = g.ld_out;
      return bgnn_run_dense_rows(ctx, g.in_type, r);
    }
  DevTmp tx, tw[2], tin;
  Maps maps;
  g.a_mn = g.b_mn = 0;
  g.nkb[0] = blocks_of(k, g.in_type == BGNN_E4M3 ? 128 : 64);
  g.nkb[1] = 0;
  const bool f32_out = g.out_type == BGNN_F32;  // the pieces' registers hold 256 columns
  const Shape sh = pick_shape(ctx, g.m, g.n, 1, TWO, TWO ? 64 : 32, g.nkb[0],
                              EPI == EPI_LINEAR_BWD || EPI == EPI_GATED_BWD || !f32_out);
  set_tile(&g, sh);
  if (k) {
    BGNN_TRY(tma_ready(ctx, g.in_type, &x, tx));
    BGNN_TRY(make_map(ctx, &maps.a[0], g.in_type, x, BM));
    for (int i = 0; i < (TWO ? 2 : 1); i++) {
      Mat wi = w[i];
      BGNN_TRY(tma_ready(ctx, g.in_type, &wi, tw[i]));
      BGNN_TRY(make_map(ctx, &maps.b[i], g.in_type, wi,
                        g.bn > 256 ? 128 : TWO ? g.bn / 2 : g.bn / sh.cg));
    }
  }
  if (g.other) {
    Mat in = {g.other, g.m, g.n, g.ld_other};
    BGNN_TRY(tma_ready(ctx, g.other_type, &in, tin));
    BGNN_TRY(make_chunk_map(ctx, &maps.in, g.other_type, in));
  }
  if constexpr (EPI == EPI_LINEAR)
    if (f32_out) return launch<EPI_LINEAR_F32>(ctx, maps, g, sh);
  if constexpr (EPI == EPI_GATED)
    if (f32_out && g.nkb[0] > PIECE) return launch<EPI_GATED_F32>(ctx, maps, g, sh);
  return launch<EPI>(ctx, maps, g, sh);
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
  const Shape sh = pick_shape(ctx, m, k, 1, false, 64, blocks_of(n, 64) * terms, true);
  set_tile(&g, sh);
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
  return launch<EPI_LINEAR>(ctx, maps, g, sh);
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
  Shape sh = {k <= 64 ? 64u : k <= 128 ? 128u : 256u, 1};
  if (sh.bn == 256 && n > BM) sh.cg = 2;
  g.nkb[0] = blocks_of(m, 64);
  if (sh.cg == 2) {
    const Shape wide = pick_shape(ctx, n, k, terms, false, 64, g.nkb[0], true);
    if (wide.bn == 512) sh = wide;
  }
  set_tile(&g, sh);
  // ranges so that every SM has a tile, each of at least 8 k blocks, and of at
  // most MAX_PER
  const uint64_t tiles = (uint64_t)blocks_of(n, BM * sh.cg) * blocks_of(k, g.bn) * terms;
  uint64_t s = tiles * sh.cg >= (uint64_t)ctx->num_sms ? 1 : ctx->num_sms / (tiles * sh.cg);
  if (s > (g.nkb[0] + 7) / 8) s = (g.nkb[0] + 7) / 8;
  if (s < 1) s = 1;
  g.per = blocks_of(g.nkb[0], (uint32_t)s);
  if (g.per < 1) g.per = 1;
  if (g.per > MAX_PER) g.per = MAX_PER;
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
  g.out_type = type;
  g.out[0] = dw[0];
  g.out[1] = dw[1];
  g.ld_out = k;
  if (g.splits == 1) return launch<EPI_PARTIAL>(ctx, maps, g, sh);
  g.ld_out = (k + 3) / 4 * 4;
  BGNN_TRY(bgnn_tmp_alloc(ctx, part, (uint64_t)n * g.ld_out * terms * g.splits * sizeof(float)));
  g.part = part.as<float>();
  BGNN_TRY(launch<EPI_PARTIAL>(ctx, maps, g, sh));
  const int chains = g.splits >= 16 ? 8 : 1;
  const uint64_t el = 256 / chains;
  const uint64_t want = ((uint64_t)n * k * terms + el - 1) / el, cap = (uint64_t)ctx->num_sms * 16;
  const unsigned grid = (unsigned)(want < cap ? want : cap);
  auto add = [&](auto kernel) {
    kernel<<<grid, 256, 0, ctx->stream>>>(g.part, g.splits, (uint32_t)terms, (uint32_t)g.ld_out, n,
                                          k, dw[0], dw[1], type);
  };
  if (chains == 8) add(k_add_splits<8>);
  else add(k_add_splits<1>);
  BGNN_LAUNCHED(ctx);
  return BGNN_OK;
}

int run_db(bgnn_ctx* ctx, int type, const Mat& dz, void* db, int db_type) {
  if (dz.rows == 0) {
    BGNN_CUDA(ctx, cudaMemsetAsync(db, 0, dz.cols * dtype_size(db_type), ctx->stream));
    return BGNN_OK;
  }
  if (type == BGNN_F32 && dz.ld == dz.cols && dz.rows <= 2048)  // few sums: one kernel
    return bgnn_run_sum_parts(ctx, static_cast<const float*>(dz.p), (uint32_t)dz.rows, dz.cols, db,
                              db_type);
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

// what the gradients of few rows share
RowsArgs rows_backward(const void* grad, uint64_t ld_grad, const void* x, uint64_t ld_x, uint64_t m,
                       uint32_t k, uint32_t n, int bias_type, int act, double act_param) {
  RowsArgs a = {};
  a.x = x;
  a.ld_x = ld_x;
  a.m = (uint32_t)m;
  a.k = k;
  a.n = n;
  a.bias_type = bias_type;
  a.act = act;
  a.act_p = (float)act_param;
  a.grad = grad;
  a.ld_grad = ld_grad;
  return a;
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
  BGNN_REQUIRE(ctx, residual != out || (res_type == out_type && (m == 1 || ld_res == ld_out)),
               "linear_fused: out in the residual's buffer needs its type and row stride");
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
  if (act != BGNN_ACT_NONE && m && few_rows_backward(m, k)) {
    RowsArgs a = rows_backward(grad, ld_grad, x, ld_x, m, k, n, bias_type, act, act_param);
    a.w[0] = w;
    a.ld_w[0] = ld_w;
    a.bias[0] = bias;
    return bgnn_run_dense_rows_backward(ctx, type, a,
                                        {grad_x, {grad_w, nullptr}, {grad_bias, nullptr}});
  }
  const uint32_t ldz = (n + 7) / 8 * 8;
  Mat dz[2] = {{grad, m, n, ld_grad}, {}};
  DevTmp tz, tg;
  // what the bias gradient sums: dz in f32, 32 rows at a time, or the gradient
  Mat bsum = dz[0];
  int bsum_type = type;
  if (m) BGNN_TRY(tma_ready(ctx, type, &dz[0], tg));  // once for every product that reads it
  if (act != BGNN_ACT_NONE && m) {
    const uint64_t parts = grad_bias ? (m + 31) / 32 : 0;
    BGNN_TRY(bgnn_tmp_alloc(ctx, tz, m * ldz * 2 + parts * n * sizeof(float)));
    GemmArgs g = {};
    g.m = (uint32_t)m;
    g.n = n;
    g.in_type = type;
    g.bias[0] = bias;
    g.bias_type = bias_type;
    g.act = act;
    g.act_p = (float)act_param;
    g.other = dz[0].p;
    g.other_type = type;
    g.ld_other = dz[0].ld;
    g.out_type = type;
    g.out[0] = tz.p;
    g.ld_out = ldz;
    if (grad_bias) {
      g.bsum[0] = reinterpret_cast<float*>(tz.as<uint16_t>() + m * ldz);
      bsum = {g.bsum[0], parts, n, n};
      bsum_type = BGNN_F32;
    }
    const Mat ws[2] = {{w, n, k, ld_w}, {w, n, k, ld_w}};
    BGNN_TRY(run_nt<EPI_LINEAR_BWD>(ctx, g, {x, m, k, ld_x}, ws, k));
    dz[0] = {tz.p, m, n, ldz};
  }
  const Mat ws[2] = {{w, n, k, ld_w}, {}};
  if (grad_x && m && k) BGNN_TRY(run_dx(ctx, type, (uint32_t)m, n, k, dz, ws, 1, grad_x));
  if (grad_w && k) {
    void* const dw[2] = {grad_w, nullptr};
    BGNN_TRY(run_dw(ctx, type, (uint32_t)m, n, k, dz, {x, m, k, ld_x}, 1, dw));
  }
  if (grad_bias) BGNN_TRY(run_db(ctx, bsum_type, bsum, grad_bias, bias_type));
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
  if (m && few_rows_backward(m, k)) {
    RowsArgs a = rows_backward(grad, ld_grad, x, ld_x, m, k, n, bias_type, act, act_param);
    a.two = 1;
    a.w[0] = w_gate;
    a.w[1] = w_up;
    a.ld_w[0] = ld_gate;
    a.ld_w[1] = ld_up;
    a.bias[0] = bias_gate;
    a.bias[1] = bias_up;
    return bgnn_run_dense_rows_backward(
        ctx, type, a, {grad_x, {grad_w_gate, grad_w_up}, {grad_bias_gate, grad_bias_up}});
  }
  const uint32_t ldz = (n + 7) / 8 * 8;
  DevTmp tz;  // dg, du, then the bias gradients' sums of 32 rows
  const uint64_t parts = (m + 31) / 32;
  BGNN_TRY(bgnn_tmp_alloc(ctx, tz, 2 * m * ldz * 2 +
                                       (grad_bias_gate || grad_bias_up ? 2 * parts * n * 4 : 0)));
  uint16_t* z0 = tz.as<uint16_t>();
  uint16_t* z1 = z0 + m * ldz;
  float* sums[2];
  sums[0] = reinterpret_cast<float*>(z1 + m * ldz);
  sums[1] = sums[0] + parts * n;
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
    g.bsum[0] = grad_bias_gate ? sums[0] : nullptr;
    g.bsum[1] = grad_bias_up ? sums[1] : nullptr;
    BGNN_TRY(run_nt<EPI_GATED_BWD>(ctx, g, {x, m, k, ld_x}, ws, k));
  }
  const Mat dz[2] = {{z0, m, n, ldz}, {z1, m, n, ldz}};
  if (grad_x && m && k) BGNN_TRY(run_dx(ctx, type, (uint32_t)m, n, k, dz, ws, 2, grad_x));
  if (grad_w_gate && k) {
    void* const dw[2] = {grad_w_gate, grad_w_up};
    BGNN_TRY(run_dw(ctx, type, (uint32_t)m, n, k, dz, {x, m, k, ld_x}, 2, dw));
  }
  if (grad_bias_gate)
    BGNN_TRY(run_db(ctx, BGNN_F32, {sums[0], parts, n, n}, grad_bias_gate, bias_type));
  if (grad_bias_up)
    BGNN_TRY(run_db(ctx, BGNN_F32, {sums[1], parts, n, n}, grad_bias_up, bias_type));
  return BGNN_OK;
}
