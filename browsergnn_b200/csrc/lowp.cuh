// Element types of the mixed-precision operators (bgnn_dtype): loads to f32,
// one rounding on the way out, and the launch-side guard and checks that
// their entry points share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "bgnn_internal.cuh"

inline size_t dtype_size(int t) { return t == BGNN_F32 ? 4 : t == BGNN_E4M3 ? 1 : 2; }
inline bool dtype_float(int t) { return t == BGNN_F32 || t == BGNN_BF16 || t == BGNN_F16; }
inline bool dtype_half(int t) { return t == BGNN_BF16 || t == BGNN_F16; }

// Makes the context's device current for one entry point and puts the
// caller's device back on return.
struct DeviceGuard {
  int before = -1;
  int status = BGNN_OK;
  explicit DeviceGuard(bgnn_ctx* ctx) {
    if (!ctx) {
      status = BGNN_ERR_INVALID_ARG;
      return;
    }
    cudaError_t e = cudaGetDevice(&before);
    if (e == cudaSuccess && before != ctx->device) e = cudaSetDevice(ctx->device);
    else before = -1;
    if (e != cudaSuccess)
      status = bgnn_set_error(ctx, BGNN_ERR_CUDA, "cudaSetDevice(%d): %s", ctx->device,
                              cudaGetErrorString(e));
  }
  ~DeviceGuard() {
    if (before >= 0) cudaSetDevice(before);
  }
  DeviceGuard(const DeviceGuard&) = delete;
  DeviceGuard& operator=(const DeviceGuard&) = delete;
};
#define BGNN_ON_DEVICE(ctx) \
  DeviceGuard device_guard_(ctx); \
  if (device_guard_.status != BGNN_OK) return device_guard_.status

// Columns of a row are counted in 32 bits with room for a block's step.
#define BGNN_REQUIRE_COLS(ctx, name, cols) \
  BGNN_REQUIRE(ctx, (cols) <= 0x7fffffffu, "%s: a row of %u elements, 2^31 or more", name, cols)

// out[c] = the sum of column c over `parts` rows of f32 partial sums, in a
// fixed order (rownorm.cu)
int bgnn_run_sum_parts(bgnn_ctx* ctx, const float* part, uint32_t parts, uint64_t cols, void* out,
                       int out_type);

// one element type at compile time
template <int DT>
struct Elt;
template <>
struct Elt<BGNN_F32> {
  using type = float;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Elt<BGNN_BF16> {
  using type = __nv_bfloat16;
  static __device__ __forceinline__ float get(type v) { return __bfloat162float(v); }
  static __device__ __forceinline__ type put(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elt<BGNN_F16> {
  using type = __half;
  static __device__ __forceinline__ float get(type v) { return __half2float(v); }
  static __device__ __forceinline__ type put(float v) { return __float2half_rn(v); }
};
template <>
struct Elt<BGNN_E4M3> {  // round to nearest even, saturating at +-448; NaN stays NaN
  using type = __nv_fp8_storage_t;
  static __device__ __forceinline__ type put(float v) {
    return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
  }
};
template <int DT>
using elt_t = typename Elt<DT>::type;

// what an element of the type holds after one rounding, back in f32
template <int DT>
__device__ __forceinline__ float rounded(float v) {
  return Elt<DT>::get(Elt<DT>::put(v));
}

// eight consecutive elements; p is aligned to 16 bytes (8 elements)
template <int DT>
__device__ __forceinline__ void load8(const elt_t<DT>* p, float (&v)[8]) {
  if constexpr (DT == BGNN_F32) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    const float4 b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (DT == BGNN_BF16) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
  }
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == BGNN_BF16) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
  } else {
    const __half2 t = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
  }
}

// eight consecutive elements; p aligned to 16 bytes (e4m3: to 8)
template <int DT>
__device__ __forceinline__ void store8(elt_t<DT>* p, const float (&v)[8]) {
  if constexpr (DT == BGNN_F32) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else if constexpr (DT == BGNN_E4M3) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i], v[4 * i + 1]),
                                                   __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i + 2], v[4 * i + 3]),
                                                   __NV_SATFINITE, __NV_E4M3);
      w[i] = lo | (hi << 16);
    }
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]),
                                              pack2<DT>(v[4], v[5]), pack2<DT>(v[6], v[7]));
  }
}

// one element of a type known at run time (biases, norm weights, residuals)
__device__ __forceinline__ float load_any(const void* p, int dt, uint64_t i) {
  if (dt == BGNN_F32) return static_cast<const float*>(p)[i];
  if (dt == BGNN_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int dt, uint64_t i, float v) {
  if (dt == BGNN_F32) static_cast<float*>(p)[i] = v;
  else if (dt == BGNN_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// ---- f32 arithmetic that the kernels share ---------------------------------------
constexpr float LOG2E = 1.4426950408889634f;
// 2^x, two units in the last place; results below the normal range are 0
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two f32 operations in one instruction
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n"
      " mul.rn.f32x2 z, x, y;\n mov.b64 {%0, %1}, z;\n}\n"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n"
      " add.rn.f32x2 z, x, y;\n mov.b64 {%0, %1}, z;\n}\n"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n .reg .b64 x, y, z, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n"
      " mov.b64 w, {%6, %7};\n fma.rn.f32x2 z, x, y, w;\n mov.b64 {%0, %1}, z;\n}\n"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
