// Activations (bgnn_act) in f32 and their derivatives, for the epilogues of the
// mixed-precision products.
#pragma once

#include <type_traits>

#include "lowp.cuh"

__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// the logistic function 1 / (1 + 2^t), t = -x log2(e)
__device__ __forceinline__ float sigmoid_t(float t) { return rcp(1.0f + ex2(t)); }
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
// ... of two arguments.  (One reciprocal for both, 1/a = b/(ab), saves a
// quarter of the special-function work but costs three more instructions a
// pair and a clamp; the epilogue is bound by instructions, not by that unit.)
__device__ __forceinline__ float2 sigmoid_t2(float2 t) {
  const float2 a = add2(make_float2(ex2(t.x), ex2(t.y)), both(1.0f));
  return make_float2(rcp(a.x), rcp(a.y));
}
constexpr float GELU_C = 0.7978845608028654f;  // sqrt(2/pi)
template <int ACT>
constexpr bool GATES = ACT == BGNN_ACT_SILU || ACT == BGNN_ACT_GELU;  // z sigmoid(..)
// the gates' t: -z log2(e); gelu: 0.5 (1 + tanh v) = sigmoid(2 v),
// v = sqrt(2/pi) (z + 0.044715 z^3)
template <int ACT>
__device__ __forceinline__ float2 gate_t2(float2 z) {
  if constexpr (ACT == BGNN_ACT_SILU) return mul2(z, both(-LOG2E));
  constexpr float C = -2.0f * LOG2E * GELU_C;
  return mul2(z, fma2(mul2(z, z), both(C * 0.044715f), both(C)));
}
template <int ACT>
__device__ __forceinline__ float act_one(float z, float p) {
  if constexpr (ACT == BGNN_ACT_RELU) return z > 0.0f ? z : 0.0f;
  if constexpr (ACT == BGNN_ACT_RELU_MAX) return z != z ? z : (z > 0.0f ? z : 0.0f);
  if constexpr (ACT == BGNN_ACT_ELU) return z > 0.0f ? z : p * expm1f(z);
  if constexpr (ACT == BGNN_ACT_LEAKY_RELU) return z > 0.0f ? z : p * z;
  if constexpr (ACT == BGNN_ACT_SIGMOID) return sigmoid_t(-LOG2E * z);
  if constexpr (ACT == BGNN_ACT_TANH) return tanhf(z);
  return z;
}
// two activations
template <int ACT>
__device__ __forceinline__ float2 act_two(float2 z, float p) {
  if constexpr (GATES<ACT>) return mul2(z, sigmoid_t2(gate_t2<ACT>(z)));
  return make_float2(act_one<ACT>(z.x, p), act_one<ACT>(z.y, p));
}
// act(z) and act'(z); s: sigmoid(..) of the gates
template <int ACT>
__device__ __forceinline__ float2 act_grad(float z, float s, float p) {
  if constexpr (ACT == BGNN_ACT_SILU) return make_float2(z * s, s * fmaf(z, 1.0f - s, 1.0f));
  if constexpr (ACT == BGNN_ACT_GELU) {
    const float dv = 2.0f * GELU_C * fmaf(3.0f * 0.044715f * z, z, 1.0f);
    // far out s (1 - s) is 0; dv must not make a NaN of it
    const float q = s * (1.0f - s);
    return make_float2(z * s, q == 0.0f ? s : fmaf(z * q, dv, s));
  }
  if constexpr (ACT == BGNN_ACT_RELU)
    return z > 0.0f ? make_float2(z, 1.0f) : make_float2(0.0f, 0.0f);
  if constexpr (ACT == BGNN_ACT_RELU_MAX)
    return z != z ? make_float2(z, z) : z > 0.0f ? make_float2(z, 1.0f) : make_float2(0.0f, 0.0f);
  if constexpr (ACT == BGNN_ACT_ELU) {
    const float e = p * expm1f(z);
    return z > 0.0f ? make_float2(z, 1.0f) : make_float2(e, e + p);
  }
  if constexpr (ACT == BGNN_ACT_LEAKY_RELU)
    return z > 0.0f ? make_float2(z, 1.0f) : make_float2(p * z, p);
  if constexpr (ACT == BGNN_ACT_SIGMOID) {
    const float g = sigmoid_t(-LOG2E * z);
    return make_float2(g, g * sigmoid_t(LOG2E * z));
  }
  if constexpr (ACT == BGNN_ACT_TANH) {
    const float t = tanhf(z);
    return make_float2(t, (1.0f - t) * (1.0f + t));
  }
  return make_float2(z, 1.0f);
}
template <int ACT>
__device__ __forceinline__ void act_grad_two(float2 z, float p, float2& f0, float2& f1) {
  float2 s = make_float2(0.0f, 0.0f);
  if constexpr (GATES<ACT>) s = sigmoid_t2(gate_t2<ACT>(z));
  f0 = act_grad<ACT>(z.x, s.x, p);
  f1 = act_grad<ACT>(z.y, s.y, p);
}
// Runs f(Act<..>) for an activation known at run time.  One branch a chunk of
// 32 elements: the switch inside the element loop made the code of every
// activation part of every element (7.8 ms instead of 2.45 at 2.45M x 256 -> 512).
template <int ACT>
using Act = std::integral_constant<int, ACT>;
template <class F>
__device__ __forceinline__ void with_act(int act, F&& f) {
  switch (act) {
    case BGNN_ACT_RELU: f(Act<BGNN_ACT_RELU>{}); break;
    case BGNN_ACT_RELU_MAX: f(Act<BGNN_ACT_RELU_MAX>{}); break;
    case BGNN_ACT_ELU: f(Act<BGNN_ACT_ELU>{}); break;
    case BGNN_ACT_LEAKY_RELU: f(Act<BGNN_ACT_LEAKY_RELU>{}); break;
    case BGNN_ACT_SIGMOID: f(Act<BGNN_ACT_SIGMOID>{}); break;
    case BGNN_ACT_TANH: f(Act<BGNN_ACT_TANH>{}); break;
    case BGNN_ACT_GELU: f(Act<BGNN_ACT_GELU>{}); break;
    case BGNN_ACT_SILU: f(Act<BGNN_ACT_SILU>{}); break;
    default: f(Act<BGNN_ACT_NONE>{}); break;
  }
}
