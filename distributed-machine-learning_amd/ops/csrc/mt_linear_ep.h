// What the dense layer's kernels (linear_ep.hip) do to an accumulator: y = act(acc + bias) + residual in f32, rounded once;
// z = acc + bias is kept when the backward pass needs it.
#pragma once
#include "mt_common.h"

#define MT_ACT_NONE 0
#define MT_ACT_RELU 1
#define MT_ACT_GELU 2
struct MtLinearEp {
  const void* bias;        // [J] f32, or bf16 with bias_bf16; may be null
  const void* residual;    // [I][ldr], the output's type; may be null
  void* z;                 // [I][ldz], the output's type; may be null
  int32_t bias_bf16, act, ldr, ldz;
};
__device__ __forceinline__ float mt_ep_bias(const MtLinearEp& ep, int col) {
  return ep.bias_bf16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(ep.bias)[col])
                      : reinterpret_cast<const float*>(ep.bias)[col];
}
__device__ __forceinline__ float mt_ep_act(float v, int act) {
  if (act == MT_ACT_RELU) return v < 0.f ? 0.f : v;                                   // NaN stays NaN
  if (act == MT_ACT_GELU) return 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
  return v;
}

// d act(z) / dz
__device__ __forceinline__ float mt_ep_slope(float z, int act) {
  if (act == MT_ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if (act == MT_ACT_GELU)
    return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * 0.39894228040143268f * __expf(-0.5f * z * z);
  return 1.f;
}
