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
  float* part;             // [I][J] f32: the bare accumulators go here instead (one part of a split contraction); may be null
  int32_t bias_bf16, act, ldr, ldz;
};
__device__ __forceinline__ float mt_ep_bias(const MtLinearEp& ep, int col) {
  return ep.bias_bf16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(ep.bias)[col])
                      : reinterpret_cast<const float*>(ep.bias)[col];
}
// Four accumulator columns of a row, at whatever alignment the row has; columns past J are left alone.
__device__ __forceinline__ void mt_ep_put_part(float* part, int64_t row, int col, int J, f32x4 v) {
  float* p = part + row * J + col;
  if (col + 4 <= J) {
    __builtin_memcpy(p, &v, 16);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col + j < J) p[j] = v[j];
  }
}
__device__ __forceinline__ void mt_ep_put_db(void* db, int row, float v, int bf16) {
  if (bf16) reinterpret_cast<uint16_t*>(db)[row] = (uint16_t)f32_to_bf16_bits(v);
  else reinterpret_cast<float*>(db)[row] = v;
}
// erf for values that end up in bf16: 1 - (a1 t + ... + a5 t^5) exp(-x^2), t = 1 / (1 + 0.3275911 |x|), Abramowitz and Stegun
// 7.1.26, off by at most 1.5e-7: a hundredth of a bf16 step of gelu wherever that is not already below 1e-6 of its input.
// A third of erff's instructions, which the epilogue of a 256-tile runs 128 times per lane with nothing to hide behind.
__device__ __forceinline__ float mt_erf_short(float x) {
  const float a = fabsf(x);
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, a, 1.f));
  float p = __builtin_fmaf(1.061405429f, t, -1.453152027f);
  p = __builtin_fmaf(p, t, 1.421413741f);
  p = __builtin_fmaf(p, t, -0.284496736f);
  p = __builtin_fmaf(p, t, 0.254829592f);
  const float e = __builtin_amdgcn_exp2f(-1.4426950408889634f * x * x);
  return copysignf(__builtin_fmaf(-p * t, e, 1.f), x);
}
template <bool SHORT> __device__ __forceinline__ float mt_ep_act(float v, int act) {
  if (act == MT_ACT_RELU) return v < 0.f ? 0.f : v;                                   // NaN stays NaN
  if (act == MT_ACT_GELU) {
    const float r = v * 0.70710678118654752f;
    return 0.5f * v * (1.f + (SHORT ? mt_erf_short(r) : erff(r)));
  }
  return v;
}

// d act(z) / dz
template <bool SHORT> __device__ __forceinline__ float mt_ep_slope(float z, int act) {
  if (act == MT_ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if (act == MT_ACT_GELU) {
    const float r = z * 0.70710678118654752f;
    return 0.5f * (1.f + (SHORT ? mt_erf_short(r) : erff(r))) + z * 0.39894228040143268f * __expf(-0.5f * z * z);
  }
  return 1.f;
}
