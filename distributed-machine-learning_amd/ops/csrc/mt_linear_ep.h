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
// Phi(z) = 0.5 (1 + erf(z / sqrt 2)), with e = exp(-z^2 / 2).  The lower tail is computed as such, Phi(-a) = P(t) e with
// t = 1 / (1 + p a), and the upper is 1 less it: where 0.5 (1 + erf) is a difference of nearly equal numbers (f32: up to 5 % off at
// z = -5, all of it at -5.6) a product keeps its relative precision.  P is a minimax fit of exp(a^2 / 2) Phi(-a) on 0 <= a <= 14, made
// for these kernels.  SHORT, for values that end up in bf16: seven terms, within 2e-7, and below z = 0 within 1e-5 of Phi itself (most
// of it the rounding of the exponent), a four-hundredth of a bf16 step.  Otherwise ten terms and an exponent that keeps what rounding
// took off it: within 9 units of 2^-24 of Phi below 0, of 1 above.  No branches: the epilogue of a 256-tile runs this 128 times per
// lane with nothing to hide behind.
template <bool SHORT> __device__ __forceinline__ float mt_ep_phi(float z, float& e) {
  constexpr float HALF_LOG2E = 0.72134752f, REST = 9.6298e-9f, LN2 = 0.69314718f;
  float a = fabsf(z), v;
  if constexpr (SHORT) {
    e = __builtin_amdgcn_exp2f(-HALF_LOG2E * z * z);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.35f, a, 1.f));
    v = __builtin_fmaf(0.04461544f, t, -0.18442905f);
    v = __builtin_fmaf(v, t, 0.21108223f);
    v = __builtin_fmaf(v, t, 0.00892729f);
    v = __builtin_fmaf(v, t, 0.14315635f);
    v = __builtin_fmaf(v, t, 0.13687132f);
    v = __builtin_fmaf(v, t, 0.13977645f) * t;
  } else {
    a = fminf(a, 15.f);                      // e = 0 from there on, and infinity is no number less itself
    const float s = a * a, h = -HALF_LOG2E * s;
    const float left = __builtin_fmaf(-HALF_LOG2E, s, -h) - __builtin_fmaf(REST, s, HALF_LOG2E * __builtin_fmaf(a, a, -s));
    e = __builtin_amdgcn_exp2f(h);
    e = __builtin_fmaf(e * LN2, left, e);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.375f, a, 1.f));
    v = __builtin_fmaf(0.0208994f, t, -0.1340013f);
    v = __builtin_fmaf(v, t, 0.34483624f);
    v = __builtin_fmaf(v, t, -0.42400947f);
    v = __builtin_fmaf(v, t, 0.21556373f);
    v = __builtin_fmaf(v, t, -0.05615849f);
    v = __builtin_fmaf(v, t, 0.10810973f);
    v = __builtin_fmaf(v, t, 0.12528306f);
    v = __builtin_fmaf(v, t, 0.14988403f);
    v = __builtin_fmaf(v, t, 0.14959307f) * t;
  }
  return z < 0.f ? v * e : __builtin_fmaf(-v, e, 1.f);
}
template <bool SHORT> __device__ __forceinline__ float mt_ep_act(float v, int act) {
  if (act == MT_ACT_RELU) return v < 0.f ? 0.f : v;                                   // NaN stays NaN
  if (act == MT_ACT_GELU) {
    float e;
    return v * mt_ep_phi<SHORT>(v, e);
  }
  return v;
}

// f(MtAct<the launch's activation>): the loops over an accumulator are there once per activation, each a
// straight run of instructions (asked per element, a small launch spends its time fetching code around the branches not taken).
template <int N> struct MtAct { static constexpr int value = N; };
template <typename F> __device__ __forceinline__ void mt_ep_for_act(int act, F&& f) {
  if (act == MT_ACT_GELU) f(MtAct<MT_ACT_GELU>{});
  else if (act == MT_ACT_RELU) f(MtAct<MT_ACT_RELU>{});
  else f(MtAct<MT_ACT_NONE>{});
}

// d act(z) / dz
template <bool SHORT> __device__ __forceinline__ float mt_ep_slope(float z, int act) {
  if (act == MT_ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if (act == MT_ACT_GELU) {
    float e;
    const float phi = mt_ep_phi<SHORT>(z, e);
    return __builtin_fmaf(z * 0.39894228040143268f, e, phi);
  }
  return 1.f;
}
