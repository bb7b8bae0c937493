// Device helpers shared by the single operators: value types, activations
// and e4m3 codes.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>
#include <type_traits>

#include "ops.h"

namespace iec {

__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }

template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }

// Two values rounded to T in one instruction (single conversions go through
// a unit with an eighth of the rate).
template <class T>
__device__ __forceinline__ uint32_t pack_2(float lo, float hi) {
  uint32_t v;
  if constexpr (std::is_same<T, __half>::value)
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
  return v;
}

// Activations. Two kinds of accuracy: FAST for results that are rounded to 16
// bits (a few units of f32), exact to about one unit for f32 results and for
// values that are quantised (where every unit moves more of them across a
// rounding boundary).
//
// e^-v for -43.6 <= v: t = -v log2(e), 2^t by the special-function unit, and
// for the exact kind the rounding of t put back: 2^(t + d) = 2^t (1 + d ln 2).
// Arguments are clamped from below, where v / (1 + e^-v) is less than 1e-17
// either way, so that two denominators multiply without overflow
// (op_sigmoid_pair), and for the exact kind from above, where 1 + e^-v is 1.
template <bool FAST>
__device__ __forceinline__ float op_exp_neg(float v) {
  v = fmaxf(v, -43.6f);
  if (!FAST) v = fminf(v, 87.0f);
  constexpr float L = -1.4426950408889634f, L_LO = -1.925963033500e-8f;  // log2(e) = -(L + L_LO)
  const float t = v * L;
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  if (!FAST) e = fmaf(e * 0.6931471805599453f, fmaf(v, L_LO, fmaf(v, L, -t)), e);
  return e;
}

// 1 / d; one Newton step for the exact kind.
template <bool FAST>
__device__ __forceinline__ float op_rcp(float d) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  if (!FAST) r = fmaf(r, fmaf(-d, r, 1.0f), r);
  return r;
}

template <bool FAST>
__device__ __forceinline__ float op_sigmoid(float v) { return op_rcp<FAST>(1.0f + op_exp_neg<FAST>(v)); }

// Two sigmoids by one reciprocal, of the denominators' product: the unit for
// exponentials and reciprocals has an eighth of the multiplies' rate and
// bounds these activations.
template <bool FAST>
__device__ __forceinline__ void op_sigmoid_pair(float v, float w, float* sv, float* sw) {
  const float a = 1.0f + op_exp_neg<FAST>(v), b = 1.0f + op_exp_neg<FAST>(w), r = op_rcp<FAST>(a * b);
  *sv = r * b;
  *sw = r * a;
}

// GELU for FAST, as max(v, 0) - |v| / (2 P^16) (igemm_sm100.cuh); |error| at
// most 1.5e-7 |v|.
__device__ __forceinline__ float op_gelu_fast(float v) {
  const float av = fabsf(v), a = av * 0.70710678118654752f;
  float q = fmaf(fmaf(fmaf(fmaf(fmaf(fmaf(4.30638e-5f, a, 2.765672e-4f), a, 1.520143e-4f), a, 9.2705272e-3f), a,
                          4.22820123e-2f),
                     a, 7.05230784e-2f),
                a, 1.0f);
  q *= q;
  q *= q;
  q *= q;
  q *= q;
  return fmaf(-0.5f * av, op_rcp<true>(q), fmaxf(v, 0.0f));
}

// The activation of N values. The products that end an activation are not
// contracted with what is added to them, so that every kernel and path
// rounds the same. NaN stays NaN.
template <int ACT, bool FAST, int N>
__device__ __forceinline__ void op_act_vec(float* v) {
  if constexpr (ACT == OP_RELU) {
#pragma unroll
    for (int e = 0; e < N; e++) v[e] = v[e] < 0.0f ? 0.0f : v[e];
  } else if constexpr (ACT == OP_GELU) {
#pragma unroll
    for (int e = 0; e < N; e++)
      v[e] = FAST ? op_gelu_fast(v[e]) : __fmul_rn(0.5f * v[e], 1.0f + erff(v[e] * 0.70710678118654752f));
  } else if constexpr (ACT == OP_SIGMOID || ACT == OP_SILU) {
    float s[N];
    if constexpr (N % 2 == 0) {
#pragma unroll
      for (int e = 0; e < N; e += 2) op_sigmoid_pair<FAST>(v[e], v[e + 1], &s[e], &s[e + 1]);
    } else {
#pragma unroll
      for (int e = 0; e < N; e++) s[e] = op_sigmoid<FAST>(v[e]);
    }
#pragma unroll
    for (int e = 0; e < N; e++) v[e] = ACT == OP_SILU ? __fmul_rn(v[e], s[e]) : v[e] != v[e] ? v[e] : s[e];
  }
}

// Calls f(std::integral_constant<int, ACT>()) for the activation `act`: the
// choice is made once, outside the loops over values.
template <class F>
__device__ __forceinline__ void op_act_switch(int act, F&& f) {
  switch (act) {
    case OP_RELU: f(std::integral_constant<int, OP_RELU>()); break;
    case OP_GELU: f(std::integral_constant<int, OP_GELU>()); break;
    case OP_SIGMOID: f(std::integral_constant<int, OP_SIGMOID>()); break;
    case OP_SILU: f(std::integral_constant<int, OP_SILU>()); break;
    default: f(std::integral_constant<int, OP_NONE>());
  }
}

constexpr int FP8_BLOCK = 128;  // values along k that share a scale

// The magnitudes' bits order as unsigned integers the way the magnitudes do,
// with infinity above every finite value and NaN above infinity, so an
// integer maximum keeps both where fmaxf would drop a NaN.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// A block's factor (values to codes) and scale (codes to values) from its
// largest magnitude: 448 / amax and amax / 448, or 1 and 1 below 2^-100,
// where the factor would leave f32's range and every code rounds to zero.
__device__ __forceinline__ void fp8_scale(uint32_t amax_bits, float* factor, float* scale) {
  const float amax = __uint_as_float(amax_bits);
  const bool tiny = amax < 7.888609052210118e-31f;  // 2^-100; false for NaN
  *factor = tiny ? 1.0f : 448.0f / amax;
  *scale = tiny ? 1.0f : amax / 448.0f;
}

// Two values to two e4m3 codes (`lo` in the low byte), round to nearest
// even. The factor puts every value within 448 (1 + 2^-22), which rounds to
// 448; NaN (also 0 * inf of an infinite value) becomes the NaN code.
__device__ __forceinline__ uint16_t e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

}  // namespace iec
