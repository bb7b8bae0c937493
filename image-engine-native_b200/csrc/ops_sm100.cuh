// Device helpers shared by the single operators: value types, activations
// and e4m3 codes.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

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

// 1 / (1 + e^-v). e^-v overflows to infinity for v below about -88, whose
// reciprocal is the limit 0.
__device__ __forceinline__ float op_sigmoid(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }

// The products that end an activation are not contracted with what is added
// to them, so that every kernel and path rounds the same.
template <int ACT>
__device__ __forceinline__ float op_act(float v) {
  if (ACT == OP_RELU) return v < 0.0f ? 0.0f : v;  // NaN stays
  if (ACT == OP_GELU) return __fmul_rn(0.5f * v, 1.0f + erff(v * 0.70710678118654752f));
  if (ACT == OP_SIGMOID) return op_sigmoid(v);
  if (ACT == OP_SILU) return __fmul_rn(v, op_sigmoid(v));
  return v;
}

__device__ __forceinline__ float op_act_any(float v, int act) {
  if (act == OP_RELU) return op_act<OP_RELU>(v);
  if (act == OP_GELU) return op_act<OP_GELU>(v);
  if (act == OP_SIGMOID) return op_act<OP_SIGMOID>(v);
  if (act == OP_SILU) return op_act<OP_SILU>(v);
  return v;
}

// The activation of N values, one branch for all of them.
template <int N>
__device__ __forceinline__ void op_act_n(float* v, int act) {
#define IEC_OP_ACT(A_)                                  \
  if (act == A_) {                                      \
    _Pragma("unroll") for (int e = 0; e < N; e++) v[e] = op_act<A_>(v[e]); \
  }
  IEC_OP_ACT(OP_RELU)
  else IEC_OP_ACT(OP_GELU)
  else IEC_OP_ACT(OP_SIGMOID)
  else IEC_OP_ACT(OP_SILU)
#undef IEC_OP_ACT
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
