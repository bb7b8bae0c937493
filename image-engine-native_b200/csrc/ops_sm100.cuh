// Device helpers shared by the single operators: value types, activations
// and e4m3 codes.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>
#include <type_traits>

#include "ops.h"
#include "sm100.cuh"

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

__device__ __forceinline__ float op_ex2(float t) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return e;
}
__device__ __forceinline__ float op_rcp(float d) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// Two products, those below 2^-126 as zeros.
__device__ __forceinline__ float2 fmul2_ftz(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.ftz.f32x2 %0, %1, %2;" : "=l"(d) : "l"(pack_f32x2(a.x, a.y)), "l"(pack_f32x2(b.x, b.y)));
  return unpack_f32x2(d);
}

// The sigmoids 1 / d, d = 1 + e^-v, of two values for results of 8 and 16
// bits, on packed pairs (their instructions bound these kernels next to memory)
// and with one reciprocal r for both (the unit for exponentials and reciprocals
// has an eighth of the multiplies' rate: with one each, 4 x 64 x 64 x 512 f16
// takes 12.5 us instead of 11.9). With u = 2^-126,
//   1 / d0 = (d1 u) r,  1 / d1 = (d0 u) r,  r = 1 / (d0 (d1 u)),
// which stay in f32's range for all d up to 2^126.5, where v is clamped. They
// are good to 2^-20 of themselves up to |v| = 8, to 2^-18 up to 87 (v log2(e) is
// rounded once), and 0 below -87.3, where they are less than 2^-126; of a NaN
// they are 0 too. Quantised, no more e4m3 codes come out beside the nearest one
// than with exact exponentials and quotients in f32 (SiLU of 4 x 128 x 128 x 256
// values: 26 and 34 of 16.8 M).
__device__ __forceinline__ float2 op_sigmoid_pair(float2 v) {
  const float2 t = fmul2(make_float2(fmaxf(v.x, -87.68f), fmaxf(v.y, -87.68f)), both(-1.4426950408889634f));
  const float2 e = make_float2(op_ex2(t.x), op_ex2(t.y));
  const float2 d = fadd2(e, both(1.0f)), du = fmul2(d, both(0x1p-126f));
  return fmul2_ftz(make_float2(du.y, du.x), both(op_rcp(d.x * du.y)));
}

// GELU = v Phi(v) of two values for results of 16 bits, as max(v, 0) - a
// Phi(-a), a = |v|. Phi(-a) = 2^(s(a) - a^2 log2(e) / 2), where s = log2(e^(a^2 /
// 2) Phi(-a)) goes from -1 to -5 over 0 to 13.2 and is a polynomial here, fitted
// to it (least largest error, by linear programming over 1500 Chebyshev points):
// good to 2^-14 of Phi(-a) and better. For f16 up to a = 5.85, where a Phi(-a) is
// less than half its smallest step; for bf16 up to 13.2, and 0 beyond, below
// 2^-126. (With a degree less the tails are off by 2^-11 and 2^-13 of themselves.)
// A quarter to a third of erfcf's instructions. NaN stays NaN.
template <class R>
__device__ __forceinline__ float2 op_gelu_pair(float2 v) {
  constexpr bool F16 = std::is_same<R, __half>::value;
  constexpr float most = F16 ? 5.85f : 13.2f;
  const float2 m = make_float2(fmaxf(-fabsf(v.x), -most), fmaxf(-fabsf(v.y), -most));  // -a
  float2 s;
  if constexpr (F16) {
    s = ffma2(both(1.831785198e-6f), m, both(6.154859875e-5f));
    s = ffma2(s, m, both(9.302141261e-4f));
    s = ffma2(s, m, both(8.506965823e-3f));
    s = ffma2(s, m, both(5.395872518e-2f));
    s = ffma2(s, m, both(2.628822327e-1f));
    s = ffma2(s, m, both(1.151250839f));
    s = ffma2(s, m, both(-9.999953508e-1f));
  } else {
    s = ffma2(both(1.923425197e-9f), m, both(1.403363541e-7f));
    s = ffma2(s, m, both(4.502811407e-6f));
    s = ffma2(s, m, both(8.410552982e-5f));
    s = ffma2(s, m, both(1.024093712e-3f));
    s = ffma2(s, m, both(8.679608814e-3f));
    s = ffma2(s, m, both(5.398480967e-2f));
    s = ffma2(s, m, both(2.625868917e-1f));
    s = ffma2(s, m, both(1.150994f));
    s = ffma2(s, m, both(-1.000029564f));
  }
  s = ffma2(fmul2(m, both(-0.72134752f)), m, s);
  return ffma2(m, make_float2(op_ex2(s.x), op_ex2(s.y)), make_float2(max_nan(v.x, 0.0f), max_nan(v.y, 0.0f)));
}

// The same for results of 8 and 32 bits, with Phi(-a) = e^(-a^2 / 2) t q(y), t
// = 1 / (1 + p a), y = p a t, and q a polynomial fitted in the same way (to
// 2^-26) with q(0) = 1 / 2. Good to 2^-20 of Phi(-a) up to a = 4, 2^-18 up to 6,
// 2^-16 up to 13.2, since the exponent is rounded, and 0 beyond; v (1 + erf(v /
// sqrt 2)) / 2 in f32 is off by 2^-10 of itself at -4. 8 x 128 x 128 x 256 f16 to
// e4m3: 58 us (68 with erff, 89 with erfcf), 26 codes of 16.8 M beside the nearest
// one in 4 x 128 x 128 x 256 (38 with erff); a product of 8192 x 4096 x 1024 to
// f32: 75 us (155 with erfcf).
__device__ __forceinline__ float2 op_gelu_pair_32(float2 v) {
  const float2 m = make_float2(fmaxf(-fabsf(v.x), -13.3f), fmaxf(-fabsf(v.y), -13.3f));  // -a
  const float2 pa = fmul2(m, both(-0.264f)), d = fadd2(pa, both(1.0f));
  const float2 t = make_float2(op_rcp(d.x), op_rcp(d.y)), y = fmul2(pa, t);
  const float2 x = fmul2(fmul2(m, m), both(-0.72134752f));
  float2 q = ffma2(both(3.112974390e-2f), y, both(-1.013756022e-1f));
  q = ffma2(q, y, both(6.575393677e-2f));
  q = ffma2(q, y, both(1.177721322e-1f));
  q = ffma2(q, y, both(-6.130456924e-2f));
  q = ffma2(q, y, both(-5.002308488e-1f));
  q = ffma2(q, y, both(1.064747930f));
  q = ffma2(q, y, both(-1.011145711f));
  q = ffma2(q, y, both(0.5f));
  const float2 g = fmul2(make_float2(op_ex2(x.x), op_ex2(x.y)), t);
  return ffma2(m, fmul2(q, g), make_float2(max_nan(v.x, 0.0f), max_nan(v.y, 0.0f)));
}

// The activation of N values for results of type R (uint8_t: e4m3 codes). The
// products that end an activation are not contracted with what is added to
// them, so that every kernel and path rounds the same. NaN stays NaN.
template <int ACT, class R, int N>
__device__ __forceinline__ void op_act_vec(float* v) {
  constexpr bool SHORT = sizeof(R) == 2;
  if constexpr (ACT == OP_RELU) {
#pragma unroll
    for (int e = 0; e < N; e++) v[e] = v[e] < 0.0f ? 0.0f : v[e];
  } else if constexpr (ACT != OP_NONE && ACT != OP_GELU && sizeof(R) == 4) {
    // A reciprocal each (of what is above 2^126 it is 0): no value's last bits
    // depend on its neighbour's.
#pragma unroll
    for (int e = 0; e < N; e++) {
      const float s = op_rcp(1.0f + expf(-v[e]));
      v[e] = ACT == OP_SILU ? __fmul_rn(v[e], s) : s;
    }
  } else if constexpr (ACT != OP_NONE) {
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const float2 x = make_float2(v[e], v[N == 1 ? e : e + 1]);
      float2 y;
      if constexpr (ACT == OP_GELU && SHORT)
        y = op_gelu_pair<R>(x);
      else if constexpr (ACT == OP_GELU)
        y = op_gelu_pair_32(x);
      else
        y = op_sigmoid_pair(x);
      if constexpr (ACT == OP_SILU) y = fmul2(x, y);
      if constexpr (ACT == OP_SIGMOID) y = make_float2(x.x != x.x ? x.x : y.x, x.y != x.y ? x.y : y.y);
      v[e] = y.x;
      if (N > 1) v[e + 1] = y.y;
    }
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

// max(|a|, b), NaN if one of them is.
__device__ __forceinline__ float max_abs(float a, float b) {
  float m;
  asm("{\n\t.reg .f32 t;\n\tabs.f32 t, %1;\n\tmax.NaN.f32 %0, t, %2;\n\t}" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

constexpr int FP8_BLOCK = 128;  // values along k that share a scale

// The magnitudes' bits order as unsigned integers the way the magnitudes do,
// with infinity above every finite value and NaN above infinity, so an
// integer maximum keeps both.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// A block's factor (values to codes) and scale (codes to values) from its
// largest magnitude: 448 / amax and amax / 448, or 1 and 1 below 2^-100, where
// the factor would leave f32's range and every code rounds to zero. Each is a
// product with an approximate reciprocal and one correction by the quotient's
// remainder (Markstein), which an fma gives without rounding: as good as a
// division to within 2^-24 of half a unit, for all 128 values of a block, at a
// quarter of the instructions of its general form. Where the reciprocal or amax
// is not a normal number the division itself.
__device__ __forceinline__ void fp8_scale(uint32_t amax_bits, float* factor, float* scale) {
  const float amax = __uint_as_float(amax_bits), r = op_rcp(amax), q = 448.0f * r, s = amax * (1.0f / 448.0f);
  *factor = fmaf(fmaf(-amax, q, 448.0f), r, q);
  *scale = fmaf(fmaf(-448.0f, s, amax), 1.0f / 448.0f, s);
  if (!(amax <= 8.0e37f)) {  // also infinity and NaN
    *factor = 448.0f / amax;
    *scale = amax / 448.0f;
  }
  if (amax < 7.888609052210118e-31f) *factor = *scale = 1.0f;  // 2^-100
}

// Two values to two e4m3 codes (`lo` in the low byte), round to nearest
// even. The factor puts every value within 448 (1 + 2^-22), which rounds to
// 448; NaN (also 0 * inf of an infinite value) becomes the NaN code.
__device__ __forceinline__ uint16_t e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// VE values of T next to each other: 16 bytes where the map has a multiple
// of them as channels (AL: its base and strides let them be read at once),
// else one value.
template <class T, int VE, bool AL>
struct Vec {
  using Raw = std::conditional_t<VE == 1, T, uint4>;
  static __device__ __forceinline__ Raw zero() {
    if constexpr (VE == 1)
      return from_f32<T>(0.0f);
    else
      return make_uint4(0, 0, 0, 0);
  }
  static __device__ __forceinline__ Raw fetch(const T* p) {
    if constexpr (VE == 1 || AL) {
      return *reinterpret_cast<const Raw*>(p);
    } else {
      T v[VE];
#pragma unroll
      for (int e = 0; e < VE; e++) v[e] = p[e];
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4)
          w[i] = __float_as_uint(v[i]);
        else
          w[i] = (uint32_t) reinterpret_cast<const uint16_t&>(v[2 * i]) |
                 (uint32_t) reinterpret_cast<const uint16_t&>(v[2 * i + 1]) << 16;
      }
      return make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  static __device__ __forceinline__ void expand(Raw q, float* v) {
    if constexpr (VE == 1) {
      v[0] = to_f32(q);
    } else {
      expand_16(q, v);
    }
  }
  // The values of the i-th 32-bit word (VE 1: the one value).
  static __device__ __forceinline__ void word(Raw q, int i, float* v) {
    if constexpr (VE == 1) {
      v[0] = to_f32(q);
    } else {
      const uint32_t w = i == 0 ? q.x : i == 1 ? q.y : i == 2 ? q.z : q.w;
      if constexpr (sizeof(T) == 4) {
        v[0] = __uint_as_float(w);
      } else {
        const uint16_t lo = (uint16_t)(w & 0xffffu), hi = (uint16_t)(w >> 16);
        v[0] = to_f32(reinterpret_cast<const T&>(lo));
        v[1] = to_f32(reinterpret_cast<const T&>(hi));
      }
    }
  }
  // Channels 2 i and 2 i + 1 (VE 1: the one value, twice).
  static __device__ __forceinline__ float2 pair(Raw q, int i) {
    float v[2];
    if constexpr (VE == 1) {
      v[0] = v[1] = to_f32(q);
    } else if constexpr (VE == 8) {
      word(q, i, v);
    } else {
      word(q, 2 * i, v);
      word(q, 2 * i + 1, v + 1);
    }
    return make_float2(v[0], v[1]);
  }
  static __device__ __forceinline__ void expand_16(uint4 q, float* v) {
#pragma unroll
    for (int i = 0; i < 4; i++) word(q, i, v + i * (VE / 4));
  }
  static __device__ __forceinline__ void store(T* p, const float* v) {
    if constexpr (VE == 1 || !AL) {
#pragma unroll
      for (int e = 0; e < VE; e++) p[e] = from_f32<T>(v[e]);
    } else if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      *reinterpret_cast<uint4*>(p) =
          make_uint4(pack_2<T>(v[0], v[1]), pack_2<T>(v[2], v[3]), pack_2<T>(v[4], v[5]), pack_2<T>(v[6], v[7]));
    }
  }
};

}  // namespace iec
