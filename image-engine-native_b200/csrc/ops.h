// Single operators for networks built next to the models: group
// normalisation over channels-last maps (ops_norm.cu), e4m3 quantisation
// (ops_quant.cu) and the block-scaled e4m3 product (ops_fp8.cu). Arguments
// are checked here and in capi.cpp; everything is queued on the caller's
// stream.
#pragma once

#include "runtime.h"

namespace iec {

enum DType { DT_F16 = 0, DT_BF16 = 1, DT_F32 = 2 };
enum OpAct { OP_NONE = 0, OP_RELU = 1, OP_GELU = 2, OP_SIGMOID = 3, OP_SILU = 4 };
inline size_t dtype_bytes(int t) { return t == DT_F32 ? 4 : 2; }

// 8-bit rows: codes (row stride in bytes) and the scales of their blocks of
// 128 (block b of row r, or of 128 rows r, at scales[b * scale_stride + r]).
struct Fp8Out {
  uint8_t* codes = nullptr;
  size_t code_stride = 0;
  float* scales = nullptr;
  size_t scale_stride = 0;
};

struct NormSpec {
  const void* x = nullptr;
  int dtype = DT_F16;
  int n = 0, c = 0, groups = 1;
  long long pixels = 0;
  long long x_stride = 0, x_map_stride = 0;
  const float* gamma = nullptr;
  const float* beta = nullptr;
  float eps = 0;
  int act = OP_NONE;
  void* out = nullptr;  // null: quantised to `q`
  long long out_stride = 0, out_map_stride = 0;
  Fp8Out q;
};
void group_norm(Device& dev, const NormSpec& spec, cudaStream_t s);

struct QuantSpec {
  const void* x = nullptr;
  int dtype = DT_F16;
  long long rows = 0, x_stride = 0;
  int k = 0, block_rows = 1;
  Fp8Out q;
};
void quantize_fp8(Device& dev, const QuantSpec& spec, cudaStream_t s);

struct Fp8MatmulSpec {
  const uint8_t* a = nullptr;
  const uint8_t* w = nullptr;
  const float* a_scales = nullptr;
  const float* w_scales = nullptr;
  long long a_stride = 0, w_stride = 0, a_scale_stride = 0, w_scale_stride = 0;
  const float* bias = nullptr;
  const void* residual = nullptr;
  void* out = nullptr;
  long long residual_stride = 0, out_stride = 0;
  int m = 0, n = 0, k = 0, act = OP_NONE, dtype = DT_F16;
};
void matmul_fp8(Device& dev, const Fp8MatmulSpec& spec, cudaStream_t s);

}  // namespace iec
