// Rows of 16- or 32-bit values to e4m3 codes with an f32 scale for each
// block of 128 values of a row (activations), or of 128 rows and 128 values
// (weights).
#include "ops_sm100.cuh"

namespace iec {

namespace {

// One warp per row and block.
template <class T>
__global__ void __launch_bounds__(256) quant_rows(QuantSpec p) {
  const int kb = (p.k + FP8_BLOCK - 1) / FP8_BLOCK, lane = threadIdx.x & 31;
  const long long total = p.rows * kb;
  for (long long t = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); t < total; t += (long long)gridDim.x * 8) {
    const long long row = t / kb;
    const int b = (int)(t - row * kb);
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    float v[4];
    uint32_t top = 0;
    for (int j = 0; j < 4; j++) {
      const int ch = b * FP8_BLOCK + j * 32 + lane;
      v[j] = ch < p.k ? to_f32(x[ch]) : 0.0f;
      top = max(top, abs_bits(v[j]));
    }
    top = __reduce_max_sync(~0u, top);
    float factor, scale;
    fp8_scale(top, &factor, &scale);
    for (int j = 0; j < 4; j++) {
      const int ch = b * FP8_BLOCK + j * 32 + lane;
      if (ch < p.k) p.q.codes[row * p.q.code_stride + ch] = (uint8_t)e4m3x2(v[j] * factor, 0.0f);
    }
    if (lane == 0) p.q.scales[b * p.q.scale_stride + row] = scale;
  }
}

// One CTA per block of 128 x 128, read twice.
template <class T>
__global__ void __launch_bounds__(256) quant_blocks(QuantSpec p) {
  __shared__ uint32_t red[8];
  const int b = blockIdx.x, rb = blockIdx.y;
  const int col = b * FP8_BLOCK + (threadIdx.x & 127);
  uint32_t top = 0;
  for (int r = threadIdx.x >> 7; r < FP8_BLOCK; r += 2) {
    const long long row = (long long)rb * FP8_BLOCK + r;
    if (row < p.rows && col < p.k) top = max(top, abs_bits(to_f32(static_cast<const T*>(p.x)[row * p.x_stride + col])));
  }
  top = __reduce_max_sync(~0u, top);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
  __syncthreads();
  for (int i = 0; i < 8; i++) top = max(top, red[i]);
  float factor, scale;
  fp8_scale(top, &factor, &scale);
  for (int r = threadIdx.x >> 7; r < FP8_BLOCK; r += 2) {
    const long long row = (long long)rb * FP8_BLOCK + r;
    if (row < p.rows && col < p.k)
      p.q.codes[row * p.q.code_stride + col] =
          (uint8_t)e4m3x2(to_f32(static_cast<const T*>(p.x)[row * p.x_stride + col]) * factor, 0.0f);
  }
  if (threadIdx.x == 0) p.q.scales[b * p.q.scale_stride + rb] = scale;
}

template <class T>
void run(Device& dev, const QuantSpec& p, cudaStream_t s) {
  const int kb = (p.k + FP8_BLOCK - 1) / FP8_BLOCK;
  const double values = (double)p.rows * p.k;
  timed_launch("quantize_fp8", 2 * values, values * (sizeof(T) + 1), s, [&] {
    if (p.block_rows == 1)
      quant_rows<T><<<dev.sms() * 8, 256, 0, s>>>(p);
    else
      quant_blocks<T><<<dim3(kb, (unsigned)((p.rows + FP8_BLOCK - 1) / FP8_BLOCK)), 256, 0, s>>>(p);
    IEC_CUDA(cudaGetLastError());
  });
}

}  // namespace

void quantize_fp8(Device& dev, const QuantSpec& p, cudaStream_t s) {
  if (p.rows == 0 || p.k == 0) return;
  if (p.dtype == DT_F16) return run<__half>(dev, p, s);
  if (p.dtype == DT_BF16) return run<__nv_bfloat16>(dev, p, s);
  run<float>(dev, p, s);
}

}  // namespace iec
