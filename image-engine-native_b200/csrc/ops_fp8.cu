// The block-scaled e4m3 product: out = act(a w^T + bias) + residual, with
// a[m][k] w[n][k] summed per block of 128 along k, multiplied by the block's
// two scales and added up in f32.
#include "ops_sm100.cuh"

namespace iec {

namespace {

__device__ __forceinline__ float e4m3_f32(uint8_t code) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(code, __NV_E4M3)));
}

// 64 x 64 outputs per CTA, 4 x 4 per thread, K steps of 16.
template <class T>
__global__ void __launch_bounds__(256) matmul_simple(Fp8MatmulSpec p) {
  __shared__ float sa[16][65], sw[16][65];
  const int m0 = blockIdx.x * 64, n0 = blockIdx.y * 64;
  const int tm = threadIdx.x / 16, tn = threadIdx.x % 16;
  float acc[4][4] = {}, part[4][4] = {};
  for (int k0 = 0; k0 < p.k; k0 += 16) {
    for (int e = threadIdx.x; e < 1024; e += 256) {
      const int r = e / 16, kk = k0 + e % 16;
      sa[e % 16][r] = m0 + r < p.m && kk < p.k ? e4m3_f32(p.a[(m0 + r) * p.a_stride + kk]) : 0.0f;
      sw[e % 16][r] = n0 + r < p.n && kk < p.k ? e4m3_f32(p.w[(n0 + r) * p.w_stride + kk]) : 0.0f;
    }
    __syncthreads();
    for (int kk = 0; kk < 16; kk++)
      for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) part[i][j] = fmaf(sa[kk][tm + 16 * i], sw[kk][tn + 16 * j], part[i][j]);
    __syncthreads();
    if ((k0 + 16) % FP8_BLOCK == 0 || k0 + 16 >= p.k) {
      const int b = k0 / FP8_BLOCK;
      for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) {
          const int row = m0 + tm + 16 * i, col = n0 + tn + 16 * j;
          if (row < p.m && col < p.n)
            acc[i][j] = fmaf(part[i][j],
                             p.a_scales[b * p.a_scale_stride + row] * p.w_scales[b * p.w_scale_stride + col / FP8_BLOCK],
                             acc[i][j]);
          part[i][j] = 0.0f;
        }
    }
  }
  for (int i = 0; i < 4; i++)
    for (int j = 0; j < 4; j++) {
      const long long row = m0 + tm + 16 * i, col = n0 + tn + 16 * j;
      if (row >= p.m || col >= p.n) continue;
      float v = op_act_any(acc[i][j] + (p.bias ? p.bias[col] : 0.0f), p.act);
      if (p.residual) v += to_f32(static_cast<const T*>(p.residual)[row * p.residual_stride + col]);
      static_cast<T*>(p.out)[row * p.out_stride + col] = from_f32<T>(v);
    }
}

template <class T>
void run(Device&, const Fp8MatmulSpec& p, cudaStream_t s) {
  const double m = p.m, n = p.n, k = p.k;
  timed_launch("matmul_fp8", 2 * m * n * k, m * k + n * k + m * n * sizeof(T) * (p.residual ? 2 : 1), s, [&] {
    matmul_simple<T><<<dim3((p.m + 63) / 64, (p.n + 63) / 64), 256, 0, s>>>(p);
    IEC_CUDA(cudaGetLastError());
  });
}

}  // namespace

void matmul_fp8(Device& dev, const Fp8MatmulSpec& p, cudaStream_t s) {
  if (p.m == 0 || p.n == 0) return;
  if (p.dtype == DT_F16) return run<__half>(dev, p, s);
  if (p.dtype == DT_BF16) return run<__nv_bfloat16>(dev, p, s);
  run<float>(dev, p, s);
}

}  // namespace iec
