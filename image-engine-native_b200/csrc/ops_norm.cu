// Group normalisation with an activation over channels-last maps.
//
//   mean = sum x / N, variance = sum (x - mean)^2 / N over the N = pixels *
//   c / groups values of a group, out = act((x - mean) rstd gamma + beta)
//
// One CTA per map and group computes the statistics (two passes, so that a
// mean far from zero costs no digits), a second kernel applies them.
#include "ops_sm100.cuh"

namespace iec {

namespace {

__device__ __forceinline__ float block_sum(float v, float* red) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.0f;
  for (int i = 0; i < (int)blockDim.x / 32; i++) t += red[i];
  return t;
}

template <class T>
__global__ void __launch_bounds__(512) norm_stats(NormSpec p, float2* stats) {
  __shared__ float red[16];
  const int g = blockIdx.x, i = blockIdx.y, cg = p.c / p.groups;
  const T* x = static_cast<const T*>(p.x) + i * p.x_map_stride + g * cg;
  const long long count = p.pixels * cg;
  float s = 0.0f;
  for (long long e = threadIdx.x; e < count; e += blockDim.x) s += to_f32(x[e / cg * p.x_stride + e % cg]);
  const float mean = block_sum(s, red) / (float)count;
  float q = 0.0f;
  for (long long e = threadIdx.x; e < count; e += blockDim.x) {
    const float d = to_f32(x[e / cg * p.x_stride + e % cg]) - mean;
    q = fmaf(d, d, q);
  }
  const float var = block_sum(q, red) / (float)count;
  if (threadIdx.x == 0) stats[i * p.groups + g] = make_float2(mean, 1.0f / sqrtf(var + p.eps));
}

template <class T>
__device__ __forceinline__ float normed(const NormSpec& p, const float2* stats, long long row, int ch) {
  const int i = (int)(row / p.pixels);
  const long long px = row - i * p.pixels;
  const float2 st = stats[i * p.groups + ch / (p.c / p.groups)];
  const float v = to_f32(static_cast<const T*>(p.x)[i * p.x_map_stride + px * p.x_stride + ch]);
  const float y = (v - st.x) * st.y * (p.gamma ? p.gamma[ch] : 1.0f) + (p.beta ? p.beta[ch] : 0.0f);
  return op_act_any(y, p.act);
}

template <class T>
__global__ void __launch_bounds__(256) norm_apply(NormSpec p, const float2* stats) {
  const long long total = p.n * p.pixels * p.c;
  for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long long)gridDim.x * 256) {
    const long long row = e / p.c;
    const int ch = (int)(e - row * p.c), i = (int)(row / p.pixels);
    const float y = normed<T>(p, stats, row, ch);
    static_cast<T*>(p.out)[i * p.out_map_stride + (row - i * p.pixels) * p.out_stride + ch] = from_f32<T>(y);
  }
}

// One warp per pixel and block of 128 channels.
template <class T>
__global__ void __launch_bounds__(256) norm_apply_fp8(NormSpec p, const float2* stats) {
  const int kb = (p.c + FP8_BLOCK - 1) / FP8_BLOCK, lane = threadIdx.x & 31;
  const long long total = p.n * p.pixels * kb;
  for (long long t = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); t < total; t += (long long)gridDim.x * 8) {
    const long long row = t / kb;
    const int b = (int)(t - row * kb);
    float v[4];
    uint32_t top = 0;
    for (int j = 0; j < 4; j++) {
      const int ch = b * FP8_BLOCK + j * 32 + lane;
      v[j] = ch < p.c ? normed<T>(p, stats, row, ch) : 0.0f;
      top = max(top, abs_bits(v[j]));
    }
    top = __reduce_max_sync(~0u, top);
    float factor, scale;
    fp8_scale(top, &factor, &scale);
    for (int j = 0; j < 4; j++) {
      const int ch = b * FP8_BLOCK + j * 32 + lane;
      if (ch < p.c) p.q.codes[row * p.q.code_stride + ch] = (uint8_t)e4m3x2(v[j] * factor, 0.0f);
    }
    if (lane == 0) p.q.scales[b * p.q.scale_stride + row] = scale;
  }
}

template <class T>
void run(Device& dev, const NormSpec& p, cudaStream_t s) {
  float2* stats = static_cast<float2*>(dev.scratch((size_t)p.n * p.groups * sizeof(float2), s));
  const double values = (double)p.n * p.pixels * p.c;
  timed_launch("norm_stats", 3 * values, values * sizeof(T), s, [&] {
    norm_stats<T><<<dim3(p.groups, p.n), 512, 0, s>>>(p, stats);
    IEC_CUDA(cudaGetLastError());
  });
  timed_launch("norm_apply", 8 * values, values * (sizeof(T) + (p.out ? sizeof(T) : 1)), s, [&] {
    if (p.out)
      norm_apply<T><<<dev.sms() * 8, 256, 0, s>>>(p, stats);
    else
      norm_apply_fp8<T><<<dev.sms() * 8, 256, 0, s>>>(p, stats);
    IEC_CUDA(cudaGetLastError());
  });
}

}  // namespace

void group_norm(Device& dev, const NormSpec& p, cudaStream_t s) {
  if (p.n == 0 || p.pixels == 0) return;
  if (p.dtype == DT_F16) return run<__half>(dev, p, s);
  if (p.dtype == DT_BF16) return run<__nv_bfloat16>(dev, p, s);
  run<float>(dev, p, s);
}

}  // namespace iec
