// Host side of the block-scaled e4m3 product (fp8_sm100.cuh): tile choice,
// tensor maps and launches.
#include <algorithm>

#include "fp8_sm100.cuh"

namespace iec {

namespace {

// `rows` x `k` codes as boxes of `box_rows` rows x 128 values, 128-byte
// swizzled; values past k and rows past the last read as zero.
CUtensorMap code_map(const uint8_t* codes, long long stride, int rows, int k, int box_rows) {
  CUtensorMap map;
  const uint64_t dims[2] = {(uint64_t)k, (uint64_t)rows};
  const uint64_t strides[1] = {rows > 1 ? (uint64_t)stride : ((uint64_t)k + 15) / 16 * 16};
  const uint32_t box[2] = {FP8_BLOCK, (uint32_t)box_rows};
  encode_tensor_map(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, codes, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  return map;
}

template <auto Kernel>
void allow_smem(Device& dev, int bytes) {
  static bool done[64] = {};
  bool& d = done[dev.ordinal() & 63];
  if (!d) IEC_CUDA(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  d = true;
}

template <class T, int BN>
void run_tiles(Device& dev, const Fp8MatmulSpec& q, Fp8Params p, cudaStream_t s) {
  using L = Fp8Smem<BN>;
  constexpr auto kernel = fp8_gemm_sm100<T, BN>;
  allow_smem<kernel>(dev, L::DYN_BYTES);
  CUtensorMap a_map = {}, w_map = {};
  if (q.k) {
    a_map = code_map(q.a, q.a_stride, q.m, q.k, 128);
    w_map = code_map(q.w, q.w_stride, q.n, q.k, BN);
  }
  p.tiles_m = (q.m + 127) / 128;
  p.tiles_n = (q.n + BN - 1) / BN;
  if ((long long)p.tiles_m * p.tiles_n > INT32_MAX / 2) throw Error(ERR_INPUT, "product too large for one launch");
  p.tiles = p.tiles_m * p.tiles_n;
  launch_pdl(kernel, dim3(std::min(p.tiles, dev.sms())), dim3(FP8_THREADS), (size_t)L::DYN_BYTES, s, a_map, w_map, p);
}

template <class T>
void run(Device& dev, const Fp8MatmulSpec& q, cudaStream_t s) {
  Fp8Params p = {};
  p.m = q.m;
  p.n = q.n;
  p.kblocks = (q.k + FP8_BLOCK - 1) / FP8_BLOCK;
  p.act = q.act;
  p.a_scales = q.a_scales;
  p.w_scales = q.w_scales;
  p.a_scale_stride = q.a_scale_stride;
  p.w_scale_stride = q.w_scale_stride;
  p.bias = q.bias;
  p.residual = q.residual;
  p.out = q.out;
  p.residual_stride = q.residual_stride;
  p.out_stride = q.out_stride;
  auto rows_on_32 = [](const void* ptr, long long stride) {
    return reinterpret_cast<uintptr_t>(ptr) % 32 == 0 && stride * (long long)sizeof(T) % 32 == 0;
  };
  p.wide = rows_on_32(q.out, q.out_stride) && (!q.residual || rows_on_32(q.residual, q.residual_stride));
  p.dev_err = dev.dev_err();
  const double m = q.m, n = q.n, k = q.k;
  char name[96];
  const long long wide = (long long)((q.m + 127) / 128) * ((q.n + 255) / 256);
  const int bn = wide >= dev.sms() ? 256 : 128;
  snprintf(name, sizeof name, "fp8_gemm_sm100<%d> %dx%dx%d", bn, q.m, q.n, q.k);
  timed_launch(name, 2 * m * n * k, m * k + n * k + m * n * sizeof(T) * (q.residual ? 2 : 1), s, [&] {
    if (bn == 256)
      run_tiles<T, 256>(dev, q, p, s);
    else
      run_tiles<T, 128>(dev, q, p, s);
  });
}

}  // namespace

void matmul_fp8(Device& dev, const Fp8MatmulSpec& q, cudaStream_t s) {
  if (q.m == 0 || q.n == 0) return;
  if (q.dtype == DT_F16) return run<__half>(dev, q, s);
  if (q.dtype == DT_BF16) return run<__nv_bfloat16>(dev, q, s);
  run<float>(dev, q, s);
}

}  // namespace iec
