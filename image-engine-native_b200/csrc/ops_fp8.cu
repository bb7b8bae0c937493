// Host side of the block-scaled e4m3 product (fp8_sm100.cuh): tile choice,
// tensor maps and launches.
#include <algorithm>
#include <type_traits>

#include "fp8_sm100.cuh"
#include "ops_launch.h"

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

// out (or residual) as boxes of 32 rows x 128 bytes, 128-byte swizzled.
template <class T>
CUtensorMap value_map(const void* values, long long stride, int rows, int cols) {
  CUtensorMap map;
  const uint64_t dims[2] = {(uint64_t)cols, (uint64_t)rows};
  const uint64_t bytes = rows > 1 ? (uint64_t)stride * sizeof(T) : ((uint64_t)cols * sizeof(T) + 15) / 16 * 16;
  const uint64_t strides[1] = {bytes};
  const uint32_t box[2] = {128 / sizeof(T), 32};
  const CUtensorMapDataType type = std::is_same<T, float>::value    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                    : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  encode_tensor_map(&map, type, 2, values, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  return map;
}

// The rows of a matrix start on 16 bytes, as tensor maps need.
template <class T>
bool on_16(const void* values, long long stride, int rows) {
  return reinterpret_cast<uintptr_t>(values) % 16 == 0 && (rows == 1 || stride * (long long)sizeof(T) % 16 == 0);
}

template <class T, int MODE>
void run_tiles(Device& dev, const Fp8MatmulSpec& q, Fp8Params p, cudaStream_t s) {
  using L = Fp8Smem;
  constexpr auto kernel = fp8_gemm_sm100<T, MODE>;
  constexpr int edge = MODE == FP8_PAIR ? 256 : 128;
  const int cluster = MODE == FP8_PAIR ? 2 : p.splits;
  allow_smem<kernel>(dev, L::DYN_BYTES);
  CUtensorMap a_map = {}, w_map = {}, out_map = {}, res_map = {};
  if (q.k) {
    a_map = code_map(q.a, q.a_stride, q.m, q.k, 128);
    w_map = code_map(q.w, q.w_stride, q.n, q.k, 128);
  }
  p.tma_out = MODE != FP8_SPLIT && on_16<T>(q.out, q.out_stride, q.m) &&
              (!q.residual || on_16<T>(q.residual, q.residual_stride, q.m));
  if (p.tma_out) {
    out_map = value_map<T>(q.out, q.out_stride, q.m, q.n);
    if (q.residual) res_map = value_map<T>(q.residual, q.residual_stride, q.m, q.n);
  }
  p.tiles_m = (q.m + edge - 1) / edge;
  p.tiles_n = (q.n + edge - 1) / edge;
  // (2^20 columns are at most 2^13 tiles, a group of them 2^16: within what FastDiv divides by)
  if ((long long)p.tiles_m * p.tiles_n >= 1 << 24) throw Error(ERR_INPUT, "product too large for one launch");
  p.tiles = p.tiles_m * p.tiles_n;
  p.div_group = FastDiv((uint32_t)(FP8_GROUP * p.tiles_n));
  p.div_rest = FastDiv((uint32_t)std::max(1, p.tiles_m % FP8_GROUP));
  int grid = p.tiles * cluster;
  if (MODE != FP8_SPLIT) grid = std::min(grid, resident_ctas<kernel>(dev, FP8_THREADS, L::DYN_BYTES, cluster));
  launch_ops(kernel, dim3(grid), FP8_THREADS, (size_t)L::DYN_BYTES, cluster, s, a_map, w_map, out_map, res_map, p);
}

// CTAs that share a tile's blocks along k: where the tiles leave at least
// half the SMs idle, as many as fill them, of at least two blocks each.
template <class T>
int splits_of(Device& dev, int tiles, int kblocks) {
  constexpr auto kernel = fp8_gemm_sm100<T, FP8_SPLIT>;
  int n = std::min({16, dev.sms() / std::max(tiles, 1), kblocks / 2});
  // clusters that do not all run at once would take turns
  while (n > 1 && resident_ctas<kernel>(dev, FP8_THREADS, Fp8Smem::DYN_BYTES, n) < tiles * n) n--;
  return std::max(n, 1);
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
  p.dev_err = dev.dev_err();
  const double m = q.m, n = q.n, k = q.k;
  // The least rounds of 128 x 128 outputs an SM: pairs of CTAs take two at a
  // time, at 1.3 times the rate (9472 x 2048 x 1024, whole rounds either way:
  // 31 us in pairs, 39 in single tiles; 4096 x 1536 x 384, four rounds in
  // pairs and three single: 16.9 and 15.2 us).
  const int sms = dev.sms();
  const long long pairs = (long long)((q.m + 255) / 256) * ((q.n + 255) / 256);
  const long long tiles = (long long)((q.m + 127) / 128) * ((q.n + 127) / 128);
  p.splits = tiles * 2 <= sms ? splits_of<T>(dev, (int)tiles, p.kblocks) : 1;
  p.split_blocks = (p.kblocks + p.splits - 1) / p.splits;
  const long long by_pairs = 2 * ((pairs + sms / 2 - 1) / (sms / 2)), by_tiles = (tiles + sms - 1) / sms;
  const int mode = p.splits > 1 ? FP8_SPLIT : 10 * by_pairs <= 13 * by_tiles ? FP8_PAIR : FP8_SINGLE;
  char name[96] = "";
  if (dev.timing()) snprintf(name, sizeof name, "fp8_gemm_sm100<%d> %dx%dx%d", mode, q.m, q.n, q.k);
  timed_launch(name, 2 * m * n * k, m * k + n * k + m * n * sizeof(T) * (q.residual ? 2 : 1), s, [&] {
    if (mode == FP8_PAIR)
      run_tiles<T, FP8_PAIR>(dev, q, p, s);
    else if (mode == FP8_SPLIT)
      run_tiles<T, FP8_SPLIT>(dev, q, p, s);
    else
      run_tiles<T, FP8_SINGLE>(dev, q, p, s);
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
