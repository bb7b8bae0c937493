// Rows of 16- or 32-bit values to e4m3 codes with an f32 scale for each
// block of 128 values of a row (activations), or of 128 rows and 128 values
// (weights). Bound by memory: a value is read once, a byte written, some
// five instructions between.
#include "ops_launch.h"
#include "ops_sm100.cuh"

namespace iec {

namespace {

constexpr int QUANT_THREADS = 256;

struct QuantShape {
  int blocks;            // of a row
  long long items;       // (columns of) rows x blocks
  // An item is a row (a column of rows) and a block of it; a warp takes one
  // item after another, `stride` items on: so many rows and blocks further.
  long long stride, stride_rows;
  int stride_blocks;
};

__device__ __forceinline__ uint32_t group_max(uint32_t top, int lanes) {
  for (int o = lanes / 2; o; o >>= 1) top = max(top, __shfl_xor_sync(~0u, top, o));
  return top;
}

// The magnitude's bits of the largest of a vector's values, NaN above all.
template <class T, int VE>
__device__ __forceinline__ uint32_t vector_top(uint4 q) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  if constexpr (sizeof(T) == 4) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) top = max(top, w[i] & 0x7fffffffu);
    return top;
  } else {
    // 16-bit magnitudes order as integers too, two at a time
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
    const uint16_t one = (uint16_t)max(m & 0xffffu, m >> 16);
    return __float_as_uint(to_f32(reinterpret_cast<const T&>(one)));
  }
}

// Scaled vectors as codes.
template <class T, int VE>
__device__ __forceinline__ void store_codes(uint8_t* out, uint4 raw, float factor) {
  float v[VE];
  Vec<T, VE, true>::expand(raw, v);
  uint32_t w[VE / 4];
#pragma unroll
  for (int e = 0; e < VE; e += 4) {
    const float2 a = fmul2(make_float2(v[e], v[e + 1]), both(factor));
    const float2 b = fmul2(make_float2(v[e + 2], v[e + 3]), both(factor));
    w[e / 4] = (uint32_t)e4m3x2(a.x, a.y) | (uint32_t)e4m3x2(b.x, b.y) << 16;
  }
  if constexpr (VE == 8)
    *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
  else
    *reinterpret_cast<uint32_t*>(out) = w[0];
}

// Rows of whole, aligned vectors: 128 / VE lanes take a row's block, a vector
// each, and a warp four blocks of rows below one another at a time for each
// such group of lanes (an item here is such a column of blocks, its rows U *
// 32 / LANES), whose scales then lie side by side and are stored together.
// 49152 x 1536 f16 (229 MB with codes and scales): 40 us in a graph, 5.8 TB/s,
// 89 % of a copy's rate, 41 to 43 as calls of their own (one block an item, its
// scale stored alone: 44 us in a graph; a division per value: 127).
constexpr int QUANT_UNROLL = 4;
template <class T>
__global__ void __launch_bounds__(QUANT_THREADS) quant_rows(const QuantSpec p, const QuantShape q) {
  constexpr int VE = 16 / (int)sizeof(T), LANES = FP8_BLOCK / VE, GROUPS = 32 / LANES, U = QUANT_UNROLL;
  griddep_launch_dependents();
  griddep_wait();
  long long item = ((long long)blockIdx.x * QUANT_THREADS + threadIdx.x) / 32;
  const int lane = threadIdx.x % LANES, group = threadIdx.x % 32 / LANES;
  long long row = item / q.blocks;
  int block = (int)(item - row * q.blocks);
  const T* x = static_cast<const T*>(p.x);
  for (; item < q.items; item += q.stride) {
    // step u of a group of lanes is row row0 + u * GROUPS
    const long long row0 = row * (U * GROUPS) + group;
    const bool inside = block * FP8_BLOCK + lane * VE < p.k;
    const T* at = x + row0 * p.x_stride + block * FP8_BLOCK + lane * VE;
    uint4 raw[U];
    float scale[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      raw[u] = make_uint4(0, 0, 0, 0);
      if (inside && row0 + u * GROUPS < p.rows) raw[u] = *reinterpret_cast<const uint4*>(at + u * GROUPS * p.x_stride);
    }
    uint8_t* out = p.q.codes + row0 * (long long)p.q.code_stride + block * FP8_BLOCK + lane * VE;
#pragma unroll
    for (int u = 0; u < U; u++) {
      float factor;
      fp8_scale(group_max(vector_top<T, VE>(raw[u]), LANES), &factor, &scale[u]);
      if (inside && row0 + u * GROUPS < p.rows)
        store_codes<T, VE>(out + u * GROUPS * (long long)p.q.code_stride, raw[u], factor);
    }
    float mine = scale[0];
#pragma unroll
    for (int u = 1; u < U; u++) mine = lane == u ? scale[u] : mine;
    if (lane < U && row0 + lane * GROUPS < p.rows)
      p.q.scales[block * (long long)p.q.scale_stride + row0 + lane * GROUPS] = mine;
    row += q.stride_rows;
    block += q.stride_blocks;
    if (block >= q.blocks) {
      block -= q.blocks;
      row++;
    }
  }
}

// Four values of a row from `col` on, wherever it starts; beyond its end the
// last one again, which leaves the block's maximum as it is. (Each load has an
// address of its own and stands under no condition: many are under way.)
template <class T>
__device__ __forceinline__ void load_four(const T* row, int block, int lane, int k, T* v) {
  const int col = block * FP8_BLOCK + lane * 4;
  if ((block + 1) * FP8_BLOCK <= k) {
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = row[col + e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = row[min(col + e, k - 1)];
  }
}
template <class T>
__device__ __forceinline__ uint32_t four_top(const T* v) {
  float most = 0.0f;
#pragma unroll
  for (int e = 0; e < 4; e++) most = max_abs(to_f32(v[e]), most);
  return abs_bits(most);
}
// Their codes; `words`: rows of codes start on words.
template <class T>
__device__ __forceinline__ void store_four(uint8_t* row, int col, int k, bool words, const T* v, float factor) {
  const uint32_t w = (uint32_t)e4m3x2(to_f32(v[0]) * factor, to_f32(v[1]) * factor) |
                     (uint32_t)e4m3x2(to_f32(v[2]) * factor, to_f32(v[3]) * factor) << 16;
  if (words && col + 4 <= k) {
    *reinterpret_cast<uint32_t*>(row + col) = w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (col + e < k) row[col + e] = (uint8_t)(w >> (8 * e));
  }
}
__device__ __forceinline__ bool on_words(const Fp8Out& q) {
  return ((reinterpret_cast<uintptr_t>(q.codes) | (uintptr_t)q.code_stride) & 3) == 0;
}

// Any rows: a warp an item, four values a lane, U items at a time (6607 x 7287
// bf16: 49 us; with two items, a lane's values 32 apart and codes stored one by
// one: 65).
template <class T, int U>
__global__ void __launch_bounds__(QUANT_THREADS) quant_rows_odd(const QuantSpec p, const QuantShape q) {
  griddep_launch_dependents();
  griddep_wait();
  long long item = ((long long)blockIdx.x * QUANT_THREADS + threadIdx.x) / 32;
  const int lane = threadIdx.x % 32;
  const bool words = on_words(p.q);
  long long row = item / q.blocks;
  int block = (int)(item - row * q.blocks);
  while (item < q.items) {
    T v[U][4];
    long long rows[U];
    int blocks[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      rows[u] = row;
      blocks[u] = block;
      load_four(static_cast<const T*>(p.x) + min(row, p.rows - 1) * p.x_stride, block, lane, p.k, v[u]);
      row += q.stride_rows;
      block += q.stride_blocks;
      if (block >= q.blocks) {
        block -= q.blocks;
        row++;
      }
    }
    item += U * q.stride;
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (rows[u] >= p.rows) break;
      float factor, scale;
      fp8_scale(__reduce_max_sync(~0u, four_top(v[u])), &factor, &scale);
      store_four(p.q.codes + rows[u] * (long long)p.q.code_stride, blocks[u] * FP8_BLOCK + lane * 4, p.k, words, v[u],
                 factor);
      if (lane == 0) p.q.scales[blocks[u] * (long long)p.q.scale_stride + rows[u]] = scale;
    }
  }
}

// Rows of one block: a warp a row, a lane's values 32 apart, so that in short
// rows most lanes have some (40000 x 31 f16: 6.4 us, 9.3 side by side).
template <class T>
__global__ void __launch_bounds__(QUANT_THREADS) quant_rows_short(const QuantSpec p, const QuantShape q) {
  constexpr int U = 2;
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x % 32;
  for (long long row = ((long long)blockIdx.x * QUANT_THREADS + threadIdx.x) / 32; row < p.rows; row += U * q.stride) {
    float v[U][4];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const T* x = static_cast<const T*>(p.x) + (row + u * q.stride) * p.x_stride + lane;
#pragma unroll
      for (int j = 0; j < 4; j++)
        v[u][j] = row + u * q.stride < p.rows && j * 32 + lane < p.k ? to_f32(x[j * 32]) : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const long long at = row + u * q.stride;
      if (at >= p.rows) break;
      float most = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; j++) most = max_abs(v[u][j], most);
      float factor, scale;
      fp8_scale(__reduce_max_sync(~0u, abs_bits(most)), &factor, &scale);
      uint8_t* out = p.q.codes + at * (long long)p.q.code_stride + lane;
      const uint32_t a = e4m3x2(v[u][0] * factor, v[u][1] * factor), b = e4m3x2(v[u][2] * factor, v[u][3] * factor);
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (j * 32 + lane < p.k) out[j * 32] = (uint8_t)((j < 2 ? a : b) >> (8 * (j & 1)));
      if (lane == 0) p.q.scales[at] = scale;
    }
  }
}

__device__ __forceinline__ uint32_t cta_max(uint32_t top) {
  __shared__ uint32_t red[QUANT_THREADS / 32];
  top = __reduce_max_sync(~0u, top);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < QUANT_THREADS / 32; i++) top = max(top, red[i]);
  return top;
}

// A CTA a block of 128 x 128, its vectors in registers between the maximum
// and the codes. 16384 x 4096 bf16 (201 MB): 31 us, 6.6 TB/s, a copy's rate.
template <class T>
__global__ void __launch_bounds__(QUANT_THREADS) quant_blocks(const QuantSpec p) {
  constexpr int VE = 16 / (int)sizeof(T), LANES = FP8_BLOCK / VE, ROWS = QUANT_THREADS / LANES, N = FP8_BLOCK / ROWS;
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x % LANES, col = blockIdx.x * FP8_BLOCK + lane * VE;
  const long long row = (long long)blockIdx.y * FP8_BLOCK + threadIdx.x / LANES;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride + col;
  uint4 raw[N];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < N; i++) {
    raw[i] = make_uint4(0, 0, 0, 0);
    if (row + i * ROWS < p.rows && col < p.k) raw[i] = *reinterpret_cast<const uint4*>(x + i * ROWS * p.x_stride);
  }
#pragma unroll
  for (int i = 0; i < N; i++) top = max(top, vector_top<T, VE>(raw[i]));
  float factor, scale;
  fp8_scale(cta_max(top), &factor, &scale);
#pragma unroll
  for (int i = 0; i < N; i++)
    if (row + i * ROWS < p.rows && col < p.k)
      store_codes<T, VE>(p.q.codes + (row + i * ROWS) * (long long)p.q.code_stride + col, raw[i], factor);
  if (threadIdx.x == 0) p.q.scales[blockIdx.x * (long long)p.q.scale_stride + blockIdx.y] = scale;
}

// The same for any rows, four values a lane (62949 x 587 bf16: 45 us; a
// column a thread, read twice: 64).
template <class T>
__global__ void __launch_bounds__(QUANT_THREADS) quant_blocks_odd(const QuantSpec p) {
  griddep_launch_dependents();
  griddep_wait();
  constexpr int ROWS = QUANT_THREADS / 32, N = FP8_BLOCK / ROWS;
  const int lane = threadIdx.x % 32;
  const long long row = (long long)blockIdx.y * FP8_BLOCK + threadIdx.x / 32;
  const bool words = on_words(p.q);
  T v[N][4];
#pragma unroll
  for (int i = 0; i < N; i++)
    load_four(static_cast<const T*>(p.x) + min(row + i * ROWS, p.rows - 1) * p.x_stride, (int)blockIdx.x, lane, p.k, v[i]);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < N; i++) top = max(top, four_top(v[i]));
  float factor, scale;
  fp8_scale(cta_max(top), &factor, &scale);
#pragma unroll
  for (int i = 0; i < N; i++)
    if (row + i * ROWS < p.rows)
      store_four(p.q.codes + (row + i * ROWS) * (long long)p.q.code_stride, (int)blockIdx.x * FP8_BLOCK + lane * 4, p.k,
                 words, v[i], factor);
  if (threadIdx.x == 0) p.q.scales[blockIdx.x * (long long)p.q.scale_stride + blockIdx.y] = scale;
}

template <class T>
void run(Device& dev, const QuantSpec& p, cudaStream_t s) {
  constexpr int VE = 16 / (int)sizeof(T);
  const int blocks = (p.k + FP8_BLOCK - 1) / FP8_BLOCK;
  const bool wide = reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && p.x_stride % VE == 0 && p.k % VE == 0 &&
                    reinterpret_cast<uintptr_t>(p.q.codes) % VE == 0 && p.q.code_stride % VE == 0;
  const double values = (double)p.rows * p.k;
  timed_launch("quantize_fp8", 2 * values, values * (sizeof(T) + 1), s, [&] {
    if (p.block_rows == 1) {
      QuantShape q;
      q.blocks = blocks;
      // a warp an item
      const int column = wide ? QUANT_UNROLL * 32 * VE / FP8_BLOCK : 1, per = QUANT_THREADS / 32;
      q.items = (p.rows + column - 1) / column * blocks;
      // as many CTAs an SM as fit, or fewer where the items run out; several
      // items at a time only where each warp has them
      const long long want = (q.items + per - 1) / per, most = 8LL * dev.sms();
      const bool brief = !wide && blocks == 1, few = brief || want <= 8 * most;
      const int grid = (int)std::max<long long>(1, std::min<long long>(want, wide || few ? most : most / 2));
      q.stride = (long long)grid * per;
      q.stride_rows = q.stride / blocks;
      q.stride_blocks = (int)(q.stride - q.stride_rows * blocks);
      if (wide)
        launch_pdl(quant_rows<T>, dim3(grid), dim3(QUANT_THREADS), 0, s, p, q);
      else if (brief)
        launch_pdl(quant_rows_short<T>, dim3(grid), dim3(QUANT_THREADS), 0, s, p, q);
      else if (few)
        launch_pdl(quant_rows_odd<T, 1>, dim3(grid), dim3(QUANT_THREADS), 0, s, p, q);
      else
        launch_pdl(quant_rows_odd<T, 4>, dim3(grid), dim3(QUANT_THREADS), 0, s, p, q);
    } else {
      const long long row_blocks = (p.rows + FP8_BLOCK - 1) / FP8_BLOCK;
      // a grid is at most 65535 high
      for (long long done = 0; done < row_blocks; done += 65535) {
        QuantSpec part = p;
        part.x = static_cast<const T*>(p.x) + done * FP8_BLOCK * p.x_stride;
        part.rows = p.rows - done * FP8_BLOCK;
        part.q.codes = p.q.codes + (size_t)done * FP8_BLOCK * p.q.code_stride;
        part.q.scales = p.q.scales + done;
        const dim3 grid((unsigned)blocks, (unsigned)std::min<long long>(row_blocks - done, 65535));
        if (wide)
          launch_pdl(quant_blocks<T>, grid, dim3(QUANT_THREADS), 0, s, part);
        else
          launch_pdl(quant_blocks_odd<T>, grid, dim3(QUANT_THREADS), 0, s, part);
      }
    }
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
