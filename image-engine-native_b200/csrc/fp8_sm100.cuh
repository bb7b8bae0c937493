// The block-scaled e4m3 product on sm_100a tensor cores:
//   out[m][n] = act(sum_b sa[b][m] sw[b][n / 128] (sum_{k in block b}
//               a[m][k] w[n][k]) + bias[n]) + residual[m][n]
//
// A block of 128 values along k is one 128-byte row of a swizzled tile and
// four tcgen05 instructions (K 32 each). Its product lies in one of two TMEM
// accumulators; while the tensor core computes the next block into the
// other, the epilogue warps read it, multiply it by the block's scales and
// add it to the tile's sums, which stay in registers in f32: thread t of a
// lane quarter holds row t, so the scale of a is one register and that of w
// is the same for all its columns.
//
// fp8_gemm_sm100<T, MODE>: FP8_PAIR takes tiles of 256 x 256 by two CTAs of a
// cluster (cta_group::2: each loads its 128 rows of a and half the rows of w
// and holds its rows' accumulators), FP8_SINGLE tiles of 128 x 128 by one;
// FP8_SPLIT, for few tiles, has the CTAs of a cluster take a stretch of k
// each of one 128 x 128 tile and add up their sums through distributed shared
// memory, always in the same order. CTAs of 12 warps walk the tiles: warp 0 loads (TMA, 128-byte swizzle), warp
// 1 issues the MMAs, warps 4..11 (two per TMEM lane quarter, half the columns
// each) scale and add the blocks and write the tile; they take the registers
// that the others give up (setmaxnreg), 128 of them for the sums of a row's
// 128 columns. A tile is written through shared memory by TMA, each warp its
// own 32 rows, and the residual comes in the same way while the tile's MMAs
// run; where the rows of out or residual do not start on 16 bytes, they are
// written through shared memory with plain accesses. All waits are bounded.
//
// What it measured: 16384 x 8192 x 2048 to bf16 280 us in a burst (1,965
// TFLOP/s), 320 sustained under the power cap; 8192^3 485 and 561 us. The
// bound is the accumulators' way back: per SM and block 128 x 256 values read
// from TMEM and added, next to 512 cycles of MMAs (with the loads and MMAs
// alone, and the output: 226 us). 256 x 256 is the largest tile whose sums (128
// registers a thread) and two accumulators (512 TMEM columns) fit, and has the
// least traffic from L2 for its MMAs: 64 bytes a cycle and SM. The sums are
// read 16 columns at a time, the next 16 on their way (32 at a time: 531 us
// at 8192^3, 64: 535).
#pragma once

#include "ops_sm100.cuh"
#include "sm100.cuh"

namespace iec {

struct Fp8Params {
  int m, n, kblocks, act;
  int tiles_m, tiles_n, tiles;
  FastDiv div_group, div_rest;  // by the tiles of a group of M tiles, and by the M tiles of the last one
  const float* a_scales;
  const float* w_scales;
  long long a_scale_stride, w_scale_stride;
  const float* bias;
  const void* residual;
  void* out;
  long long residual_stride, out_stride;
  int tma_out;  // out and residual have tensor maps
  int splits, split_blocks;  // FP8_SPLIT: CTAs of a tile, blocks along k of one
  int* dev_err;
};

enum Fp8Mode { FP8_SINGLE = 0, FP8_PAIR = 1, FP8_SPLIT = 2 };

constexpr int FP8_THREADS = 384;
constexpr int FP8_EPI_WARPS = 8;
constexpr int FP8_GROUP = 8;  // M tiles walked together, so that L2 serves their w tiles

struct Fp8Smem {
  static constexpr int HALF_BYTES = 128 * 128, STAGE = 2 * HALF_BYTES;  // a's rows, w's rows
  static constexpr int NSTAGE = 4;
  static constexpr int OUT_OFF = NSTAGE * STAGE, OUT_WARP = 8192;  // a warp's patch of the output
  static constexpr int BIAS_OFF = OUT_OFF + FP8_EPI_WARPS * OUT_WARP;
  static constexpr int BAR_OFF = BIAS_OFF + FP8_EPI_WARPS * 128 * 4;
  static constexpr int MISC_OFF = BAR_OFF + (2 * NSTAGE + 4 + FP8_EPI_WARPS) * 8;
  static constexpr int DYN_BYTES = MISC_OFF + 16 + 1024;
  static_assert(DYN_BYTES <= 232448, "shared memory of a CTA");
};

// Tile -> (M tile, N tile), in groups of FP8_GROUP M tiles.
__device__ __forceinline__ void fp8_tile(const Fp8Params& p, int tile, int* mt, int* nt) {
  const int g = (int)p.div_group.div((uint32_t)tile), r = tile - g * FP8_GROUP * p.tiles_n;
  const bool last = (g + 1) * FP8_GROUP > p.tiles_m;
  const int rows = last ? p.tiles_m - g * FP8_GROUP : FP8_GROUP;
  *nt = last ? (int)p.div_rest.div((uint32_t)r) : r / FP8_GROUP;
  *mt = g * FP8_GROUP + r - *nt * rows;
}

// 16 bytes of T: add to f32, or make from f32.
template <class T>
__device__ __forceinline__ void add_16(float* f, uint4 v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (sizeof(T) == 4) {
      f[i] += __uint_as_float(w[i]);
    } else {
      const uint16_t lo = (uint16_t)(w[i] & 0xffffu), hi = (uint16_t)(w[i] >> 16);
      f[2 * i] += to_f32(reinterpret_cast<const T&>(lo));
      f[2 * i + 1] += to_f32(reinterpret_cast<const T&>(hi));
    }
  }
}
template <class T>
__device__ __forceinline__ uint4 make_16(const float* f) {
  if constexpr (sizeof(T) == 4)
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  else
    return make_uint4(pack_2<T>(f[0], f[1]), pack_2<T>(f[2], f[3]), pack_2<T>(f[4], f[5]), pack_2<T>(f[6], f[7]));
}

// A block's two scales in one. Of finite ones it is cut off at f32's largest
// value, so that a sum of zero stays zero. (Sums multiplied by the scales one
// after the other would reach further, but any more work, or a choice, per block
// in the sums' loop costs 16384 x 8192 x 2048 13 % and more.)
__device__ __forceinline__ float fp8_scale_product(float a, float w) {
  const float s = a * w, most = 3.4028235e38f;
  return fabsf(s) > most && fmaxf(fabsf(a), fabsf(w)) <= most ? copysignf(most, s) : s;
}

template <int REGS>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS));
}
template <int REGS>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS));
}

// A row of a patch's box (128 bytes: 128 / sizeof(T) columns from `col`) to or
// from global memory at `row`, by one warp, wherever the row starts: a lane
// takes one 32-bit word, and where the row's words straddle global memory's,
// the halves of two lanes' words.
__device__ __forceinline__ uint32_t* fp8_word(uint8_t* box, int r, int lane) {
  return reinterpret_cast<uint32_t*>(box + r * 128 + ((((lane >> 2) ^ r) & 7) << 4) + (lane & 3) * 4);
}
template <class T>
__device__ __forceinline__ void fp8_drain_row(uint8_t* box, int r, int lane, T* row, int col, int n) {
  const uint32_t word = *fp8_word(box, r, lane);
  if constexpr (sizeof(T) == 4) {
    if (col + lane < n) reinterpret_cast<uint32_t*>(row)[col + lane] = word;
  } else {
    uint16_t* at = reinterpret_cast<uint16_t*>(row) + col + 2 * lane;
    const int left = n - col - 2 * lane;  // columns from this lane's first on
    if ((reinterpret_cast<uintptr_t>(at) & 3) == 0) {
      if (left > 1) *reinterpret_cast<uint32_t*>(at) = word;
      if (left == 1) at[0] = (uint16_t)word;
    } else {
      const uint32_t next = __shfl_down_sync(~0u, word, 1);
      if (lane == 0 && left > 0) at[0] = (uint16_t)word;
      if (lane < 31 && left > 2)
        *reinterpret_cast<uint32_t*>(at + 1) = word >> 16 | next << 16;
      else if (left > 1)
        at[1] = (uint16_t)(word >> 16);
    }
  }
}
// A box of `rows` rows in: 4 rows at a time, from addresses that always hold
// something, so that no load waits for another (what comes from beside the
// rows' ends stands where nothing is written out). 1738 x 6738 x 764 to f16
// with a residual: 57 us, 116 with loads under conditions; 8 rows at a time, 48
// us, but the sums' loop lost registers to it (16384 x 8192 x 2048 in a burst:
// 294 us, 277 now).
template <class T>
__device__ __forceinline__ void fp8_fill_box(uint8_t* box, int lane, const T* in, long long stride, int rows, int col, int n) {
  constexpr int U = 4, PER = 4 / sizeof(T);
  if (col >= n) return;
  const T* lo = in + min(col + PER * lane, n - 1);
  const T* hi = in + min(col + PER * lane + PER - 1, n - 1);
#pragma unroll 1
  for (int r0 = 0; r0 < rows; r0 += U) {
    T w[U][PER];
#pragma unroll
    for (int i = 0; i < U; i++) {
      const long long at = min(r0 + i, rows - 1) * stride;
      w[i][0] = lo[at];
      if (PER > 1) w[i][PER - 1] = hi[at];
    }
#pragma unroll
    for (int i = 0; i < U; i++) memcpy(fp8_word(box, r0 + i, lane), w[i], 4);
  }
}

// `BOXES` boxes of 4 KB next to each other in a row. (Out of line: inlined
// where it is used, it took registers from the sums.)
template <int BOXES, int BOX_COLS>
__device__ __noinline__ void fp8_load_boxes(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int col, int row) {
  mbar_arrive_expect_tx(bar, BOXES * 4096);
#pragma unroll
  for (int b = 0; b < BOXES; b++) tma_load_2d(dst + b * 4096, map, bar, col + b * BOX_COLS, row);
}

template <class T, int MODE>
__global__ void __launch_bounds__(FP8_THREADS, 1)
    fp8_gemm_sm100(const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap w_map,
                   const __grid_constant__ CUtensorMap out_map, const __grid_constant__ CUtensorMap res_map,
                   const Fp8Params p) {
  using L = Fp8Smem;
  constexpr bool PAIR = MODE == FP8_PAIR, SPLIT = MODE == FP8_SPLIT;
  constexpr int BM = PAIR ? 256 : 128, BN = BM, CW = BN / 2;  // CW: columns of a thread
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);  // of a pair, only the first CTA's is used
  uint64_t* empty = full + L::NSTAGE;
  uint64_t* acc_full = empty + L::NSTAGE;
  uint64_t* acc_empty = acc_full + 2;  // of a pair, only the first CTA's is used
  uint64_t* res_full = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC_OFF);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::MISC_OFF + 4);
  const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_rank() : 0;
  const uint32_t split = SPLIT ? cluster_rank() : 0;
  const int first = PAIR ? blockIdx.x >> 1 : SPLIT ? blockIdx.x / p.splits : blockIdx.x;
  const int step = PAIR ? gridDim.x >> 1 : SPLIT ? p.tiles : gridDim.x;
  const int kb0 = SPLIT ? min((int)split * p.split_blocks, p.kblocks) : 0;
  const int kb1 = SPLIT ? min(kb0 + p.split_blocks, p.kblocks) : p.kblocks;

  if (threadIdx.x == 64 && p.kblocks) {
    prefetch_tensor_map(&a_map);
    prefetch_tensor_map(&w_map);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < L::NSTAGE; s++) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; a++) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], FP8_EPI_WARPS * (PAIR ? 2 : 1));
    }
    for (int w = 0; w < FP8_EPI_WARPS; w++) mbar_init(&res_full[w], 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    if (PAIR) {
      tmem_alloc_pair(tmem_slot, 2 * BN);
    } else {
      tmem_alloc(tmem_slot, 2 * BN);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();  // the other CTA's barriers are ready
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  griddep_launch_dependents();
  griddep_wait();

  if (warp < 4) {
    regs_dec<104>();
    if (warp == 0 && lane == 0) {
      // ------------------------------------------------------------ producer
      int s = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = first; tile < p.tiles && ok; tile += step) {
        int mt, nt;
        fp8_tile(p, tile, &mt, &nt);
        const int row = mt * BM + (int)rank * 128, col = nt * BN + (int)rank * 128;
        for (int kb = kb0; kb < kb1; kb++) {
          if (!mbar_wait(&empty[s], phase ^ 1, abort_flag, p.dev_err, DEV_ERR_WAIT_EMPTY)) {
            ok = false;
            break;
          }
          uint8_t* st = smem + s * L::STAGE;
          if (PAIR) {
            // both CTAs' bytes complete on the first one's barrier
            const uint32_t bar = cluster_map(&full[s], 0);
            if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * L::STAGE);
            tma_load_2d_pair(st, &a_map, bar, kb * FP8_BLOCK, row);
            tma_load_2d_pair(st + L::HALF_BYTES, &w_map, bar, kb * FP8_BLOCK, col);
          } else {
            mbar_arrive_expect_tx(&full[s], L::STAGE);
            tma_load_2d(st, &a_map, &full[s], kb * FP8_BLOCK, row);
            tma_load_2d(st + L::HALF_BYTES, &w_map, &full[s], kb * FP8_BLOCK, col);
          }
          issued++;
          if (++s == L::NSTAGE) {
            s = 0;
            phase ^= 1;
          }
        }
      }
      // the stages in flight are consumed before this CTA's memory goes
      for (int i = max(0, issued - L::NSTAGE); i < issued; i++)
        mbar_wait(&empty[i % L::NSTAGE], (uint32_t)(i / L::NSTAGE) & 1, abort_flag, p.dev_err, 0);
    } else if (warp == 1 && rank == 0) {
      // ---------------------------------------------------------- MMA issuer
      // (the whole warp walks the loop, one lane issues: see elect_one)
      constexpr uint32_t idesc = idesc_e4m3_f32(BM, BN);
      const uint64_t desc0 = smem_desc_sw128(smem_u32(smem));
      int s = 0, i = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = first; tile < p.tiles && ok; tile += step)
        for (int kb = kb0; kb < kb1; kb++, i++) {
          ok = __all_sync(~0u, mbar_wait(&full[s], phase, abort_flag, p.dev_err, DEV_ERR_WAIT_FULL));
          if (!ok) break;
          const int a = i & 1;
          ok = __all_sync(~0u, mbar_wait(&acc_empty[a], ((uint32_t)(i >> 1) & 1) ^ 1, abort_flag, p.dev_err,
                                         DEV_ERR_WAIT_ACC_EMPTY));
          if (!ok) break;
          tc_fence_after();
          const uint64_t adesc = desc0 + (uint32_t)(s * (L::STAGE >> 4)), bdesc = adesc + (L::HALF_BYTES >> 4);
          const uint32_t d = tmem_base + (uint32_t)(a * BN);
          if (elect_one()) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
              if (PAIR)
                umma_f8_pair(d, adesc + 2 * j, bdesc + 2 * j, idesc, j != 0);
              else
                umma_f8(d, adesc + 2 * j, bdesc + 2 * j, idesc, j != 0);
            }
            if (PAIR) {
              umma_commit_pair(&empty[s]);
              umma_commit_pair(&acc_full[a]);
            } else {
              umma_commit(&empty[s]);
              umma_commit(&acc_full[a]);
            }
          }
          if (++s == L::NSTAGE) {
            s = 0;
            phase ^= 1;
          }
        }
      // the MMAs in flight end before TMEM is freed
      for (int q = max(0, i - 2); q < i; q++)
        mbar_wait(&acc_full[q & 1], (uint32_t)(q >> 1) & 1, abort_flag, p.dev_err, 0);
    }
  } else {
    // ------------------------------------------- scaling, sums and epilogue
    regs_inc<200>();
    // The output patch in shared memory: boxes of 32 rows x 128 bytes,
    // 128-byte swizzled, BOXES at a time, ROUNDS times.
    constexpr int BOX_COLS = 128 / (int)sizeof(T), BOXES = CW * (int)sizeof(T) / 128 < 2 ? 1 : 2;
    constexpr int ROUNDS = CW / (BOXES * BOX_COLS), V = 16 / (int)sizeof(T);
    const int e = warp - 4, quarter = warp & 3, part = e >> 2;
    uint8_t* patch = smem + L::OUT_OFF + e * L::OUT_WARP;
    float* sbias = reinterpret_cast<float*>(smem + L::BIAS_OFF) + e * 128;
    const uint32_t lanes = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(part * CW);
    const uint32_t acc_bar = PAIR ? cluster_map(acc_empty, 0) : 0;
    int i = 0;
    uint32_t res_phase = 0;
    bool ok = true, res_flying = false;

    // Round `r` of a tile's residual into the patch (lane 0; the patch free).
    auto load_residual = [&](int row, int col, int r) {
      res_flying = true;
      fp8_load_boxes<BOXES, BOX_COLS>(patch, &res_map, &res_full[e], col + r * BOXES * BOX_COLS, row);
    };

    // A tile's first row and column of this warp, its first scales and bias.
    int row0 = 0, col0 = 0;
    const float* sa = p.a_scales;
    const float* sw = p.w_scales;
    float sa_next = 0.0f, sw_next = 0.0f, bias_r[CW / 32];
    auto enter_tile = [&](int tile) {
      int mt, nt;
      fp8_tile(p, tile, &mt, &nt);
      row0 = mt * BM + (int)rank * 128 + quarter * 32;
      col0 = nt * BN + part * CW;
      sa = p.a_scales + min(row0 + lane, p.m - 1);
      sw = p.w_scales + min(col0, p.n - 1) / FP8_BLOCK;
      if (kb0 < kb1) {
        sa += kb0 * p.a_scale_stride;
        sw += kb0 * p.w_scale_stride;
        sa_next = *sa;
        sw_next = *sw;
      }
#pragma unroll
      for (int c = 0; c < CW / 32; c++) {
        const int col = col0 + c * 32 + lane;
        bias_r[c] = p.bias && col < p.n ? p.bias[col] : 0.0f;
      }
    };
    if (first < p.tiles) enter_tile(first);

    for (int tile = first; tile < p.tiles && ok; tile += step) {
      const int row_t = row0, col_t = col0;
      const bool any = row_t < p.m && col_t < p.n;
      __syncwarp();
#pragma unroll
      for (int c = 0; c < CW / 32; c++) sbias[c * 32 + lane] = bias_r[c];
      uint64_t acc[CW / 2];  // f32 pairs
#pragma unroll
      for (int c = 0; c < CW / 2; c++) acc[c] = 0;
      for (int kb = kb0; kb < kb1; kb++, i++) {
        const float s1 = fp8_scale_product(sa_next, sw_next);
        const uint64_t s2 = pack_f32x2(s1, s1);
        if (kb + 1 < kb1) {
          sa += p.a_scale_stride;
          sw += p.w_scale_stride;
          sa_next = *sa;
          sw_next = *sw;
        }
        const int a = i & 1;
        if (!mbar_wait(&acc_full[a], (uint32_t)(i >> 1) & 1, abort_flag, p.dev_err, DEV_ERR_WAIT_ACC_FULL)) ok = false;
        if (__any_sync(~0u, !ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t t = lanes + (uint32_t)(a * BN);
        uint32_t r[2][16];
        // Rows past the last only hand the accumulator back. (Looked at only
        // where there are few rows: the test takes registers.)
        const bool work = MODE == FP8_SPLIT ? any : true;
        if (work) tmem_ld16(t, r[0]);
#pragma unroll
        for (int c = 0; c < CW / 16; c++) {
          if (!work && c + 1 < CW / 16) continue;
          tmem_wait_ld();
          if (c + 1 < CW / 16) {
            tmem_ld16(t + (uint32_t)(16 * (c + 1)), r[(c + 1) & 1]);
          } else {
            tc_fence_before();
            if (lane == 0) {
              if (PAIR)
                mbar_arrive_cluster(acc_bar + (uint32_t)(a * 8));
              else
                mbar_arrive(&acc_empty[a]);
            }
          }
#pragma unroll
          for (int q = 0; q < 8; q++)
            if (work) ffma2_acc(acc[c * 8 + q], r[c & 1][2 * q], r[c & 1][2 * q + 1], s2);
        }
        // The residual, once the last tile has left the patch: behind the
        // first block, so that the wait for the patch delays nothing.
        if (!SPLIT && kb == 0 && p.tma_out && p.residual && any && lane == 0) {
          bulk_wait_read();
          load_residual(row_t, col_t, 0);
        }
      }
      if constexpr (SPLIT) {
        // This CTA's sums in fours, four q of row `lane` at q ^ (lane % 16).
        ulonglong2* mine = reinterpret_cast<ulonglong2*>(patch) + lane * (CW / 4);
        if (any)
#pragma unroll
          for (int q = 0; q < CW / 4; q++) mine[q ^ (lane & 15)] = make_ulonglong2(acc[2 * q], acc[2 * q + 1]);
        break;
      }
      if (!ok) break;
      if (tile + step < p.tiles) enter_tile(tile + step);  // its first scales and bias are on their way
      if (!any) continue;
      if (lane == 0) {
        bulk_wait_read();  // the last tile has left the patch
        if (p.kblocks == 0 && p.tma_out && p.residual) load_residual(row_t, col_t, 0);
      }
      __syncwarp();
      // ---- bias, activation, residual, rounding
      // One copy of the code per activation, with and without a residual,
      // chosen once a tile: with the choices made per chunk, the unrolled
      // code of all of them put the executed part out of the instruction
      // cache's reach and kept chunks from overlapping (a 128-column row
      // took 9,000 cycles, against 1,500).
      auto write_tile = [&](auto act_c, auto res_c) {
        constexpr int ACT = decltype(act_c)::value;
        constexpr bool RES = decltype(res_c)::value;
        const int rows = min(32, p.m - row_t);
#pragma unroll
        for (int h = 0; h < ROUNDS; h++) {
          const int col_h = col_t + h * BOXES * BOX_COLS;
          if (p.tma_out) {
            if (h) {
              if (lane == 0) {
                bulk_wait_read();
                if (RES) load_residual(row_t, col_t, h);
              }
              __syncwarp();
            }
            if (RES) {
              if (!mbar_wait(&res_full[e], res_phase, abort_flag, p.dev_err, DEV_ERR_WAIT_FULL)) ok = false;
              res_phase ^= 1;
              res_flying = false;
            }
          } else if (RES) {
            const T* res = static_cast<const T*>(p.residual) + (long long)row_t * p.residual_stride;
#pragma unroll 1
            for (int b = 0; b < BOXES; b++)
              fp8_fill_box<T>(patch + b * 4096, lane, res, p.residual_stride, rows, col_h + b * BOX_COLS, p.n);
            __syncwarp();
          }
#pragma unroll
          for (int j = 0; j < BOXES * 8; j++) {
            const int at = h * BOXES * BOX_COLS + j * V;  // the chunk's first column
            float v[V];
#pragma unroll
            for (int q = 0; q < V; q += 4) {
              const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(sbias + at + q);
              const float2 x = unpack_f32x2(fadd2_pair(acc[(at + q) / 2], b.x));
              const float2 y = unpack_f32x2(fadd2_pair(acc[(at + q) / 2 + 1], b.y));
              v[q] = x.x;
              v[q + 1] = x.y;
              v[q + 2] = y.x;
              v[q + 3] = y.y;
            }
            op_act_vec<ACT, T, V>(v);
            uint4* chunk = reinterpret_cast<uint4*>(patch + (j >> 3) * 4096 + lane * 128 + (((j ^ lane) & 7) << 4));
            if (RES) add_16<T>(v, *chunk);
            *chunk = make_16<T>(v);
          }
          if (p.tma_out) {
            fence_proxy_async_shared();
            __syncwarp();
            if (lane == 0) {
#pragma unroll
              for (int b = 0; b < BOXES; b++)
                if (col_h + b * BOX_COLS < p.n) tma_store_2d(&out_map, patch + b * 4096, col_h + b * BOX_COLS, row_t);
              bulk_commit();
            }
          } else {
            __syncwarp();
            T* out = static_cast<T*>(p.out) + (long long)row_t * p.out_stride;
#pragma unroll 1
            for (int b = 0; b < BOXES; b++)
#pragma unroll 4
              for (int r = 0; r < rows; r++)
                fp8_drain_row<T>(patch + b * 4096, r, lane, out + r * p.out_stride, col_h + b * BOX_COLS, p.n);
            __syncwarp();
          }
        }
      };
      op_act_switch(p.act, [&](auto act_c) {
        if (p.residual)
          write_tile(act_c, std::true_type());
        else
          write_tile(act_c, std::false_type());
      });
      __syncwarp();  // the patch is read
    }
    if constexpr (SPLIT) {
      // The warps of the cluster take the tile's rows in turn: four columns a
      // lane, the CTAs' sums added in their order.
      int mt, nt;
      fp8_tile(p, first, &mt, &nt);
      const int rows = min(128, p.m - mt * 128), col = nt * 128 + 4 * lane, cols = min(4, p.n - col);
      float bias[4];
#pragma unroll
      for (int q = 0; q < 4; q++) bias[q] = p.bias ? p.bias[min(col + q, p.n - 1)] : 0.0f;
      cluster_sync();  // every CTA's sums are in its shared memory
      op_act_switch(p.act, [&](auto act_c) {
        constexpr int ACT = decltype(act_c)::value;
        constexpr int U = 4;  // rows at a time, for their loads to overlap
        const int stride = p.splits * FP8_EPI_WARPS;
#pragma unroll 1
        for (int r0 = (int)split * FP8_EPI_WARPS + e; ok && r0 < rows; r0 += U * stride) {
          float v[U][4], more[U][4];
#pragma unroll
          for (int u = 0; u < U; u++) {
            const int r = r0 + u * stride;
            const T* res = static_cast<const T*>(p.residual) + (mt * 128 + min(r, rows - 1)) * p.residual_stride;
#pragma unroll
            for (int q = 0; q < 4; q++) {
              v[u][q] = bias[q];
              // never under a condition of its own: the loads overlap
              more[u][q] = p.residual ? to_f32(res[min(col + q, p.n - 1)]) : 0.0f;
            }
          }
#pragma unroll 4
          for (int k = 0; k < p.splits; k++)
#pragma unroll
            for (int u = 0; u < U; u++) {
              const int r = r0 + u * stride;
              if (r >= rows) break;
              const uint8_t* at = smem + L::OUT_OFF + ((lane >> 4) * 4 + (r >> 5)) * L::OUT_WARP;
              const float4 x = ld_cluster_f32x4(
                  reinterpret_cast<const float4*>(at) + (r & 31) * (CW / 4) + ((lane ^ r) & 15), (uint32_t)k);
              v[u][0] += x.x;
              v[u][1] += x.y;
              v[u][2] += x.z;
              v[u][3] += x.w;
            }
#pragma unroll
          for (int u = 0; u < U; u++) {
            const int r = r0 + u * stride;
            op_act_vec<ACT, T, 4>(v[u]);
            T* out = static_cast<T*>(p.out) + (mt * 128 + r) * p.out_stride + col;
            if (r < rows)
#pragma unroll
              for (int q = 0; q < 4; q++)
                if (q < cols) out[q] = from_f32<T>(p.residual ? v[u][q] + more[u][q] : v[u][q]);
          }
        }
      });
    }
    if (lane == 0) {
      bulk_wait();
      // after an abort: a residual still on its way lands first
      if (res_flying) mbar_wait(&res_full[e], res_phase, abort_flag, p.dev_err, 0);
    }
  }
  if (SPLIT && warp < 4) cluster_sync();  // (of the epilogue's first one above)
  tc_fence_before();
  __syncthreads();
  if (PAIR || SPLIT) cluster_sync();  // nothing of another CTA is in flight to this one, or reads it
  if (warp == 1) {
    if (PAIR)
      tmem_dealloc_pair(tmem_base, 2 * BN);
    else
      tmem_dealloc(tmem_base, 2 * BN);
  }
}

}  // namespace iec
