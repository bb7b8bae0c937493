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
// Persistent CTAs of 320 threads walk the tiles: warp 0 loads (TMA, 128-byte
// swizzle), warp 1 issues the MMAs, warps 2..9 (two per TMEM lane quarter,
// half the columns each) scale and add the blocks and write the tile. All
// waits are bounded.
#pragma once

#include "ops_sm100.cuh"
#include "sm100.cuh"

namespace iec {

struct Fp8Params {
  int m, n, kblocks, act;
  int tiles_m, tiles_n, tiles;
  const float* a_scales;
  const float* w_scales;
  long long a_scale_stride, w_scale_stride;
  const float* bias;
  const void* residual;
  void* out;
  long long residual_stride, out_stride;
  int wide;  // rows of out (and residual) start on 32 bytes
  int* dev_err;
};

constexpr int FP8_THREADS = 320;
constexpr int FP8_GROUP = 8;  // M tiles walked together, so that L2 serves their w tiles

template <int BN>
struct Fp8Smem {
  static constexpr int A_BYTES = 128 * 128, B_BYTES = BN * 128, STAGE = A_BYTES + B_BYTES;
  static constexpr int NSTAGE = BN == 256 ? 4 : 6;
  static constexpr int STG_PITCH = 33;  // a warp's 32 x 32 patch of the output, one float of padding a row
  static constexpr int STG_OFF = NSTAGE * STAGE, STG_BYTES = 8 * 32 * STG_PITCH * 4;
  static constexpr int BAR_OFF = STG_OFF + STG_BYTES;
  static constexpr int MISC_OFF = BAR_OFF + (2 * NSTAGE + 4) * 8;
  static constexpr int BYTES = MISC_OFF + 16;
  static constexpr int DYN_BYTES = BYTES + 1024;
};

// Tile -> (M tile, N tile), in groups of FP8_GROUP M tiles.
__device__ __forceinline__ void fp8_tile(const Fp8Params& p, int tile, int* mt, int* nt) {
  const int per = FP8_GROUP * p.tiles_n, g = tile / per, r = tile - g * per;
  const int rows = min(FP8_GROUP, p.tiles_m - g * FP8_GROUP);
  *nt = r / rows;
  *mt = g * FP8_GROUP + r - *nt * rows;
}

// 32 bytes to or from global memory, 32-byte aligned.
__device__ __forceinline__ void st_global_32(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ void ld_global_32(const void* p, uint32_t* v) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "l"(p)
               : "memory");
}

// 32 bytes of T to f32 and back.
template <class T>
__device__ __forceinline__ void unpack_32(const uint32_t* v, float* f) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = __uint_as_float(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      T lo, hi;
      reinterpret_cast<uint16_t&>(lo) = (uint16_t)(v[i] & 0xffffu);
      reinterpret_cast<uint16_t&>(hi) = (uint16_t)(v[i] >> 16);
      f[2 * i] = to_f32(lo);
      f[2 * i + 1] = to_f32(hi);
    }
  }
}
template <class T>
__device__ __forceinline__ void pack_32(const float* f, uint32_t* v) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = __float_as_uint(f[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const T lo = from_f32<T>(f[2 * i]), hi = from_f32<T>(f[2 * i + 1]);
      v[i] = (uint32_t) reinterpret_cast<const uint16_t&>(lo) | (uint32_t) reinterpret_cast<const uint16_t&>(hi) << 16;
    }
  }
}

template <class T, int BN>
__global__ void __launch_bounds__(FP8_THREADS, 1)
    fp8_gemm_sm100(const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap w_map,
                   const Fp8Params p) {
  using L = Fp8Smem<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);
  uint64_t* empty = full + L::NSTAGE;
  uint64_t* acc_full = empty + L::NSTAGE;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC_OFF);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::MISC_OFF + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::NSTAGE; s++) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; a++) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 8);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 2 * BN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  griddep_launch_dependents();
  griddep_wait();

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------------------ producer
      int s = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x) {
        int mt, nt;
        fp8_tile(p, tile, &mt, &nt);
        for (int kb = 0; kb < p.kblocks; kb++) {
          if (!mbar_wait(&empty[s], phase ^ 1, abort_flag, p.dev_err, DEV_ERR_WAIT_EMPTY)) {
            ok = false;
            break;
          }
          uint8_t* st = smem + s * L::STAGE;
          mbar_arrive_expect_tx(&full[s], L::STAGE);
          tma_load_2d(st, &a_map, &full[s], kb * FP8_BLOCK, mt * 128);
          tma_load_2d(st + L::A_BYTES, &w_map, &full[s], kb * FP8_BLOCK, nt * BN);
          issued++;
          if (++s == L::NSTAGE) {
            s = 0;
            phase ^= 1;
          }
        }
      }
      // the copies in flight land before the CTA's shared memory goes
      for (int i = max(0, issued - L::NSTAGE); i < issued; i++)
        mbar_wait(&full[i % L::NSTAGE], (uint32_t)(i / L::NSTAGE) & 1, abort_flag, p.dev_err, 0);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      // ---------------------------------------------------------- MMA issuer
      constexpr uint32_t idesc = idesc_e4m3_f32(128, BN);
      int s = 0, i = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x)
        for (int kb = 0; kb < p.kblocks; kb++, i++) {
          const int a = i & 1;
          if (!mbar_wait(&acc_empty[a], ((uint32_t)(i >> 1) & 1) ^ 1, abort_flag, p.dev_err, DEV_ERR_WAIT_ACC_EMPTY) ||
              !mbar_wait(&full[s], phase, abort_flag, p.dev_err, DEV_ERR_WAIT_FULL)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t adesc = smem_desc_sw128(smem_u32(smem + s * L::STAGE));
          const uint64_t bdesc = smem_desc_sw128(smem_u32(smem + s * L::STAGE + L::A_BYTES));
#pragma unroll
          for (int j = 0; j < 4; j++)
            umma_f8(tmem_base + (uint32_t)(a * BN), adesc + 2 * j, bdesc + 2 * j, idesc, j != 0);
          umma_commit(&empty[s]);
          umma_commit(&acc_full[a]);
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
    constexpr int CW = BN / 2;  // columns of a thread
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    float* stg = reinterpret_cast<float*>(smem + L::STG_OFF) + (warp - 2) * 32 * L::STG_PITCH;
    const uint32_t lanes = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * CW);
    int i = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x) {
      int mt, nt;
      fp8_tile(p, tile, &mt, &nt);
      const int row0 = mt * 128 + quarter * 32, row = row0 + lane, col0 = nt * BN + half * CW;
      const float* sa = p.a_scales + min(row, p.m - 1);
      const float* sw = p.w_scales + min(col0, p.n - 1) / FP8_BLOCK;
      float2 acc[CW / 2];
#pragma unroll
      for (int c = 0; c < CW / 2; c++) acc[c] = make_float2(0.0f, 0.0f);
      float sa_next = 0.0f, sw_next = 0.0f;
      if (p.kblocks) {
        sa_next = sa[0];
        sw_next = sw[0];
      }
      for (int kb = 0; kb < p.kblocks; kb++, i++) {
        const float s1 = sa_next * sw_next;
        const float2 s2 = make_float2(s1, s1);
        if (kb + 1 < p.kblocks) {
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
        tmem_ld16(t, r[0]);
#pragma unroll
        for (int c = 0; c < CW / 16; c++) {
          tmem_wait_ld16(r[c & 1]);
          if (c + 1 < CW / 16) {
            tmem_ld16(t + (uint32_t)(16 * (c + 1)), r[(c + 1) & 1]);
          } else {
            tc_fence_before();
            if (lane == 0) mbar_arrive(&acc_empty[a]);
          }
#pragma unroll
          for (int e = 0; e < 8; e++)
            acc[c * 8 + e] = ffma2(make_float2(__uint_as_float(r[c & 1][2 * e]), __uint_as_float(r[c & 1][2 * e + 1])), s2,
                                   acc[c * 8 + e]);
        }
      }
      if (!ok) break;
      // ---- bias, activation, residual, rounding
      constexpr int V = 32 / (int)sizeof(T);
      const bool whole = p.wide && col0 + CW <= p.n;
      if (whole) {
        if (row < p.m) {
          T* out = static_cast<T*>(p.out) + row * p.out_stride + col0;
          const T* res = static_cast<const T*>(p.residual) + (p.residual ? row * p.residual_stride + col0 : 0);
#pragma unroll
          for (int c = 0; c < CW / V; c++) {
            float v[V];
#pragma unroll
            for (int e = 0; e < V; e++) {
              const float2 pr = acc[(c * V + e) / 2];
              v[e] = e & 1 ? pr.y : pr.x;
            }
            if (p.bias)
#pragma unroll
              for (int e = 0; e < V; e++) v[e] += p.bias[col0 + c * V + e];
            op_act_n<V>(v, p.act);
            uint32_t w[8];
            if (p.residual) {
              float f[V];
              ld_global_32(res + c * V, w);
              unpack_32<T>(w, f);
#pragma unroll
              for (int e = 0; e < V; e++) v[e] += f[e];
            }
            pack_32<T>(v, w);
            st_global_32(out + c * V, w);
          }
        }
      } else {
        // Through shared memory, 32 x 32 at a time, so that a warp's accesses
        // are runs of a row wherever the rows start.
#pragma unroll
        for (int c = 0; c < CW / 32; c++) {
          if (col0 + c * 32 >= p.n) break;
          __syncwarp();
#pragma unroll
          for (int e = 0; e < 16; e++) {
            stg[lane * L::STG_PITCH + 2 * e] = acc[c * 16 + e].x;
            stg[lane * L::STG_PITCH + 2 * e + 1] = acc[c * 16 + e].y;
          }
          __syncwarp();
          const int col = col0 + c * 32 + lane;
          if (col < p.n) {
            const float b = p.bias ? p.bias[col] : 0.0f;
            const int rows = min(32, p.m - row0);
            for (int r = 0; r < rows; r++) {
              float v = op_act_any(stg[r * L::STG_PITCH + lane] + b, p.act);
              if (p.residual) v += to_f32(static_cast<const T*>(p.residual)[(row0 + r) * p.residual_stride + col]);
              static_cast<T*>(p.out)[(row0 + r) * p.out_stride + col] = from_f32<T>(v);
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem_base, 2 * BN);
}

}  // namespace iec
