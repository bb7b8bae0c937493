// Group normalisation with an activation over channels-last maps.
//
//   mean = sum x / N, variance = sum (x - mean)^2 / N over the N = pixels *
//   c / groups values of a group, out = act((x - mean) rstd gamma + beta)
//
// Bound by memory: a value is read and written once and costs some ten
// instructions, with SiLU one and a half of them on the special-function unit.
//
// norm_resident: maps whose values fit into the shared memory of a cluster
// per channel segment (a run of whole groups). Each thread copies its own
// vectors there (cp.async), and sums, squared deviations and results are
// computed from there, so a value crosses HBM once each way, in one launch,
// and the variance is the exact two-pass one. The CTAs of a cluster split the
// pixels and add their group sums over distributed shared memory, in a fixed
// order.
//
// norm_stats + norm_apply: larger maps. The first kernel reduces chunks of
// pixels, per channel around the channel's first value (so that a mean far
// from zero costs no digits), to (mean, sum of squared deviations) per
// group; the second joins the chunks' pairs and applies them, walking the
// pixels backwards, since the last ones are the likeliest to be in L2 still.
#pragma once

#include "ops_sm100.cuh"
#include "sm100.cuh"

namespace iec {

// VE values of T next to each other as f32: 16 bytes where the map's
// channels, strides and base allow, else one at a time.
template <class T, int VE>
struct Vec {
  using Raw = std::conditional_t<VE == 1, T, uint4>;
  static __device__ __forceinline__ Raw zero() {
    if constexpr (VE == 1)
      return from_f32<T>(0.0f);
    else
      return make_uint4(0, 0, 0, 0);
  }
  static __device__ __forceinline__ Raw fetch(const T* p) { return *reinterpret_cast<const Raw*>(p); }
  static __device__ __forceinline__ void load(const T* p, float* v) { expand(fetch(p), v); }
  static __device__ __forceinline__ void expand(Raw q, float* v) {
    if constexpr (VE == 1) {
      v[0] = to_f32(q);
    } else {
      expand_16(q, v);
    }
  }
  static __device__ __forceinline__ void expand_16(uint4 q, float* v) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (sizeof(T) == 4) {
        v[i] = __uint_as_float(w[i]);
      } else {
        const uint16_t lo = (uint16_t)(w[i] & 0xffffu), hi = (uint16_t)(w[i] >> 16);
        v[2 * i] = to_f32(reinterpret_cast<const T&>(lo));
        v[2 * i + 1] = to_f32(reinterpret_cast<const T&>(hi));
      }
    }
  }
  static __device__ __forceinline__ void store(T* p, const float* v) {
    if constexpr (VE == 1) {
      *p = from_f32<T>(v[0]);
    } else if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      *reinterpret_cast<uint4*>(p) =
          make_uint4(pack_2<T>(v[0], v[1]), pack_2<T>(v[2], v[3]), pack_2<T>(v[4], v[5]), pack_2<T>(v[6], v[7]));
    }
  }
};

// A thread's VE values of a pixel as e4m3 codes with the scale of their block
// of 128: the block's threads are 128 / VE consecutive lanes. `live`: the
// thread's channels exist.
template <int VE>
__device__ __forceinline__ void store_fp8(const Fp8Out& q, long long row, int ch, bool live, const float* v) {
  constexpr int LANES = FP8_BLOCK / VE;
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < VE; e++) top = max(top, abs_bits(v[e]));
  if (!live) top = 0;
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) top = max(top, __shfl_xor_sync(~0u, top, o));
  float factor, scale;
  fp8_scale(top, &factor, &scale);
  if (!live) return;
  uint32_t w[VE / 4];
#pragma unroll
  for (int e = 0; e < VE; e += 4)
    w[e / 4] = (uint32_t)e4m3x2(v[e] * factor, v[e + 1] * factor) |
               (uint32_t)e4m3x2(v[e + 2] * factor, v[e + 3] * factor) << 16;
  uint8_t* out = q.codes + row * (long long)q.code_stride + ch;
  if constexpr (VE == 8)
    *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
  else
    *reinterpret_cast<uint32_t*>(out) = w[0];
  if (ch % FP8_BLOCK == 0) q.scales[(long long)(ch / FP8_BLOCK) * (long long)q.scale_stride + row] = scale;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// ---------------------------------------------------------------- resident
struct NormResident {
  int seg_c, vecs, rows;  // channels of a segment, their vectors, pixels a CTA takes per step
  int slots;              // threads of a pixel: vecs, rounded up to whole blocks of 128 channels with fp8
  int pixels;             // of a CTA
};

constexpr int NORM_THREADS = 512;

__device__ __forceinline__ void cp_async_16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(const float* p, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_map(p, rank)) : "memory");
  return v;
}

template <class T, bool FP8>
__global__ void __launch_bounds__(NORM_THREADS, 1) norm_resident(const NormSpec p, const NormResident q) {
  constexpr bool FAST = !FP8 && sizeof(T) == 2;
  constexpr int VE = 16 / (int)sizeof(T);
  extern __shared__ __align__(16) uint8_t smem[];
  const int rank = blockIdx.x, ctas = gridDim.x, seg = blockIdx.y, map = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cg = p.c / p.groups, groups = q.seg_c / cg;
  // [step][thread] vectors, then per-channel sums of the rows of threads,
  // then the group sums of the two reductions and the group's results.
  uint4* data = reinterpret_cast<uint4*>(smem);
  const int steps = (q.pixels + q.rows - 1) / q.rows;
  float* red = reinterpret_cast<float*>(smem + (size_t)steps * NORM_THREADS * 16);
  float* sums = red + NORM_THREADS * VE;  // [2][groups]
  float* stat = sums + 2 * groups;        // [2][groups]: mean, rstd
  const int slot = threadIdx.x % q.slots, r = threadIdx.x / q.slots;
  const bool live = r < q.rows && slot < q.vecs;
  const int first = rank * q.pixels, last = (int)min((long long)first + q.pixels, p.pixels);
  const int ch0 = seg * q.seg_c, ch = ch0 + slot * VE;
  griddep_launch_dependents();
  griddep_wait();

  const T* x = static_cast<const T*>(p.x) + map * p.x_map_stride + ch;
  for (int s = 0; s < steps; s++) {
    const int px = first + s * q.rows + r;
    if (live && px < last) cp_async_16(&data[s * NORM_THREADS + threadIdx.x], x + px * p.x_stride);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");

  // A group's total over this CTA of each thread's per-channel sums, the
  // whole cluster's totals being ready when it returns.
  auto group_total = [&](const float* v, float* own) {
    if (live)
#pragma unroll
      for (int e = 0; e < VE; e++) red[r * q.seg_c + slot * VE + e] = v[e];
    __syncthreads();
    for (int ch_ = threadIdx.x; ch_ < q.seg_c; ch_ += NORM_THREADS) {
      float t = 0.0f;
      for (int k = 0; k < q.rows; k++) t += red[k * q.seg_c + ch_];
      red[ch_] = t;  // its first row, which only this thread has read
    }
    __syncthreads();
    for (int g = warp; g < groups; g += NORM_THREADS / 32) {
      float t = 0.0f;
      for (int k = lane; k < cg; k += 32) t += red[g * cg + k];
      t = warp_sum(t);
      if (lane == 0) own[g] = t;
    }
    cluster_sync();
  };
  auto joined = [&](const float* own, int g) {
    float t = 0.0f;
    for (int k = 0; k < ctas; k++) t += ld_cluster_f32(own + g, (uint32_t)k);
    return t;
  };
  const float count = (float)p.pixels * (float)cg;

  float acc[VE];
#pragma unroll
  for (int e = 0; e < VE; e++) acc[e] = 0.0f;
  for (int s = 0; s < steps; s++)
    if (live && first + s * q.rows + r < last) {
      float v[VE];
      Vec<T, VE>::expand(data[s * NORM_THREADS + threadIdx.x], v);
#pragma unroll
      for (int e = 0; e < VE; e++) acc[e] += v[e];
    }
  group_total(acc, sums);
  for (int g = threadIdx.x; g < groups; g += NORM_THREADS) stat[g] = joined(sums, g) / count;
  __syncthreads();
  float mean[VE];
#pragma unroll
  for (int e = 0; e < VE; e++) {
    mean[e] = live ? stat[(slot * VE + e) / cg] : 0.0f;
    acc[e] = 0.0f;
  }
  for (int s = 0; s < steps; s++)
    if (live && first + s * q.rows + r < last) {
      float v[VE];
      Vec<T, VE>::expand(data[s * NORM_THREADS + threadIdx.x], v);
#pragma unroll
      for (int e = 0; e < VE; e++) {
        const float d = v[e] - mean[e];
        acc[e] = fmaf(d, d, acc[e]);
      }
    }
  group_total(acc, sums + groups);
  for (int g = threadIdx.x; g < groups; g += NORM_THREADS)
    stat[groups + g] = 1.0f / sqrtf(joined(sums + groups, g) / count + p.eps);
  __syncthreads();
  float scale[VE], beta[VE];
#pragma unroll
  for (int e = 0; e < VE; e++) {
    scale[e] = live ? stat[groups + (slot * VE + e) / cg] * (p.gamma ? p.gamma[ch + e] : 1.0f) : 0.0f;
    beta[e] = live && p.beta ? p.beta[ch + e] : 0.0f;
  }
  op_act_switch(p.act, [&](auto act_c) {
    constexpr int ACT = decltype(act_c)::value;
    for (int s = 0; s < steps; s++) {
      const int px = first + s * q.rows + r;
      const bool here = live && px < last;
      // with fp8 the lanes of a block go through the shuffles together
      if (!FP8 && !here) continue;
      float v[VE];
      Vec<T, VE>::expand(here ? data[s * NORM_THREADS + threadIdx.x] : make_uint4(0, 0, 0, 0), v);
#pragma unroll
      for (int e = 0; e < VE; e++) v[e] = fmaf(v[e] - mean[e], scale[e], beta[e]);
      op_act_vec<ACT, FAST, VE>(v);
      if (FP8)
        store_fp8<VE>(p.q, map * p.pixels + px, ch, here, v);
      else
        Vec<T, VE>::store(static_cast<T*>(p.out) + map * p.out_map_stride + px * p.out_stride + ch, v);
    }
  });
  cluster_sync();  // the others have read this CTA's sums
}

// ------------------------------------------------------------- two kernels
// A tile is a run of up to NORM_THREADS vectors of channels (tile_c
// channels, the last one shorter), a chunk a run of pixels. part[map][chunk]
// [tile][slot] is the pair of the tile's slot-th group over the chunk.
struct NormChunks {
  int tiles, tile_c, chunks, slots;
  long long chunk;  // pixels
  int map0;         // the first map of this launch
  float2* part;
};

template <class T, int VE>
__global__ void __launch_bounds__(NORM_THREADS) norm_stats(const NormSpec p, const NormChunks q) {
  extern __shared__ __align__(16) float red[];  // [3][rows][channels of the tile]: value, mean, deviations
  const int tile = blockIdx.y, map = q.map0 + blockIdx.z;
  const int c0 = tile * q.tile_c, c = min(q.tile_c, p.c - c0), vecs = c / VE, cg = p.c / p.groups;
  const int slot = threadIdx.x % vecs, r = threadIdx.x / vecs, rows = NORM_THREADS / vecs;
  const bool live = r < rows;
  const long long first = blockIdx.x * q.chunk, last = min(first + q.chunk, p.pixels);
  griddep_launch_dependents();
  griddep_wait();
  const T* x = static_cast<const T*>(p.x) + map * p.x_map_stride + c0 + slot * VE;
  // Sums of the distances to this thread's first value of the channel.
  float k[VE], s[VE], d2[VE];
  int n = 0;
#pragma unroll
  for (int e = 0; e < VE; e++) k[e] = s[e] = d2[e] = 0.0f;
  if (live && first + r < last) {
    const T* at = x + (first + r) * p.x_stride;
    const long long step = (long long)rows * p.x_stride;
    Vec<T, VE>::load(at, k);
    n = (int)((last - first - r + rows - 1) / rows);
    auto add = [&](typename Vec<T, VE>::Raw raw) {
      float v[VE];
      Vec<T, VE>::expand(raw, v);
#pragma unroll
      for (int e = 0; e < VE; e++) {
        const float d = v[e] - k[e];
        s[e] += d;
        d2[e] = fmaf(d, d, d2[e]);
      }
    };
    constexpr int U = 8;
    int i = 0;
    for (; i + U <= n; i += U, at += U * step) {
      typename Vec<T, VE>::Raw raw[U];
#pragma unroll
      for (int u = 0; u < U; u++) raw[u] = Vec<T, VE>::fetch(at + u * step);
#pragma unroll
      for (int u = 0; u < U; u++) add(raw[u]);
    }
    for (; i < n; i++, at += step) add(Vec<T, VE>::fetch(at));
  }
  // (mean, deviations) of each thread's channels, joined over the rows of
  // threads (each of its own count), then over a group's channels.
  float* smean = red;
  float* sdev = red + NORM_THREADS * VE;
  if (live) {
    const float inv = n ? 1.0f / (float)n : 0.0f;
#pragma unroll
    for (int e = 0; e < VE; e++) {
      smean[r * c + slot * VE + e] = fmaf(s[e], inv, k[e]);
      // not below zero; NaN stays
      const float dev = fmaf(-s[e] * inv, s[e], d2[e]);
      sdev[r * c + slot * VE + e] = dev < 0.0f ? 0.0f : dev;
    }
  }
  __syncthreads();
  const int px = (int)(last - first), full = min(rows, px);
  const float inv_px = 1.0f / (float)px;
  for (int ch = threadIdx.x; ch < c; ch += NORM_THREADS) {
    float mean = 0.0f, dev = 0.0f;
    for (int k_ = 0; k_ < full; k_++)
      mean = fmaf((float)((px - k_ + rows - 1) / rows) * inv_px, smean[k_ * c + ch], mean);
    for (int k_ = 0; k_ < full; k_++) {
      const float d = smean[k_ * c + ch] - mean;
      dev += fmaf((float)((px - k_ + rows - 1) / rows) * d, d, sdev[k_ * c + ch]);
    }
    smean[ch] = mean;  // its first row, which only this thread has read
    sdev[ch] = dev;
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g0 = c0 / cg, g1 = (c0 + c - 1) / cg;
  for (int g = g0 + warp; g <= g1; g += NORM_THREADS / 32) {
    const int a = max(g * cg, c0) - c0, b = min((g + 1) * cg, c0 + c) - c0;
    float t = 0.0f;
    for (int ch = a + lane; ch < b; ch += 32) t += smean[ch];
    const float mean = warp_sum(t) / (float)(b - a);
    t = 0.0f;
    for (int ch = a + lane; ch < b; ch += 32) {
      const float d = smean[ch] - mean;
      t += fmaf((float)px * d, d, sdev[ch]);
    }
    t = warp_sum(t);
    if (lane == 0)
      q.part[((blockIdx.z * (long long)q.chunks + blockIdx.x) * q.tiles + tile) * q.slots + g - g0] = make_float2(mean, t);
  }
}

// Mean and rstd of group `g` of map `z` (of this launch) from the chunks'
// pairs, by one warp; every lane gets them.
__device__ __forceinline__ float2 norm_join(const NormSpec& p, const NormChunks& q, int z, int g) {
  const int cg = p.c / p.groups, lane = threadIdx.x & 31;
  const int t0 = g * cg / q.tile_c, t1 = (g * cg + cg - 1) / q.tile_c, span = t1 - t0 + 1;
  auto pair = [&](int i, float* n) {
    const int chunk = i / span, tile = t0 + i % span, c0 = tile * q.tile_c;
    const int w = min((g + 1) * cg, c0 + q.tile_c) - max(g * cg, c0);
    *n = (float)(min((chunk + 1) * q.chunk, p.pixels) - chunk * q.chunk) * (float)w;
    return q.part[((z * (long long)q.chunks + chunk) * q.tiles + tile) * q.slots + g - c0 / cg];
  };
  const float count = (float)p.pixels * (float)cg;
  float t = 0.0f, n;
  for (int i = lane; i < q.chunks * span; i += 32) {
    const float2 v = pair(i, &n);
    t = fmaf(n, v.x, t);
  }
  const float mean = warp_sum(t) / count;
  t = 0.0f;
  for (int i = lane; i < q.chunks * span; i += 32) {
    const float2 v = pair(i, &n);
    const float d = v.x - mean;
    t += fmaf(n * d, d, v.y);
  }
  return make_float2(mean, 1.0f / sqrtf(warp_sum(t) / count + p.eps));
}

template <class T, int VE, bool FP8>
__global__ void __launch_bounds__(NORM_THREADS, 2) norm_apply(const NormSpec p, const NormChunks q) {
  constexpr bool FAST = !FP8 && sizeof(T) == 2;
  extern __shared__ __align__(16) float2 stat[];  // of the tile's groups
  // the chunks backwards, the latest map first
  const int tile = blockIdx.y, z = (int)gridDim.z - 1 - (int)blockIdx.z, map = q.map0 + z;
  const int c0 = tile * q.tile_c, c = min(q.tile_c, p.c - c0), vecs = c / VE, cg = p.c / p.groups;
  const int g0 = c0 / cg, g1 = (c0 + c - 1) / cg;
  griddep_launch_dependents();
  griddep_wait();
  for (int g = g0 + (int)(threadIdx.x >> 5); g <= g1; g += NORM_THREADS / 32) {
    const float2 st = norm_join(p, q, z, g);
    if ((threadIdx.x & 31) == 0) stat[g - g0] = st;
  }
  __syncthreads();
  constexpr int LANES = FP8 ? FP8_BLOCK / VE : 1;
  const int slots = (vecs + LANES - 1) / LANES * LANES;
  const int slot = threadIdx.x % slots, r = threadIdx.x / slots, rows = NORM_THREADS / slots;
  const bool live = r < rows && slot < vecs;
  const int ch = c0 + slot * VE;
  float mean[VE], scale[VE], beta[VE];
#pragma unroll
  for (int e = 0; e < VE; e++) {
    const float2 st = live ? stat[(ch + e) / cg - g0] : make_float2(0.0f, 0.0f);
    mean[e] = st.x;
    scale[e] = live && p.gamma ? st.y * p.gamma[ch + e] : st.y;
    beta[e] = live && p.beta ? p.beta[ch + e] : 0.0f;
  }
  const long long span = (p.pixels + gridDim.x - 1) / gridDim.x;
  const long long first = ((long long)gridDim.x - 1 - blockIdx.x) * span, last = min(first + span, p.pixels);
  const T* x = static_cast<const T*>(p.x) + map * p.x_map_stride + ch;
  T* out = FP8 ? nullptr : static_cast<T*>(p.out) + map * p.out_map_stride + ch;
  const int steps = first < last ? (int)((last - first + rows - 1) / rows) : 0;
  op_act_switch(p.act, [&](auto act_c) {
    constexpr int ACT = decltype(act_c)::value;
    constexpr int U = VE == 1 ? 8 : 4;
    for (int s = (steps - 1) / U * U; s >= 0 && steps; s -= U) {
      typename Vec<T, VE>::Raw raw[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const long long px = first + (long long)(s + u) * rows + r;
        raw[u] = Vec<T, VE>::zero();
        if (live && px < last) raw[u] = Vec<T, VE>::fetch(x + px * p.x_stride);
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const long long px = first + (long long)(s + u) * rows + r;
        const bool here = live && px < last;
        float v[VE];
        Vec<T, VE>::expand(raw[u], v);
#pragma unroll
        for (int e = 0; e < VE; e++) v[e] = fmaf(v[e] - mean[e], scale[e], beta[e]);
        op_act_vec<ACT, FAST, VE>(v);
        if constexpr (FP8)
          store_fp8<VE>(p.q, map * p.pixels + px, ch, here, v);
        else if (here)
          Vec<T, VE>::store(out + px * p.out_stride, v);
      }
    }
  });
}

// 8-bit rows of maps whose channels do not fall into vectors: one warp per
// pixel and block of 128 channels, four channels a lane, 32 apart.
template <class T>
__global__ void __launch_bounds__(NORM_THREADS) norm_apply_fp8_odd(const NormSpec p, const NormChunks q) {
  extern __shared__ __align__(16) float2 stat[];  // of all groups
  const int z = (int)gridDim.z - 1 - (int)blockIdx.z, map = q.map0 + z, cg = p.c / p.groups;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, block = blockIdx.y;
  const int ga = block * FP8_BLOCK / cg, gb = min(block * FP8_BLOCK + FP8_BLOCK - 1, p.c - 1) / cg;
  griddep_launch_dependents();
  griddep_wait();
  for (int g = ga + warp; g <= gb; g += NORM_THREADS / 32) {
    const float2 st = norm_join(p, q, z, g);
    if (lane == 0) stat[g - ga] = st;
  }
  __syncthreads();
  float mean[4], scale[4], beta[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int ch = block * FP8_BLOCK + j * 32 + lane;
    const float2 st = ch < p.c ? stat[ch / cg - ga] : make_float2(0.0f, 0.0f);
    mean[j] = st.x;
    scale[j] = ch < p.c && p.gamma ? st.y * p.gamma[ch] : st.y;
    beta[j] = ch < p.c && p.beta ? p.beta[ch] : 0.0f;
  }
  const T* x = static_cast<const T*>(p.x) + map * p.x_map_stride + block * FP8_BLOCK + lane;
  op_act_switch(p.act, [&](auto act_c) {
    constexpr int ACT = decltype(act_c)::value;
    const long long step = (long long)gridDim.x * (NORM_THREADS / 32);
    for (long long px = (long long)blockIdx.x * (NORM_THREADS / 32) + warp; px < p.pixels; px += step) {
      float v[4];
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 4; j++)
        v[j] = block * FP8_BLOCK + j * 32 + lane < p.c ? to_f32(x[px * p.x_stride + j * 32]) : 0.0f;
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] = fmaf(v[j] - mean[j], scale[j], beta[j]);
      op_act_vec<ACT, false, 4>(v);
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (block * FP8_BLOCK + j * 32 + lane < p.c) top = max(top, abs_bits(v[j]));
      top = __reduce_max_sync(~0u, top);
      float factor, sc;
      fp8_scale(top, &factor, &sc);
      const long long row = map * p.pixels + px;
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (block * FP8_BLOCK + j * 32 + lane < p.c)
          p.q.codes[row * (long long)p.q.code_stride + block * FP8_BLOCK + j * 32 + lane] =
              (uint8_t)e4m3x2(v[j] * factor, 0.0f);
      if (lane == 0) p.q.scales[block * (long long)p.q.scale_stride + row] = sc;
    }
  });
}

}  // namespace iec
