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
// vectors there (cp.async) and takes statistics as they arrive, so a value
// crosses HBM once each way, in one launch; the CTAs of a cluster split the
// pixels and join their statistics over distributed shared memory.
//
// 4 x 64 x 64 x 512 f16 with SiLU (34 MB): 12 us, of which the loads take 2.6,
// the statistics 2 and results and stores 4.5, one after another; a single
// small map, 16 x 16 x 512: 4.8 us. To e4m3, where groups end inside blocks
// of 128 channels, segments of whole groups and blocks are long and few; CTAs
// then write single blocks and read the groups around them twice (32 x 32 x
// 768, groups of 24: 6.2 us in 6 x 16 CTAs, 9.7 in 2 x 16; 32 x 32 x 640,
// groups of 20: 6.6 against 13.6).
//
// norm_stats + norm_apply: larger maps. The first kernel reduces chunks of
// pixels, a cluster of CTAs each, to (mean, sum of squared deviations) per
// group; the second joins the chunks' pairs and applies them, walking the
// pixels backwards, since the last ones are the likeliest to be in L2 still.
// 2 x 768 x 512 x 128 bf16 (201 MB, twice the size of a map that L2 holds):
// 114 us, 45 and 69 of it. 8 x 128 x 128 x 256 f16 to e4m3: 47 us, of which
// norm_apply takes 25 without an activation (as to f16), 31 with SiLU and 43 with
// GELU: with 16 warps an SM (128 registers) it issues in half of its cycles, its
// warps waiting for instructions, for one another and for exponentials, whose
// unit SiLU keeps busy for 39 % of the time. Channels that are no whole vectors
// are read one by one: 3 x 137 x 153 x 321 f16 to e4m3 77 us (61 MB).
//
// Statistics: each thread takes a few pixels at a time from registers, their
// mean and the squared deviations around it, and joins that to what it has
//   mean' = mean + d k / (n + k),  dev' = dev + dev_k + d^2 n k / (n + k)
// (k values of mean mean_k after n, d = mean_k - mean), as threads, CTAs and
// chunks are joined after it (means as one of them plus weighted differences
// from it): no difference of large sums anywhere, so a mean far from zero
// costs no digits, and equal values have variance 0. The order is fixed.
#pragma once

#include "ops_sm100.cuh"
#include "sm100.cuh"

namespace iec {

constexpr int NORM_THREADS = 512;
constexpr int NORM_RING = 2;
constexpr int APPLY_THREADS = 256;

// A thread's VE values of a pixel as e4m3 codes at `out`; the scale of their
// block of 128, whose threads are 128 / VE consecutive lanes. `live`: the
// thread's channels exist.
template <int VE, bool AL>
__device__ __forceinline__ float store_fp8(uint8_t* out, bool live, const float* v) {
  constexpr int LANES = FP8_BLOCK / VE;
  float most = 0.0f;
#pragma unroll
  for (int e = 0; e < VE; e++) most = max_abs(v[e], most);
  uint32_t top = live ? abs_bits(most) : 0u;
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) top = max(top, __shfl_xor_sync(~0u, top, o));
  float factor, scale;
  fp8_scale(top, &factor, &scale);
  if (!live) return scale;
  uint32_t w[VE / 4];
#pragma unroll
  for (int e = 0; e < VE; e += 4) {
    const float2 a = fmul2(make_float2(v[e], v[e + 1]), both(factor));
    const float2 b = fmul2(make_float2(v[e + 2], v[e + 3]), both(factor));
    w[e / 4] = (uint32_t)e4m3x2(a.x, a.y) | (uint32_t)e4m3x2(b.x, b.y) << 16;
  }
  if constexpr (!AL) {
#pragma unroll
    for (int e = 0; e < VE; e++) out[e] = (uint8_t)(w[e / 4] >> (8 * (e % 4)));
  } else if constexpr (VE == 8) {
    *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
  } else {
    *reinterpret_cast<uint32_t*>(out) = w[0];
  }
  return scale;
}

__device__ __forceinline__ void cp_async_16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
template <int LEFT>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// The running statistics of a thread's VE channels.
template <int VE>
struct Running {
  float mean[VE], dev[VE];
  int n = 0;
  __device__ __forceinline__ Running() {
#pragma unroll
    for (int e = 0; e < VE; e++) mean[e] = dev[e] = 0.0f;
  }
  // U pixels, two channels at a time: few are held as f32, on packed pairs.
  template <class V, int U>
  __device__ __forceinline__ void add(const typename V::Raw* raw) {
    const float share = (float)U * op_rcp((float)(n + U)), both_n = (float)n * share;
    constexpr int P = VE == 1 ? 1 : 2;
#pragma unroll
    for (int e = 0; e < VE; e += P) {
      float2 v[U], m[U];
#pragma unroll
      for (int u = 0; u < U; u++) m[u] = v[u] = V::pair(raw[u], e / P);
      // pairs of pairs: the mean of equal values is that value
#pragma unroll
      for (int k = U / 2; k; k /= 2)
#pragma unroll
        for (int u = 0; u < k; u++) m[u] = fadd2(m[u], m[u + k]);
      m[0] = fmul2(m[0], both(1.0f / (float)U));
      float2 q = make_float2(dev[e], dev[e + P - 1]);
      const float2 old = make_float2(mean[e], mean[e + P - 1]);
      const float2 neg = make_float2(-m[0].x, -m[0].y);
#pragma unroll
      for (int u = 0; u < U; u++) {
        const float2 x = fadd2(v[u], neg);
        q = ffma2(x, x, q);
      }
      const float2 d = fadd2(old, neg);  // the other way round: its sign cancels below
      const float2 now = ffma2(d, both(-share), old);
      q = ffma2(fmul2(d, both(both_n)), d, q);
      mean[e] = now.x;
      dev[e] = q.x;
      mean[e + P - 1] = P == 2 ? now.y : now.x;
      dev[e + P - 1] = P == 2 ? q.y : q.x;
    }
    n += U;
  }
};

// The largest power of two, at most VE, that divides a group's channels: so
// many (1 << shift) of a thread's channels next to each other are of one group.
template <int VE>
__host__ __device__ __forceinline__ int norm_shift(int cg) {
  int s = 0;
  while ((1 << s) < VE && cg % (2 << s) == 0) s++;
  return s;
}

// Joins a thread's channels (each of n pixels) in runs of 1 << shift, and
// stores the statistics of the VE >> shift runs at mean[] and dev[].
template <int VE, int K>
__device__ __forceinline__ void join_runs(Running<VE>& s, float half) {
#pragma unroll
  for (int e = 0; e < VE; e += 2 * K) {
    const float x = s.mean[e] - s.mean[e + K];
    s.dev[e] = s.dev[e] + s.dev[e + K] + x * x * (half * (float)K);
    s.mean[e] = fmaf(-0.5f, x, s.mean[e]);
  }
}
template <int VE, int K>
__device__ __forceinline__ void put_runs(const Running<VE>& s, float* mean, float* dev) {
#pragma unroll
  for (int e = 0; e < VE; e += K) {
    mean[e / K] = s.mean[e];
    dev[e / K] = s.dev[e];
  }
}
template <int VE>
__device__ __forceinline__ void store_runs(Running<VE>& s, int shift, float* mean, float* dev) {
  const float half = 0.5f * (float)s.n;
  if (shift == 0) return put_runs<VE, 1>(s, mean, dev);
  if constexpr (VE > 1) {
    join_runs<VE, 1>(s, half);
    if (shift == 1) return put_runs<VE, 2>(s, mean, dev);
    join_runs<VE, 2>(s, half);
    if (shift == 2) return put_runs<VE, 4>(s, mean, dev);
    if constexpr (VE == 8) {
      join_runs<VE, 4>(s, half);
      put_runs<VE, 8>(s, mean, dev);
    }
  }
}

// What the joining of a CTA's threads needs, found on the host (a division
// on the device is a chain of a hundred cycles, and this code is one chain):
// the runs of a tile, and the same of the last, shorter tile.
struct NormJoin {
  int rows, shift;   // rows of threads; channels of a run
  int cg, runs[2];   // runs of a group, of a tile
  FastDiv by_rows, by_cg, by_runs[2];
};

// Entries that join_threads keeps: shared floats, three for each.
__host__ __device__ __forceinline__ int norm_entries(int runs) { return max(runs, NORM_THREADS); }

// Joins the statistics of a CTA's threads per group: mean[r * c + ch] and
// dev[] of the ch-th of c runs over the pixels r, r + rows, ... of `px` > 0.
// The tile starts with run c0. `entries` takes 3 norm_entries(c) floats.
// Calls put(group, mean, dev) in one lane for each group that has some of
// the tile's runs.
template <class F>
__device__ __forceinline__ void join_threads(const NormJoin& q, bool last, const float* mean, const float* dev,
                                             float* entries, int px, int c0, F&& put) {
  const int c = q.runs[last];
  float* emean = entries;
  float* edev = entries + norm_entries(c);
  float* en = entries + 2 * norm_entries(c);
  __syncthreads();
  // First each run over the rows part, part + parts, ...; row r has k0 + (r <
  // rem) pixels. Entry ch * parts + part: a group's entries are one stretch.
  const int full = min(q.rows, px);
  const int part = (int)q.by_runs[last].div(threadIdx.x), ch0 = (int)threadIdx.x - part * c;
  const int parts = max(1, min((int)q.by_runs[last].div(NORM_THREADS), full));
  const int k0 = (int)q.by_rows.div((uint32_t)px), rem = px - k0 * q.rows;
  const float few = (float)k0, more = (float)(k0 + 1), width = (float)(1 << q.shift);
  if (part < parts)
#pragma unroll 1
    for (int ch = ch0; ch < c; ch += parts == 1 ? NORM_THREADS : c) {
      const float m0 = mean[part * c + ch];
      float m = 0.0f, d = 0.0f, n = 0.0f;
      if (part + parts >= full) {  // one row
        m = m0;
        d = dev[part * c + ch];
        n = part < rem ? more : few;
      } else {
#pragma unroll 1
        for (int r = part, at = part * c + ch; r < full; r += parts, at += parts * c) {
          const float k = r < rem ? more : few;
          m = fmaf(k, mean[at] - m0, m);
          n += k;
        }
        m = fmaf(m, op_rcp(n), m0);
#pragma unroll 1
        for (int r = part, at = part * c + ch; r < full; r += parts, at += parts * c) {
          const float x = mean[at] - m;
          d += fmaf((r < rem ? more : few) * width * x, x, dev[at]);
        }
      }
      const int to = ch * parts + part;
      emean[to] = m;
      edev[to] = d;
      en[to] = n;
    }
  __syncthreads();
  // Then a group's entries, one warp a group.
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g0 = (int)q.by_cg.div((uint32_t)c0), g1 = (int)q.by_cg.div((uint32_t)(c0 + c - 1));
#pragma unroll 1
  for (int g = g0 + warp; g <= g1; g += NORM_THREADS / 32) {
    const int a = max(g * q.cg - c0, 0), w = min((g + 1) * q.cg - c0, c) - a;
    const int from = a * parts + lane, to = (a + w) * parts;
    const float m0 = emean[a * parts], inv = op_rcp((float)px * (float)w);
    float m = 0.0f, d = 0.0f;
    if (w * parts <= 4 * 32) {  // the usual case, from registers
      float v[4], n[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const bool some = from + 32 * i < to;
        v[i] = some ? emean[from + 32 * i] : m0;
        n[i] = some ? en[from + 32 * i] : 0.0f;
        d += some ? edev[from + 32 * i] : 0.0f;
        m = fmaf(n[i], v[i] - m0, m);
      }
      m = fmaf(warp_sum(m), inv, m0);
#pragma unroll
      for (int i = 0; i < 4; i++) d = fmaf(n[i] * width * (v[i] - m), v[i] - m, d);
    } else {
#pragma unroll 1
      for (int i = from; i < to; i += 32) m = fmaf(en[i], emean[i] - m0, m);
      m = fmaf(warp_sum(m), inv, m0);
#pragma unroll 1
      for (int i = from; i < to; i += 32) d += fmaf(en[i] * width * (emean[i] - m), emean[i] - m, edev[i]);
    }
    d = warp_sum(d);
    if (lane == 0) put(g, m, d);
  }
}

// The constants of a thread's VE channels from its groups' (mean, rstd):
// act((v - mean) scale + shift). (v scale + (shift - mean scale) would be an
// operation less, but rounds at the size of mean scale.)
template <int VE>
struct Affine {
  float minus[VE], scale[VE], shift[VE];  // minus the mean
  __device__ __forceinline__ void fetch(const NormSpec& p, int ch, bool live) {
#pragma unroll
    for (int e = 0; e < VE; e++) {
      scale[e] = live && p.gamma ? p.gamma[ch + e] : 1.0f;
      shift[e] = live && p.beta ? p.beta[ch + e] : 0.0f;
    }
  }
  // `ch`: the first channel; stat[0] is group `g0`'s.
  __device__ __forceinline__ void set(const float2* stat, int ch, int g0, int cg, const FastDiv& by_cg) {
    int g = (int)by_cg.div((uint32_t)ch), left = (g + 1) * cg - ch;
#pragma unroll
    for (int e = 0; e < VE; e++) {
      const float2 st = stat[g - g0];
      minus[e] = -st.x;
      scale[e] *= st.y;
      if (--left == 0) {
        g++;
        left = cg;
      }
    }
  }
  __device__ __forceinline__ void apply(float* v) const {
    if constexpr (VE == 1) {
      v[0] = fmaf(v[0] + minus[0], scale[0], shift[0]);
    } else {
#pragma unroll
      for (int e = 0; e < VE; e += 2) {
        const float2 d = fadd2(make_float2(v[e], v[e + 1]), make_float2(minus[e], minus[e + 1]));
        const float2 y = ffma2(d, make_float2(scale[e], scale[e + 1]), make_float2(shift[e], shift[e + 1]));
        v[e] = y.x;
        v[e + 1] = y.y;
      }
    }
  }
};

// 1 / sqrt(v), rounded once: rsqrtf's two units would be a whole group's.
__device__ __forceinline__ float norm_rstd(float v) { return __frsqrt_rn(v); }

// ---------------------------------------------------------------- resident
// A CTA writes a segment of seg_c channels and reads its window: the segment
// and, where groups cross its ends (only with fp8, whose x nobody writes),
// the vectors around it that complete them. Two CTAs then both read what lies
// between; in return segments may be as short as a block of 128 channels.
struct NormResident {
  int seg_c, rows;  // channels of a segment, pixels a CTA takes per step
  int vecs[2];      // vectors of a window, of the last one
  int slots;        // threads of a pixel: a segment's vectors, rounded up to whole blocks of 128 channels with fp8
  int parted;       // segments end inside groups
  int around;       // then, behind all pixels' slots, threads of a pixel for the window's other vectors
  int pixels;       // of a CTA
  int groups;       // room for a window's
  float inv;        // 1 / the values of a group
  FastDiv by_slots, by_around, by_rows, by_cg;
  NormJoin join;
};

template <class T, bool FP8, bool AL>
__global__ void __launch_bounds__(NORM_THREADS, 1) norm_resident(const NormSpec p, const NormResident q) {
  using R = std::conditional_t<FP8, uint8_t, T>;
  constexpr int VE = 16 / (int)sizeof(T);
  extern __shared__ __align__(16) uint8_t smem[];
  const int rank = blockIdx.x, ctas = gridDim.x, seg = blockIdx.y, map = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cg = q.join.cg << q.join.shift;
  const int steps = (int)q.by_rows.div((uint32_t)(q.pixels + q.rows - 1));
  // The window: `vecs` vectors from channel `lo`, `left` of them before the
  // segment's `own_vecs`; channel c0 and group g0 as counted from where groups
  // begin. The outer two groups may be in part.
  const int ch0 = seg * q.seg_c;
  bool last = false;
  int vecs = q.vecs[0], own_vecs = vecs, lo = ch0, left = 0, c0 = 0, g0 = 0, groups = q.groups;
  if (FP8 && q.parted) {
    last = seg == (int)gridDim.y - 1;
    vecs = q.vecs[last];
    own_vecs = min(q.seg_c, p.c - ch0) / VE;
    c0 = lo = min((int)q.by_cg.div((uint32_t)ch0) * cg / VE * VE, p.c - vecs * VE);
    left = (ch0 - lo) / VE;
    g0 = (int)q.by_cg.div((uint32_t)lo);
    groups = (int)q.by_cg.div((uint32_t)(lo + vecs * VE - 1)) - g0 + 1;
  }
  // [pixel][vector], the threads' statistics, the groups' statistics over this
  // CTA and their mean and rstd over the cluster.
  const int stride = q.rows * vecs;  // vectors of a step
  float* tmean = reinterpret_cast<float*>(smem + (size_t)steps * q.rows * q.vecs[0] * 16);
  float* tdev = tmean + NORM_THREADS * VE;
  float* entries = tdev + NORM_THREADS * VE;
  float2* own = reinterpret_cast<float2*>(entries + 3 * norm_entries(q.join.runs[0]));
  float2* stat = own + (q.groups + 1) / 2 * 2;
  int r = (int)q.by_slots.div(threadIdx.x), vec = (int)threadIdx.x - r * q.slots;
  const bool mine = r < q.rows && vec < own_vecs;  // a vector of the segment
  bool live = mine;
  if (FP8 && q.parted && r >= q.rows) {
    const int u = (int)threadIdx.x - q.rows * q.slots;
    r = (int)q.by_around.div((uint32_t)u);
    vec = u - r * q.around;
    live = r < q.rows && vec < vecs - own_vecs;
    if (vec >= left) vec += own_vecs;
  } else if (FP8) {
    vec += left;
  }
  uint4* data = reinterpret_cast<uint4*>(smem) + r * vecs + vec;
  const int first = rank * q.pixels, px = max(0, (int)min((long long)q.pixels, p.pixels - first));
  const int ch = lo + vec * VE;
  const int n = live && r < px ? (int)q.by_rows.div((uint32_t)(px - r + q.rows - 1)) : 0;  // this thread's vectors
  griddep_launch_dependents();
  griddep_wait();

  // The copies, in four groups; the first groups are added up while the
  // others are on their way.
  const T* x = static_cast<const T*>(p.x) + map * p.x_map_stride + (first + r) * p.x_stride + ch;
  const long long step = q.rows * p.x_stride;
  const int batch = (steps + 15) / 16 * 4;  // whole fours
  int s = 0;
#pragma unroll 1
  for (int b = 0; b < 4; b++) {
    for (const int end = min(n, (b + 1) * batch); s < end; s++)
      if constexpr (AL)
        cp_async_16(data + s * stride, x + s * step);
      else
        data[s * stride] = Vec<T, VE, AL>::fetch(x + s * step);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  Affine<VE> affine;
  affine.fetch(p, ch, mine);
  using V = Vec<T, VE, AL>;
  Running<VE> run;
  auto add_until = [&](int end) {
    int i = run.n;
    for (; i + 4 <= end; i += 4) {
      uint4 raw[4];
#pragma unroll
      for (int u = 0; u < 4; u++) raw[u] = data[(i + u) * stride];
      run.template add<V, 4>(raw);
    }
    if (end == n && i < end) {
      const uint4 two[2] = {data[i * stride], data[min(i + 1, end - 1) * stride]};
      if (i + 2 <= end) {
        run.template add<V, 2>(two);
        i += 2;
      }
      if (i < end) run.template add<V, 1>(data + i * stride);
    }
  };
  cp_async_wait<3>();
  add_until(min(n, batch));
  cp_async_wait<2>();
  add_until(min(n, 2 * batch));
  cp_async_wait<1>();
  add_until(min(n, 3 * batch));
  cp_async_wait<0>();
  add_until(n);
  if (live) {
    const int at = r * q.join.runs[last] + (vec * VE >> q.join.shift);
    store_runs<VE>(run, q.join.shift, tmean + at, tdev + at);
  }
  if (px > 0)
    join_threads(q.join, last, tmean, tdev, entries, px, c0 >> q.join.shift,
                 [&](int g, float m, float d) { own[g - g0] = make_float2(m, d); });
  cluster_sync();
#pragma unroll 1
  for (int g = warp; g < groups; g += NORM_THREADS / 32) {
    float2 v = make_float2(0.0f, 0.0f);
    float k = 0.0f;
    const int theirs = min(q.pixels, (int)p.pixels - lane * q.pixels);
    if (lane < ctas && theirs > 0) {
      k = (float)theirs * (float)cg;
      v = ld_cluster_f32x2(own + g, (uint32_t)lane);
    }
    const float m0 = __shfl_sync(~0u, v.x, 0);  // the first CTA always has pixels
    const float m = m0 + warp_sum(k * (v.x - m0)) * q.inv, d = v.x - m;
    const float dev = warp_sum(fmaf(k * d, d, v.y));
    if (lane == 0) stat[g] = make_float2(m, norm_rstd(dev * q.inv + p.eps));
  }
  __syncthreads();
  affine.set(stat, mine ? c0 + vec * VE : c0, g0, cg, q.by_cg);
  op_act_switch(p.act, [&](auto act_c) {
    constexpr int ACT = decltype(act_c)::value;
    // with fp8 the lanes of a block go through the shuffles together
    const int end = !FP8 ? n : warp * 32 < q.rows * q.slots ? steps : 0;
    const long long row0 = map * p.pixels + first + r, code_step = q.rows * (long long)p.q.code_stride;
    uint8_t* codes = FP8 ? p.q.codes + row0 * (long long)p.q.code_stride + ch : nullptr;
    float* scale_at = FP8 && mine && ch % FP8_BLOCK == 0
                          ? p.q.scales + (long long)(ch / FP8_BLOCK) * (long long)p.q.scale_stride + row0
                          : nullptr;
    T* out = FP8 ? nullptr : static_cast<T*>(p.out) + map * p.out_map_stride + (first + r) * p.out_stride + ch;
    const long long out_step = q.rows * p.out_stride;
#pragma unroll 1
    for (int i = 0; i < end; i++) {
      float v[VE];
      Vec<T, VE, AL>::expand(i < n ? data[i * stride] : make_uint4(0, 0, 0, 0), v);
      affine.apply(v);
      op_act_vec<ACT, R, VE>(v);
      if (FP8) {
        const float sc = store_fp8<VE, AL>(codes + i * code_step, mine && i < n, v);
        if (scale_at && i < n) scale_at[i * q.rows] = sc;
      } else {
        Vec<T, VE, AL>::store(out + i * out_step, v);
      }
    }
  });
  cluster_sync();  // the others have read this CTA's statistics
}

// ------------------------------------------------------------- two kernels
// A tile is a run of up to APPLY_THREADS vectors of channels (tile_c
// channels, the last one shorter), a chunk the pixels of one cluster: `span`
// for each of its `cluster` CTAs. part[map][tile][slot][chunk] is the pair of
// the tile's slot-th group over the chunk. (One pair a CTA, joined by every
// CTA of norm_apply, cost that kernel 11 us of L2 reads at 296 CTAs.)
struct NormChunks {
  int tiles, tile_c, chunks, slots, cluster;
  long long span;  // pixels of a CTA of norm_stats
  int map0;        // the first map of this launch
  float inv;       // 1 / the values of a group
  FastDiv by_cg;   // by the channels of a group
  NormJoin join;
  float2* part;
};

template <class T, int VE, bool AL>
__global__ void __launch_bounds__(NORM_THREADS, 2) norm_stats(const NormSpec p, const NormChunks q) {
  extern __shared__ __align__(16) float tmean[];  // [2][rows][channels of the tile]
  const int tile = blockIdx.y, map = q.map0 + blockIdx.z;
  const int c0 = tile * q.tile_c, c = min(q.tile_c, p.c - c0), vecs = c / VE, cg = p.c / p.groups;
  const int rows = q.join.rows, r = threadIdx.x / vecs, slot = threadIdx.x - r * vecs;
  const long long first = blockIdx.x * q.span;
  const int px = (int)max(0ll, min(q.span, p.pixels - first));
  griddep_launch_dependents();
  griddep_wait();
  using V = Vec<T, VE, AL>;
  Running<VE> run;
  const T* x = static_cast<const T*>(p.x) + map * p.x_map_stride + c0 + slot * VE + (first + r) * p.x_stride;
  const long long step = (long long)rows * p.x_stride;
  const int n = r < rows && r < px ? (px - r + rows - 1) / rows : 0;
  int i = 0;
  if constexpr (VE > 1 && AL) {
    // Through a ring of shared memory, NORM_RING fours of pixels deep, so
    // that copies are on their way all the time.
    uint4* ring = reinterpret_cast<uint4*>(tmean) + threadIdx.x;
    const int fours = n / 4;
    auto copy = [&](int f) {
      if (f < fours) {
        const T* at = x + 4 * f * step;
        uint4* to = ring + f % NORM_RING * 4 * NORM_THREADS;
#pragma unroll
        for (int u = 0; u < 4; u++) cp_async_16(to + u * NORM_THREADS, at + u * step);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int f = 0; f < NORM_RING - 1; f++) copy(f);
    for (int f = 0; f < fours; f++) {
      copy(f + NORM_RING - 1);
      cp_async_wait<NORM_RING - 1>();
      uint4 raw[4];
#pragma unroll
      for (int u = 0; u < 4; u++) raw[u] = ring[(f % NORM_RING * 4 + u) * NORM_THREADS];
      run.template add<V, 4>(raw);
    }
    i = 4 * fours;
    cp_async_wait<0>();
    __syncthreads();  // the ring becomes the threads' statistics
  } else {
    constexpr int U = VE == 1 ? 8 : 4;
    for (; i + U <= n; i += U) {
      typename V::Raw raw[U];
#pragma unroll
      for (int u = 0; u < U; u++) raw[u] = V::fetch(x + (i + u) * step);
      run.template add<V, U>(raw);
    }
  }
  for (; i < n; i++) {
    const typename V::Raw raw = V::fetch(x + i * step);
    run.template add<V, 1>(&raw);
  }
  float* tdev = tmean + NORM_THREADS * VE;
  const bool short_tile = c < q.tile_c;
  const int runs = q.join.runs[short_tile];
  if (r < rows) {
    const int at = r * runs + (slot * VE >> q.join.shift);
    store_runs<VE>(run, q.join.shift, tmean + at, tdev + at);
  }
  float* entries = tdev + NORM_THREADS * VE;
  float2* pairs = reinterpret_cast<float2*>(entries + 3 * norm_entries(runs));
  const int g0 = c0 / cg, g1 = (c0 + c - 1) / cg;
  if (px > 0)
    join_threads(q.join, short_tile, tmean, tdev, entries, px, c0 >> q.join.shift,
                 [&](int g, float m, float d) { pairs[g - g0] = make_float2(m, d); });
  cluster_sync();
  const int rank = blockIdx.x % q.cluster, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long base = first - rank * q.span;  // the cluster's first pixel
#pragma unroll 1
  for (int g = g0 + rank * (NORM_THREADS / 32) + warp; g <= g1; g += q.cluster * (NORM_THREADS / 32)) {
    const int width = min((g + 1) * cg, c0 + c) - max(g * cg, c0);
    const float k = (float)max(0ll, min(q.span, p.pixels - base - lane * q.span)) * (float)width;
    const bool some = lane < q.cluster && k > 0.0f;
    const float2 v = some ? ld_cluster_f32x2(pairs + g - g0, (uint32_t)lane) : make_float2(0.0f, 0.0f);
    const float n = warp_sum(some ? k : 0.0f), m0 = __shfl_sync(~0u, v.x, 0);
    const float m = m0 + warp_sum(some ? k * (v.x - m0) : 0.0f) / fmaxf(n, 1.0f), d = v.x - m;
    const float dev = warp_sum(some ? fmaf(k * d, d, v.y) : 0.0f);
    if (lane == 0)
      q.part[((blockIdx.z * (long long)q.tiles + tile) * q.slots + g - g0) * q.chunks + blockIdx.x / q.cluster] =
          make_float2(m, dev);
  }
  cluster_sync();  // the others have read this CTA's pairs
}

// Mean and rstd of group `g` of map `z` (of this launch) from the chunks'
// pairs, by one warp; every lane gets them.
__device__ __forceinline__ float2 norm_join(const NormSpec& p, const NormChunks& q, int z, int g) {
  const int cg = p.c / p.groups, lane = threadIdx.x & 31;
  const int t0 = g * cg / q.tile_c, t1 = (g * cg + cg - 1) / q.tile_c, span = t1 - t0 + 1;
  const long long chunk = q.span * q.cluster;
  auto pair = [&](int i, float* n) {
    const int s = span == 1 ? 0 : i / q.chunks, tile = t0 + s, k = i - s * q.chunks, c0 = tile * q.tile_c;
    const int w = min((g + 1) * cg, c0 + q.tile_c) - max(g * cg, c0);
    *n = (float)max(0ll, min(chunk, p.pixels - k * chunk)) * (float)w;
    return q.part[((z * (long long)q.tiles + tile) * q.slots + g - c0 / cg) * q.chunks + k];
  };
  const int all = q.chunks * span;
  float m = 0.0f, d = 0.0f, n;
  const float m0 = pair(0, &n).x;
  for (int i = lane; i < all; i += 32) {
    const float2 v = pair(i, &n);
    m = fmaf(n, v.x - m0, m);
  }
  m = m0 + warp_sum(m) * q.inv;
  for (int i = lane; i < all; i += 32) {
    const float2 v = pair(i, &n);
    d += fmaf(n * (v.x - m), v.x - m, v.y);
  }
  return make_float2(m, norm_rstd(warp_sum(d) * q.inv + p.eps));
}

// The same for the groups g0 .. g1 of a tile into stat[], by a CTA of `warps`
// warps. Where the map is one tile of at most 160 chunks, four groups at a
// time: one group's loads, sums and root are a chain of 1.1 us.
__device__ __forceinline__ void norm_join_all(const NormSpec& p, const NormChunks& q, int z, int g0, int g1, int warps,
                                              float2* stat) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (q.tiles > 1 || q.chunks > 5 * 32) {
    for (int g = g0 + warp; g <= g1; g += warps) {
      const float2 st = norm_join(p, q, z, g);
      if (lane == 0) stat[g - g0] = st;
    }
    return;
  }
  const long long chunk = q.span * q.cluster;
  const float inv = op_rcp((float)p.pixels), cg = (float)(q.join.cg << q.join.shift);
  float n[5];
#pragma unroll
  for (int i = 0; i < 5; i++) n[i] = (float)max(0ll, min(chunk, p.pixels - (i * 32 + lane) * chunk));
  const float2* part = q.part + (long long)z * q.slots * q.chunks + lane;
  for (int g = g0 + warp; g <= g1; g += 4 * warps) {
    float2 v[4][5];
    float m[4], d[4];
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
      for (int i = 0; i < 5; i++) {
        v[k][i] = make_float2(0.0f, 0.0f);
        if (i * 32 + lane < q.chunks && g + k * warps <= g1) v[k][i] = part[(g + k * warps) * q.chunks + i * 32];
      }
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const float m0 = __shfl_sync(~0u, v[k][0].x, 0);
      m[k] = 0.0f;
#pragma unroll
      for (int i = 0; i < 5; i++) m[k] = fmaf(n[i], v[k][i].x - m0, m[k]);
      m[k] = fmaf(warp_sum(m[k]), inv, m0);
      d[k] = 0.0f;
#pragma unroll
      for (int i = 0; i < 5; i++) d[k] += fmaf(n[i] * cg * (v[k][i].x - m[k]), v[k][i].x - m[k], v[k][i].y);
      d[k] = warp_sum(d[k]);
    }
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (lane == k && g + k * warps <= g1)
        stat[g + k * warps - g0] = make_float2(m[k], norm_rstd(d[k] * q.inv + p.eps));
  }
}

template <class T, int VE, bool FP8, bool AL>
__global__ void __launch_bounds__(APPLY_THREADS, 2) norm_apply(const NormSpec p, const NormChunks q) {
  using R = std::conditional_t<FP8, uint8_t, T>;
  using V = Vec<T, VE, AL>;
  extern __shared__ __align__(16) float2 stat[];  // of the tile's groups
  // the pixels backwards, the latest map first
  const int tile = blockIdx.y, z = (int)gridDim.z - 1 - (int)blockIdx.z, map = q.map0 + z;
  const int c0 = tile * q.tile_c, c = min(q.tile_c, p.c - c0), vecs = c / VE, cg = p.c / p.groups;
  const int g0 = c0 / cg, g1 = (c0 + c - 1) / cg;
  constexpr int LANES = FP8 ? FP8_BLOCK / VE : 1;
  const int slots = (vecs + LANES - 1) / LANES * LANES, rows = APPLY_THREADS / slots;
  const int r = threadIdx.x / slots, slot = threadIdx.x - r * slots;
  const bool live = r < rows && slot < vecs;
  const int ch = c0 + (live ? slot * VE : 0);
  griddep_launch_dependents();
  griddep_wait();
  // (gamma and beta too may come from the kernels before)
  Affine<VE> affine;
  affine.fetch(p, ch, live);
  norm_join_all(p, q, z, g0, g1, APPLY_THREADS / 32, stat);
  __syncthreads();
  affine.set(stat, ch, g0, cg, q.by_cg);
  const long long span = (p.pixels + gridDim.x - 1) / gridDim.x;
  const long long first = ((long long)gridDim.x - 1 - blockIdx.x) * span;
  const int px = (int)max(0ll, min(span, p.pixels - first));
  constexpr int U = VE == 1 ? 8 : 4;
  const int per = U * rows, full = px / per;
  // A thread's U pixels lie next to each other. Threads without a pixel of
  // their own go through the motions on row 0's.
  const long long x_step = (long long)per * p.x_stride, out_step = (long long)per * p.out_stride;
  const long long code_step = FP8 ? per * (long long)p.q.code_stride : 0;
  const long long at = first + (long long)full * per + (r < rows ? r : 0) * U, row = map * p.pixels + at;
  const T* x = static_cast<const T*>(p.x) + map * p.x_map_stride + at * p.x_stride + ch;
  T* out = FP8 ? nullptr : static_cast<T*>(p.out) + map * p.out_map_stride + at * p.out_stride + ch;
  uint8_t* codes = FP8 ? p.q.codes + row * (long long)p.q.code_stride + ch : nullptr;
  // lane u of a block stores the u-th pixel's scale
  const int lane = slot % LANES;
  float* scale_at = FP8 ? p.q.scales + (long long)((c0 + slot * VE) / FP8_BLOCK) * (long long)p.q.scale_stride + row + lane
                        : nullptr;
  const bool scales = FP8 && r < rows && lane < U && slot - lane < vecs;
  op_act_switch(p.act, [&](auto act_c) {
    constexpr int ACT = decltype(act_c)::value;
    // U pixels, the first `some` of which exist.
    auto put = [&](const typename V::Raw* raw, int some) {
      float mine = 0.0f;
#pragma unroll
      for (int u = 0; u < U; u++) {
        float v[VE];
        V::expand(raw[u], v);
        affine.apply(v);
        op_act_vec<ACT, R, VE>(v);
        if constexpr (FP8) {
          const float sc = store_fp8<VE, AL>(codes + u * (long long)p.q.code_stride, live && u < some, v);
          mine = lane == u ? sc : mine;
        } else if (live && u < some) {
          V::store(out + u * p.out_stride, v);
        }
      }
      if (scales && lane < some) *scale_at = mine;
    };
    // The last pixels, then whole steps, the next one's loads ahead of this
    // one's work. (Each load has its condition: with one around them all, 2 x
    // 768 x 512 x 128 bf16 with SiLU took 125 us instead of 115.)
    typename V::Raw raw[U], rest[U];
    const int some = px - full * per - r * U;
#pragma unroll
    for (int u = 0; u < U; u++) rest[u] = live && u < some ? V::fetch(x + u * p.x_stride) : V::zero();
    if (full) {
      x -= x_step;
#pragma unroll
      for (int u = 0; u < U; u++) raw[u] = V::fetch(x + u * p.x_stride);
    }
    if (px > full * per) put(rest, some);
    if (!FP8 && !live) return;
    for (int f = full; f > 0; f--) {
      typename V::Raw next[U];
      x -= x_step;
#pragma unroll
      for (int u = 0; u < U; u++) next[u] = f > 1 ? V::fetch(x + u * p.x_stride) : V::zero();
      out -= FP8 ? 0 : out_step;
      codes -= code_step;
      scale_at -= FP8 ? per : 0;
      put(raw, U);
#pragma unroll
      for (int u = 0; u < U; u++) raw[u] = next[u];
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
  norm_join_all(p, q, z, ga, gb, NORM_THREADS / 32, stat);
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
      op_act_vec<ACT, uint8_t, 4>(v);
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
