// Host side of the group normalisation (norm_sm100.cuh): which kernels a
// shape takes, and their launches.
#include <algorithm>
#include <numeric>

#include "norm_sm100.cuh"

namespace iec {

namespace {

constexpr int RESIDENT_BYTES = 180 * 1024;  // of a CTA's values in shared memory
constexpr int CLUSTER = 16;

template <auto Kernel>
void allow_smem(Device& dev, int bytes) {
  static int most[64] = {};
  int& m = most[dev.ordinal() & 63];
  if (m == 0) IEC_CUDA(cudaFuncSetAttribute(Kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  if (bytes > m) IEC_CUDA(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  m = std::max(m, bytes);
}

template <class... KArgs, class... Args>
void launch(void (*kernel)(KArgs...), dim3 grid, size_t smem, int cluster, cudaStream_t s, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(NORM_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {(unsigned)cluster, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  IEC_CUDA(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...));
}

// The resident kernel's shape, or false where a segment outgrows a cluster.
// A segment is the smallest run of whole groups, vectors (and with fp8 whole
// blocks) that has at least 128 bytes, so that segments read whole lines and
// there are as many clusters as possible.
template <class T>
bool plan_resident(Device& dev, const NormSpec& p, bool fp8, NormResident* q, int* cluster, size_t* smem) {
  constexpr int VE = 16 / (int)sizeof(T);
  const int cg = p.c / p.groups;
  long long unit = std::lcm<long long>(cg, VE);
  if (fp8) unit = std::lcm<long long>(unit, FP8_BLOCK);
  long long seg = p.c;
  if (unit < p.c && p.c % unit == 0) {
    seg = unit;
    while (seg < p.c && (seg * (long long)sizeof(T) < 128 || p.c % seg)) seg += unit;
  }
  q->seg_c = (int)seg;
  q->vecs = (int)seg / VE;
  const int lanes = fp8 ? FP8_BLOCK / VE : 1;
  q->slots = (q->vecs + lanes - 1) / lanes * lanes;
  if (q->slots > NORM_THREADS || p.pixels > (1 << 24)) return false;
  q->rows = NORM_THREADS / q->slots;
  const int segs = p.c / q->seg_c, most_steps = RESIDENT_BYTES / (NORM_THREADS * 16);
  const long long need = (p.pixels + (long long)most_steps * q->rows - 1) / ((long long)most_steps * q->rows);
  if (need > CLUSTER || segs > 65535) return false;
  // as many CTAs as fill the GPU, but at least two steps each
  const long long spread = dev.sms() / std::max<long long>(1, (long long)segs * p.n);
  const long long fill = (p.pixels + 2LL * q->rows - 1) / (2LL * q->rows);
  int n = (int)std::max(need, std::min({spread, fill, (long long)CLUSTER}));
  n = std::max(n, 1);
  q->pixels = (int)((p.pixels + n - 1) / n);
  *cluster = n;
  const int steps = (q->pixels + q->rows - 1) / q->rows;
  *smem = (size_t)steps * NORM_THREADS * 16 + (size_t)NORM_THREADS * VE * 8 + (size_t)(q->seg_c / cg) * 16;
  return *smem <= 220 * 1024;
}

template <class T, int VE, bool AL>
void run_chunks(Device& dev, const NormSpec& p, cudaStream_t s) {
  const int cg = p.c / p.groups;
  NormChunks q = {};
  q.tile_c = std::min(p.c, NORM_THREADS * VE);
  q.tiles = (p.c + q.tile_c - 1) / q.tile_c;
  q.slots = std::min(p.groups, (q.tile_c + cg - 2) / cg + 1);
  if (q.tiles > 65535) throw Error(ERR_INPUT, "too many channels");
  // Maps at a time: as many as their pairs take a few MB for.
  const int rows = std::max(1, NORM_THREADS / (std::min(q.tile_c, p.c) / VE));
  const long long ctas = 2LL * dev.sms();  // two an SM
  auto chunks_of = [&](long long maps) {
    const long long want = std::max<long long>(1, ctas / (maps * q.tiles));
    return std::max<long long>(1, std::min(want, (p.pixels + 8LL * rows - 1) / (8LL * rows)));
  };
  long long maps = p.n;
  while (maps > 1 && maps * chunks_of(maps) * q.tiles * q.slots > (8 << 20)) maps = (maps + 1) / 2;
  q.chunk = (p.pixels + chunks_of(maps) - 1) / chunks_of(maps);
  q.chunks = (int)((p.pixels + q.chunk - 1) / q.chunk);
  q.part = static_cast<float2*>(dev.scratch((size_t)maps * q.chunks * q.tiles * q.slots * sizeof(float2), s));
  const size_t stats_smem = (size_t)NORM_THREADS * VE * 8;
  const double values = (double)p.pixels * p.c;
  for (q.map0 = 0; q.map0 < p.n; q.map0 += (int)maps) {
    const int now = (int)std::min<long long>(maps, p.n - q.map0);
    timed_launch("norm_stats", 4 * values * now, values * now * sizeof(T), s, [&] {
      constexpr auto kernel = norm_stats<T, VE, AL>;
      launch(kernel, dim3(q.chunks, q.tiles, now), stats_smem, 1, s, p, q);
    });
    timed_launch("norm_apply", 10 * values * now, values * now * (sizeof(T) + (p.out ? sizeof(T) : 1)), s, [&] {
      const dim3 grid(q.chunks, q.tiles, now);
      const size_t smem = (size_t)q.slots * sizeof(float2);
      if (p.out) {
        constexpr auto kernel = norm_apply<T, VE, false, AL>;
        allow_smem<kernel>(dev, (int)smem);
        launch(kernel, grid, smem, 1, s, p, q);
      } else if constexpr (VE > 1) {
        constexpr auto kernel = norm_apply<T, VE, true, AL>;
        allow_smem<kernel>(dev, (int)smem);
        launch(kernel, grid, smem, 1, s, p, q);
      } else {
        constexpr auto kernel = norm_apply_fp8_odd<T>;
        const int blocks = (p.c + FP8_BLOCK - 1) / FP8_BLOCK;
        const long long want = std::max<long long>(1, 2LL * ctas / ((long long)now * blocks));
        const long long px = (p.pixels + NORM_THREADS / 32 - 1) / (NORM_THREADS / 32);
        launch(kernel, dim3((unsigned)std::min(want, px), blocks, now), FP8_BLOCK * sizeof(float2), 1, s, p, q);
      }
    });
  }
}

template <class T, bool AL>
void run_vectors(Device& dev, const NormSpec& p, cudaStream_t s) {
  constexpr int VE = 16 / (int)sizeof(T);
  const bool fp8 = p.out == nullptr;
  NormResident q;
  int cluster = 1;
  size_t smem = 0;
  if (!plan_resident<T>(dev, p, fp8, &q, &cluster, &smem)) return run_chunks<T, VE, AL>(dev, p, s);
  const double values = (double)p.n * p.pixels * p.c;
  timed_launch("norm_resident", 12 * values, values * (sizeof(T) + (fp8 ? 1 : sizeof(T))), s, [&] {
    const dim3 grid(cluster, p.c / q.seg_c, p.n);
    if (fp8) {
      constexpr auto kernel = norm_resident<T, true, AL>;
      allow_smem<kernel>(dev, (int)smem);
      launch(kernel, grid, smem, cluster, s, p, q);
    } else {
      constexpr auto kernel = norm_resident<T, false, AL>;
      allow_smem<kernel>(dev, (int)smem);
      launch(kernel, grid, smem, cluster, s, p, q);
    }
  });
}

template <class T>
void run(Device& dev, const NormSpec& p, cudaStream_t s) {
  constexpr int VE = 16 / (int)sizeof(T);
  if (p.c % VE) return run_chunks<T, 1, true>(dev, p, s);
  // 16-byte vectors of x and out, 8 or 4 bytes of codes
  auto even = [](const void* ptr, long long a, long long b, int bytes) {
    return reinterpret_cast<uintptr_t>(ptr) % bytes == 0 && a % VE == 0 && b % VE == 0;
  };
  if (even(p.x, p.x_stride, p.x_map_stride, 16) && (p.out ? even(p.out, p.out_stride, p.out_map_stride, 16)
                                                           : even(p.q.codes, (long long)p.q.code_stride, 0, VE)))
    run_vectors<T, true>(dev, p, s);
  else
    run_vectors<T, false>(dev, p, s);
}

}  // namespace

void group_norm(Device& dev, const NormSpec& p, cudaStream_t s) {
  if (p.n == 0 || p.pixels == 0) return;
  if (p.dtype == DT_F16) return run<__half>(dev, p, s);
  if (p.dtype == DT_BF16) return run<__nv_bfloat16>(dev, p, s);
  run<float>(dev, p, s);
}

}  // namespace iec
