// Host side of the group normalisation (norm_sm100.cuh): which kernels a
// shape takes, and their launches.
#include <algorithm>
#include <numeric>

#include "norm_sm100.cuh"
#include "ops_launch.h"

namespace iec {

namespace {

constexpr int RESIDENT_BYTES = 184 * 1024;  // of a CTA's values in shared memory
constexpr int CLUSTER = 16, STATS_CLUSTER = 2;

// The joining of a tile of `c` channels (and of the last one, of `c_last`)
// over `rows` rows of threads.
template <int VE>
NormJoin join_shape(int cg, int c, int c_last, int rows) {
  NormJoin j;
  j.rows = rows;
  j.shift = norm_shift<VE>(cg);
  j.cg = cg >> j.shift;
  j.by_rows = FastDiv((uint32_t)rows);
  j.by_cg = FastDiv((uint32_t)j.cg);
  const int tile[2] = {c, c_last};
  for (int i = 0; i < 2; i++) {
    j.runs[i] = tile[i] >> j.shift;
    j.by_runs[i] = FastDiv((uint32_t)j.runs[i]);
  }
  return j;
}

// The vectors that cover the whole groups of the segments of `seg` channels,
// the most of any and those of the last one.
template <int VE>
void window_vecs(int c, int cg, int seg, int* vecs) {
  const int segs = (c + seg - 1) / seg;
  // where segments begin in a group repeats
  const int every = std::min(segs - 1, cg / std::gcd(cg, seg));
  auto width = [&](int s) {
    const int lo = s * seg / cg * cg / VE, hi = std::min(c, ((std::min(c, (s + 1) * seg) + cg - 1) / cg * cg + VE - 1) / VE * VE);
    return hi / VE - lo;
  };
  vecs[1] = vecs[0] = width(segs - 1);
  for (int s = 0; s < every; s++) vecs[0] = std::max(vecs[0], width(s));
}

// The resident kernel's shape with segments of `seg` channels, of whole
// groups or not (`around`: they may end inside one, the last one may be short), and its cost, vectors that a CTA reads and
// writes; or a cost of zero where it does not fit.
struct ResidentPlan {
  NormResident q;
  int cluster;
  size_t smem;
  long long cost;
};

template <class T>
ResidentPlan plan_segment(Device& dev, const NormSpec& p, bool fp8, int seg, bool around) {
  constexpr int VE = 16 / (int)sizeof(T);
  const int cg = p.c / p.groups, lanes = fp8 ? FP8_BLOCK / VE : 1, segs = (p.c + seg - 1) / seg;
  ResidentPlan f = {};
  NormResident& q = f.q;
  q.seg_c = seg;
  q.vecs[0] = q.vecs[1] = seg / VE;
  q.slots = (seg / VE + lanes - 1) / lanes * lanes;
  if (around) {
    q.parted = 1;
    window_vecs<VE>(p.c, cg, seg, q.vecs);
    q.around = std::max(q.vecs[0] - seg / VE, q.vecs[1] - (p.c - (segs - 1) * seg) / VE);
  }
  if (q.slots + q.around > NORM_THREADS || p.pixels > (1 << 23)) return f;
  q.rows = NORM_THREADS / (q.slots + q.around);
  const int most_steps = RESIDENT_BYTES / (q.rows * q.vecs[0] * 16);
  const long long need = (p.pixels + (long long)most_steps * q.rows - 1) / ((long long)most_steps * q.rows);
  if (need > CLUSTER || segs > 65535) return f;
  q.groups = around ? (q.vecs[0] * VE + cg - 1) / cg + 1 : seg / cg;
  q.by_slots = FastDiv((uint32_t)q.slots);
  q.by_around = FastDiv((uint32_t)std::max(1, q.around));
  q.by_rows = FastDiv((uint32_t)q.rows);
  q.by_cg = FastDiv((uint32_t)cg);
  q.inv = (float)(1.0 / ((double)p.pixels * cg));
  q.join = join_shape<VE>(cg, q.vecs[0] * VE, q.vecs[1] * VE, q.rows);
  // As many CTAs as fill the GPU, but at least two steps each; a cluster size
  // that the GPU's parts divide badly is made smaller. Only where all clusters
  // run at once: one after another, their loads, statistics and stores take
  // turns (8 x 128 x 128 x 256 f16: 90 us in four waves of clusters of 16, 47
  // in chunks through L2).
  const long long spread = dev.sms() / std::max<long long>(1, (long long)segs * p.n);
  const long long fill = (p.pixels + 2LL * q.rows - 1) / (2LL * q.rows);
  constexpr auto codes = norm_resident<T, true, true>;
  constexpr auto wide = norm_resident<T, false, true>;
  for (long long n = std::max<long long>({1, need, std::min({spread, fill, (long long)CLUSTER})}); n >= std::max(1LL, need); n--) {
    q.pixels = (int)((p.pixels + n - 1) / n);
    const int steps = (q.pixels + q.rows - 1) / q.rows;
    f.smem = (size_t)steps * q.rows * q.vecs[0] * 16 + (size_t)NORM_THREADS * VE * 8 +
             (size_t)norm_entries(q.join.runs[0]) * 12 + (size_t)(q.groups + 1) * 16;
    if (f.smem > 224 * 1024) break;
    const int room = fp8 ? resident_ctas<codes>(dev, NORM_THREADS, f.smem, (int)n)
                         : resident_ctas<wide>(dev, NORM_THREADS, f.smem, (int)n);
    if (n * segs * p.n <= room) {
      f.cluster = (int)n;
      f.cost = (long long)q.pixels * (q.vecs[0] + seg / VE);
      break;
    }
  }
  return f;
}

// The resident kernel's shape: segments of whole groups and vectors (and with
// fp8 whole blocks), the smallest that have 128 bytes, so that they read
// whole lines and there are many clusters; else the largest below that. With
// fp8, where groups and blocks share no small multiple, segments of one or two
// blocks and what is around them, if each CTA has less to do then (1 x 64 x
// 64 x 320 f16: 11.6 us in three clusters of 16, 22.8 in one). CTAs that have
// too much to do of a small map lose against the chunks on all SMs: a resident
// CTA takes 5 us and 0.8 ns a vector, chunks 12 us and 1.06 per million values
// (1 x 96 x 96 x 384: 18.2 in three clusters, 15.8 in chunks).
template <class T>
ResidentPlan plan_resident(Device& dev, const NormSpec& p, bool fp8) {
  constexpr int VE = 16 / (int)sizeof(T);
  long long unit = std::lcm<long long>(p.c / p.groups, VE);
  if (fp8) unit = std::lcm<long long>(unit, FP8_BLOCK);
  ResidentPlan best = {};
  if (unit >= p.c || p.c % unit) {
    best = plan_segment<T>(dev, p, fp8, p.c, false);
  } else {
    const long long line = 128 / sizeof(T);
    for (long long seg = (line + unit - 1) / unit * unit; seg <= p.c && !best.cost; seg += unit)
      if (p.c % seg == 0) {
        best = plan_segment<T>(dev, p, fp8, (int)seg, false);
        break;
      }
    for (long long seg = (line - 1) / unit * unit; seg >= unit && !best.cost; seg -= unit)
      if (p.c % seg == 0) {
        best = plan_segment<T>(dev, p, fp8, (int)seg, false);
        break;
      }
  }
  if (fp8)
    for (int seg = FP8_BLOCK; seg <= 2 * FP8_BLOCK && seg < p.c && (unit > seg || p.c % unit); seg += FP8_BLOCK) {
      const ResidentPlan f = plan_segment<T>(dev, p, fp8, seg, true);
      if (f.cost && (!best.cost || f.cost < best.cost)) best = f;
    }
  if (fp8 && best.cost > 9000 + p.n * p.pixels * p.c / 768) best.cost = 0;
  return best;
}

template <class T, int VE, bool AL>
void run_chunks(Device& dev, const NormSpec& p, cudaStream_t s) {
  const int cg = p.c / p.groups;
  NormChunks q = {};
  q.tile_c = std::min(p.c, APPLY_THREADS * VE);
  q.tiles = (p.c + q.tile_c - 1) / q.tile_c;
  q.slots = std::min(p.groups, (q.tile_c + cg - 2) / cg + 1);
  if (q.tiles > 65535) throw Error(ERR_INPUT, "too many channels");
  const size_t ring = VE > 1 && AL ? (size_t)NORM_RING * 4 * NORM_THREADS * 16 : 0;
  const int c_last = p.c - (q.tiles - 1) * q.tile_c;
  q.join = join_shape<VE>(cg, q.tile_c, c_last, NORM_THREADS / (q.tile_c / VE));
  q.by_cg = FastDiv((uint32_t)cg);
  q.inv = (float)(1.0 / ((double)p.pixels * cg));
  // the ring, or the threads' statistics, their entries and pairs
  const size_t stats_smem = std::max(
      ring, (size_t)NORM_THREADS * VE * 8 + (size_t)norm_entries(q.join.runs[0]) * 12 + (size_t)(q.slots + 1) * 8);
  constexpr auto stats = norm_stats<T, VE, AL>;
  allow_smem<stats>(dev, stats_smem);
  const long long resident = resident_ctas<stats>(dev, NORM_THREADS, stats_smem, STATS_CLUSTER);
  // CTAs of the statistics: as many as are resident, of at least eight steps
  // each, in clusters that join their pairs. Maps at a time: as many as their pairs
  // take 64 MB for.
  const int rows = std::max(1, NORM_THREADS / (q.tile_c / VE));
  auto ctas_of = [&](long long maps) {
    const long long most = (p.pixels + 8LL * rows - 1) / (8LL * rows), room = std::max<long long>(resident / (maps * q.tiles), (p.pixels >> 23) + 1);
    if (most < STATS_CLUSTER || room < STATS_CLUSTER) return std::max<long long>(1, std::min(most, room));
    return std::min((most + STATS_CLUSTER - 1) / STATS_CLUSTER, room / STATS_CLUSTER) * STATS_CLUSTER;
  };
  long long maps = p.n;
  auto chunks_of = [&](long long n) { return (ctas_of(n) + STATS_CLUSTER - 1) / STATS_CLUSTER; };
  while (maps > 1 && maps * chunks_of(maps) * q.tiles * q.slots > (8 << 20)) maps = (maps + 1) / 2;
  const long long ctas = ctas_of(maps);
  q.cluster = (int)std::min<long long>(ctas, STATS_CLUSTER);
  q.chunks = (int)((ctas + q.cluster - 1) / q.cluster);
  q.span = (p.pixels + q.chunks * q.cluster - 1) / (q.chunks * q.cluster);
  q.part = static_cast<float2*>(dev.lasting_scratch((size_t)maps * q.chunks * q.tiles * q.slots * sizeof(float2), s));
  const double values = (double)p.pixels * p.c;
  for (q.map0 = 0; q.map0 < p.n; q.map0 += (int)maps) {
    const int now = (int)std::min<long long>(maps, p.n - q.map0);
    timed_launch("norm_stats", 4 * values * now, values * now * sizeof(T), s, [&] {
      launch_ops(stats, dim3(q.chunks * q.cluster, q.tiles, now), NORM_THREADS, stats_smem, q.cluster, s, p, q);
    });
    timed_launch("norm_apply", 10 * values * now, values * now * (sizeof(T) + (p.out ? sizeof(T) : 1)), s, [&] {
      // two CTAs an SM, of at least eight steps
      const int step = std::max(1, APPLY_THREADS / (std::min(q.tile_c, p.c) / VE));
      const long long per = std::max<long long>(1, 2LL * dev.sms() / ((long long)now * q.tiles));
      const dim3 grid((unsigned)std::min(per, (p.pixels + 8LL * step - 1) / (8LL * step)), q.tiles, now);
      const size_t smem = (size_t)q.slots * sizeof(float2);
      if (p.out) {
        constexpr auto kernel = norm_apply<T, VE, false, AL>;
        allow_smem<kernel>(dev, smem);
        launch_ops(kernel, grid, APPLY_THREADS, smem, 1, s, p, q);
      } else if constexpr (VE > 1) {
        constexpr auto kernel = norm_apply<T, VE, true, AL>;
        allow_smem<kernel>(dev, smem);
        launch_ops(kernel, grid, APPLY_THREADS, smem, 1, s, p, q);
      } else {
        constexpr auto kernel = norm_apply_fp8_odd<T>;
        const int blocks = (p.c + FP8_BLOCK - 1) / FP8_BLOCK;
        const long long want = std::max<long long>(1, 4LL * dev.sms() / ((long long)now * blocks));
        const long long px = (p.pixels + NORM_THREADS / 32 - 1) / (NORM_THREADS / 32);
        launch_ops(kernel, dim3((unsigned)std::min(want, px), blocks, now), NORM_THREADS, FP8_BLOCK * sizeof(float2), 1, s, p, q);
      }
    });
  }
}

template <class T, bool AL>
void run_vectors(Device& dev, const NormSpec& p, cudaStream_t s) {
  constexpr int VE = 16 / (int)sizeof(T);
  const bool fp8 = p.out == nullptr;
  constexpr auto wide = norm_resident<T, false, AL>;
  constexpr auto codes = norm_resident<T, true, AL>;
  const ResidentPlan f = plan_resident<T>(dev, p, fp8);
  if (!f.cost) return run_chunks<T, VE, AL>(dev, p, s);
  const double values = (double)p.n * p.pixels * p.c;
  timed_launch("norm_resident", 12 * values, values * (sizeof(T) + (fp8 ? 1 : sizeof(T))), s, [&] {
    const dim3 grid(f.cluster, (p.c + f.q.seg_c - 1) / f.q.seg_c, p.n);
    if (fp8) {
      allow_smem<codes>(dev, f.smem);
      launch_ops(codes, grid, NORM_THREADS, f.smem, f.cluster, s, p, f.q);
    } else {
      allow_smem<wide>(dev, f.smem);
      launch_ops(wide, grid, NORM_THREADS, f.smem, f.cluster, s, p, f.q);
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
