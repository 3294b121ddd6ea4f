// Group norm over channels-last images, and over rows of tokens whose groups do not fit a warp.
//
// Bound by memory: x is read once and y written once, so a group's values have to stay on chip between the statistics and the
// last pass. They stay in shared memory: a cluster of up to eight blocks holds all pixels of a slab of neighbouring groups (rows
// of about 64 bytes). Every thread copies its own rows there asynchronously and nobody else reads them, so that nothing waits
// for anything but sums; as soon as a row has gone through the last pass, the next image's row is on its way into its place.
// The sums are taken in one pass (see local_moments) and joined over the block and, by distributed shared memory, the cluster.
// The gradient holds x and dy the same way, sums g xh and g per channel, and joins those.
//
// (With the rows in registers, sixteen vectors a thread and copies a buffer ahead, the same took 37 us on 32 x 256 x 56 x 56 bf16:
// two blocks an SM, and unrolled code that the instruction cache did not hold.)
//
// 32 x 256 x 56 x 56 bf16 with silu: 36.2 us, 2.8 TB/s.
// Slabs that no cluster holds go in two launches, which read x twice.
#include <cooperative_groups.h>

#include "group_norm.cuh"

namespace fdnn {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxChunks = 64;        // pieces of an image in two launches
constexpr int kMaxGroups = 512;       // of a slab
constexpr int kThreads = 256;
constexpr int kMostShared = 224 * 1024, kSharedOfSm = 228 * 1024;
constexpr int kRowVectors = 4;        // of a slab's row, where groups are narrower and pixels not few
constexpr int kStatic = 24 * 1024;    // shared memory that the forward kernel has beside its rows, at most
constexpr int kMostRows = (kMostShared - kStatic) / (kThreads * 16);   // rows of 16-byte vectors that a thread may then hold: 50

struct Slab {
  NormParams p;
  int S;                 // pixels
  int channels, cols;    // of a slab; vectors of channels in a row of it
  int rows_at_once;      // rows that a block's threads cover
  int rows;              // of a block (cluster) or a piece (two launches)
  int slabs, cluster;
  int held;              // rows of a thread
  int slices;            // clusters that share the images
  int pieces;
  float2* part;          // forward in two launches: [N, pieces, G] mean and squared deviations
  float2* sums;          // backward: rows of [C] sums of g xh and g
};

// A thread's place: a vector of channels and every rows_at_once-th row.  (All that takes a division is taken once.)
struct Place {
  int col, r, cc;        // column, first row, first channel within the slab
  int c0;                // the slab's first channel
  int here;              // channels of this slab (the last may have fewer)
  int groups;            // and groups
  bool live;
  template <int V>
  static __device__ Place of(const Slab& s, int slab) {
    Place at;
    at.r = int(threadIdx.x) / s.cols;
    at.col = int(threadIdx.x) - at.r * s.cols;
    at.cc = at.col * V;
    at.c0 = slab * s.channels;
    at.here = min(s.channels, s.p.C - at.c0);
    at.groups = at.here / (s.p.C / s.p.G);
    at.live = at.r < s.rows_at_once && at.cc < at.here;
    return at;
  }
};

// Rows that each of a block's rows of threads has: `each` of them, the first `more` one more.
struct Rows {
  int all, each, more;
  __device__ Rows(const Slab& s, int rows) : all(rows), each(rows / s.rows_at_once), more(rows - each * s.rows_at_once) {}
  __device__ int of(int r) const { return each + (r < more ? 1 : 0); }
};

// Mean and squared deviations of a block's rows by group: out[g] in shared memory.
// A thread sums its values' distances from its own first one, and their squares, channel by channel, in one pass. Where that first
// value lies D from n - 1 others, the sums grow to n D and n D^2 and are rounded on the way to 2^-24 of what they have come to: the
// thread's squared deviations are off by up to 1.5 n^2 2^-24 D^2, and the group's are D^2 at least. n is a thread's rows, up to 50 of a
// block that holds them as vectors of 16 bytes.  LONG rows, of which a thread may have hundreds (narrow vectors) or thousands (two
// launches), are summed in runs: the first kRun from the first value (off by up to 9.2e-5 of the group's), then as many again as there
// were from the mean so far. Such a run of n that lies D from it brings the group
// n / 2 times D^2, of which 3 n 2^-24 may be lost: as much at kMostRun.  Runs, threads and channels are joined by their means.
// ONE (everywhere): the channels of a vector are all of one group.
constexpr int kRun = 32, kMostRun = 512;
template <typename T, int V, bool ONE, bool LONG, typename F>
__device__ __forceinline__ void local_moments(const Slab& s, const Place& at, F&& row, const Rows& rows, float2* red, float2* out) {
  const int cpg = s.p.C / s.p.G, count = at.live ? rows.of(at.r) : 0, run = LONG ? min(count, kRun) : count;
  constexpr int P = Pack<T, V>::kPairs;
  F2 sum[P], square[P], minus[P];
  Pack<T, V> x0;
  x0.clear();
  if (count > 0) x0 = row(0);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    sum[i] = square[i] = 0;
    minus[i] = f2_mul(x0.pair(i), f2_both(-1.0f));
  }
#pragma unroll 4
  for (int k = 1; k < run; ++k) {
    const Pack<T, V> x = row(k);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const F2 d = f2_add(x.pair(i), minus[i]);
      sum[i] = f2_add(sum[i], d);
      square[i] = f2_fma(d, d, square[i]);
    }
  }
  if (at.r < s.rows_at_once) {
    const float inv = count > 0 ? __fdividef(1.0f, float(run)) : 0.0f;
    float mean[2 * P], m2[2 * P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
      float a[2], q[2], first[2];
      f2_split(sum[i], a[0], a[1]);
      f2_split(square[i], q[0], q[1]);
      f2_split(x0.pair(i), first[0], first[1]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        mean[2 * i + j] = first[j] + a[j] * inv;
        // (a^2 may be no number where a^2 / n is one; rounding may leave less than nothing; NaN stays)
        m2[2 * i + j] = fmaxf(q[j] - a[j] * (a[j] * inv), q[j] * 0.0f);
      }
    }
    if constexpr (LONG) {
      for (int begin = kRun, end; begin < count; begin = end) {
        end = min(count, begin + min(begin, kMostRun));
#pragma unroll
        for (int i = 0; i < P; ++i) {
          sum[i] = square[i] = 0;
          minus[i] = f2_pack(-mean[2 * i], -mean[2 * i + 1]);
        }
#pragma unroll 8
        for (int k = begin; k < end; ++k) {
          const Pack<T, V> x = row(k);
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const F2 d = f2_add(x.pair(i), minus[i]);
            sum[i] = f2_add(sum[i], d);
            square[i] = f2_fma(d, d, square[i]);
          }
        }
        const float each = __fdividef(1.0f, float(end - begin)), share = __fdividef(float(end - begin), float(end));
#pragma unroll
        for (int i = 0; i < P; ++i) {
          float a[2], q[2];
          f2_split(sum[i], a[0], a[1]);
          f2_split(square[i], q[0], q[1]);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float d = a[j] * each;
            m2[2 * i + j] += fmaxf(q[j] - a[j] * d, q[j] * 0.0f) + d * (d * (float(begin) * share));
            mean[2 * i + j] += d * share;
          }
        }
      }
    }
    if constexpr (ONE) {
      float all = 0.0f, dev = 0.0f;
#pragma unroll
      for (int j = 0; j < V; ++j) all += mean[j];
      all *= 1.0f / V;
#pragma unroll
      for (int j = 0; j < V; ++j) dev += m2[j] + float(count) * (mean[j] - all) * (mean[j] - all);
      red[at.r * s.cols + at.col] = make_float2(all, dev);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) red[at.r * s.channels + at.cc + j] = make_float2(mean[j], m2[j]);
    }
  }
  __syncthreads();
  // a warp takes a group: the mean of its threads' means first, then their deviations from it
  const int pitch = ONE ? s.cols : s.channels, per = cpg / (ONE ? V : 1), lane = threadIdx.x & 31;
  const int entries = s.rows_at_once * per;
  const float part = __fdividef(1.0f, float(per)), inv = __fdividef(1.0f, float(rows.all) * float(cpg)), each = ONE ? V : 1;
  for (int g = threadIdx.x >> 5; g < at.groups; g += blockDim.x >> 5) {
    const float2* from = red + g * per;
    const float first = from[0].x;
    float t = 0.0f;
    for (int i = lane; i < entries; i += 32) {
      const int row = per == 1 ? i : int((float(i) + 0.5f) * part);   // i / per: exact for the few thousand entries there are
      t += float(rows.of(row)) * (rows.of(row) > 0 ? from[row * pitch + i - row * per].x - first : 0.0f);
    }
    const float mean = first + warp_sum(t) * each * inv;
    t = 0.0f;
    for (int i = lane; i < entries; i += 32) {
      const int row = per == 1 ? i : int((float(i) + 0.5f) * part);
      const float2 v = from[row * pitch + i - row * per];
      if (rows.of(row) > 0) t += v.y + float(rows.of(row)) * each * (v.x - mean) * (v.x - mean);
    }
    t = warp_sum(t);
    if (lane == 0) out[g] = make_float2(mean, t);
  }
  __syncthreads();
}

// The cluster's barrier, after a __syncthreads(): what the block's threads wrote (or read) before that is ordered by the first
// warp's release; a fence in each of the others would cost as much again and order nothing more.
__device__ __forceinline__ void cluster_arrive() {
  if (threadIdx.x < 32) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  else asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

template <typename T, int V, bool ONE>
__global__ void __launch_bounds__(kThreads, 3)
norm_images_kernel(const Slab s) {
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ float2 red[ONE ? kThreads : kThreads * V];
  __shared__ float2 own[kMaxGroups], all_of[kMaxGroups];   // mean and squared deviations; mean and 1 / deviation
  constexpr int M = ONE ? 1 : Pack<T, V>::kPairs, P = Pack<T, V>::kPairs;
  Pack<T, V>* held = reinterpret_cast<Pack<T, V>*>(raw) + threadIdx.x;   // this thread's rows, kThreads apart
  chained();
  const NormParams& p = s.p;
  const cg::cluster_group cluster = cg::this_cluster();
  const int rank = blockIdx.x % s.cluster, job = blockIdx.x / s.cluster, slab = job % s.slabs, slice = job / s.slabs;
  const int row0 = rank * s.rows, cpg = p.C / p.G;
  const Rows rows(s, max(0, min(s.rows, s.S - row0)));
  const Place at = Place::of<V>(s, slab);
  const int count = at.live ? rows.of(at.r) : 0, c = at.c0 + at.cc, g0 = at.c0 / cpg;
  const long long pixel = p.W > 1 ? p.x_s[3] : p.x_s[2], out_pixel = p.W > 1 ? p.y_s[3] : p.y_s[2];
  const T* x0 = static_cast<const T*>(p.x) + (count > 0 ? c + (long long)(row0 + at.r) * pixel : 0);
  T* y0 = static_cast<T*>(p.y) + (count > 0 ? c + (long long)(row0 + at.r) * out_pixel : 0);
  const long long x_step = s.rows_at_once * pixel, y_step = s.rows_at_once * out_pixel;
  int group[M][2];                                  // of a pair's two channels, within the slab
#pragma unroll
  for (int i = 0; i < M; ++i) {
    group[i][0] = at.live ? (at.cc + (ONE ? 0 : 2 * i)) / cpg : 0;
    group[i][1] = ONE || !at.live ? group[i][0] : (at.cc + min(2 * i + 1, V - 1)) / cpg;
  }
  F2 w[P], b[P];
  norm_params_of<T, V>(p, c, at.live, w, b);
  if (slice < p.N) {
    const T* from = x0 + (count > 0 ? slice * p.x_s[0] : 0);
    for (int k = 0; k < count; ++k) async_load(held + k * kThreads, from + k * x_step, true);
  }
  for (int n = slice; n < p.N; n += s.slices) {
    async_commit();
    async_wait<0>();
    local_moments<T, V, ONE, V <= 2>(s, at, [&](int k) { return held[k * kThreads]; }, rows, red, own);
    if (s.cluster > 1) {
      cluster_arrive();
      cluster_wait();
    }
    for (int g = threadIdx.x; g < at.groups; g += kThreads) {
      float2 all = own[g];
      if (s.cluster > 1) {
        float2 v[8];
        float n_of[8], t = 0.0f;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          n_of[q] = q < s.cluster ? float(max(0, min(s.rows, s.S - q * s.rows))) * float(cpg) : 0.0f;
          v[q] = n_of[q] > 0.0f ? cluster.map_shared_rank(own, q)[g] : make_float2(0.0f, 0.0f);
        }
        const float inv = __fdividef(1.0f, float(s.S) * float(cpg));
#pragma unroll
        for (int q = 1; q < 8; ++q) t += n_of[q] > 0.0f ? n_of[q] * (v[q].x - v[0].x) : 0.0f;
        all = make_float2(v[0].x + t * inv, 0.0f);
#pragma unroll
        for (int q = 0; q < 8; ++q) all.y += n_of[q] > 0.0f ? v[q].y + n_of[q] * (v[q].x - all.x) * (v[q].x - all.x) : 0.0f;
      }
      const float rstd = rsqrtf(all.y / (float(s.S) * float(cpg)) + p.eps);
      all_of[g] = make_float2(all.x, rstd);
      if (p.mean != nullptr && rank == 0) {
        p.mean[(long long)n * p.G + g0 + g] = all.x;
        p.rstd[(long long)n * p.G + g0 + g] = rstd;
      }
    }
    __syncthreads();
    if (s.cluster > 1) cluster_arrive();           // this block has read the others' moments
    F2 m[M], scale[P];                                // m: minus the mean
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float2 lo = all_of[group[ONE ? 0 : i][0]], hi = ONE ? lo : all_of[group[ONE ? 0 : i][1]];
      m[ONE ? 0 : i] = f2_pack(-lo.x, -hi.x);
      scale[i] = f2_mul(w[i], f2_pack(lo.y, hi.y));
    }
    T* to = y0 + (count > 0 ? n * p.y_s[0] : 0);
    const bool more = n + s.slices < p.N;
    const T* from = x0 + (count > 0 && more ? (n + s.slices) * p.x_s[0] : 0);
    with_activation(p.act, [&](auto act) {
#pragma unroll 4
      for (int k = 0; k < count; ++k) {
        const Pack<T, V> x = held[k * kThreads];
        Pack<T, V> y;
#pragma unroll
        for (int i = 0; i < P; ++i)
          y.set_pair(i, activate2<decltype(act)::value>(f2_fma(f2_add(x.pair(i), m[ONE ? 0 : i]), scale[i], b[i])));
        y.store(to + k * y_step);
        if (more) async_load(held + k * kThreads, from + k * x_step, true);
      }
    });
    if (s.cluster > 1) cluster_wait();             // and the others have read this one's
  }
}

// Sums over a block's rows of two values per channel: sums[channel of the slab]. red: twice as many floats as threads times V.
template <int V>
__device__ __forceinline__ void sum_by_channel(const Slab& s, const Place& at, const F2 (&a)[(V + 1) / 2], const F2 (&b)[(V + 1) / 2],
                                               float2* red, float2* sums) {
  if (at.r < s.rows_at_once) {
#pragma unroll
    for (int i = 0; i < (V + 1) / 2; ++i) {
      float x0, x1, y0, y1;
      f2_split(a[i], x0, x1);
      f2_split(b[i], y0, y1);
      red[at.r * s.channels + at.cc + 2 * i] = make_float2(x0, y0);
      if (V > 1) red[at.r * s.channels + at.cc + 2 * i + 1] = make_float2(x1, y1);
    }
  }
  __syncthreads();
  // the rows in as many parts as there are threads for, each thread a channel's; then the parts in their order
  const int parts = s.channels <= kThreads ? min(s.rows_at_once, kThreads / s.channels) : 1;
  const int part = s.channels <= kThreads ? int(threadIdx.x) / s.channels : 0;
  for (int c = int(threadIdx.x) - part * s.channels; c < s.channels && part < parts; c += kThreads) {
    float2 t = make_float2(0.0f, 0.0f);
#pragma unroll 4
    for (int row = part; row < s.rows_at_once; row += parts) {
      const float2 q = red[row * s.channels + c];
      t.x += q.x;
      t.y += q.y;
    }
    red[part * s.channels + c] = t;      // (of the rows that this thread alone has read)
  }
  __syncthreads();
  for (int c = threadIdx.x; c < s.channels; c += kThreads) {
    float2 t = red[c];
#pragma unroll 4
    for (int q = 1; q < parts; ++q) {
      const float2 v = red[q * s.channels + c];
      t.x += v.x;
      t.y += v.y;
    }
    sums[c] = t;
  }
}

// s1 / m and s2 / m of every group of the slab from its channels' sums.
__device__ __forceinline__ void group_means(const Slab& s, const Place& at, const float* weight, const float2* sums, float2* means) {
  const int cpg = s.p.C / s.p.G, lane = threadIdx.x & 31;
  const float inv = __fdividef(1.0f, float(s.S) * float(cpg));
  for (int g = threadIdx.x >> 5; g < at.groups; g += kThreads / 32) {
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = g * cpg + lane; c < (g + 1) * cpg; c += 32) {
      s2 += weight[c] * sums[c].x;
      s1 += weight[c] * sums[c].y;
    }
    s1 = warp_sum(s1);
    s2 = warp_sum(s2);
    if (lane == 0) means[g] = make_float2(s1 * inv, s2 * inv);
  }
}

// Shared memory of the backward kernels: a row of vectors bounds a slab's channels.
struct BackwardShared {
  float2 *red, *own, *all, *acc, *means;
  float* weight;
  __device__ BackwardShared(unsigned char* raw, int entries, int channels)
      : red(reinterpret_cast<float2*>(raw)), own(red + entries), all(own + channels), acc(all + channels), means(acc + channels),
        weight(reinterpret_cast<float*>(means + kMaxGroups)) {}
  static __host__ __device__ int bytes(int entries, int channels) {
    return (8 * (entries + 3 * channels + kMaxGroups) + 4 * channels + 15) / 16 * 16;
  }
};
template <typename T>
__device__ __forceinline__ void stage_weights(const NormParams& p, const Place& at, float* weight) {
  for (int i = threadIdx.x; i < at.here; i += kThreads)
    weight[i] = p.weight != nullptr ? param<T>(p.weight, p.param_f32, at.c0 + i) : 1.0f;
}

template <typename T, int V, bool ONE>
__global__ void __launch_bounds__(kThreads, 2)
norm_images_backward_kernel(const Slab s) {
  extern __shared__ __align__(16) unsigned char raw[];
  const BackwardShared sh(raw, kThreads * V, s.channels);
  constexpr int M = ONE ? 1 : Pack<T, V>::kPairs;
  chained();
  const NormParams& p = s.p;
  const cg::cluster_group cluster = cg::this_cluster();
  const int rank = blockIdx.x % s.cluster, job = blockIdx.x / s.cluster, slab = job % s.slabs, slice = job / s.slabs;
  const int row0 = rank * s.rows, cpg = p.C / p.G;
  const Rows rows(s, max(0, min(s.rows, s.S - row0)));
  const Place at = Place::of<V>(s, slab);
  const bool tall = p.W > 1;
  const long long px = tall ? p.x_s[3] : p.x_s[2], pdy = tall ? p.dy_s[3] : p.dy_s[2], pdx = tall ? p.dx_s[3] : p.dx_s[2];
  const int c = at.c0 + at.cc, first = row0 + at.r, g0 = at.c0 / cpg;
  constexpr int P = Pack<T, V>::kPairs;
  F2 w[P], b[P];
  norm_params_of<T, V>(p, c, at.live, w, b);
  int group[M][2];                                  // of a pair's two channels, within the slab
#pragma unroll
  for (int i = 0; i < M; ++i) {
    group[i][0] = at.live ? (at.cc + (ONE ? 0 : 2 * i)) / cpg : 0;
    group[i][1] = ONE || !at.live ? group[i][0] : (at.cc + min(2 * i + 1, V - 1)) / cpg;
  }
  for (int i = threadIdx.x; i < s.channels; i += kThreads) sh.acc[i] = make_float2(0.0f, 0.0f);
  stage_weights<T>(p, at, sh.weight);
  // this thread's rows, kThreads apart: x, then dy
  Pack<T, V>* held = reinterpret_cast<Pack<T, V>*>(raw + BackwardShared::bytes(kThreads * V, s.channels)) + threadIdx.x;
  Pack<T, V>* held_dy = held + s.held * kThreads;
  const int count = at.live ? rows.of(at.r) : 0;
  const long long x_step = s.rows_at_once * px, dy_step = s.rows_at_once * pdy, dx_step = s.rows_at_once * pdx;
  const T* x0 = static_cast<const T*>(p.x) + (count > 0 ? c + first * px : 0);
  const T* dy0 = static_cast<const T*>(p.dy) + (count > 0 ? c + first * pdy : 0);
  T* dx0 = static_cast<T*>(p.dx) + (count > 0 ? c + first * pdx : 0);
  for (int k = 0; k < count; ++k) {
    async_load(held + k * kThreads, x0 + slice * p.x_s[0] + k * x_step, true);
    async_load(held_dy + k * kThreads, dy0 + slice * p.dy_s[0] + k * dy_step, true);
  }
  for (int n = slice; n < p.N; n += s.slices) {
    async_commit();
    async_wait<0>();
    F2 mean[M], rstd[M], gx[P], gs[P];               // mean: minus the mean
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const long long lo = (long long)n * p.G + g0 + group[i][0], hi = (long long)n * p.G + g0 + group[i][1];
      mean[i] = f2_pack(-p.mean[lo], -p.mean[hi]);
      rstd[i] = f2_pack(p.rstd[lo], p.rstd[hi]);
    }
#pragma unroll
    for (int i = 0; i < P; ++i) gx[i] = gs[i] = 0;
    with_activation(p.act, [&](auto act) {
#pragma unroll 2
      for (int k = 0; k < count; ++k) {
        const Pack<T, V> x = held[k * kThreads], dy = held_dy[k * kThreads];
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const F2 xh = f2_mul(f2_add(x.pair(i), mean[ONE ? 0 : i]), rstd[ONE ? 0 : i]);
          const F2 g = f2_mul(dy.pair(i), slope2<decltype(act)::value>(f2_fma(xh, w[i], b[i])));
          gx[i] = f2_fma(g, xh, gx[i]);
          gs[i] = f2_add(gs[i], g);
        }
      }
    });
    sum_by_channel<V>(s, at, gx, gs, sh.red, sh.own);
    __syncthreads();
    if (s.cluster > 1) {
      cluster_arrive();
      cluster_wait();
    }
    for (int i = threadIdx.x; i < s.channels; i += kThreads) {
      float2 t = sh.own[i];
      if (s.cluster > 1) {
        float2 v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = q < s.cluster ? cluster.map_shared_rank(sh.own, q)[i] : make_float2(0.0f, 0.0f);
        t = v[0];
#pragma unroll
        for (int q = 1; q < 8; ++q) {
          t.x += v[q].x;
          t.y += v[q].y;
        }
      }
      sh.all[i] = t;
      sh.acc[i].x += t.x;
      sh.acc[i].y += t.y;
    }
    __syncthreads();
    if (s.cluster > 1) cluster_arrive();
    group_means(s, at, sh.weight, sh.all, sh.means);
    __syncthreads();
    F2 s1[M], s2[M];                                 // minus s1 / m, minus s2 / m
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const float2 lo = sh.means[group[i][0]], hi = sh.means[group[i][1]];
      s1[i] = f2_pack(-lo.x, -hi.x);
      s2[i] = f2_pack(-lo.y, -hi.y);
    }
    const bool more = n + s.slices < p.N;
    const T* next_x = x0 + (more ? (n + s.slices) * p.x_s[0] : 0);
    const T* next_dy = dy0 + (more ? (n + s.slices) * p.dy_s[0] : 0);
    with_activation(p.act, [&](auto act) {
#pragma unroll 2
      for (int k = 0; k < count; ++k) {
        const Pack<T, V> x = held[k * kThreads], dy = held_dy[k * kThreads];
        if (p.dx != nullptr) {
          Pack<T, V> dx;
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const F2 xh = f2_mul(f2_add(x.pair(i), mean[ONE ? 0 : i]), rstd[ONE ? 0 : i]);
            const F2 g = f2_mul(dy.pair(i), slope2<decltype(act)::value>(f2_fma(xh, w[i], b[i])));
            dx.set_pair(i, f2_mul(rstd[ONE ? 0 : i], f2_fma(xh, s2[ONE ? 0 : i], f2_fma(g, w[i], s1[ONE ? 0 : i]))));
          }
          dx.store(dx0 + n * p.dx_s[0] + k * dx_step);
        }
        if (more) {
          async_load(held + k * kThreads, next_x + k * x_step, true);
          async_load(held_dy + k * kThreads, next_dy + k * dy_step, true);
        }
      }
    });
    if (s.cluster > 1) cluster_wait();           // before sh.own is written again, or the block ends
  }
  if (rank == 0)
    for (int i = threadIdx.x; i < at.here; i += kThreads) s.sums[(long long)slice * p.C + at.c0 + i] = sh.acc[i];
}

// ---- in two launches: a block takes a piece of an image's pixels of a slab -----------------------------------------

constexpr int kSplitRows = 32;        // rows of a thread

template <typename T, int V, bool ONE>
__global__ void __launch_bounds__(kThreads)
norm_split_stats_kernel(const Slab s) {
  __shared__ float2 red[ONE ? kThreads : kThreads * V];
  __shared__ float2 own[kMaxGroups];
  chained();
  const NormParams& p = s.p;
  const int piece = blockIdx.x % s.pieces, job = blockIdx.x / s.pieces, slab = job % s.slabs, n = job / s.slabs;
  const int row0 = piece * s.rows, cpg = p.C / p.G;
  const Place at = Place::of<V>(s, slab);
  const long long pixel = p.W > 1 ? p.x_s[3] : p.x_s[2];
  const T* x0 = static_cast<const T*>(p.x) + n * p.x_s[0] + at.c0 + at.cc + (long long)(row0 + at.r) * pixel;
  local_moments<T, V, ONE, true>(s, at, [&](int k) {
    Pack<T, V> x;
    x.load(x0 + (long long)k * s.rows_at_once * pixel);
    return x;
  }, Rows(s, min(s.S - row0, s.rows)), red, own);
  for (int g = threadIdx.x; g < at.groups; g += kThreads) s.part[((long long)n * s.pieces + piece) * p.G + at.c0 / cpg + g] = own[g];
}

template <typename T, int V, bool ONE>
__global__ void __launch_bounds__(kThreads)
norm_split_apply_kernel(const Slab s) {
  __shared__ float2 all_of[kMaxGroups];
  constexpr int M = ONE ? 1 : Pack<T, V>::kPairs;
  chained();
  const NormParams& p = s.p;
  const int piece = blockIdx.x % s.pieces, job = blockIdx.x / s.pieces, slab = job % s.slabs, n = job / s.slabs;
  const int row0 = piece * s.rows, end = min(s.S, row0 + s.rows), cpg = p.C / p.G;
  const Place at = Place::of<V>(s, slab);
  const int g0 = at.c0 / cpg;
  for (int g = threadIdx.x; g < at.groups; g += kThreads) {
    Moments all{0.0f, 0.0f, 0.0f};
    for (int q = 0; q < s.pieces; ++q) {
      const float2 v = s.part[((long long)n * s.pieces + q) * p.G + g0 + g];
      all = joined(all, Moments{float(min(s.S, (q + 1) * s.rows) - q * s.rows) * float(cpg), v.x, v.y});
    }
    const float rstd = rsqrtf(all.m2 / all.n + p.eps);
    all_of[g] = make_float2(all.mean, rstd);
    if (p.mean != nullptr && piece == 0) {
      p.mean[(long long)n * p.G + g0 + g] = all.mean;
      p.rstd[(long long)n * p.G + g0 + g] = rstd;
    }
  }
  __syncthreads();
  if (!at.live) return;
  const long long px = p.W > 1 ? p.x_s[3] : p.x_s[2], py = p.W > 1 ? p.y_s[3] : p.y_s[2];
  constexpr int P = Pack<T, V>::kPairs;
  F2 w[P], b[P], m[M];                              // m: minus the mean
  norm_params_of<T, V>(p, at.c0 + at.cc, true, w, b);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const float2 lo = all_of[at.live ? (at.cc + (ONE ? 0 : 2 * i)) / cpg : 0];
    const float2 hi = ONE ? lo : all_of[at.live ? (at.cc + min(2 * i + 1, V - 1)) / cpg : 0];
    m[ONE ? 0 : i] = f2_pack(-lo.x, -hi.x);
    w[i] = f2_mul(w[i], f2_pack(lo.y, hi.y));
  }
  const T* x0 = static_cast<const T*>(p.x) + n * p.x_s[0] + at.c0 + at.cc;
  T* y0 = static_cast<T*>(p.y) + n * p.y_s[0] + at.c0 + at.cc;
  with_activation(p.act, [&](auto act) {
#pragma unroll 4
    for (long long row = row0 + at.r; row < end; row += s.rows_at_once) {
      Pack<T, V> x, y;
      x.load(x0 + row * px);
#pragma unroll
      for (int i = 0; i < P; ++i) y.set_pair(i, activate2<decltype(act)::value>(f2_fma(f2_add(x.pair(i), m[ONE ? 0 : i]), w[i], b[i])));
      y.store(y0 + row * py);
    }
  });
}

template <typename T, int V, bool ONE>
__global__ void __launch_bounds__(kThreads)
norm_split_sums_kernel(const Slab s) {
  extern __shared__ __align__(16) unsigned char raw[];
  const BackwardShared sh(raw, kThreads * V, s.channels);
  constexpr int M = ONE ? 1 : Pack<T, V>::kPairs;
  chained();
  const NormParams& p = s.p;
  const int piece = blockIdx.x % s.pieces, job = blockIdx.x / s.pieces, slab = job % s.slabs, n = job / s.slabs;
  const int row0 = piece * s.rows, end = min(s.S, row0 + s.rows), cpg = p.C / p.G;
  const Place at = Place::of<V>(s, slab);
  const long long px = p.W > 1 ? p.x_s[3] : p.x_s[2], pdy = p.W > 1 ? p.dy_s[3] : p.dy_s[2];
  const int c = at.c0 + at.cc;
  constexpr int P = Pack<T, V>::kPairs;
  F2 w[P], b[P], mean[M], rstd[M], gx[P], gs[P];    // mean: minus the mean
  norm_params_of<T, V>(p, c, at.live, w, b);
#pragma unroll
  for (int i = 0; i < M; ++i) {
    const long long lo = (long long)n * p.G + (at.live ? (c + 2 * i) / cpg : 0);
    const long long hi = ONE ? lo : (long long)n * p.G + (at.live ? (c + min(2 * i + 1, V - 1)) / cpg : 0);
    mean[i] = f2_pack(-p.mean[lo], -p.mean[hi]);
    rstd[i] = f2_pack(p.rstd[lo], p.rstd[hi]);
  }
#pragma unroll
  for (int i = 0; i < P; ++i) gx[i] = gs[i] = 0;
  const T* x0 = static_cast<const T*>(p.x) + n * p.x_s[0] + c;
  const T* dy0 = static_cast<const T*>(p.dy) + n * p.dy_s[0] + c;
  if (at.live)
    with_activation(p.act, [&](auto act) {
#pragma unroll 4
      for (long long row = row0 + at.r; row < end; row += s.rows_at_once) {
        Pack<T, V> x, dy;
        x.load(x0 + row * px);
        dy.load(dy0 + row * pdy);
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const F2 xh = f2_mul(f2_add(x.pair(i), mean[ONE ? 0 : i]), rstd[ONE ? 0 : i]);
          const F2 g = f2_mul(dy.pair(i), slope2<decltype(act)::value>(f2_fma(xh, w[i], b[i])));
          gx[i] = f2_fma(g, xh, gx[i]);
          gs[i] = f2_add(gs[i], g);
        }
      }
    });
  sum_by_channel<V>(s, at, gx, gs, sh.red, sh.own);
  __syncthreads();
  for (int i = threadIdx.x; i < at.here; i += kThreads) s.sums[((long long)n * s.pieces + piece) * p.C + at.c0 + i] = sh.own[i];
}

template <typename T, int V, bool ONE>
__global__ void __launch_bounds__(kThreads)
norm_split_dx_kernel(const Slab s) {
  extern __shared__ __align__(16) unsigned char raw[];
  const BackwardShared sh(raw, kThreads * V, s.channels);
  constexpr int M = ONE ? 1 : Pack<T, V>::kPairs;
  chained();
  const NormParams& p = s.p;
  const int piece = blockIdx.x % s.pieces, job = blockIdx.x / s.pieces, slab = job % s.slabs, n = job / s.slabs;
  const int row0 = piece * s.rows, end = min(s.S, row0 + s.rows), cpg = p.C / p.G;
  const Place at = Place::of<V>(s, slab);
  for (int i = threadIdx.x; i < at.here; i += kThreads) {
    float2 t = make_float2(0.0f, 0.0f);
    for (int q = 0; q < s.pieces; ++q) {
      const float2 v = s.sums[((long long)n * s.pieces + q) * p.C + at.c0 + i];
      t.x += v.x;
      t.y += v.y;
    }
    sh.all[i] = t;
  }
  stage_weights<T>(p, at, sh.weight);
  __syncthreads();
  group_means(s, at, sh.weight, sh.all, sh.means);
  __syncthreads();
  if (!at.live) return;
  const bool tall = p.W > 1;
  const long long px = tall ? p.x_s[3] : p.x_s[2], pdy = tall ? p.dy_s[3] : p.dy_s[2], pdx = tall ? p.dx_s[3] : p.dx_s[2];
  const int c = at.c0 + at.cc;
  constexpr int P = Pack<T, V>::kPairs;
  F2 w[P], b[P], mean[M], rstd[M], s1[M], s2[M];    // minus the mean, minus s1 / m, minus s2 / m
  norm_params_of<T, V>(p, c, true, w, b);
#pragma unroll
  for (int i = 0; i < M; ++i) {
    const int glo = (c + 2 * i) / cpg, ghi = ONE ? glo : (c + min(2 * i + 1, V - 1)) / cpg;
    const long long at_n = (long long)n * p.G;
    mean[i] = f2_pack(-p.mean[at_n + glo], -p.mean[at_n + ghi]);
    rstd[i] = f2_pack(p.rstd[at_n + glo], p.rstd[at_n + ghi]);
    const float2 lo = sh.means[glo - at.c0 / cpg], hi = sh.means[ghi - at.c0 / cpg];
    s1[i] = f2_pack(-lo.x, -hi.x);
    s2[i] = f2_pack(-lo.y, -hi.y);
  }
  const T* x0 = static_cast<const T*>(p.x) + n * p.x_s[0] + c;
  const T* dy0 = static_cast<const T*>(p.dy) + n * p.dy_s[0] + c;
  T* dx0 = static_cast<T*>(p.dx) + n * p.dx_s[0] + c;
  with_activation(p.act, [&](auto act) {
#pragma unroll 4
    for (long long row = row0 + at.r; row < end; row += s.rows_at_once) {
      Pack<T, V> x, dy, dx;
      x.load(x0 + row * px);
      dy.load(dy0 + row * pdy);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const F2 xh = f2_mul(f2_add(x.pair(i), mean[ONE ? 0 : i]), rstd[ONE ? 0 : i]);
        const F2 g = f2_mul(dy.pair(i), slope2<decltype(act)::value>(f2_fma(xh, w[i], b[i])));
        dx.set_pair(i, f2_mul(rstd[ONE ? 0 : i], f2_fma(xh, s2[ONE ? 0 : i], f2_fma(g, w[i], s1[ONE ? 0 : i]))));
      }
      dx.store(dx0 + row * pdx);
    }
  });
}

// ---- which slab, how many blocks ------------------------------------------------------------------------------------

struct ImagePlan {
  Slab s;
  int V;
  bool split;            // two launches
  int smem;              // else: a block's
};

int gcd(int a, int b) { return b == 0 ? a : gcd(b, a % b); }

// False: a row of the slab is wider than a block's threads.
bool slab_of(ImagePlan* plan, const NormParams& p, int V, int channels) {
  Slab& s = plan->s;
  s.p = p;
  s.S = p.H * p.W;
  s.channels = channels;
  s.cols = channels / V;
  if (s.cols > kThreads || s.cols < 1) return false;
  s.rows_at_once = kThreads / s.cols;
  s.slabs = (p.C + channels - 1) / channels;
  s.slices = s.pieces = s.cluster = 1;
  s.held = 0;
  s.part = nullptr;
  s.sums = nullptr;
  plan->V = V;
  plan->split = false;
  return channels / (p.C / p.G) <= kMaxGroups;
}

// The slab: whole groups and whole vectors, rows of about 64 bytes (4 vectors: narrower rows waste what a DRAM access brings,
// wider ones leave too few blocks), narrower where no cluster holds it; few pixels take wider rows, or threads have none.
// The cluster: the fewest blocks that hold the slab with three (gradient: two) to an SM, more where SMs would be idle, and with
// one to an SM where eight blocks are too few.
bool image_plan(int dtype, const NormParams& p, bool backward, ImagePlan* plan) {
  const int cpg = p.C / p.G, es = dtype == FDNN_F32 ? 4 : 2, sms = current_sm_count();
  int V = norm_vector(dtype, p, backward, p.C);
  if (V == 0) return false;
  if (V == 2 && cpg % 2 != 0) V = 1;
  const long long S = (long long)p.H * p.W;
  if (S > 0x1fffffff) return false;
  const int unit = cpg / gcd(cpg, V) * V, units = p.C / unit;   // whole groups and whole vectors
  const long long wide = S < 64 ? kThreads / S : kRowVectors;
  int k = int(wide * V / unit);
  if (k < 1) k = 1;
  if (k > units) k = units;
  Slab& s = plan->s;
  for (;; k /= 2) {
    if (!slab_of(plan, p, V, k * unit)) {
      if (k == 1) return false;
      continue;
    }
    const int fixed = backward ? BackwardShared::bytes(kThreads * V, s.channels) : 0;
    const int row = kThreads * V * es * (backward ? 2 : 1);       // bytes of a row of a block's threads
    // (forward: beside 10 to 24 KB of static shared memory)
    const int few = ((backward ? 112 : 74) * 1024 - (backward ? fixed : (cpg % V == 0 ? 11 : 25) * 1024)) / row;
    const int most = (kMostShared - (backward ? fixed : kStatic)) / row;
    const long long at_once = s.rows_at_once;
    int cluster = 1;
    while (cluster < 8 && cluster * at_once * few < S) cluster *= 2;
    while (cluster < 8 && (long long)p.N * s.slabs * cluster < sms && cluster * at_once * 2 <= S) cluster *= 2;
    const long long need = (S + cluster * at_once - 1) / (cluster * at_once);
    // (not under 32 bytes to have three blocks to an SM, 64 x 64 x 112 x 112 bf16 97 us and 209; the gradient goes in two launches
    // rather than with one block to an SM, 195 us and 345)
    if (need > most || (need > few && (backward || (k > 1 && k * unit / V > 2)))) {
      if (k > 1 && k * unit / V > 2) continue;                     // narrower
      if (k > 1 && !backward) continue;
      break;
    }
    // The gradient of a few large images goes in two launches, which cut them finer: 1 x 4 x 163 x 170 bf16 in 4 groups 14.3 us, held by
    // clusters 20.2 (but 3 x 4 x 147 x 150 in one group 13.9 and 12.2; most are not held as it is). Forward the one launch is ahead on
    // 35 of 37 such shapes: 1 x 128 x 177 x 170 bf16 in 16 groups 13.5 us, cut 28.6; 1 x 16 x 194 x 189 in one 13.8 and 12.8.
    if (backward && 2ll * p.N * s.slabs * cluster <= sms && need > 16) break;
    s.cluster = cluster;
    s.rows = int((S + cluster - 1) / cluster);
    s.held = int((s.rows + at_once - 1) / at_once);
    plan->smem = fixed + s.held * row;
    // as many clusters as the SMs hold at once, or fewer that have equally many images each
    int per_sm = kSharedOfSm / (plan->smem + 1024 + (backward ? 0 : (cpg % V == 0 ? 10 : 24) * 1024));
    if (per_sm > (backward ? 2 : 3)) per_sm = backward ? 2 : 3;
    long long room = (long long)per_sm * sms / ((long long)s.slabs * cluster);
    if (room < 1) room = 1;
    const long long rounds = (p.N + room - 1) / room;
    s.slices = int((p.N + rounds - 1) / rounds);
    return true;
  }
  // no cluster holds a slab
  plan->split = true;
  // up to 32 rows a thread, fewer (down to 4) where that leaves SMs without blocks
  long long rows = (long long)p.N * s.slabs * S / (2ll * sms * s.rows_at_once);
  rows = rows > kSplitRows ? kSplitRows : rows < 4 ? 4 : rows;
  long long pieces = (S + rows * s.rows_at_once - 1) / (rows * s.rows_at_once);
  if (pieces > kMaxChunks) pieces = kMaxChunks;
  s.rows = int((S + pieces - 1) / pieces);
  s.pieces = int((S + s.rows - 1) / s.rows);
  return true;
}

template <typename T, int V, bool ONE>
cudaError_t forward(ImagePlan& plan, cudaStream_t stream) {
  Slab& s = plan.s;
  const NormParams& p = s.p;
  if (plan.split) {
    const long long blocks = (long long)p.N * s.slabs * s.pieces;
    if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    if (8ll * p.N * s.pieces * p.G > p.workspace_bytes) return cudaErrorInvalidValue;
    s.part = static_cast<float2*>(p.workspace);
    const cudaError_t e = launch_seq(norm_split_stats_kernel<T, V, ONE>, dim3(unsigned(blocks)), kThreads, 0, 1, stream, s);
    if (e != cudaSuccess) return e;
    return launch_seq(norm_split_apply_kernel<T, V, ONE>, dim3(unsigned(blocks)), kThreads, 0, 1, stream, s);
  }
  static std::atomic<uint64_t> done;
  auto* kernel = norm_images_kernel<T, V, ONE>;
  const cudaError_t e = allow_smem(kernel, kMostShared - kStatic, done);   // (beside the static part)
  if (e != cudaSuccess) return e;
  return launch_seq(kernel, dim3(unsigned((long long)s.slices * s.slabs * s.cluster)), kThreads, plan.smem, s.cluster, stream, s);
}

template <typename T, int V, bool ONE>
cudaError_t run_split(const Slab& s, long long blocks, cudaStream_t stream) {
  static std::atomic<uint64_t> sums_done, dx_done;
  const int smem = BackwardShared::bytes(kThreads * V, s.channels), most = BackwardShared::bytes(kThreads * V, kThreads * V);
  cudaError_t e = allow_smem(norm_split_sums_kernel<T, V, ONE>, most, sums_done);
  if (e == cudaSuccess) e = allow_smem(norm_split_dx_kernel<T, V, ONE>, most, dx_done);
  if (e == cudaSuccess) e = launch_seq(norm_split_sums_kernel<T, V, ONE>, dim3(unsigned(blocks)), kThreads, smem, 1, stream, s);
  if (e == cudaSuccess && s.p.dx != nullptr)
    e = launch_seq(norm_split_dx_kernel<T, V, ONE>, dim3(unsigned(blocks)), kThreads, smem, 1, stream, s);
  return e;
}

template <typename T, int V, bool ONE>
cudaError_t backward(ImagePlan& plan, cudaStream_t stream) {
  Slab& s = plan.s;
  const NormParams& p = s.p;
  s.sums = static_cast<float2*>(p.workspace);
  const long long rows = plan.split ? (long long)p.N * s.pieces : s.slices;
  if (8 * rows * p.C > p.workspace_bytes) return cudaErrorInvalidValue;
  cudaError_t e;
  if (plan.split) {
    const long long blocks = (long long)p.N * s.slabs * s.pieces;
    if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    e = run_split<T, V, ONE>(s, blocks, stream);
  } else {
    static std::atomic<uint64_t> done;
    auto* kernel = norm_images_backward_kernel<T, V, ONE>;
    e = allow_smem(kernel, kMostShared, done);
    if (e == cudaSuccess)
      e = launch_seq(kernel, dim3(unsigned((long long)s.slices * s.slabs * s.cluster)), kThreads, plan.smem, s.cluster, stream, s);
  }
  if (e != cudaSuccess || (p.dweight == nullptr && p.dbias == nullptr)) return e;
  return launch_norm_dparams<T>(p, s.sums, rows, stream);
}

}  // namespace

bool norm_images_take(int dtype, const NormParams& p, bool backward) {
  ImagePlan plan;
  return image_plan(dtype, p, backward, &plan);
}

// Upper bounds for any alignment: slices of the images, or pieces of them.
long long norm_images_workspace(int dtype, const NormParams& p, bool backward) {
  (void)dtype;
  const long long S = (long long)p.H * p.W, pieces = S < kMaxChunks ? S : kMaxChunks;
  const long long slices = 4ll * current_sm_count() < p.N ? 4ll * current_sm_count() : p.N;
  // Two launches: only where eight blocks do not hold kMostRows rows of vectors (backward 4, beside the sums of 2048 channels) for each
  // of their threads, of which at least 129 have work. A row has as many vectors as a group has channels, at most, or kRowVectors (of
  // several narrow groups; the wider rows of images of a few pixels are held by one block).
  const long long cols = p.C / p.G > kRowVectors ? p.C / p.G : kRowVectors;
  const bool split = S * cols > 8 * 128 * (backward ? 4 : kMostRows);
  const long long rows = split ? (p.N * pieces > slices ? p.N * pieces : slices) : slices;
  return 8 * rows * (backward ? p.C : split ? p.G : 0);
}

cudaError_t launch_norm_images(int dtype, const NormParams& p, bool back, cudaStream_t stream) {
  ImagePlan plan;
  if (!image_plan(dtype, p, back, &plan)) return cudaErrorInvalidValue;
  const bool one = p.C / p.G % plan.V == 0;
  return norm_by_vector(dtype, plan.V, [&](auto type, auto v) {
    using T = typename decltype(type)::type;
    constexpr int V = decltype(v)::value;
    if constexpr (V > 2)
      if (!one) return back ? backward<T, V, false>(plan, stream) : forward<T, V, false>(plan, stream);
    return back ? backward<T, V, true>(plan, stream) : forward<T, V, true>(plan, stream);
  });
}

}  // namespace fdnn
