// The selective state space scan over prompts.
//
//   dt = delta + delta_bias, softplus of it if asked
//   h_t = exp(dt A) h_(t-1) + dt u_t B_t,  y_t = (sum over the states of C_t h_t + D u_t) silu(z_t)
//
// per channel, with a decay rate of its own for each of its S states; B_t and C_t are shared by the channels of a group.
// The states are fp32 throughout.
//
// What bounds it is the special function unit: an exponential per token, channel and state (8 cycles per warp and SM
// quarter), beside three packed multiplications; the bytes of 8192 x 4096 values of bf16 take 41 us, their 16 exponentials
// each 118.  So a block keeps one half of its warps on nothing but the recurrence and has the other half do the rest:
//
//   warps 4-7 (fill)  load u, delta, z, B, C of the next 32 tokens, take softplus and the gate, leave (dt, dt u)
//                     and fp32 B, C in shared memory, two tiles deep; later add D u, gate and store what the scan left
//   warps 0-3 (scan)  LANES neighbouring parts of a channel's states per channel, NPT states a thread in registers, packed
//                     in pairs; a tile's sums over the states are exchanged between the lanes four tokens at a time
//
// Hand-over is by named barriers (full and done for each buffer).  Few channels would leave SMs idle: rows are then cut into
// chunks, a first launch scans each but the last from zeros and keeps its end state and its sum of dt (the decay over the
// whole chunk is exp(A sum dt)), and the second begins each chunk with the states before it joined in their order.
#include <math.h>

#include "f32x2.cuh"
#include "sequence_internal.h"
#include "sequence_launch.h"
#include "sequence_math.cuh"

namespace fdnn {
namespace {


constexpr int kScan = 128, kFill = 128;    // threads that scan, threads that fill

struct Cut {
  int chunks, tokens;                      // chunks of a row, tokens of each (the last may have fewer)
};

struct ScanJob {
  ScanParams p;
  Cut cut;
  int blocks_per_group;
  float* ends;                             // [N, chunks - 1, C, S] end states of the chunks
  float* sums;                             // [N, chunks - 1, C] sums of dt
};

__device__ __forceinline__ int length_of(const int* lengths, int n, int L) {
  return lengths == nullptr ? L : min(max(lengths[n], 0), L);
}
template <int ID>
__device__ __forceinline__ void bar_sync(int which) { asm volatile("bar.sync %0, %1;" ::"r"(ID + which), "n"(kScan + kFill) : "memory"); }
// (Orders this thread's accesses to shared memory before those behind the others' bar_sync: the producer's half of the PTX
// manual's own example. A fence in front of it would wait for the stores of y.)
template <int ID>
__device__ __forceinline__ void bar_arrive(int which) { asm volatile("bar.arrive %0, %1;" ::"r"(ID + which), "n"(kScan + kFill) : "memory"); }
constexpr int kFull = 1, kDone = 3;

// Eight neighbouring values (of channels or of states), as loaded.
template <typename T>
struct Eight {
  static constexpr int kWords = sizeof(T) / 2;
  uint4 q[kWords];
  __device__ __forceinline__ float at(int k) const { return to_f32<T>(reinterpret_cast<const T*>(q)[k]); }
  __device__ __forceinline__ void set(int k, T v) { reinterpret_cast<T*>(q)[k] = v; }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int w = 0; w < kWords; ++w) q[w] = make_uint4(0, 0, 0, 0);
  }
  // VEC: all eight are there, dense and 16-byte aligned; otherwise the first `count`, `stride` apart
  template <bool VEC>
  __device__ __forceinline__ void load(const T* p, long long stride, int count) {
    if constexpr (VEC) {
#pragma unroll
      for (int w = 0; w < kWords; ++w) q[w] = __ldg(reinterpret_cast<const uint4*>(p) + w);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) set(k, k < count ? p[k * stride] : from_f32<T>(0.0f));
    }
  }
};

// A tile is eight channels of a token for each filling thread.
template <int NPT, int LANES>
struct Tile {
  static constexpr int kChannels = kScan / LANES;
  static constexpr int kChunks = kChannels / 8;                      // eights of channels
  static constexpr int kStates = NPT * LANES;
  static constexpr int kTokens = 8 * kFill / kChannels < kFill / 4 ? 8 * kFill / kChannels : kFill / 4;
  static constexpr int kPieces = 2 * kStates / 8;                    // eights of a token's B and C
  // Sixteen threads of a warp store their k-th channels at once, and the scanning lanes read eight neighbours: channel k of an
  // eight lies at k ^ turn, so that neither meets a bank twice.
  static __device__ __forceinline__ int turn(int t, int chunk) { return ((t * kChunks + chunk) >> 1) & 7; }
  float2 step[kTokens][kChannels];                                   // dt, dt u
  float bc[kTokens][2 * kStates];                                    // B, then C
  float y[kChunks][kTokens * 8 + 8];                                 // [token][channel of the eight]
};

// What a filling thread has on its way from memory: its eights of u, delta, z and of the table of B and C, several tiles ahead.
// The slots are its own (no other thread reads them), u and z stay until the tile's y has been stored.
constexpr int kPrefetch = 3, kSlots = kPrefetch + 1, kLongSlots = kPrefetch + 3;
template <typename T, int PIECES>
struct Ring {
  static constexpr int kWords = Eight<T>::kWords;
  uint4 u[kLongSlots][kWords][kFill];
  uint4 z[kLongSlots][kWords][kFill];
  uint4 delta[kSlots][kWords][kFill];
  uint4 bc[kSlots][PIECES > 0 ? PIECES : 1][kWords][kFill];
};
// Asynchronously, 16 bytes at a time, zeros past `count` values.
template <typename T>
__device__ __forceinline__ void fetch(uint4 (&slot)[Eight<T>::kWords][kFill], int tid, const T* p, int count) {
#pragma unroll
  for (int w = 0; w < Eight<T>::kWords; ++w)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(uint32_t(__cvta_generic_to_shared(&slot[w][tid]))),
                 "l"(reinterpret_cast<const uint4*>(p) + w), "r"(count > w * 16 / int(sizeof(T)) ? 16 : 0)
                 : "memory");
}
template <typename T>
__device__ __forceinline__ void put(uint4 (&slot)[Eight<T>::kWords][kFill], int tid, const Eight<T>& v) {
#pragma unroll
  for (int w = 0; w < Eight<T>::kWords; ++w) slot[w][tid] = v.q[w];
}
template <typename T>
__device__ __forceinline__ Eight<T> fetched(const uint4 (&slot)[Eight<T>::kWords][kFill], int tid) {
  Eight<T> v;
#pragma unroll
  for (int w = 0; w < Eight<T>::kWords; ++w) v.q[w] = slot[w][tid];
  return v;
}

template <typename T, int NPT, int LANES>
struct Loads {
  using Buf = Tile<NPT, LANES>;
  static constexpr int kTable = Buf::kTokens * Buf::kPieces;          // eights of a tile's B and C
  static constexpr int kMine = (kTable + kFill - 1) / kFill;            // of a filling thread
  static constexpr bool kFetched = Buf::kStates >= 8 && kMine <= 4;
  using R = Ring<T, kFetched ? kMine : 0>;
  static constexpr int kSmem = 2 * int(sizeof(Buf)) + int(sizeof(R));
};

// ENDS: the first launch of a row in chunks (end states and sums of dt, no y).  VEC: every tensor can be read by 16 bytes.  ALONE:
// no other block on the SM.
template <typename T, int NPT, int LANES, bool ALONE, bool ENDS, bool VEC>
__global__ void __launch_bounds__(kScan + kFill)
scan_kernel(const ScanJob job) {
  using Buf = Tile<NPT, LANES>;
  using Load = Loads<T, NPT, LANES>;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Buf* buf = reinterpret_cast<Buf*>(smem_raw);
  chained();
  const ScanParams& p = job.p;
  const int blocks = p.G * job.blocks_per_group, runs = ENDS ? job.cut.chunks - 1 : job.cut.chunks;
  const int cb = int(blockIdx.x % unsigned(blocks)), rest = int(blockIdx.x / unsigned(blocks));
  const int chunk = rest % runs, n = rest / runs;
  const int per_group = p.C / p.G, g = cb / job.blocks_per_group;
  const int c0 = g * per_group + (cb % job.blocks_per_group) * Buf::kChannels, c1 = (g + 1) * per_group;
  const int len = length_of(p.lengths, n, p.L);
  const int t0 = chunk * job.cut.tokens, t1 = min(t0 + job.cut.tokens, p.L), te = min(t1, len);
  const int tiles = te > t0 ? (te - t0 + Buf::kTokens - 1) / Buf::kTokens : 0;

  if (threadIdx.x >= kScan) {
    // A filling thread has one token of a tile and eight channels.
    const int tid = threadIdx.x - kScan;
    const int dt0 = tid / Buf::kChunks, eight = tid % Buf::kChunks;
    const int c = c0 + eight * 8;
    const int have = dt0 < Buf::kTokens ? min(max(c1 - c, 0), 8) : 0;   // channels of this thread
    const long long first = t0 + dt0;
    const T* u = static_cast<const T*>(p.u) + n * p.u_s[0] + c * p.u_s[2] + first * p.u_s[1];
    const T* delta = static_cast<const T*>(p.delta) + n * p.delta_s[0] + c * p.delta_s[2] + first * p.delta_s[1];
    const T* z = p.z == nullptr ? nullptr : static_cast<const T*>(p.z) + n * p.z_s[0] + c * p.z_s[2] + first * p.z_s[1];
    T* y = static_cast<T*>(p.y) + n * p.y_s[0] + c * p.y_s[2] + first * p.y_s[1];
    float D[8], bias[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      D[k] = !ENDS && k < have && p.D != nullptr ? p.D[c + k] : 0.0f;
      bias[k] = k < have && p.delta_bias != nullptr ? p.delta_bias[c + k] : 0.0f;
    }
    // eights of the table of B and C: fetched ahead where they are few, else loaded when they are stored
    constexpr int kMine = Load::kMine;
    auto& ring = *reinterpret_cast<typename Load::R*>(smem_raw + 2 * sizeof(Buf));
    auto source = [&](int i, int m, const T*& from, long long& stride) -> int {
      const int e = tid + m * kFill, dt = e / Buf::kPieces, j = e % Buf::kPieces * 8, t = t0 + i * Buf::kTokens + dt;
      const bool is_c = j >= Buf::kStates;
      const int s = is_c ? j - Buf::kStates : j;
      const bool in = e < Load::kTable && t < te && s < p.S && !(ENDS && is_c);
      const long long* st = is_c ? p.c_s : p.b_s;
      stride = st[3];
      from = static_cast<const T*>(is_c ? p.Cm : p.B) + (in ? n * st[0] + t * st[1] + g * st[2] + s * st[3] : 0);
      return in ? min(p.S - s, 8) : 0;
    };
    auto tabulate = [&](int i, int m, const Eight<T>& v) {
      const int e = tid + m * kFill;
      if (e >= Load::kTable) return;
      float4* to = reinterpret_cast<float4*>(&buf[i & 1].bc[e / Buf::kPieces][e % Buf::kPieces * 8]);
      to[0] = make_float4(v.at(0), v.at(1), v.at(2), v.at(3));
      to[1] = make_float4(v.at(4), v.at(5), v.at(6), v.at(7));
    };
    // values that cannot be copied asynchronously wait in registers until the next tile is asked for
    constexpr int kEights = Load::kFetched ? kMine : 1;
    Eight<T> wait_u, wait_d, wait_z, wait_bc[kEights];
    auto settle = [&](int i) {
      if (i < 0 || i >= tiles) return;
      put(ring.u[i % kLongSlots], tid, wait_u);
      put(ring.delta[i % kSlots], tid, wait_d);
      if (!ENDS && p.z != nullptr) put(ring.z[i % kLongSlots], tid, wait_z);
      if constexpr (Load::kFetched) {
#pragma unroll
        for (int m = 0; m < kMine; ++m) put(ring.bc[i % kSlots][m], tid, wait_bc[m]);
      }
    };
    auto load = [&](int i) {
      if constexpr (!VEC) settle(i - 1);
      if (i < tiles) {
        const int got = first + (long long)i * Buf::kTokens < te ? have : 0;
        const long long at = got > 0 ? (long long)i * Buf::kTokens : 0;
        if constexpr (VEC) {   // (an address inside the tensor, read or not)
          fetch<T>(ring.u[i % kLongSlots], tid, got > 0 ? u + at * p.u_s[1] : static_cast<const T*>(p.u), got);
          fetch<T>(ring.delta[i % kSlots], tid, got > 0 ? delta + at * p.delta_s[1] : static_cast<const T*>(p.delta), got);
          if (!ENDS && p.z != nullptr) fetch<T>(ring.z[i % kLongSlots], tid, got > 0 ? z + at * p.z_s[1] : static_cast<const T*>(p.z), got);
        } else {
          wait_u.template load<false>(u + at * p.u_s[1], p.u_s[2], got);
          wait_d.template load<false>(delta + at * p.delta_s[1], p.delta_s[2], got);
          if (!ENDS && p.z != nullptr) wait_z.template load<false>(z + at * p.z_s[1], p.z_s[2], got);
        }
        if constexpr (Load::kFetched) {
#pragma unroll
          for (int m = 0; m < kMine; ++m) {
            const T* from;
            long long stride;
            const int count = source(i, m, from, stride);
            if constexpr (VEC) fetch<T>(ring.bc[i % kSlots][m], tid, from, count);
            else wait_bc[m].template load<false>(from, stride, count);
          }
        }
      }
      if constexpr (VEC) asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto fill = [&](int i) {
      Buf& b = buf[i & 1];
      if constexpr (VEC) asm volatile("cp.async.wait_group %0;" ::"n"(kPrefetch - 1) : "memory");
      if constexpr (Load::kFetched) {
#pragma unroll
        for (int m = 0; m < kMine; ++m) tabulate(i, m, fetched<T>(ring.bc[i % kSlots][m], tid));
      } else if constexpr (Buf::kStates >= 8) {
        for (int m = 0; m < kMine; m += 4) {
          Eight<T> v[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const T* from;
            long long stride;
            const int count = source(i, m + q, from, stride);
            if (count > 0) v[q].template load<VEC>(from, stride, count);
            else v[q].clear();
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) tabulate(i, m + q, v[q]);
        }
      } else {
        const int t = t0 + i * Buf::kTokens + tid;                       // at most four states: an eight is a token's B and C
        Eight<T> v;
        v.clear();
        if (tid < Buf::kTokens && t < te) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int s = k % Buf::kStates;
            const long long* st = k >= Buf::kStates ? p.c_s : p.b_s;
            if (s < p.S)
              v.set(k, (static_cast<const T*>(k >= Buf::kStates ? p.Cm : p.B) + n * st[0] + t * st[1] + g * st[2])[s * st[3]]);
          }
        }
        tabulate(i, 0, v);
      }
      if (dt0 < Buf::kTokens) {
        const int got = first + (long long)i * Buf::kTokens < te ? have : 0, turn = Buf::turn(dt0, eight);
        const Eight<T> ru = fetched<T>(ring.u[i % kLongSlots], tid), rd = fetched<T>(ring.delta[i % kSlots], tid);
        float d[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) d[k] = rd.at(k) + bias[k];
        if (p.softplus) {
#pragma unroll
          for (int k = 0; k < 8; ++k) d[k] = softplus(d[k]);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float dk = k < got ? d[k] : 0.0f;                      // past the row: a step of no time
          const float du = dk * ru.at(k);
          b.step[dt0][eight * 8 + (k ^ turn)] = make_float2(dk, du);
        }
      }
    };
    auto store = [&](int i) {
      if (dt0 < Buf::kTokens && first + (long long)i * Buf::kTokens < te && have > 0) {
        const float4* from = reinterpret_cast<const float4*>(&buf[i & 1].y[eight][dt0 * 8]);
        const float4 lo = from[0], hi = from[1];
        float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        const Eight<T> ku = fetched<T>(ring.u[i % kLongSlots], tid);
        if (p.D != nullptr) {   // (zero times an infinite u is not nothing)
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] += D[k] * ku.at(k);
        }
        if (p.z != nullptr) {
          const Eight<T> kz = fetched<T>(ring.z[i % kLongSlots], tid);
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] *= silu(kz.at(k));
        }
        if constexpr (VEC) {
          Eight<T> out;
#pragma unroll
          for (int k = 0; k < 8; ++k) out.set(k, from_f32<T>(v[k]));
#pragma unroll
          for (int w = 0; w < Eight<T>::kWords; ++w)
            if (have > w * 16 / int(sizeof(T))) reinterpret_cast<uint4*>(y)[w] = out.q[w];
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k < have) y[k * p.y_s[2]] = from_f32<T>(v[k]);
        }
      }
      y += Buf::kTokens * p.y_s[1];
    };
    for (int i = 0; i < kPrefetch; ++i) load(i);
    for (int i = 0; i < tiles; ++i) {
      if (i >= 2) {
        bar_sync<kDone>(i & 1);
        if constexpr (!ENDS) store(i - 2);
      }
      fill(i);
      bar_arrive<kFull>(i & 1);
      load(i + kPrefetch);   // into the slots of tile i - 1 (delta, B, C) and i - 3 (u, z: stored)
    }
    for (int i = tiles > 2 ? tiles - 2 : 0; i < tiles; ++i) {
      bar_sync<kDone>(i & 1);
      if constexpr (!ENDS) store(i);
    }
    if constexpr (!ENDS) {
      // padding
      T* row = static_cast<T*>(p.y) + n * p.y_s[0];
      const int span = min(c1 - c0, Buf::kChannels);
      for (long long e = tid; e < (long long)(t1 - max(t0, len)) * span; e += kFill)
        row[(max(t0, len) + e / span) * p.y_s[1] + (c0 + e % span) * p.y_s[2]] = from_f32<T>(0.0f);
    }
    return;
  }

  constexpr int kPerWarp = 32 / LANES, kPairs = NPT / 2, kQ = LANES >= 8 ? 8 : 4;
  const int lane = threadIdx.x & 31, cl = (threadIdx.x >> 5) * kPerWarp + lane % kPerWarp, part = lane / kPerWarp;
  const int c = c0 + cl, s0 = part * NPT;
  const bool live = c < c1;
  F2 a[kPairs], h[kPairs];
  {
    float av[NPT], hv[NPT];
    const long long row = (long long)n * p.C + c;
#pragma unroll
    for (int s = 0; s < NPT; ++s) {
      const bool in = live && s0 + s < p.S;
      av[s] = in ? rate_of(p.A[(long long)c * p.S + s0 + s]) : 0.0f;
      hv[s] = !ENDS && in && p.initial != nullptr ? p.initial[row * p.S + s0 + s] : 0.0f;
    }
    if constexpr (!ENDS) {
      for (int k = 0; live && k < chunk; ++k) {
        const long long at = ((long long)n * (job.cut.chunks - 1) + k) * p.C + c;
        const float sum = job.sums[at];
#pragma unroll
        for (int s = 0; s < NPT; ++s)
          if (s0 + s < p.S)   // (a state of nothing stays nothing, even if e^(A sum dt) is no number)
            hv[s] = hv[s] * decay_of(hv[s] == 0.0f ? 0.0f : sum, av[s]) + job.ends[at * p.S + s0 + s];
      }
    }
#pragma unroll
    for (int s = 0; s < kPairs; ++s) {
      a[s] = f2_pack(av[2 * s], av[2 * s + 1]);
      h[s] = f2_pack(hv[2 * s], hv[2 * s + 1]);
    }
  }
  const F2 middle = f2_both(kDecayMiddle);
  const int eight = cl / 8, in_eight = cl % 8;
  float sum = 0.0f;
  for (int i = 0; i < tiles; ++i) {
    bar_sync<kFull>(i & 1);
    Buf& b = buf[i & 1];
    auto decay = [&](int t, F2 (&e)[kPairs], float& du) {
      const float2 st = b.step[t][eight * 8 + (in_eight ^ Buf::turn(t, eight))];
      du = st.y;
      if constexpr (ENDS) sum += st.x;
#pragma unroll
      for (int s = 0; s < kPairs; ++s) {
        float x0, x1;
        f2_split(f2_fma(f2_pack(st.x, st.x), a[s], middle), x0, x1);
        e[s] = f2_pack(ex2(x0), ex2(x1));
      }
    };
    auto advance = [&](int t, const F2 (&e)[kPairs], float du) -> float {
      F2 B2[kPairs], C2[kPairs];
      const float *Bt = &b.bc[t][s0], *Ct = &b.bc[t][Buf::kStates + s0];
      if constexpr (kPairs == 1) {
        B2[0] = *reinterpret_cast<const F2*>(Bt);
        if constexpr (!ENDS) C2[0] = *reinterpret_cast<const F2*>(Ct);
      } else {
#pragma unroll
        for (int s = 0; s < kPairs; s += 2) {
          const ulonglong2 q = reinterpret_cast<const ulonglong2*>(Bt)[s / 2];
          B2[s] = q.x;
          B2[s + 1] = q.y;
          if constexpr (!ENDS) {
            const ulonglong2 r = reinterpret_cast<const ulonglong2*>(Ct)[s / 2];
            C2[s] = r.x;
            C2[s + 1] = r.y;
          }
        }
      }
      F2 y2 = 0;
#pragma unroll
      for (int s = 0; s < kPairs; ++s) {
        h[s] = f2_fma(h[s], e[s], f2_mul(f2_pack(du, du), B2[s]));
        if constexpr (!ENDS) y2 = s == 0 ? f2_mul(h[s], C2[s]) : f2_fma(h[s], C2[s], y2);
      }
      float y0, y1;
      f2_split(y2, y0, y1);
      return y0 + y1;
    };
    // the lanes of a channel exchange their sums of kQ tokens: each keeps half of them, then a quarter, ...
    auto give = [&](int t, float (&v)[kQ]) {
      int at = t;
      constexpr int kKeep = kQ > LANES ? kQ / LANES : 1;
#pragma unroll
      for (int m = kQ / 2, o = kPerWarp, bit = 1; o < 32; m /= 2, o *= 2, bit *= 2) {
        const bool upper = (part & bit) != 0;
        if (m >= kKeep && m > 0) {
#pragma unroll
          for (int q = 0; q < m; ++q)
            v[q] = (upper ? v[q + m] : v[q]) + __shfl_xor_sync(0xffffffffu, upper ? v[q] : v[q + m], o);
          at += upper ? m : 0;
        } else {
          v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
        }
      }
      float* to = &b.y[eight][in_eight];
#pragma unroll
      for (int q = 0; q < kKeep; ++q)
        if (part < kQ) to[(at + q) * 8] = v[q];
    };
    if constexpr (ALONE) {
      // One scanning warp to an SM quarter has only itself to hide latencies behind: what it reads of four tokens, and their decays,
      // are on their way, in this order, while the states go through the four before them (8192 x 4096: 279 us, 304 as below).
      struct Ahead {
        float dt[kQ], du[kQ];
        F2 B[kQ][kPairs], C[kQ][kPairs];
      };
      auto lds2 = [](const void* p, float& a, float& b) {
        asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(a), "=f"(b) : "r"(uint32_t(__cvta_generic_to_shared(p))));
      };
      auto lds4 = [](const void* p, F2& a, F2& b) {
        asm volatile("ld.shared.v2.b64 {%0,%1}, [%2];" : "=l"(a), "=l"(b) : "r"(uint32_t(__cvta_generic_to_shared(p))));
      };
      auto vex2 = [](float v) {
        float r;
        asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
        return r;
      };
      auto ahead = [&](int t, Ahead& n) {
#pragma unroll
        for (int q = 0; q < kQ; ++q) lds2(&b.step[t + q][eight * 8 + (in_eight ^ Buf::turn(t + q, eight))], n.dt[q], n.du[q]);
#pragma unroll
        for (int q = 0; q < kQ; ++q) {
#pragma unroll
          for (int s = 0; s < kPairs; s += 2) {
            lds4(&b.bc[t + q][s0 + 2 * s], n.B[q][s], n.B[q][s + 1]);
            if constexpr (!ENDS) lds4(&b.bc[t + q][Buf::kStates + s0 + 2 * s], n.C[q][s], n.C[q][s + 1]);
          }
        }
      };
      Ahead now, next;
      F2 e[kQ][kPairs], f[kQ][kPairs];
      float v[kQ], w[kQ];
      ahead(0, now);
#pragma unroll
      for (int q = 0; q < kQ; ++q) {
        if constexpr (ENDS) sum += now.dt[q];
#pragma unroll
        for (int s = 0; s < kPairs; ++s) {
          float x0, x1;
          f2_split(f2_fma(f2_pack(now.dt[q], now.dt[q]), a[s], middle), x0, x1);
          e[q][s] = f2_pack(vex2(x0), vex2(x1));
        }
      }
#pragma unroll
      for (int t = 0; t < Buf::kTokens; t += kQ) {
        const bool more = t + kQ < Buf::kTokens;
        if (more) ahead(t + kQ, next);
#pragma unroll
        for (int q = 0; q < kQ; ++q) {
          F2 y2 = 0;
#pragma unroll
          for (int s = 0; s < kPairs; ++s) {
            if (more) {
              float x0, x1;
              f2_split(f2_fma(f2_pack(next.dt[q], next.dt[q]), a[s], middle), x0, x1);
              f[q][s] = f2_pack(vex2(x0), vex2(x1));
            }
            h[s] = f2_fma(h[s], e[q][s], f2_mul(f2_pack(now.du[q], now.du[q]), now.B[q][s]));
            if constexpr (!ENDS) y2 = s == 0 ? f2_mul(h[s], now.C[q][s]) : f2_fma(h[s], now.C[q][s], y2);
          }
          if constexpr (ENDS) { if (more) sum += next.dt[q]; }
          float y0, y1;
          f2_split(y2, y0, y1);
          w[q] = y0 + y1;
        }
        if (!ENDS && t > 0) give(t - kQ, v);
#pragma unroll
        for (int q = 0; q < kQ; ++q) {
          v[q] = w[q];
#pragma unroll
          for (int s = 0; s < kPairs; ++s) e[q][s] = f[q][s];
        }
        now = next;
      }
      if constexpr (!ENDS) give(Buf::kTokens - kQ, v);
    } else if constexpr (NPT <= 4) {
      // The decays of kQ tokens are taken while the states go through the kQ before them, and sums are exchanged kQ tokens late.
      F2 e[kQ][kPairs];
      float v[kQ], du[kQ];
#pragma unroll
      for (int q = 0; q < kQ; ++q) decay(q, e[q], du[q]);
#pragma unroll
      for (int t = 0; t < Buf::kTokens; t += kQ) {
        F2 now[kQ][kPairs];
        float w[kQ], now_du[kQ];
#pragma unroll
        for (int q = 0; q < kQ; ++q) {
#pragma unroll
          for (int s = 0; s < kPairs; ++s) now[q][s] = e[q][s];
          now_du[q] = du[q];
        }
#pragma unroll
        for (int q = 0; q < kQ; ++q) {
          if (t + kQ < Buf::kTokens) decay(t + kQ + q, e[q], du[q]);
          w[q] = advance(t + q, now[q], now_du[q]);
        }
        if (!ENDS && t > 0) give(t - kQ, v);
#pragma unroll
        for (int q = 0; q < kQ; ++q) v[q] = w[q];
      }
      if constexpr (!ENDS) give(Buf::kTokens - kQ, v);
    } else {
      for (int t = 0; t < Buf::kTokens; t += kQ) {
        float v[kQ];
#pragma unroll
        for (int q = 0; q < kQ; ++q) {
          F2 e[kPairs];
          float du;
          decay(t + q, e, du);
          v[q] = advance(t + q, e, du);
        }
        if constexpr (!ENDS) give(t, v);
      }
    }
    bar_arrive<kDone>(i & 1);
  }
  if (!live) return;
  float* out = nullptr;
  if constexpr (ENDS) {
    const long long at = ((long long)n * (job.cut.chunks - 1) + chunk) * p.C + c;
    out = job.ends + at * p.S;
    if (part == 0) job.sums[at] = sum;
  } else if (p.final_state != nullptr && chunk == job.cut.chunks - 1) {
    out = p.final_state + ((long long)n * p.C + c) * p.S;
  }
  if (out == nullptr) return;
#pragma unroll
  for (int s = 0; s < NPT; ++s) {
    float lo, hi;
    f2_split(h[s / 2], lo, hi);
    if (s0 + s < p.S) out[s0 + s] = s % 2 == 0 ? lo : hi;
  }
}

// Threads of a channel.
int lanes_of(int S) { return S <= 4 ? 1 : S <= 8 ? 2 : S <= 32 ? 4 : S <= 128 ? 8 : 16; }

// How many chunks a row is cut into: the fewest clocks by what was measured for 16 states. A token costs the m blocks that
// share an SM 57 m + 16 clocks (73 for one alone, where latencies show), the first launch of a row in chunks 0.65 of that for
// all but the last chunk, and there is some 4 us in a second launch. 8192 x 1024: 280 us whole, 145 in 4, 116 in 12 chunks;
// 8192 x 4096: 279 us whole, 380 in 4, 361 in 12; 2048 x 256: 73 whole, 19 in 16.
// With more states a token costs more (alone on an SM 64 clocks for 16, 140 for 32, 129 for 64, 216 for 128, 330 for 256), which weighs
// only against the second launch: ten shapes of 32 to 256 states are cut alike with these factors and without. 4096 x 256 x 32: 307 us
// whole, 50 in the 16 chunks chosen; 4096 x 1024 x 64: 284, 205 in 16 (191 in 10); 8192 x 256 x 256: 1440, 568.
Cut cut_of(const ScanParams& p) {
  const int channels = kScan / lanes_of(p.S), per_group = p.C / p.G, sms = current_sm_count();
  const double blocks = double(p.N) * p.G * ((per_group + channels - 1) / channels);
  const double states = p.S <= 16 ? 1.0 : p.S <= 32 ? 1.5 : p.S <= 64 ? 1.9 : 3.8;   // what a block's token costs with more states
  auto token = [&](double b) { return (57.0 * ceil(b / sms) + 16.0) * states; };
  Cut best{1, p.L};
  double least = p.L * token(blocks);
  for (int k = 2; k <= 16; ++k) {
    const int tokens = (p.L / k + 64) / 64 * 64;
    if (tokens < 128) break;
    const int chunks = (p.L - 1) / tokens + 1;
    if (chunks != k) continue;
    const double clocks = tokens * (token(blocks * k) + 0.65 * token(blocks * (k - 1))) + 8000.0;
    if (clocks < least) {
      least = clocks;
      best = Cut{chunks, tokens};
    }
  }
  return best;
}

// Whether every tensor can be read (and y written) by 16 bytes: channels and states dense, aligned and whole numbers of them.
template <typename T>
bool by_eights(const ScanParams& p) {
  const int per = 16 / int(sizeof(T));
  auto ok = [&](const void* q, const long long* st, int last, int strides) {
    if ((reinterpret_cast<uintptr_t>(q) & 15u) != 0 || st[last] != 1) return false;
    for (int i = 0; i < strides; ++i)
      if (i != last && st[i] % per != 0) return false;
    return true;
  };
  return p.C / p.G % per == 0 && p.S % 8 == 0 && (p.S & (p.S - 1)) == 0 && ok(p.u, p.u_s, 2, 3) && ok(p.delta, p.delta_s, 2, 3) &&
         ok(p.y, p.y_s, 2, 3) && (p.z == nullptr || ok(p.z, p.z_s, 2, 3)) && ok(p.B, p.b_s, 3, 4) && ok(p.Cm, p.c_s, 3, 4);
}

template <typename T, int NPT, int LANES, bool ALONE, bool ENDS, bool VEC>
cudaError_t run(const ScanJob& job, long long blocks, cudaStream_t stream) {
  static std::atomic<uint64_t> done;
  // No more blocks than SMs: each asks for more than half of an SM's shared memory, or two may share one beside an idle one.
  constexpr int kAlone = 116 * 1024, kNeeds = Loads<T, NPT, LANES>::kSmem, kMost = kNeeds > kAlone ? kNeeds : kAlone;
  auto* kernel = scan_kernel<T, NPT, LANES, ALONE, ENDS, VEC>;
  const cudaError_t e = allow_smem(kernel, kMost, done);
  if (e != cudaSuccess) return e;
  return launch_seq(kernel, dim3(unsigned(blocks)), kScan + kFill, blocks <= current_sm_count() ? kMost : kNeeds, 1, stream, job);
}

template <typename T, int NPT, int LANES, bool ENDS>
cudaError_t run(const ScanJob& job, bool vec, cudaStream_t stream) {
  const long long blocks = (long long)job.p.N * (ENDS ? job.cut.chunks - 1 : job.cut.chunks) * job.p.G * job.blocks_per_group;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  if constexpr (NPT == 4)
    if (vec && blocks <= current_sm_count()) return run<T, NPT, LANES, true, ENDS, NPT * LANES >= 8>(job, blocks, stream);
  constexpr bool kVec = NPT * LANES >= 8;
  return vec ? run<T, NPT, LANES, false, ENDS, kVec>(job, blocks, stream) : run<T, NPT, LANES, false, ENDS, false>(job, blocks, stream);
}

template <typename T, int NPT, int LANES>
cudaError_t go(const ScanParams& p, cudaStream_t stream) {
  ScanJob job;
  job.p = p;
  job.cut = cut_of(p);
  const int per_group = p.C / p.G, channels = kScan / LANES;
  job.blocks_per_group = (per_group + channels - 1) / channels;
  job.ends = static_cast<float*>(p.workspace);
  job.sums = job.ends == nullptr ? nullptr : job.ends + (long long)p.N * (job.cut.chunks - 1) * p.C * p.S;
  const bool vec = NPT * LANES >= 8 && by_eights<T>(p);
  if (job.cut.chunks > 1) {
    const cudaError_t e = run<T, NPT, LANES, true>(job, vec, stream);
    if (e != cudaSuccess) return e;
  }
  return run<T, NPT, LANES, false>(job, vec, stream);
}

template <typename T>
cudaError_t scan(const ScanParams& p, cudaStream_t stream) {
  if (p.S <= 4) return go<T, 4, 1>(p, stream);
  if (p.S <= 8) return go<T, 4, 2>(p, stream);
  if (p.S <= 16) return go<T, 4, 4>(p, stream);
  if (p.S <= 32) return go<T, 8, 4>(p, stream);
  if (p.S <= 64) return go<T, 8, 8>(p, stream);
  if (p.S <= 128) return go<T, 16, 8>(p, stream);
  return go<T, 16, 16>(p, stream);
}

}  // namespace

long long selective_scan_workspace(int dtype, const ScanParams& p) {
  (void)dtype;
  const long long ends = (long long)p.N * (cut_of(p).chunks - 1) * p.C;
  return 4 * ends * (p.S + 1);
}

cudaError_t launch_selective_scan(int dtype, const ScanParams& p, cudaStream_t stream) {
  switch (dtype) {
    case FDNN_F16: return scan<__half>(p, stream);
    case FDNN_BF16: return scan<__nv_bfloat16>(p, stream);
    default: return scan<float>(p, stream);
  }
}

}  // namespace fdnn
