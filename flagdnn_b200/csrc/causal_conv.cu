// The short causal convolution in front of a state space scan, over prompts and for single tokens.
//
//   y[t] = act(b + sum_j w[j] xs[t + j]),  xs = the width - 1 inputs before the first token, then x
//
// Tokens lie one after another with their channels together ([N, L, C], as a product of tokens with a weight matrix leaves
// them); the state between calls is the last width - 1 inputs, [N, width - 1, C].
//
// Bound by memory, short of it by latencies: the registers of a thread (128) leave 13 warps to an SM, which fill 53 % of its issue
// slots. A thread takes a vector of 16 bytes of channels and walks a run of tokens, four at a time: the width - 1 before
// them are still in its registers, and every value is widened to fp32 once. The next twelve tokens' vectors are on their way
// into slots of shared memory that are the thread's own. What a run reads of its predecessor's tokens is in the cache.
// 4 x 2048 x 4096 bf16 with silu: 34.1 us, 3.9 TB/s.
#include "group_norm.cuh"

namespace fdnn {
namespace {

constexpr int kThreads = 256, kLanes = 32;      // a block: 32 vectors of channels x 8 runs
constexpr int kStep = 4, kAhead = 3;            // tokens at a time, and how many times that is on its way

__device__ __forceinline__ int length_of(const int* lengths, int n, int L) {
  return lengths == nullptr ? L : min(max(lengths[n], 0), L);
}

struct ConvJob {
  CausalConvParams p;
  int vectors;           // of a token's channels
  int run, runs;         // tokens of a run, runs of a row (one more for the final state)
  long long items;       // runs of all rows
};

// Input number i of a row's vector of channels, counted from the first of the state.
template <typename T, int V, int W>
__device__ __forceinline__ Pack<T, V> input_at(const CausalConvParams& p, int n, int i, int c) {
  Pack<T, V> v;
  v.clear();
  if (i >= W - 1) {
    const T* from = static_cast<const T*>(p.x) + n * p.x_s[0] + (long long)(i - (W - 1)) * p.x_s[1] + c * p.x_s[2];
    v.load(from);
  } else if (p.initial != nullptr) {
    v.load(static_cast<const T*>(p.initial) + ((long long)n * (W - 1) + i) * p.C + c);
  }
  return v;
}

// The filter and bias of a vector of channels as pairs.
template <typename T, int V, int W>
__device__ __forceinline__ void taps_of(const CausalConvParams& p, int c, F2 (&w)[W][Pack<T, V>::kPairs], F2 (&b)[Pack<T, V>::kPairs]) {
  const T* from = static_cast<const T*>(p.weight) + (long long)c * W;
  Pack<T, V> raw[W];                            // [V][W] values
#pragma unroll
  for (int k = 0; k < W; ++k) raw[k].load(from + k * V);
#pragma unroll
  for (int i = 0; i < Pack<T, V>::kPairs; ++i) {
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const int e0 = 2 * i * W + j, e1 = V == 1 ? e0 : (2 * i + 1) * W + j;
      w[j][i] = f2_pack(raw[e0 / V].at(e0 % V), raw[e1 / V].at(e1 % V));
    }
  }
  Pack<T, V> bias;
  bias.clear();
  if (p.bias != nullptr) bias.load(static_cast<const T*>(p.bias) + c);
#pragma unroll
  for (int i = 0; i < Pack<T, V>::kPairs; ++i) b[i] = bias.pair(i);
}

template <typename T, int V, int W>
__global__ void __launch_bounds__(kThreads, 2)
causal_conv_kernel(const ConvJob job) {
  extern __shared__ __align__(16) unsigned char raw[];
  chained();
  const CausalConvParams& p = job.p;
  constexpr int P = Pack<T, V>::kPairs;
  const int tiles = (job.vectors + kLanes - 1) / kLanes;
  const int vec = int(blockIdx.x % unsigned(tiles)) * kLanes + int(threadIdx.x) % kLanes;
  const long long item = (long long)(blockIdx.x / unsigned(tiles)) * (kThreads / kLanes) + threadIdx.x / kLanes;
  if (vec >= job.vectors || item >= job.items) return;
  const int c = vec * V, n = int(item / job.runs), run = int(item % job.runs);
  const int len = length_of(p.lengths, n, p.L), t0 = run * job.run;
  if (t0 >= p.L) {                              // the row's last run: the state after it
    if (p.final_state == nullptr || run != job.runs - 1) return;
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
      input_at<T, V, W>(p, n, len + j, c).store(static_cast<T*>(p.final_state) + ((long long)n * (W - 1) + j) * p.C + c);
    return;
  }
  const int t1 = min(t0 + job.run, p.L), te = min(t1, len);
  T* y = static_cast<T*>(p.y) + n * p.y_s[0] + c * p.y_s[2];
  if (te > t0) {
    F2 w[W][P], b[P];
    taps_of<T, V, W>(p, c, w, b);
    Pack<T, V> x[W - 1 + kStep];
    const T* from = static_cast<const T*>(p.x) + n * p.x_s[0] + c * p.x_s[2];
    Pack<T, V>* slot = reinterpret_cast<Pack<T, V>*>(raw) + threadIdx.x;   // this thread's, kThreads apart
    auto ask = [&](int t, int at) {
#pragma unroll
      for (int q = 0; q < kStep; ++q)
        async_load(slot + (at + q) * kThreads, from + (t + q < te ? (long long)(t + q) * p.x_s[1] : 0), t + q < te);
      async_commit();
    };
#pragma unroll
    for (int k = 0; k < kAhead; ++k) ask(t0 + k * kStep, k * kStep);
#pragma unroll
    for (int j = 0; j < W - 1; ++j) x[j] = input_at<T, V, W>(p, n, t0 + j, c);
    int at = 0;
    with_activation(p.act, [&](auto act) {
      for (int t = t0; t < te; t += kStep) {
        async_wait<kAhead - 1>();
#pragma unroll
        for (int q = 0; q < kStep; ++q) x[W - 1 + q] = slot[(at + q) * kThreads];
        ask(t + kAhead * kStep, at);
        at = at == (kAhead - 1) * kStep ? 0 : at + kStep;
        Pack<T, V> out[kStep];
#pragma unroll
        for (int i = 0; i < P; ++i) {
          F2 f[W - 1 + kStep];
#pragma unroll
          for (int j = 0; j < W - 1 + kStep; ++j) f[j] = x[j].pair(i);
#pragma unroll
          for (int q = 0; q < kStep; ++q) {
            F2 v = b[i];
#pragma unroll
            for (int j = 0; j < W; ++j) v = f2_fma(w[j][i], f[q + j], v);
            out[q].set_pair(i, activate2<decltype(act)::value>(v));
          }
        }
#pragma unroll
        for (int q = 0; q < kStep; ++q)
          if (t + q < te) out[q].store(y + (long long)(t + q) * p.y_s[1]);
#pragma unroll
        for (int j = 0; j < W - 1; ++j) x[j] = x[kStep + j];
      }
    });
  }
  Pack<T, V> zero;
  zero.clear();
  for (int t = max(t0, te); t < t1; ++t) zero.store(y + (long long)t * p.y_s[1]);   // padding
}

// One token of each row: its state moves on by one input.
template <typename T, int V, int W>
__global__ void __launch_bounds__(kThreads)
causal_conv_step_kernel(const ConvJob job, T* state, int n_slots, const int* slots) {
  chained();
  const CausalConvParams& p = job.p;
  constexpr int P = Pack<T, V>::kPairs;
  const long long i0 = blockIdx.x * (long long)kThreads + threadIdx.x;
  if (i0 >= job.items) return;
  const int c = int(i0 % job.vectors) * V, n = int(i0 / job.vectors);
  T* y = static_cast<T*>(p.y) + n * p.y_s[0] + c * p.y_s[2];
  const int slot = slots != nullptr ? slots[n] : n;
  Pack<T, V> out;
  if (slot < 0 || slot >= n_slots) {
    out.clear();
    out.store(y);
    return;
  }
  T* st = state + (long long)slot * (W - 1) * p.C + c;
  Pack<T, V> x[W];
#pragma unroll
  for (int j = 0; j < W - 1; ++j) x[j].q = *reinterpret_cast<const typename Pack<T, V>::Word*>(st + (long long)j * p.C);
  x[W - 1].load(static_cast<const T*>(p.x) + n * p.x_s[0] + c * p.x_s[2]);
  F2 w[W][P], b[P];
  taps_of<T, V, W>(p, c, w, b);
#pragma unroll
  for (int j = 0; j < W - 1; ++j) x[j + 1].store(st + (long long)j * p.C);
  with_activation(p.act, [&](auto act) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      F2 v = b[i];
#pragma unroll
      for (int j = 0; j < W; ++j) v = f2_fma(w[j][i], x[j].pair(i), v);
      out.set_pair(i, activate2<decltype(act)::value>(v));
    }
  });
  out.store(y);
}

// Whether vectors of 16 bytes can be used: channels dense and whole numbers of them, every address a multiple.
template <typename T>
bool by_vectors(const CausalConvParams& p, const void* state, bool step) {
  constexpr int V = 16 / int(sizeof(T));
  const void* q[] = {p.x, p.y, p.weight, p.bias, p.initial, p.final_state, state};
  for (const void* a : q)
    if ((reinterpret_cast<uintptr_t>(a) & 15u) != 0) return false;
  const bool tokens = step || p.L <= 1 || (p.x_s[1] % V == 0 && p.y_s[1] % V == 0);
  return p.C % V == 0 && p.x_s[2] == 1 && p.y_s[2] == 1 && (p.N == 1 || (p.x_s[0] % V == 0 && p.y_s[0] % V == 0)) && tokens;
}

template <typename T, int V, int W>
cudaError_t go(const CausalConvParams& p, cudaStream_t stream) {
  ConvJob job;
  job.p = p;
  job.vectors = p.C / V;
  const int tiles = (job.vectors + kLanes - 1) / kLanes;
  // runs of 32 tokens (the 3 before one are read again); shorter where that leaves SMs idle
  job.run = 32;
  while (job.run > 8 && (long long)p.N * ((p.L + job.run - 1) / job.run) * tiles < 16ll * current_sm_count()) job.run /= 2;
  job.runs = p.L / job.run + (p.L % job.run != 0) + (p.final_state != nullptr && W > 1 ? 1 : 0);
  job.items = (long long)p.N * job.runs;
  if (job.items == 0) return cudaSuccess;
  const long long blocks = (job.items + kThreads / kLanes - 1) / (kThreads / kLanes) * tiles;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  return launch_seq(causal_conv_kernel<T, V, W>, dim3(unsigned(blocks)), kThreads, kAhead * kStep * kThreads * Pack<T, V>::kBytes, 1, stream,
                    job);
}

template <typename T, int V, int W>
cudaError_t step(const CausalConvParams& p, void* state, int n_slots, const int* slots, cudaStream_t stream) {
  ConvJob job;
  job.p = p;
  job.vectors = p.C / V;
  job.run = job.runs = 1;
  job.items = (long long)p.N * job.vectors;
  const long long blocks = (job.items + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  return launch_seq(causal_conv_step_kernel<T, V, W>, dim3(unsigned(blocks)), kThreads, 0, 1, stream, job, static_cast<T*>(state), n_slots, slots);
}

// f(TypeOf<T>, V, W) for a run-time type, vector and filter width.
template <typename F>
cudaError_t by_width(int width, F&& f) {
  switch (width) {
    case 1: return f(std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 2>{});
    case 3: return f(std::integral_constant<int, 3>{});
    case 4: return f(std::integral_constant<int, 4>{});
    case 5: return f(std::integral_constant<int, 5>{});
    case 6: return f(std::integral_constant<int, 6>{});
    case 7: return f(std::integral_constant<int, 7>{});
    default: return f(std::integral_constant<int, 8>{});
  }
}
template <typename F>
cudaError_t by_type(int dtype, F&& f) {
  if (dtype == FDNN_F16) return f(TypeOf<__half>{});
  if (dtype == FDNN_BF16) return f(TypeOf<__nv_bfloat16>{});
  return f(TypeOf<float>{});
}

}  // namespace

cudaError_t launch_causal_conv(int dtype, const CausalConvParams& p, cudaStream_t stream) {
  return by_type(dtype, [&](auto type) {
    using T = typename decltype(type)::type;
    return by_width(p.width, [&](auto w) {
      constexpr int W = decltype(w)::value, V = 16 / int(sizeof(T));
      return by_vectors<T>(p, nullptr, false) ? go<T, V, W>(p, stream) : go<T, 1, W>(p, stream);
    });
  });
}

cudaError_t launch_causal_conv_step(int dtype, const CausalConvParams& p, void* state, int n_slots, const int* slots,
                                    cudaStream_t stream) {
  return by_type(dtype, [&](auto type) {
    using T = typename decltype(type)::type;
    return by_width(p.width, [&](auto w) {
      constexpr int W = decltype(w)::value, V = 16 / int(sizeof(T));
      return by_vectors<T>(p, state, true) ? step<T, V, W>(p, state, n_slots, slots, stream) : step<T, 1, W>(p, state, n_slots, slots, stream);
    });
  });
}

}  // namespace fdnn
