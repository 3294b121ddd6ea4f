// The short causal convolution in front of a state space scan, over prompts and for single tokens.
//
//   y[t] = act(b + sum_j w[j] xs[t + j]),  xs = the width - 1 inputs before the first token, then x
//
// Tokens lie one after another with their channels together ([N, L, C], as a product of tokens with a weight matrix leaves
// them); the state between calls is the last width - 1 inputs, [N, width - 1, C].
#include "sequence_internal.h"
#include "sequence_launch.h"
#include "sequence_math.cuh"

namespace fdnn {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ int length_of(const int* lengths, int n, int L) {
  return lengths == nullptr ? L : min(max(lengths[n], 0), L);
}

// Input number i of a row, counted from the first of the state.
template <typename T>
__device__ __forceinline__ T input_at(const CausalConvParams& p, int n, int i, int c) {
  const int before = p.width - 1;
  if (i >= before) return static_cast<const T*>(p.x)[n * p.x_s[0] + (i - before) * p.x_s[1] + c * p.x_s[2]];
  if (p.initial == nullptr) return from_f32<T>(0.0f);
  return static_cast<const T*>(p.initial)[((long long)n * before + i) * p.C + c];
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
causal_conv_kernel(const CausalConvParams p) {
  chained();
  const T* w = static_cast<const T*>(p.weight);
  const long long total = (long long)p.N * p.L * p.C;
  for (long long i = blockIdx.x * (long long)kThreads + threadIdx.x; i < total; i += (long long)gridDim.x * kThreads) {
    const int c = int(i % p.C);
    const long long nt = i / p.C;
    const int t = int(nt % p.L), n = int(nt / p.L);
    T* y = static_cast<T*>(p.y) + n * p.y_s[0] + t * p.y_s[1] + c * p.y_s[2];
    if (t >= length_of(p.lengths, n, p.L)) {
      *y = from_f32<T>(0.0f);
      continue;
    }
    float v = p.bias != nullptr ? to_f32<T>(static_cast<const T*>(p.bias)[c]) : 0.0f;
    for (int j = 0; j < p.width; ++j)
      v += to_f32<T>(w[(long long)c * p.width + j]) * to_f32<T>(input_at<T>(p, n, t + j, c));
    with_activation(p.act, [&](auto act) { *y = from_f32<T>(activate<decltype(act)::value>(v)); });
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
causal_conv_state_kernel(const CausalConvParams p) {
  chained();
  const int before = p.width - 1;
  const long long total = (long long)p.N * before * p.C;
  for (long long i = blockIdx.x * (long long)kThreads + threadIdx.x; i < total; i += (long long)gridDim.x * kThreads) {
    const int c = int(i % p.C);
    const int j = int(i / p.C % before), n = int(i / p.C / before);
    static_cast<T*>(p.final_state)[i] = input_at<T>(p, n, length_of(p.lengths, n, p.L) + j, c);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
causal_conv_step_kernel(const CausalConvParams p, T* state, int n_slots, const int* slots) {
  chained();
  const int before = p.width - 1;
  const T* w = static_cast<const T*>(p.weight);
  const long long total = (long long)p.N * p.C;
  for (long long i = blockIdx.x * (long long)kThreads + threadIdx.x; i < total; i += (long long)gridDim.x * kThreads) {
    const int c = int(i % p.C), n = int(i / p.C);
    T* y = static_cast<T*>(p.y) + n * p.y_s[0] + c * p.y_s[2];
    const int slot = slots != nullptr ? slots[n] : n;
    if (slot < 0 || slot >= n_slots) {
      *y = from_f32<T>(0.0f);
      continue;
    }
    T* st = state + (long long)slot * before * p.C + c;
    const T x = static_cast<const T*>(p.x)[n * p.x_s[0] + c * p.x_s[2]];
    float v = p.bias != nullptr ? to_f32<T>(static_cast<const T*>(p.bias)[c]) : 0.0f;
    for (int j = 0; j < before; ++j) {
      const T old = st[(long long)j * p.C];
      v += to_f32<T>(w[(long long)c * p.width + j]) * to_f32<T>(old);
      if (j > 0) st[(long long)(j - 1) * p.C] = old;
    }
    if (before > 0) st[(long long)(before - 1) * p.C] = x;
    v += to_f32<T>(w[(long long)c * p.width + before]) * to_f32<T>(x);
    with_activation(p.act, [&](auto act) { *y = from_f32<T>(activate<decltype(act)::value>(v)); });
  }
}

unsigned grid_of(long long values) {
  const long long blocks = (values + kThreads - 1) / kThreads;
  return unsigned(blocks < (1ll << 30) ? blocks : (1ll << 30));
}

template <typename T>
cudaError_t go(const CausalConvParams& p, cudaStream_t stream) {
  cudaError_t e = cudaSuccess;
  if (p.L > 0) e = launch_seq(causal_conv_kernel<T>, dim3(grid_of((long long)p.N * p.L * p.C)), kThreads, 0, 1, stream, p);
  if (e != cudaSuccess || p.final_state == nullptr || p.width == 1) return e;
  return launch_seq(causal_conv_state_kernel<T>, dim3(grid_of((long long)p.N * (p.width - 1) * p.C)), kThreads, 0, 1, stream, p);
}

template <typename T>
cudaError_t step(const CausalConvParams& p, void* state, int n_slots, const int* slots, cudaStream_t stream) {
  return launch_seq(causal_conv_step_kernel<T>, dim3(grid_of((long long)p.N * p.C)), kThreads, 0, 1, stream, p,
                    static_cast<T*>(state), n_slots, slots);
}

}  // namespace

cudaError_t launch_causal_conv(int dtype, const CausalConvParams& p, cudaStream_t stream) {
  switch (dtype) {
    case FDNN_F16: return go<__half>(p, stream);
    case FDNN_BF16: return go<__nv_bfloat16>(p, stream);
    default: return go<float>(p, stream);
  }
}

cudaError_t launch_causal_conv_step(int dtype, const CausalConvParams& p, void* state, int n_slots, const int* slots,
                                    cudaStream_t stream) {
  switch (dtype) {
    case FDNN_F16: return step<__half>(p, state, n_slots, slots, stream);
    case FDNN_BF16: return step<__nv_bfloat16>(p, state, n_slots, slots, stream);
    default: return step<float>(p, state, n_slots, slots, stream);
  }
}

}  // namespace fdnn
