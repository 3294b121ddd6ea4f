// The selective state space scan over prompts and for single tokens.
//
//   dt = delta + delta_bias, softplus of it if asked
//   h_t = exp(dt A) h_(t-1) + dt u_t B_t,  y_t = (sum over the states of C_t h_t + D u_t) silu(z_t)
//
// per channel, with a decay rate of its own for each of its S states; B_t and C_t are shared by the channels of a group.
// The states are fp32 throughout.
#include "sequence_internal.h"
#include "sequence_launch.h"
#include "sequence_math.cuh"

namespace fdnn {
namespace {

constexpr int kThreads = 128;

__device__ __forceinline__ int length_of(const int* lengths, int n, int L) {
  return lengths == nullptr ? L : min(max(lengths[n], 0), L);
}

// LANES threads share a channel, NPT states each; states past S are zeros.
template <typename T, int NPT, int LANES>
__global__ void __launch_bounds__(kThreads)
scan_kernel(const ScanParams p) {
  chained();
  const int c = int((blockIdx.x * (long long)kThreads + threadIdx.x) / LANES), n = blockIdx.y;
  const int part = threadIdx.x % LANES, s0 = part * NPT;
  const bool live = c < p.C;
  const int cc = live ? c : 0;
  const int g = cc / (p.C / p.G);
  const int len = length_of(p.lengths, n, p.L);
  float a[NPT], h[NPT];
#pragma unroll
  for (int s = 0; s < NPT; ++s) {
    const bool in = s0 + s < p.S;
    a[s] = in ? p.A[(long long)cc * p.S + s0 + s] * kLog2e : 0.0f;
    h[s] = in && p.initial != nullptr ? p.initial[((long long)n * p.C + cc) * p.S + s0 + s] : 0.0f;
  }
  const float D = p.D != nullptr ? p.D[cc] : 0.0f, bias = p.delta_bias != nullptr ? p.delta_bias[cc] : 0.0f;
  for (int t = 0; t < len; ++t) {
    const float u = to_f32<T>(static_cast<const T*>(p.u)[n * p.u_s[0] + t * p.u_s[1] + cc * p.u_s[2]]);
    float dt = to_f32<T>(static_cast<const T*>(p.delta)[n * p.delta_s[0] + t * p.delta_s[1] + cc * p.delta_s[2]]) + bias;
    if (p.softplus) dt = softplus(dt);
    const T* B = static_cast<const T*>(p.B) + n * p.b_s[0] + t * p.b_s[1] + g * p.b_s[2];
    const T* Cm = static_cast<const T*>(p.Cm) + n * p.c_s[0] + t * p.c_s[1] + g * p.c_s[2];
    const float du = dt * u;
    float y = 0.0f;
#pragma unroll
    for (int s = 0; s < NPT; ++s)
      if (s0 + s < p.S) {
        h[s] = h[s] * ex2(dt * a[s]) + du * to_f32<T>(B[(s0 + s) * p.b_s[3]]);
        y += h[s] * to_f32<T>(Cm[(s0 + s) * p.c_s[3]]);
      }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
    if (live && part == 0) {
      y += D * u;
      if (p.z != nullptr) y *= silu(to_f32<T>(static_cast<const T*>(p.z)[n * p.z_s[0] + t * p.z_s[1] + c * p.z_s[2]]));
      static_cast<T*>(p.y)[n * p.y_s[0] + t * p.y_s[1] + c * p.y_s[2]] = from_f32<T>(y);
    }
  }
  if (!live) return;
  if (part == 0)
    for (int t = len; t < p.L; ++t) static_cast<T*>(p.y)[n * p.y_s[0] + t * p.y_s[1] + c * p.y_s[2]] = from_f32<T>(0.0f);
  if (p.final_state != nullptr)
#pragma unroll
    for (int s = 0; s < NPT; ++s)
      if (s0 + s < p.S) p.final_state[((long long)n * p.C + c) * p.S + s0 + s] = h[s];
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
scan_step_kernel(const ScanParams p, float* state, int n_slots, const int* slots) {
  chained();
  const long long total = (long long)p.N * p.C;
  for (long long i = blockIdx.x * (long long)kThreads + threadIdx.x; i < total; i += (long long)gridDim.x * kThreads) {
    const int c = int(i % p.C), n = int(i / p.C), g = c / (p.C / p.G);
    T* out = static_cast<T*>(p.y) + n * p.y_s[0] + c * p.y_s[2];
    const int slot = slots != nullptr ? slots[n] : n;
    if (slot < 0 || slot >= n_slots) {
      *out = from_f32<T>(0.0f);
      continue;
    }
    const float u = to_f32<T>(static_cast<const T*>(p.u)[n * p.u_s[0] + c * p.u_s[2]]);
    float dt = to_f32<T>(static_cast<const T*>(p.delta)[n * p.delta_s[0] + c * p.delta_s[2]]);
    if (p.delta_bias != nullptr) dt += p.delta_bias[c];
    if (p.softplus) dt = softplus(dt);
    const T* B = static_cast<const T*>(p.B) + n * p.b_s[0] + g * p.b_s[2];
    const T* Cm = static_cast<const T*>(p.Cm) + n * p.c_s[0] + g * p.c_s[2];
    float* h = state + ((long long)slot * p.C + c) * p.S;
    float y = 0.0f;
    for (int s = 0; s < p.S; ++s) {
      const float v = h[s] * ex2(dt * kLog2e * p.A[(long long)c * p.S + s]) + dt * u * to_f32<T>(B[s * p.b_s[3]]);
      h[s] = v;
      y += v * to_f32<T>(Cm[s * p.c_s[3]]);
    }
    if (p.D != nullptr) y += p.D[c] * u;
    if (p.z != nullptr) y *= silu(to_f32<T>(static_cast<const T*>(p.z)[n * p.z_s[0] + c * p.z_s[2]]));
    *out = from_f32<T>(y);
  }
}

template <typename T, int NPT, int LANES>
cudaError_t go(const ScanParams& p, cudaStream_t stream) {
  const long long threads = (long long)p.C * LANES;
  return launch_seq(scan_kernel<T, NPT, LANES>, dim3(unsigned((threads + kThreads - 1) / kThreads), unsigned(p.N)), kThreads, 0, 1,
                    stream, p);
}

template <typename T>
cudaError_t scan(const ScanParams& p, cudaStream_t stream) {
  if (p.S <= 4) return go<T, 4, 1>(p, stream);
  if (p.S <= 8) return go<T, 8, 1>(p, stream);
  if (p.S <= 16) return go<T, 16, 1>(p, stream);
  if (p.S <= 32) return go<T, 16, 2>(p, stream);
  if (p.S <= 64) return go<T, 16, 4>(p, stream);
  if (p.S <= 128) return go<T, 16, 8>(p, stream);
  return go<T, 16, 16>(p, stream);
}

template <typename T>
cudaError_t step(const ScanParams& p, float* state, int n_slots, const int* slots, cudaStream_t stream) {
  const long long blocks = ((long long)p.N * p.C + kThreads - 1) / kThreads;
  return launch_seq(scan_step_kernel<T>, dim3(unsigned(blocks < (1ll << 30) ? blocks : (1ll << 30))), kThreads, 0, 1, stream, p,
                    state, n_slots, slots);
}

}  // namespace

long long selective_scan_workspace(int dtype, const ScanParams& p) {
  (void)dtype;
  (void)p;
  return 0;
}

cudaError_t launch_selective_scan(int dtype, const ScanParams& p, cudaStream_t stream) {
  switch (dtype) {
    case FDNN_F16: return scan<__half>(p, stream);
    case FDNN_BF16: return scan<__nv_bfloat16>(p, stream);
    default: return scan<float>(p, stream);
  }
}

cudaError_t launch_selective_scan_step(int dtype, const ScanParams& p, float* state, int n_slots, const int* slots,
                                       cudaStream_t stream) {
  switch (dtype) {
    case FDNN_F16: return step<__half>(p, state, n_slots, slots, stream);
    case FDNN_BF16: return step<__nv_bfloat16>(p, state, n_slots, slots, stream);
    default: return step<float>(p, state, n_slots, slots, stream);
  }
}

}  // namespace fdnn
