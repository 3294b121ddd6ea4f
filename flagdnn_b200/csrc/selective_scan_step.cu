// The selective state space scan for single tokens: one step of h = exp(dt A) h + dt u B for each row, its state in place.
//
// Bound by memory: a state is read and written, everything else is small beside it.  16 states of a channel are four lanes' 16
// bytes, so that a warp moves 512 contiguous bytes; a thread keeps its channel's A and walks several rows, with the states of
// the next rows on their way.
#include "sequence_internal.h"
#include "sequence_launch.h"
#include "sequence_math.cuh"

namespace fdnn {
namespace {

constexpr int kThreads = 128;

// Four neighbouring values, those past `count` zero.
template <typename T>
__device__ __forceinline__ float4 four(const T* p, long long stride, int count) {
  float4 v;
  v.x = count > 0 ? to_f32<T>(p[0]) : 0.0f;
  v.y = count > 1 ? to_f32<T>(p[stride]) : 0.0f;
  v.z = count > 2 ? to_f32<T>(p[2 * stride]) : 0.0f;
  v.w = count > 3 ? to_f32<T>(p[3 * stride]) : 0.0f;
  return v;
}
template <bool WHOLE>
__device__ __forceinline__ float4 four_states(const float* p, int count) {
  if constexpr (WHOLE) return *reinterpret_cast<const float4*>(p);
  else return four<float>(p, 1, count);
}

// LANES threads share a channel, four states each and as often as S needs (more than 128 states: CHUNKS of them).  WHOLE: S is
// a multiple of four and so are all addresses.
template <typename T, int LANES, int CHUNKS, bool WHOLE, int ROWS>
__global__ void __launch_bounds__(kThreads)
scan_step_kernel(const ScanParams p, float* state, int n_slots, const int* slots) {
  chained();
  const long long slot_of_thread = blockIdx.x * (long long)kThreads + threadIdx.x;
  const int c = int(slot_of_thread / LANES), part = int(slot_of_thread % LANES);
  const bool live = c < p.C;
  const int cc = live ? c : 0;
  const int g = cc / (p.C / p.G);
  float4 a[CHUNKS];
#pragma unroll
  for (int k = 0; k < CHUNKS; ++k) {
    const int s = (k * LANES + part) * 4;
    a[k] = s < p.S ? four_states<WHOLE>(p.A + (long long)cc * p.S + s, p.S - s) : make_float4(0, 0, 0, 0);
    a[k].x *= kLog2e; a[k].y *= kLog2e; a[k].z *= kLog2e; a[k].w *= kLog2e;
  }
  const float D = p.D != nullptr ? p.D[cc] : 0.0f, bias = p.delta_bias != nullptr ? p.delta_bias[cc] : 0.0f;
  for (int n0 = blockIdx.y * ROWS; n0 < p.N; n0 += gridDim.y * ROWS) {
    float4 h[ROWS][CHUNKS], b[ROWS][CHUNKS], m[ROWS][CHUNKS];
    float u[ROWS], dt[ROWS], z[ROWS];
    float* at[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int n = n0 + r;
      const int slot = n < p.N ? (slots != nullptr ? slots[n] : n) : -1;
      at[r] = live && slot >= 0 && slot < n_slots ? state + ((long long)slot * p.C + cc) * p.S : nullptr;
      u[r] = dt[r] = z[r] = 0.0f;
#pragma unroll
      for (int k = 0; k < CHUNKS; ++k) {
        const int s = (k * LANES + part) * 4;
        h[r][k] = b[r][k] = m[r][k] = make_float4(0, 0, 0, 0);
        if (at[r] != nullptr && s < p.S) {
          h[r][k] = four_states<WHOLE>(at[r] + s, p.S - s);
          b[r][k] = four<T>(static_cast<const T*>(p.B) + n * p.b_s[0] + g * p.b_s[2] + s * p.b_s[3], p.b_s[3], p.S - s);
          m[r][k] = four<T>(static_cast<const T*>(p.Cm) + n * p.c_s[0] + g * p.c_s[2] + s * p.c_s[3], p.c_s[3], p.S - s);
        }
      }
      if (at[r] != nullptr) {
        u[r] = to_f32<T>(static_cast<const T*>(p.u)[n * p.u_s[0] + cc * p.u_s[2]]);
        dt[r] = to_f32<T>(static_cast<const T*>(p.delta)[n * p.delta_s[0] + cc * p.delta_s[2]]) + bias;
        if (p.z != nullptr) z[r] = to_f32<T>(static_cast<const T*>(p.z)[n * p.z_s[0] + cc * p.z_s[2]]);
      }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int n = n0 + r;
      const float d = p.softplus ? softplus(dt[r]) : dt[r], du = d * u[r];
      float y = 0.0f;
#pragma unroll
      for (int k = 0; k < CHUNKS; ++k) {
        const int s = (k * LANES + part) * 4;
        float4 v;
        v.x = h[r][k].x * ex2(d * a[k].x) + du * b[r][k].x;
        v.y = h[r][k].y * ex2(d * a[k].y) + du * b[r][k].y;
        v.z = h[r][k].z * ex2(d * a[k].z) + du * b[r][k].z;
        v.w = h[r][k].w * ex2(d * a[k].w) + du * b[r][k].w;
        // (states past S: b and m are zero, but zero times an infinite du is not)
        y += (s < p.S ? v.x * m[r][k].x : 0.0f) + (s + 1 < p.S ? v.y * m[r][k].y : 0.0f) + (s + 2 < p.S ? v.z * m[r][k].z : 0.0f) +
             (s + 3 < p.S ? v.w * m[r][k].w : 0.0f);
        if (at[r] != nullptr && s < p.S) {
          if constexpr (WHOLE) {
            *reinterpret_cast<float4*>(at[r] + s) = v;
          } else {
            at[r][s] = v.x;
            if (s + 1 < p.S) at[r][s + 1] = v.y;
            if (s + 2 < p.S) at[r][s + 2] = v.z;
            if (s + 3 < p.S) at[r][s + 3] = v.w;
          }
        }
      }
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
      if (live && part == 0 && n < p.N) {
        y += D * u[r];
        if (p.z != nullptr) y *= silu(z[r]);
        static_cast<T*>(p.y)[n * p.y_s[0] + c * p.y_s[2]] = from_f32<T>(at[r] != nullptr ? y : 0.0f);
      }
    }
  }
}

template <typename T, int LANES, int CHUNKS>
cudaError_t go(const ScanParams& p, float* state, int n_slots, const int* slots, cudaStream_t stream) {
  constexpr int kRows = CHUNKS == 1 ? 2 : 1;
  const long long blocks = ((long long)p.C * LANES + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  // about sixteen blocks an SM; rows beyond them are walked
  long long slices = (p.N + kRows - 1) / kRows, room = 16ll * current_sm_count() / blocks;
  if (room < 1) room = 1;
  if (slices > room) slices = room;
  if (slices > 65535) slices = 65535;
  auto even = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; };
  const bool whole = p.S % 4 == 0 && even(state) && even(p.A);
  auto* kernel = whole ? scan_step_kernel<T, LANES, CHUNKS, true, kRows> : scan_step_kernel<T, LANES, CHUNKS, false, kRows>;
  return launch_seq(kernel, dim3(unsigned(blocks), unsigned(slices)), kThreads, 0, 1, stream, p, state, n_slots, slots);
}

template <typename T>
cudaError_t step(const ScanParams& p, float* state, int n_slots, const int* slots, cudaStream_t stream) {
  if (p.S <= 4) return go<T, 1, 1>(p, state, n_slots, slots, stream);
  if (p.S <= 8) return go<T, 2, 1>(p, state, n_slots, slots, stream);
  if (p.S <= 16) return go<T, 4, 1>(p, state, n_slots, slots, stream);
  if (p.S <= 32) return go<T, 8, 1>(p, state, n_slots, slots, stream);
  if (p.S <= 64) return go<T, 16, 1>(p, state, n_slots, slots, stream);
  if (p.S <= 128) return go<T, 32, 1>(p, state, n_slots, slots, stream);
  return go<T, 32, 2>(p, state, n_slots, slots, stream);
}

}  // namespace

cudaError_t launch_selective_scan_step(int dtype, const ScanParams& p, float* state, int n_slots, const int* slots,
                                       cudaStream_t stream) {
  switch (dtype) {
    case FDNN_F16: return step<__half>(p, state, n_slots, slots, stream);
    case FDNN_BF16: return step<__nv_bfloat16>(p, state, n_slots, slots, stream);
    default: return step<float>(p, state, n_slots, slots, stream);
  }
}

}  // namespace fdnn
