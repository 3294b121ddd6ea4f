// Activations, their slopes and small reductions shared by the group norm and state space kernels.  All in fp32.
#pragma once
#include <math.h>

#include <type_traits>

#include "../../include/flagdnn_b200.h"
#include "conv_convert.cuh"
#include "f32x2.cuh"
#include "sm100_ptx.cuh"

namespace fdnn {

constexpr float kLog2e = 1.4426950408889634f;

// 2^v by the special function unit (relative error 2^-22, subnormal results flushed)
__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// A step's decay e^(dt A), for a = A log2 e.  The unit cuts its argument and its result downwards: between -0.1 and 0 the mean error
// is -1.2e-8 to -2.3e-8 of the decay, which a state that forgets slowly adds up over hundreds of steps (-1.8e-6 of it after 300).
// An argument larger by kDecayMiddle has a mean error within 1e-8 of zero there; 2^kDecayMiddle is 1, so a step of no time leaves a
// state as it is.
constexpr float kDecayMiddle = 2.5e-8f;
// (A as decay_of takes it. Minus infinity becomes the lowest number: e^(dt A) is zero all the same, but for a step of no time, which past
// a row's end stands for no step and would make the state NaN.)
__device__ __forceinline__ float rate_of(float A) {
  float a;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(A * kLog2e), "f"(-3.402823466e38f));   // (NaN stays)
  return a;
}
__device__ __forceinline__ float decay_of(float dt, float a) { return ex2(fmaf(dt, a, kDecayMiddle)); }
// 1 / v by the special function unit (one unit in the last place)
__device__ __forceinline__ float rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// 1 / (1 + e^-v): the denominator is infinite below -88, whose reciprocal is zero
__device__ __forceinline__ float logistic(float v) { return rcp(1.0f + ex2(-kLog2e * v)); }
__device__ __forceinline__ float silu(float v) { return v * logistic(v); }
// log(1 + e^v) = max(v, 0) + log(1 + e), e = e^-|v| at most 1.  log(1 + e) / e is a polynomial of degree 9, fitted to the
// smallest relative error on [0, 1] (4.8e-8 with these fp32 coefficients; 1.3e-7 in fp32 arithmetic): no result is lost where e is small, and no second call of
// the special function unit, which bounds the scan.
__device__ __forceinline__ float softplus(float v) {
  const float e = ex2(-kLog2e * fabsf(v));
  float p = -0.0032440070062875748f;
  p = fmaf(p, e, 0.019851384684443474f);
  p = fmaf(p, e, -0.056959398090839386f);
  p = fmaf(p, e, 0.10603642463684082f);
  p = fmaf(p, e, -0.15305586159229279f);
  p = fmaf(p, e, 0.19675937294960022f);
  p = fmaf(p, e, -0.24954132735729218f);
  p = fmaf(p, e, 0.3332996368408203f);
  p = fmaf(p, e, -0.4999990165233612f);
  p = fmaf(p, e, 1.0f);
  return fmaf(p, e, fmaxf(v, 0.0f));   // NaN stays: e is NaN then
}

constexpr float kSqrtHalf = 0.70710678118654752f;
constexpr float kGeluTanhScale = 0.79788456080286536f;   // sqrt(2 / pi)
constexpr float kGeluTanhCubic = 0.044715f;

template <int ACT>
__device__ __forceinline__ float activate(float v) {
  if constexpr (ACT == FDNN_ACT_RELU) return v < 0.0f ? 0.0f : v;   // NaN stays
  if constexpr (ACT == FDNN_ACT_GELU) return 0.5f * v * erfcf(-kSqrtHalf * v);
  if constexpr (ACT == FDNN_ACT_GELU_TANH)   // (1 + tanh a) / 2 is the logistic function of 2 a
    return v * logistic(2.0f * kGeluTanhScale * (v + kGeluTanhCubic * v * v * v));
  if constexpr (ACT == FDNN_ACT_SILU) return silu(v);
  return v;
}

// d activate(v) / dv
template <int ACT>
__device__ __forceinline__ float slope(float v) {
  if constexpr (ACT == FDNN_ACT_RELU) return v > 0.0f ? 1.0f : 0.0f;
  if constexpr (ACT == FDNN_ACT_GELU)
    return 0.5f * erfcf(-kSqrtHalf * v) + 0.3989422804014327f * v * ex2(-0.5f * kLog2e * v * v);
  if constexpr (ACT == FDNN_ACT_GELU_TANH) {
    const float p = logistic(2.0f * kGeluTanhScale * (v + kGeluTanhCubic * v * v * v));
    const float rest = p * (1.0f - p);   // zero far out, where the cube may have no finite value
    return p + (rest == 0.0f ? 0.0f : v * rest * (2.0f * kGeluTanhScale) * (1.0f + 3.0f * kGeluTanhCubic * v * v));
  }
  if constexpr (ACT == FDNN_ACT_SILU) {
    const float p = logistic(v);
    return p * (1.0f + v * (1.0f - p));
  }
  return 1.0f;
}

// The same for two values: the cheap ones stay packed.
template <int ACT>
__device__ __forceinline__ F2 activate2(F2 v) {
  if constexpr (ACT == FDNN_ACT_NONE) return v;
  float lo, hi;
  f2_split(v, lo, hi);
  return f2_pack(activate<ACT>(lo), activate<ACT>(hi));
}
template <int ACT>
__device__ __forceinline__ F2 slope2(F2 v) {
  if constexpr (ACT == FDNN_ACT_NONE) return f2_both(1.0f);
  if constexpr (ACT == FDNN_ACT_SILU) {
    float lo, hi;
    f2_split(f2_mul(v, f2_both(-kLog2e)), lo, hi);
    f2_split(f2_add(f2_pack(ex2(lo), ex2(hi)), f2_both(1.0f)), lo, hi);
    const F2 p = f2_pack(rcp(lo), rcp(hi));
    return f2_mul(p, f2_fma(v, f2_fma(p, f2_both(-1.0f), f2_both(1.0f)), f2_both(1.0f)));
  }
  float lo, hi;
  f2_split(v, lo, hi);
  return f2_pack(slope<ACT>(lo), slope<ACT>(hi));
}

// Runs f(std::integral_constant<int, ACT>) for a run-time activation: the branch is taken once, not per element.
template <typename F>
__device__ __forceinline__ void with_activation(int act, F&& f) {
  switch (act) {
    case FDNN_ACT_RELU: f(std::integral_constant<int, FDNN_ACT_RELU>{}); break;
    case FDNN_ACT_GELU: f(std::integral_constant<int, FDNN_ACT_GELU>{}); break;
    case FDNN_ACT_GELU_TANH: f(std::integral_constant<int, FDNN_ACT_GELU_TANH>{}); break;
    case FDNN_ACT_SILU: f(std::integral_constant<int, FDNN_ACT_SILU>{}); break;
    default: f(std::integral_constant<int, FDNN_ACT_NONE>{}); break;
  }
}

// Mean and sum of squared deviations of two sets together (n_a + n_b > 0).
struct Moments {
  float n, mean, m2;
};
__device__ __forceinline__ Moments joined(const Moments& a, const Moments& b) {
  const float n = a.n + b.n, d = b.mean - a.mean, share = b.n / n;
  return Moments{n, a.mean + d * share, a.m2 + b.m2 + d * d * a.n * share};
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Sum over a block of whole warps (at most 32); `scratch` holds 33 floats.  Every thread gets it.
__device__ __forceinline__ float block_sum(float v, float* scratch) {
  const int warps = blockDim.x >> 5;
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x < 32) {
    const float t = warp_sum(int(threadIdx.x) < warps ? scratch[threadIdx.x] : 0.0f);
    if (threadIdx.x == 0) scratch[32] = t;
  }
  __syncthreads();
  const float r = scratch[32];
  __syncthreads();
  return r;
}

template <typename T>
__device__ __forceinline__ float param(const void* p, int f32, long long i) {
  return f32 ? static_cast<const float*>(p)[i] : to_f32<T>(static_cast<const T*>(p)[i]);
}
template <typename T>
__device__ __forceinline__ void put_param(void* p, int f32, long long i, float v) {
  if (f32) static_cast<float*>(p)[i] = v;
  else static_cast<T*>(p)[i] = from_f32<T>(v);
}

// One launch after another on a stream without a gap: see griddep_wait().  First statement of every kernel here.
__device__ __forceinline__ void chained() {
  griddep_launch_dependents();
  griddep_wait();
}

}  // namespace fdnn
