// The gated delta rule token by token: single tokens over a cache of states, and prompts that are short or have wide keys.
//
// A state's rows (one for each value channel) do not meet: row i takes S k and S q, sums over the keys' channels, and adds its own
// multiple of k.  Eight threads hold a row in 16-byte pieces (128 bytes of it side by side), a warp four times ROWS rows, all loads of
// which are on their way together; a sum takes three exchanges for four rows (32 threads to a row took five for one: 128 rows of 32
// heads of 128 x 128 104.5 us, 84.0 now: 6.4 TB/s).  Both sums are taken of the state before the token, y = a (S q) + u (k q), so that they go through the
// warp side by side.  Its bytes are the states, read and written.
#include "delta_rule.cuh"

namespace fdnn {
namespace {

constexpr int kThreads = 128, kLanes = 8, kSubs = 32 / kLanes;

__device__ __forceinline__ float dot(float4 a, float4 b) { return a.x * b.x + a.y * b.y + a.z * b.z + a.w * b.w; }
__device__ __forceinline__ float& part_of(float4& v, int j) { return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w; }

// What a token brings, as it is loaded.
template <typename T, int CHUNKS, int ROWS>
struct Token {
  Pack<T, 4> q[CHUNKS], k[CHUNKS];
  T v[ROWS];
  float delta, beta;
};

// STEP: one token a row, `cache` [n_slots, H, V, K] updated in place.  Otherwise prompts from `initial` to `final_state`.
// WHOLE: four neighbouring channels of q, k and the states are loaded at once; otherwise neighbouring threads take neighbouring channels.
template <typename T, int CHUNKS, bool WHOLE, int ROWS, bool STEP>
__global__ void __launch_bounds__(kThreads)
delta_tokens_kernel(const DeltaParams p, float* cache, int n_slots, const int* slots) {
  chained();
  constexpr int kBlockRows = kThreads / kLanes * ROWS;
  const int parts = (p.V + kBlockRows - 1) / kBlockRows;
  const int h = blockIdx.x / parts, part = threadIdx.x % kLanes;
  const int row0 = (blockIdx.x % parts) * kBlockRows + (threadIdx.x >> 5) * kSubs * ROWS + (threadIdx.x & 31) / kLanes;   // and every fourth from it on
  auto row = [&](int i) { return row0 + i * kSubs; };
  auto channel = [&](int c, int j) { return WHOLE ? (c * kLanes + part) * 4 + j : (c * 4 + j) * kLanes + part; };
  const int g = h / (p.H / p.G);
  const float A = p.A != nullptr ? p.A[h] : 1.0f, bias = p.delta_bias != nullptr ? p.delta_bias[h] : 0.0f;
  for (long long n = blockIdx.y; n < p.N; n += gridDim.y) {
    float* to;
    const float* from;
    int end;
    if constexpr (STEP) {
      const int slot = slots != nullptr ? slots[n] : int(n);
      const bool live = slot >= 0 && slot < n_slots;
      to = live ? cache + ((long long)slot * p.H + h) * p.V * p.K : nullptr;
      from = to;
      end = live ? 1 : 0;
    } else {
      const long long at = (n * p.H + h) * p.V * p.K;
      to = p.final_state != nullptr ? p.final_state + at : nullptr;
      from = p.initial != nullptr ? p.initial + at : nullptr;
      end = p.lengths != nullptr ? min(max(p.lengths[n], 0), p.L) : p.L;
    }
    float4 s[ROWS][CHUNKS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        s[i][c] = make_float4(0, 0, 0, 0);
        if (from != nullptr && row(i) < p.V) {
          const float* at = from + (long long)row(i) * p.K;
          if constexpr (WHOLE) {
            if (channel(c, 0) < p.K) s[i][c] = __ldcs(reinterpret_cast<const float4*>(at + channel(c, 0)));   // (read and written once)
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (channel(c, j) < p.K) part_of(s[i][c], j) = __ldcs(at + channel(c, j));
          }
        }
      }
    const T* q0 = static_cast<const T*>(p.q) + n * p.q_s[0] + g * p.q_s[2];
    const T* k0 = static_cast<const T*>(p.k) + n * p.k_s[0] + g * p.k_s[2];
    const T* v0 = static_cast<const T*>(p.v) + n * p.v_s[0] + h * p.v_s[2];
    T* y0 = static_cast<T*>(p.y) + n * p.y_s[0] + h * p.y_s[2];
    const long long d0 = n * p.delta_s[0] + h * p.delta_s[2], b0 = n * p.beta_s[0] + h * p.beta_s[2];
    auto load = [&](Token<T, CHUNKS, ROWS>& x, long long t) {
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        x.q[c].clear();
        x.k[c].clear();
        const T *qp = q0 + t * p.q_s[1], *kp = k0 + t * p.k_s[1];
        if constexpr (WHOLE) {
          if (channel(c, 0) < p.K) {
            x.q[c].load(qp + channel(c, 0));
            x.k[c].load(kp + channel(c, 0));
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (channel(c, j) < p.K) {
              reinterpret_cast<T*>(&x.q[c].q)[j] = qp[channel(c, j) * p.q_s[3]];
              reinterpret_cast<T*>(&x.k[c].q)[j] = kp[channel(c, j) * p.k_s[3]];
            }
        }
      }
#pragma unroll
      for (int i = 0; i < ROWS; ++i) x.v[i] = row(i) < p.V ? v0[t * p.v_s[1] + row(i) * p.v_s[3]] : from_f32<T>(0.0f);
      x.delta = gate_at<T>(p, p.delta, d0 + t * p.delta_s[1]);
      x.beta = gate_at<T>(p, p.beta, b0 + t * p.beta_s[1]);
    };
    Token<T, CHUNKS, ROWS> next;
    if (end > 0) load(next, 0);
    for (int t = 0; t < end; ++t) {
      const Token<T, CHUNKS, ROWS> x = next;
      if (!STEP && t + 1 < end) load(next, t + 1);
      float qq = 0.0f, kk = 0.0f, qk = 0.0f, sk[ROWS] = {}, sq[ROWS] = {};
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        const float4 q = make_float4(x.q[c].at(0), x.q[c].at(1), x.q[c].at(2), x.q[c].at(3));
        const float4 k = make_float4(x.k[c].at(0), x.k[c].at(1), x.k[c].at(2), x.k[c].at(3));
        qq += dot(q, q);
        kk += dot(k, k);
        qk += dot(q, k);
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          sk[i] += dot(s[i][c], k);
          sq[i] += dot(s[i][c], q);
        }
      }
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) {
        if (p.norm) {
          qq += __shfl_xor_sync(0xffffffffu, qq, o);
          kk += __shfl_xor_sync(0xffffffffu, kk, o);
        }
        qk += __shfl_xor_sync(0xffffffffu, qk, o);
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          sk[i] += __shfl_xor_sync(0xffffffffu, sk[i], o);
          sq[i] += __shfl_xor_sync(0xffffffffu, sq[i], o);
        }
      }
      const float a = expf(log_decay(p, x.delta, bias, A)), b = step_size(p, x.beta);
      const float kn = p.norm ? 1.0f / sqrtf(kk + kKeyEps) : 1.0f, qn = p.scale * (p.norm ? 1.0f / sqrtf(qq + kKeyEps) : 1.0f);
      T* y = y0 + t * p.y_s[1];
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const float u = b * (to_f32<T>(x.v[i]) - a * (kn * sk[i])) * kn;   // (times k as it came)
        if (part == i % kLanes && row(i) < p.V) y[row(i) * p.y_s[3]] = from_f32<T>(qn * (a * sq[i] + u * qk));
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          s[i][c].x = a * s[i][c].x + u * x.k[c].at(0);
          s[i][c].y = a * s[i][c].y + u * x.k[c].at(1);
          s[i][c].z = a * s[i][c].z + u * x.k[c].at(2);
          s[i][c].w = a * s[i][c].w + u * x.k[c].at(3);
        }
      }
    }
    if (to != nullptr) {
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
          if (row(i) < p.V) {
            float* at = to + (long long)row(i) * p.K;
            if constexpr (WHOLE) {
              if (channel(c, 0) < p.K) __stcs(reinterpret_cast<float4*>(at + channel(c, 0)), s[i][c]);
            } else {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (channel(c, j) < p.K) __stcs(at + channel(c, j), part_of(s[i][c], j));
            }
          }
    }
    // an idle row, and tokens behind a row's end
    for (int t = end; t < (STEP ? 1 : p.L); ++t)
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
        if (part == i % kLanes && row(i) < p.V) y0[t * p.y_s[1] + row(i) * p.y_s[3]] = from_f32<T>(0.0f);
  }
}

template <typename T, int CHUNKS, int ROWS, bool STEP>
cudaError_t go(const DeltaParams& p, float* cache, int n_slots, const int* slots, cudaStream_t stream) {
  constexpr int kBlockRows = kThreads / kLanes * ROWS;
  const long long blocks = (long long)p.H * ((p.V + kBlockRows - 1) / kBlockRows);
  if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  auto even = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; };
  const bool whole = p.K % 4 == 0 && even(cache) && even(p.initial) && even(p.final_state) && fours<T>(p.q, p.q_s) && fours<T>(p.k, p.k_s);
  auto* kernel = whole ? delta_tokens_kernel<T, CHUNKS, true, ROWS, STEP> : delta_tokens_kernel<T, CHUNKS, false, ROWS, STEP>;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(p.N < 65535 ? p.N : 65535));
  return launch_seq(kernel, grid, kThreads, 0, 1, stream, p, cache, n_slots, slots);
}

// 32 channels a chunk; some 32 registers of state a thread.
template <typename T, bool STEP>
cudaError_t by_width(const DeltaParams& p, float* cache, int n_slots, const int* slots, cudaStream_t stream) {
  if (p.K <= 32) return go<T, 1, 4, STEP>(p, cache, n_slots, slots, stream);
  if (p.K <= 64) return go<T, 2, 4, STEP>(p, cache, n_slots, slots, stream);
  if (p.K <= 96) return go<T, 3, 2, STEP>(p, cache, n_slots, slots, stream);
  if (p.K <= 128) return go<T, 4, 2, STEP>(p, cache, n_slots, slots, stream);
  if (p.K <= 192) return go<T, 6, 1, STEP>(p, cache, n_slots, slots, stream);
  return go<T, 8, 1, STEP>(p, cache, n_slots, slots, stream);
}

template <bool STEP>
cudaError_t by_type(int dtype, const DeltaParams& p, float* cache, int n_slots, const int* slots, cudaStream_t stream) {
  switch (dtype) {
    case FDNN_F16: return by_width<__half, STEP>(p, cache, n_slots, slots, stream);
    case FDNN_BF16: return by_width<__nv_bfloat16, STEP>(p, cache, n_slots, slots, stream);
    default: return by_width<float, STEP>(p, cache, n_slots, slots, stream);
  }
}

}  // namespace

cudaError_t launch_delta_rule_step(int dtype, const DeltaParams& p, float* state, int n_slots, const int* slots, cudaStream_t stream) {
  return by_type<true>(dtype, p, state, n_slots, slots, stream);
}
cudaError_t launch_delta_rule_tokens(int dtype, const DeltaParams& p, cudaStream_t stream) {
  return by_type<false>(dtype, p, nullptr, 0, nullptr, stream);
}

}  // namespace fdnn
