// The selective state space scan for single tokens: one step of h = exp(dt A) h + dt u B for each row, its state in place.
//
// Its bytes are the states, read and written; what takes longer is instructions (73 % of the issue slots): each lane of a channel reads u,
// delta and z and takes softplus for its four states.  16 states of a channel are four lanes' 16 bytes, so that a warp moves 512
// contiguous bytes; a thread keeps its channel's A and walks several rows, with the states of the next rows on their way.
// 256 rows of 4096 x 16, f16, with the convolution's step before it: 39.3 us, 4.1 TB/s.
#include "group_norm.cuh"

namespace fdnn {
namespace {

constexpr int kThreads = 128;

// Four neighbouring states, those past `count` zero.
template <bool WHOLE>
__device__ __forceinline__ float4 four_states(const float* p, int count) {
  if constexpr (WHOLE) return *reinterpret_cast<const float4*>(p);
  return make_float4(p[0], count > 1 ? p[1] : 0.0f, count > 2 ? p[2] : 0.0f, count > 3 ? p[3] : 0.0f);
}

// LANES threads share a channel, four states each and as often as S needs (more than 128 states: CHUNKS of them).  WHOLE: S is
// a multiple of four and all addresses of four values; then nothing is loaded one by one.
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
    a[k] = make_float4(rate_of(a[k].x), rate_of(a[k].y), rate_of(a[k].z), rate_of(a[k].w));
  }
  const float D = p.D != nullptr ? p.D[cc] : 0.0f, bias = p.delta_bias != nullptr ? p.delta_bias[cc] : 0.0f;
  const T* u0 = static_cast<const T*>(p.u) + cc * p.u_s[2];
  const T* d0 = static_cast<const T*>(p.delta) + cc * p.delta_s[2];
  const T* z0 = p.z == nullptr ? nullptr : static_cast<const T*>(p.z) + cc * p.z_s[2];
  const T* B0 = static_cast<const T*>(p.B) + g * p.b_s[2] + part * 4 * p.b_s[3];
  const T* C0 = static_cast<const T*>(p.Cm) + g * p.c_s[2] + part * 4 * p.c_s[3];
  float* h0 = state + (long long)cc * p.S + part * 4;
  for (int n0 = blockIdx.y * ROWS; n0 < p.N; n0 += gridDim.y * ROWS) {
    float4 h[ROWS][CHUNKS];
    Pack<T, 4> b[ROWS][CHUNKS], m[ROWS][CHUNKS];
    T u[ROWS], dt[ROWS], z[ROWS];
    float* at[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int n = n0 + r;
      const int slot = n < p.N ? (slots != nullptr ? slots[n] : n) : -1;
      at[r] = live && slot >= 0 && slot < n_slots ? h0 + (long long)slot * p.C * p.S : nullptr;
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const long long n = n0 + r;
      u[r] = dt[r] = z[r] = from_f32<T>(0.0f);
#pragma unroll
      for (int k = 0; k < CHUNKS; ++k) {
        const int s = (k * LANES + part) * 4;
        h[r][k] = make_float4(0, 0, 0, 0);
        b[r][k].clear();
        m[r][k].clear();
        if (at[r] != nullptr && s < p.S) {
          h[r][k] = four_states<WHOLE>(at[r] + k * LANES * 4, p.S - s);
          const T* bp = B0 + n * p.b_s[0] + k * LANES * 4 * p.b_s[3];
          const T* mp = C0 + n * p.c_s[0] + k * LANES * 4 * p.c_s[3];
          if constexpr (WHOLE) {
            b[r][k].load(bp);
            m[r][k].load(mp);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (s + j < p.S) {
                reinterpret_cast<T*>(&b[r][k].q)[j] = bp[j * p.b_s[3]];
                reinterpret_cast<T*>(&m[r][k].q)[j] = mp[j * p.c_s[3]];
              }
          }
        }
      }
      if (at[r] != nullptr) {
        u[r] = u0[n * p.u_s[0]];
        dt[r] = d0[n * p.delta_s[0]];
        if (p.z != nullptr) z[r] = z0[n * p.z_s[0]];
      }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int n = n0 + r;
      const float uv = to_f32<T>(u[r]), raw = to_f32<T>(dt[r]) + bias, d = p.softplus ? softplus(raw) : raw, du = d * uv;
      float y = 0.0f;
#pragma unroll
      for (int k = 0; k < CHUNKS; ++k) {
        const int s = (k * LANES + part) * 4;
        float4 v;
        v.x = h[r][k].x * decay_of(d, a[k].x) + du * b[r][k].at(0);
        v.y = h[r][k].y * decay_of(d, a[k].y) + du * b[r][k].at(1);
        v.z = h[r][k].z * decay_of(d, a[k].z) + du * b[r][k].at(2);
        v.w = h[r][k].w * decay_of(d, a[k].w) + du * b[r][k].at(3);
        // (states past S: b and m are zero, but zero times an infinite du is not)
        if (WHOLE ? s < p.S : s + 3 < p.S) {
          y += v.x * m[r][k].at(0) + v.y * m[r][k].at(1) + v.z * m[r][k].at(2) + v.w * m[r][k].at(3);
        } else if (!WHOLE) {
          y += (s < p.S ? v.x * m[r][k].at(0) : 0.0f) + (s + 1 < p.S ? v.y * m[r][k].at(1) : 0.0f) + (s + 2 < p.S ? v.z * m[r][k].at(2) : 0.0f);
        }
        if (at[r] != nullptr && s < p.S) {
          float* to = at[r] + k * LANES * 4;
          if constexpr (WHOLE) {
            *reinterpret_cast<float4*>(to) = v;
          } else {
            to[0] = v.x;
            if (s + 1 < p.S) to[1] = v.y;
            if (s + 2 < p.S) to[2] = v.z;
            if (s + 3 < p.S) to[3] = v.w;
          }
        }
      }
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
      if (live && part == 0 && n < p.N) {
        if (p.D != nullptr) y += D * uv;   // (zero times an infinite u is not nothing)
        if (p.z != nullptr) y *= silu(to_f32<T>(z[r]));
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
  auto fours = [](const void* q, const long long* st) {
    return reinterpret_cast<uintptr_t>(q) % (4 * sizeof(T)) == 0 && st[0] % 4 == 0 && st[2] % 4 == 0 && st[3] == 1;
  };
  const bool whole = p.S % 4 == 0 && even(state) && even(p.A) && fours(p.B, p.b_s) && fours(p.Cm, p.c_s);
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
