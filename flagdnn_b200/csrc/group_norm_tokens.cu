// Group norm over rows of tokens: x [N, C] with its channels together, statistics over the c = C / G values of a group of one row.
//
// Bound by memory.  A group is an even share of a warp (up to 32 lanes, as many vectors of 16 bytes a lane as registers
// hold), so that a token's groups are reduced by shuffles alone; a lane keeps its channels' parameters and walks over tokens, the values of
// the next ones on their way.  Mean first, then squared deviations from it, both from registers: x is read once.
//
// The gradient's row sums need nothing else.  dweight and dbias are sums over the rows: a lane adds up those of its channels in
// fp32 over the tokens that it walks, each slice of the tokens leaves one row of [C] pairs, and a last launch adds the slices in
// their order.
#include "group_norm.cuh"

namespace fdnn {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;

struct TokenParams {
  NormParams p;
  int units, lanes;      // vectors of a group, lanes that share it (a power of two)
  int side;              // tokens of a block side by side, where all groups leave room for more (else 1)
  int slices;            // of the tokens
  float2* rows;          // backward: [slices, C]
};

// Sums over the lanes of a group, of several values at once: their shuffles do not wait for one another.
template <int K>
__device__ __forceinline__ void lane_sums(float (&v)[K], int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  }
}

// Where a thread works: its token of those side by side (SIDE), its group and its vectors of it.
template <int EACH, bool SIDE>
struct Seat {
  int token, g, u0;
  bool live;
  __device__ Seat(const TokenParams& t) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, groups = 32 / t.lanes;
    g = (blockIdx.x * kWarps + warp) * groups + lane / t.lanes;
    token = 0;
    if (SIDE) {
      token = g / t.p.G;
      g -= token * t.p.G;
    }
    u0 = lane % t.lanes;
    live = g < t.p.G && (!SIDE || token < t.side);
    if (!live) g = token = 0;
  }
  __device__ bool in(const TokenParams& t, int e) const { return live && u0 + e * t.lanes < t.units; }
};

template <typename T, int V, int EACH, int TOKENS, bool SIDE = false>
__global__ void __launch_bounds__(kThreads, EACH == 1 ? 4 : 1)
norm_tokens_kernel(const TokenParams t) {
  chained();
  const NormParams& p = t.p;
  const Seat<EACH, SIDE> seat(t);
  const int side = SIDE ? t.side : 1;
  const int cpg = p.C / p.G;
  constexpr int P = Pack<T, V>::kPairs;
  F2 w[EACH][P], b[EACH][P];
  int at[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    at[e] = seat.in(t, e) ? seat.g * cpg + (seat.u0 + e * t.lanes) * V : 0;
    norm_params_of<T, V>(p, at[e], seat.in(t, e), w[e], b[e]);
  }
  const float inv = 1.0f / float(cpg);
  const int step = gridDim.y * TOKENS * side;
  with_activation(p.act, [&](auto act) {
    // tokens n, n + side, ...: the same number of rounds for all of a warp, whose lanes sum together
    for (long long first = (long long)blockIdx.y * TOKENS * side; first < p.N; first += step) {
      const int n0 = int(first) + seat.token;
      Pack<T, V> x[TOKENS][EACH];
#pragma unroll
      for (int k = 0; k < TOKENS; ++k) {
        const int n = n0 + k * side < p.N ? n0 + k * side : p.N - 1;
        const T* from = static_cast<const T*>(p.x) + n * p.x_s[0];
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
          x[k][e].clear();
          if (seat.in(t, e)) x[k][e].load(from + at[e]);
        }
      }
      float mean[TOKENS], rstd[TOKENS];
#pragma unroll
      for (int k = 0; k < TOKENS; ++k) {
        F2 sum = 0;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
#pragma unroll
          for (int i = 0; i < P; ++i) sum = f2_add(sum, x[k][e].pair(i));
        }
        mean[k] = f2_sum(sum);
      }
      lane_sums(mean, t.lanes);
#pragma unroll
      for (int k = 0; k < TOKENS; ++k) {
        mean[k] *= inv;
        const F2 minus = f2_pack(-mean[k], V == 1 ? 0.0f : -mean[k]);
        rstd[k] = 0.0f;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
          F2 square = 0;
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const F2 d = f2_add(x[k][e].pair(i), minus);
            square = f2_fma(d, d, square);
          }
          rstd[k] += seat.in(t, e) ? f2_sum(square) : 0.0f;
        }
      }
      lane_sums(rstd, t.lanes);
#pragma unroll
      for (int k = 0; k < TOKENS; ++k) {
        rstd[k] = rsqrtf(rstd[k] * inv + p.eps);
        const F2 minus = f2_both(-mean[k]), scale = f2_both(rstd[k]);
        const int n = n0 + k * side;
        if (n < p.N) {
          if (p.mean != nullptr && seat.live && seat.u0 == 0) {
            p.mean[(long long)n * p.G + seat.g] = mean[k];
            p.rstd[(long long)n * p.G + seat.g] = rstd[k];
          }
          T* to = static_cast<T*>(p.y) + n * p.y_s[0];
#pragma unroll
          for (int e = 0; e < EACH; ++e) {
            if (!seat.in(t, e)) continue;
            Pack<T, V> y;
#pragma unroll
            for (int i = 0; i < P; ++i)
              y.set_pair(i, activate2<decltype(act)::value>(f2_fma(f2_mul(f2_add(x[k][e].pair(i), minus), scale), w[e][i], b[e][i])));
            y.store(to + at[e]);
          }
        }
      }
    }
  });
}

template <typename T, int V, int EACH, int TOKENS, bool SIDE = false>
__global__ void __launch_bounds__(kThreads, EACH == 1 ? 2 : 1)
norm_tokens_backward_kernel(const TokenParams t) {
  chained();
  const NormParams& p = t.p;
  const Seat<EACH, SIDE> seat(t);
  const int side = SIDE ? t.side : 1;
  const int cpg = p.C / p.G;
  constexpr int P = Pack<T, V>::kPairs;
  F2 w[EACH][P], b[EACH][P], dw[EACH][P], db[EACH][P];
  int at[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    at[e] = seat.in(t, e) ? seat.g * cpg + (seat.u0 + e * t.lanes) * V : 0;
    norm_params_of<T, V>(p, at[e], seat.in(t, e), w[e], b[e]);
#pragma unroll
    for (int i = 0; i < P; ++i) dw[e][i] = db[e][i] = 0;
  }
  const float inv = 1.0f / float(cpg);
  const int step = gridDim.y * TOKENS * side;
  with_activation(p.act, [&](auto act) {
    for (long long first = (long long)blockIdx.y * TOKENS * side; first < p.N; first += step) {
      const int n0 = int(first) + seat.token;
      Pack<T, V> x[TOKENS][EACH], dy[TOKENS][EACH];
      float mean[TOKENS], rstd[TOKENS], s[2 * TOKENS];
#pragma unroll
      for (int k = 0; k < TOKENS; ++k) {
        const bool there = n0 + k * side < p.N;
        const int n = there ? n0 + k * side : p.N - 1;
        mean[k] = p.mean[(long long)n * p.G + seat.g];
        rstd[k] = p.rstd[(long long)n * p.G + seat.g];
        const T *xn = static_cast<const T*>(p.x) + n * p.x_s[0], *dyn = static_cast<const T*>(p.dy) + n * p.dy_s[0];
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
          x[k][e].clear();
          dy[k][e].clear();
          if (seat.in(t, e) && there) {
            x[k][e].load(xn + at[e]);
            dy[k][e].load(dyn + at[e]);
          }
        }
      }
      F2 xh[TOKENS][EACH][P], g[TOKENS][EACH][P];
#pragma unroll
      for (int k = 0; k < TOKENS; ++k) {
        const F2 minus = f2_both(-mean[k]), scale = f2_both(rstd[k]);
        F2 t1 = 0, t2 = 0;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
          const bool in = n0 + k * side < p.N && seat.in(t, e);
#pragma unroll
          for (int i = 0; i < P; ++i) {
            xh[k][e][i] = in ? f2_mul(f2_add(x[k][e].pair(i), minus), scale) : 0;
            g[k][e][i] = in ? f2_mul(dy[k][e].pair(i), slope2<decltype(act)::value>(f2_fma(xh[k][e][i], w[e][i], b[e][i]))) : 0;
            dw[e][i] = f2_fma(g[k][e][i], xh[k][e][i], dw[e][i]);
            db[e][i] = f2_add(db[e][i], g[k][e][i]);
            g[k][e][i] = f2_mul(g[k][e][i], w[e][i]);
            t1 = f2_add(t1, g[k][e][i]);
            t2 = f2_fma(g[k][e][i], xh[k][e][i], t2);
          }
        }
        s[2 * k] = f2_sum(t1);
        s[2 * k + 1] = f2_sum(t2);
      }
      lane_sums(s, t.lanes);
#pragma unroll
      for (int k = 0; k < TOKENS; ++k) {
        const F2 m1 = f2_both(-s[2 * k] * inv), m2 = f2_both(-s[2 * k + 1] * inv), scale = f2_both(rstd[k]);
        const int n = n0 + k * side;
        if (n < p.N && p.dx != nullptr) {
          T* to = static_cast<T*>(p.dx) + n * p.dx_s[0];
#pragma unroll
          for (int e = 0; e < EACH; ++e) {
            if (!seat.in(t, e)) continue;
            Pack<T, V> dx;
#pragma unroll
            for (int i = 0; i < P; ++i) dx.set_pair(i, f2_mul(scale, f2_fma(xh[k][e][i], m2, f2_add(g[k][e][i], m1))));
            dx.store(to + at[e]);
          }
        }
      }
    }
  });
  // the block's part of a row of sums; every channel has one lane, or one for each of the tokens side by side
  float2* row = t.rows + (long long)blockIdx.y * p.C;
  extern __shared__ __align__(16) unsigned char raw[];
  float2* to = SIDE ? reinterpret_cast<float2*>(raw) + seat.token * p.C : row;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    if (!seat.in(t, e)) continue;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      float w0, w1, b0, b1;
      f2_split(dw[e][i], w0, w1);
      f2_split(db[e][i], b0, b1);
      to[at[e] + 2 * i] = make_float2(w0, b0);
      if (V > 1) to[at[e] + 2 * i + 1] = make_float2(w1, b1);
    }
  }
  if (!SIDE) return;
  __syncthreads();
  for (int c = threadIdx.x; c < p.C; c += kThreads) {
    float2 v = make_float2(0.0f, 0.0f);
    for (int k = 0; k < side; ++k) {
      const float2 q = reinterpret_cast<const float2*>(raw)[k * p.C + c];
      v.x += q.x;
      v.y += q.y;
    }
    row[c] = v;
  }
}

// How a problem is cut; EACH vectors a lane.
struct TokenPlan {
  TokenParams t;
  int each, blocks;
};
// Vectors a lane may have: what its registers hold.
constexpr int most_each(int V, bool backward) { return V >= 8 ? 4 : backward ? (V == 4 ? 4 : V == 2 ? 8 : 16) : V == 4 ? 8 : 16; }

TokenPlan plan_of(const NormParams& p, int V, int tokens, int per_sm) {
  TokenPlan plan;
  plan.t.p = p;
  plan.t.units = p.C / p.G / V;
  plan.t.lanes = 1;
  while (plan.t.lanes < 32 && plan.t.lanes < plan.t.units) plan.t.lanes *= 2;
  const int each = (plan.t.units + plan.t.lanes - 1) / plan.t.lanes;
  for (plan.each = 1; plan.each < each;) plan.each *= 2;
  const int groups = kWarps * (32 / plan.t.lanes);
  plan.blocks = (p.G + groups - 1) / groups;
  // few groups: several tokens to a block, as far as their sums of the parameters' gradients fit a block's 48 KB
  plan.t.side = groups / p.G;
  if (plan.t.side > 49152 / 8 / p.C) plan.t.side = 49152 / 8 / p.C;
  if (plan.t.side > p.N) plan.t.side = p.N;
  if (plan.t.side < 1) plan.t.side = 1;
  // enough blocks for every SM; more tokens are walked
  const long long at_once = (long long)tokens * plan.t.side;
  long long slices = (p.N + at_once - 1) / at_once, room = (long long)per_sm * current_sm_count() / plan.blocks;
  if (room < 1) room = 1;
  plan.t.slices = int(slices < room ? slices : room);
  plan.t.rows = static_cast<float2*>(p.workspace);
  return plan;
}

// Blocks an SM is given (they walk the tokens) and tokens a lane holds at once, as measured for one vector a lane.  Four tokens
// and as many blocks as the registers leave room for: 16384 x 4096 bf16 46.5 us (two tokens 52.4, five blocks 62, three 49), the
// gradient with two blocks 78.3 (two tokens 91, three blocks of them 85, one block 111).  fp32 takes fewer registers: eight blocks,
// 4096 x 2048 11.5 us (four 12.1).  A second round of blocks that do not fit costs most: 78 us.
template <typename T>
constexpr int per_sm(bool backward) { return backward ? 2 : sizeof(T) == 4 ? 8 : 4; }
template <typename T>
constexpr int tokens_at_once(int each, bool backward) { return each == 1 ? 4 : each == 2 && !backward ? 2 : 1; }

// One token at a time of each block's, or several side by side.
template <typename T, int V, int EACH>
cudaError_t forward_as(const TokenPlan& plan, cudaStream_t stream) {
  constexpr int tokens = tokens_at_once<T>(EACH, false);
  const dim3 grid(unsigned(plan.blocks), unsigned(plan.t.slices));
  if (plan.t.side == 1) return launch_seq(norm_tokens_kernel<T, V, EACH, tokens>, grid, kThreads, 0, 1, stream, plan.t);
  return launch_seq(norm_tokens_kernel<T, V, EACH, tokens, true>, grid, kThreads, 0, 1, stream, plan.t);
}

template <typename T, int V, int EACH>
cudaError_t backward_as(const TokenPlan& plan, cudaStream_t stream) {
  constexpr int tokens = tokens_at_once<T>(EACH, true);
  const dim3 grid(unsigned(plan.blocks), unsigned(plan.t.slices));
  if (plan.t.side == 1) return launch_seq(norm_tokens_backward_kernel<T, V, EACH, tokens>, grid, kThreads, 0, 1, stream, plan.t);
  return launch_seq(norm_tokens_backward_kernel<T, V, EACH, tokens, true>, grid, kThreads, 8 * plan.t.side * plan.t.p.C, 1, stream, plan.t);
}

template <typename T, int V>
cudaError_t forward(const NormParams& p, cudaStream_t stream) {
  TokenPlan plan = plan_of(p, V, 1, 1);
  plan = plan_of(p, V, tokens_at_once<T>(plan.each, false), per_sm<T>(false));
  switch (plan.each) {
    case 1: return forward_as<T, V, 1>(plan, stream);
    case 2: return forward_as<T, V, 2>(plan, stream);
    case 4: return forward_as<T, V, 4>(plan, stream);
    default: break;
  }
  if constexpr (most_each(V, false) >= 8)
    if (plan.each == 8) return forward_as<T, V, 8>(plan, stream);
  if constexpr (most_each(V, false) >= 16)
    if (plan.each == 16) return forward_as<T, V, 16>(plan, stream);
  return cudaErrorInvalidValue;
}

template <typename T, int V>
TokenPlan backward_plan(const NormParams& p) {
  const TokenPlan plan = plan_of(p, V, 1, 1);
  return plan_of(p, V, tokens_at_once<T>(plan.each, true), per_sm<T>(true));
}

template <typename T, int V>
cudaError_t backward(const NormParams& p, cudaStream_t stream) {
  const TokenPlan plan = backward_plan<T, V>(p);
  if (8ll * p.C * plan.t.slices > p.workspace_bytes) return cudaErrorInvalidValue;
  cudaError_t e = cudaErrorInvalidValue;
  switch (plan.each) {
    case 1: e = backward_as<T, V, 1>(plan, stream); break;
    case 2: e = backward_as<T, V, 2>(plan, stream); break;
    case 4: e = backward_as<T, V, 4>(plan, stream); break;
    default: break;
  }
  if constexpr (most_each(V, true) >= 8)
    if (plan.each == 8) e = backward_as<T, V, 8>(plan, stream);
  if constexpr (most_each(V, true) >= 16)
    if (plan.each == 16) e = backward_as<T, V, 16>(plan, stream);
  if (e != cudaSuccess || (p.dweight == nullptr && p.dbias == nullptr)) return e;
  return launch_norm_dparams<T>(p, plan.t.rows, plan.t.slices, stream);
}

}  // namespace

// Rows of tokens whose groups fit a warp.
bool norm_tokens_take(int dtype, const NormParams& p, bool backward) {
  const int V = norm_vector(dtype, p, backward, p.C / p.G);
  return V > 0 && p.H == 1 && p.W == 1 && p.C / p.G <= 32 * most_each(V, backward) * V;
}

long long norm_tokens_workspace(int dtype, const NormParams& p, bool backward) {
  (void)dtype;
  if (!backward) return 0;
  // (an upper bound that does not depend on the tensors' alignment)
  const long long slices = p.N < 65535 ? p.N : 65535, room = 8ll * current_sm_count();
  return 8ll * p.C * (slices < room ? slices : room);
}

cudaError_t launch_norm_tokens(int dtype, const NormParams& p, bool back, cudaStream_t stream) {
  return norm_by_vector(dtype, norm_vector(dtype, p, back, p.C / p.G), [&](auto type, auto v) {
    using T = typename decltype(type)::type;
    return back ? backward<T, decltype(v)::value>(p, stream) : forward<T, decltype(v)::value>(p, stream);
  });
}

}  // namespace fdnn
