// Group norm with an activation, and its gradient, for any strides.
//
//   y = act((x - mean) rstd w + b),  mean and rstd over the m = C / G * H * W values of an image's group
//   g = dy act'(.),  db = sum g,  dw = sum g xh,  dx = rstd (g w - (s1 + xh s2) / m),
//   xh = (x - mean) rstd,  s1 = sum over the group of g w,  s2 = of g w xh
//
// Statistics here are a mean and then a sum of squared deviations from it: values whose mean is thousands of times their spread keep
// their precision.  All sums are fp32 in a fixed order, so that equal calls give equal results.
//
// Values are taken one by one, with a division for each one's place: 32 x 256 x 56 x 56 bf16 with silu, contiguous, 247 us, and its
// gradient 229 (channels last, through the other files: 36 and 75).
#include "group_norm.cuh"

namespace fdnn {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 16384;       // values of a group that one block takes
constexpr int kMaxChunks = 64;      // of one group

// The values of a group in the order in which they lie in memory.
template <typename I>
struct GroupWalk {
  I cpg, S, W;
  bool c_fast;
  const long long* s;
  __device__ GroupWalk(const NormParams& p, const long long* strides)
      : cpg(I(p.C / p.G)), S(I(p.H) * I(p.W)), W(I(p.W)), c_fast(p.x_s[1] <= p.x_s[3]), s(strides) {}
  __device__ void at(I e, int& c, I& pixel) const {
    if (c_fast) {
      c = int(e % cpg);
      pixel = e / cpg;
    } else {
      pixel = e % S;
      c = int(e / S);
    }
  }
  __device__ long long offset(int c, I pixel, const long long* st) const {
    return c * st[1] + (long long)(pixel / W) * st[2] + (long long)(pixel % W) * st[3];
  }
};

struct Chunks {
  long long m, size;
  int count;
};
__host__ __device__ inline Chunks chunks_of(const NormParams& p) {
  Chunks c;
  c.m = (long long)(p.C / p.G) * p.H * p.W;
  long long n = (c.m + kChunk - 1) / kChunk;
  if (n > kMaxChunks) n = kMaxChunks;
  c.size = (c.m + n - 1) / n;
  c.count = int((c.m + c.size - 1) / c.size);
  return c;
}

// Mean and squared deviations of every chunk of every group.
template <typename T, typename I>
__global__ void __launch_bounds__(kThreads)
norm_stats_kernel(const NormParams p) {
  chained();
  __shared__ float scratch[33];
  const Chunks ch = chunks_of(p);
  const GroupWalk<I> walk(p, p.x_s);
  float2* part = static_cast<float2*>(p.workspace);
  const long long items = (long long)p.N * p.G * ch.count;
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    const long long ng = item / ch.count;
    const int n = int(ng / p.G), g = int(ng % p.G);
    const T* x = static_cast<const T*>(p.x) + n * p.x_s[0] + (long long)g * (p.C / p.G) * p.x_s[1];
    const long long e0 = (item % ch.count) * ch.size, e1 = min(ch.m, e0 + ch.size);
    float sum = 0.0f;
    for (long long e = e0 + threadIdx.x; e < e1; e += kThreads) {
      int c;
      I pix;
      walk.at(I(e), c, pix);
      sum += to_f32<T>(x[walk.offset(c, pix, p.x_s)]);
    }
    const float mean = block_sum(sum, scratch) / float(e1 - e0);
    float m2 = 0.0f;
    for (long long e = e0 + threadIdx.x; e < e1; e += kThreads) {
      int c;
      I pix;
      walk.at(I(e), c, pix);
      const float d = to_f32<T>(x[walk.offset(c, pix, p.x_s)]) - mean;
      m2 += d * d;
    }
    m2 = block_sum(m2, scratch);
    if (threadIdx.x == 0) part[item] = make_float2(mean, m2);
  }
}

template <typename T, typename I>
__global__ void __launch_bounds__(kThreads)
norm_apply_kernel(const NormParams p) {
  chained();
  const Chunks ch = chunks_of(p);
  const GroupWalk<I> walk(p, p.x_s);
  const float2* part = static_cast<const float2*>(p.workspace);
  const long long items = (long long)p.N * p.G * ch.count;
  const int cpg = p.C / p.G;
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    const long long ng = item / ch.count;
    const int n = int(ng / p.G), g = int(ng % p.G);
    Moments all{0.0f, 0.0f, 0.0f};
    for (int k = 0; k < ch.count; ++k) {
      const float2 v = part[ng * ch.count + k];
      all = joined(all, Moments{float(min(ch.m, (k + 1) * ch.size) - k * ch.size), v.x, v.y});
    }
    const float mean = all.mean, rstd = rsqrtf(all.m2 / float(ch.m) + p.eps);
    if (p.mean != nullptr && item % ch.count == 0 && threadIdx.x == 0) {
      p.mean[ng] = mean;
      p.rstd[ng] = rstd;
    }
    const T* x = static_cast<const T*>(p.x) + n * p.x_s[0] + (long long)g * cpg * p.x_s[1];
    T* y = static_cast<T*>(p.y) + n * p.y_s[0] + (long long)g * cpg * p.y_s[1];
    const long long e0 = (item % ch.count) * ch.size, e1 = min(ch.m, e0 + ch.size);
    with_activation(p.act, [&](auto act) {
      for (long long e = e0 + threadIdx.x; e < e1; e += kThreads) {
        int c;
        I pix;
        walk.at(I(e), c, pix);
        const float w = p.weight != nullptr ? param<T>(p.weight, p.param_f32, g * cpg + c) : 1.0f;
        const float b = p.bias != nullptr ? param<T>(p.bias, p.param_f32, g * cpg + c) : 0.0f;
        const float v = (to_f32<T>(x[walk.offset(c, pix, p.x_s)]) - mean) * rstd * w + b;
        y[walk.offset(c, pix, p.y_s)] = from_f32<T>(activate<decltype(act)::value>(v));
      }
    });
  }
}

// Per image and channel: sum of g xh and of g over the pixels, into the workspace as [N, C] pairs.
template <typename T, typename I>
__global__ void __launch_bounds__(kThreads)
norm_channel_sums_kernel(const NormParams p) {
  chained();
  __shared__ float scratch[33];
  float2* sums = static_cast<float2*>(p.workspace);
  const I S = I(p.H) * I(p.W), W = I(p.W);
  const long long items = (long long)p.N * p.C;
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    const int n = int(item / p.C), c = int(item % p.C);
    const long long ng = (long long)n * p.G + c / (p.C / p.G);
    const float mean = p.mean[ng], rstd = p.rstd[ng];
    const float w = p.weight != nullptr ? param<T>(p.weight, p.param_f32, c) : 1.0f;
    const float b = p.bias != nullptr ? param<T>(p.bias, p.param_f32, c) : 0.0f;
    const T* x = static_cast<const T*>(p.x) + n * p.x_s[0] + c * p.x_s[1];
    const T* dy = static_cast<const T*>(p.dy) + n * p.dy_s[0] + c * p.dy_s[1];
    float gx = 0.0f, gs = 0.0f;
    with_activation(p.act, [&](auto act) {
      for (I i = threadIdx.x; i < S; i += kThreads) {
        const long long h = i / W, q = i % W;
        const float xh = (to_f32<T>(x[h * p.x_s[2] + q * p.x_s[3]]) - mean) * rstd;
        const float g = to_f32<T>(dy[h * p.dy_s[2] + q * p.dy_s[3]]) * slope<decltype(act)::value>(xh * w + b);
        gx += g * xh;
        gs += g;
      }
    });
    gx = block_sum(gx, scratch);
    gs = block_sum(gs, scratch);
    if (threadIdx.x == 0) sums[item] = make_float2(gx, gs);
  }
}

// The same for images of a few pixels: a thread per channel.
template <typename T>
__global__ void __launch_bounds__(kThreads)
norm_channel_sums_thin_kernel(const NormParams p) {
  chained();
  float2* sums = static_cast<float2*>(p.workspace);
  const long long items = (long long)p.N * p.C;
  with_activation(p.act, [&](auto act) {
    for (long long item = blockIdx.x * (long long)kThreads + threadIdx.x; item < items; item += (long long)gridDim.x * kThreads) {
      const int n = int(item / p.C), c = int(item % p.C);
      const long long ng = (long long)n * p.G + c / (p.C / p.G);
      const float mean = p.mean[ng], rstd = p.rstd[ng];
      const float w = p.weight != nullptr ? param<T>(p.weight, p.param_f32, c) : 1.0f;
      const float b = p.bias != nullptr ? param<T>(p.bias, p.param_f32, c) : 0.0f;
      const T* x = static_cast<const T*>(p.x) + n * p.x_s[0] + c * p.x_s[1];
      const T* dy = static_cast<const T*>(p.dy) + n * p.dy_s[0] + c * p.dy_s[1];
      float2 t = make_float2(0.0f, 0.0f);
      for (int h = 0; h < p.H; ++h)
        for (int q = 0; q < p.W; ++q) {
          const float xh = (to_f32<T>(x[h * p.x_s[2] + q * p.x_s[3]]) - mean) * rstd;
          const float g = to_f32<T>(dy[h * p.dy_s[2] + q * p.dy_s[3]]) * slope<decltype(act)::value>(xh * w + b);
          t.x += g * xh;
          t.y += g;
        }
      sums[item] = t;
    }
  });
}

template <typename T, typename I>
__global__ void __launch_bounds__(kThreads)
norm_dx_kernel(const NormParams p) {
  chained();
  __shared__ float scratch[33];
  const Chunks ch = chunks_of(p);
  const GroupWalk<I> walk(p, p.x_s);
  const float2* sums = static_cast<const float2*>(p.workspace);
  const long long items = (long long)p.N * p.G * ch.count;
  const int cpg = p.C / p.G;
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    const long long ng = item / ch.count;
    const int n = int(ng / p.G), g = int(ng % p.G);
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = threadIdx.x; c < cpg; c += kThreads) {
      const float2 v = sums[(long long)n * p.C + g * cpg + c];
      const float w = p.weight != nullptr ? param<T>(p.weight, p.param_f32, g * cpg + c) : 1.0f;
      s2 += w * v.x;
      s1 += w * v.y;
    }
    s1 = block_sum(s1, scratch) / float(ch.m);
    s2 = block_sum(s2, scratch) / float(ch.m);
    const float mean = p.mean[ng], rstd = p.rstd[ng];
    const T* x = static_cast<const T*>(p.x) + n * p.x_s[0] + (long long)g * cpg * p.x_s[1];
    const T* dy = static_cast<const T*>(p.dy) + n * p.dy_s[0] + (long long)g * cpg * p.dy_s[1];
    T* dx = static_cast<T*>(p.dx) + n * p.dx_s[0] + (long long)g * cpg * p.dx_s[1];
    const long long e0 = (item % ch.count) * ch.size, e1 = min(ch.m, e0 + ch.size);
    with_activation(p.act, [&](auto act) {
      for (long long e = e0 + threadIdx.x; e < e1; e += kThreads) {
        int c;
        I pix;
        walk.at(I(e), c, pix);
        const float w = p.weight != nullptr ? param<T>(p.weight, p.param_f32, g * cpg + c) : 1.0f;
        const float b = p.bias != nullptr ? param<T>(p.bias, p.param_f32, g * cpg + c) : 0.0f;
        const float xh = (to_f32<T>(x[walk.offset(c, pix, p.x_s)]) - mean) * rstd;
        const float gr = to_f32<T>(dy[walk.offset(c, pix, p.dy_s)]) * slope<decltype(act)::value>(xh * w + b);
        dx[walk.offset(c, pix, p.dx_s)] = from_f32<T>(rstd * (gr * w - s1 - xh * s2));
      }
    });
  }
}

// 32 channels a block, each of its 32 warps every 32nd row; then the warps' sums in their order.
template <typename T>
__global__ void __launch_bounds__(1024)
norm_dparams_kernel(const NormParams p, const float2* rows, long long count) {
  chained();
  __shared__ float2 part[32][32];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float2 v = make_float2(0.0f, 0.0f);
  if (c < p.C) {
#pragma unroll 8
    for (long long r = slice; r < count; r += 32) {
      const float2 q = rows[r * p.C + c];
      v.x += q.x;
      v.y += q.y;
    }
  }
  part[slice][lane] = v;
  __syncthreads();
  if (slice != 0 || c >= p.C) return;
#pragma unroll 8
  for (int k = 1; k < 32; ++k) {
    v.x += part[k][lane].x;
    v.y += part[k][lane].y;
  }
  if (p.dweight != nullptr) put_param<T>(p.dweight, p.param_f32, c, v.x);
  if (p.dbias != nullptr) put_param<T>(p.dbias, p.param_f32, c, v.y);
}

unsigned grid_of(long long items) { return unsigned(items < (1ll << 30) ? items : (1ll << 30)); }

template <typename T, typename I>
cudaError_t forward(const NormParams& p, cudaStream_t stream) {
  if (8ll * p.N * p.G * chunks_of(p).count > p.workspace_bytes) return cudaErrorInvalidValue;
  const long long items = (long long)p.N * p.G * chunks_of(p).count;
  cudaError_t e = launch_seq(norm_stats_kernel<T, I>, dim3(grid_of(items)), kThreads, 0, 1, stream, p);
  if (e != cudaSuccess) return e;
  return launch_seq(norm_apply_kernel<T, I>, dim3(grid_of(items)), kThreads, 0, 1, stream, p);
}

template <typename T, typename I>
cudaError_t backward(const NormParams& p, cudaStream_t stream) {
  if (8ll * p.N * p.C > p.workspace_bytes) return cudaErrorInvalidValue;
  const long long channels = (long long)p.N * p.C;
  cudaError_t e = (long long)p.H * p.W <= 32
                      ? launch_seq(norm_channel_sums_thin_kernel<T>, dim3(grid_of((channels + kThreads - 1) / kThreads)), kThreads, 0, 1, stream, p)
                      : launch_seq(norm_channel_sums_kernel<T, I>, dim3(grid_of(channels)), kThreads, 0, 1, stream, p);
  if (e != cudaSuccess) return e;
  if (p.dx != nullptr) {
    e = launch_seq(norm_dx_kernel<T, I>, dim3(grid_of((long long)p.N * p.G * chunks_of(p).count)), kThreads, 0, 1, stream, p);
    if (e != cudaSuccess) return e;
  }
  if (p.dweight == nullptr && p.dbias == nullptr) return cudaSuccess;
  return launch_norm_dparams<T>(p, static_cast<const float2*>(p.workspace), p.N, stream);
}

bool small(const NormParams& p) { return (long long)(p.C / p.G) * p.H * p.W < (1ll << 31); }

template <typename T>
cudaError_t forward_t(const NormParams& p, cudaStream_t stream) {
  return small(p) ? forward<T, uint32_t>(p, stream) : forward<T, unsigned long long>(p, stream);
}
template <typename T>
cudaError_t backward_t(const NormParams& p, cudaStream_t stream) {
  return small(p) ? backward<T, uint32_t>(p, stream) : backward<T, unsigned long long>(p, stream);
}

}  // namespace

template <typename T>
cudaError_t launch_norm_dparams(const NormParams& p, const float2* rows, long long count, cudaStream_t stream) {
  return launch_seq(norm_dparams_kernel<T>, dim3(unsigned((p.C + 31) / 32)), 1024, 0, 1, stream, p, rows, count);
}
template cudaError_t launch_norm_dparams<__half>(const NormParams&, const float2*, long long, cudaStream_t);
template cudaError_t launch_norm_dparams<__nv_bfloat16>(const NormParams&, const float2*, long long, cudaStream_t);
template cudaError_t launch_norm_dparams<float>(const NormParams&, const float2*, long long, cudaStream_t);

// Known without the tensors' addresses: the most that any kernel which may take the problem needs.
long long group_norm_workspace(int dtype, const NormParams& p, bool backward) {
  const long long here = 8ll * p.N * (backward ? p.C : p.G * chunks_of(p).count);
  if (!norm_rows(p, backward) || (long long)p.H * p.W > 0x1fffffff) return here;
  const long long images = norm_images_workspace(dtype, p, backward);
  const long long tokens = p.H == 1 && p.W == 1 ? norm_tokens_workspace(dtype, p, backward) : 0;
  // groups that may be wider than a block of the images' kernels has threads
  const long long wide = p.C / p.G > 256 ? here : 0;
  const long long most = tokens > images ? tokens : images;
  return most > wide ? most : wide;
}

cudaError_t launch_group_norm(int dtype, const NormParams& p, cudaStream_t stream) {
  if (norm_tokens_take(dtype, p, false)) return launch_norm_tokens(dtype, p, false, stream);
  if (norm_images_take(dtype, p, false)) return launch_norm_images(dtype, p, false, stream);
  switch (dtype) {
    case FDNN_F16: return forward_t<__half>(p, stream);
    case FDNN_BF16: return forward_t<__nv_bfloat16>(p, stream);
    default: return forward_t<float>(p, stream);
  }
}

cudaError_t launch_group_norm_backward(int dtype, const NormParams& p, cudaStream_t stream) {
  if (norm_tokens_take(dtype, p, true)) return launch_norm_tokens(dtype, p, true, stream);
  if (norm_images_take(dtype, p, true)) return launch_norm_images(dtype, p, true, stream);
  switch (dtype) {
    case FDNN_F16: return backward_t<__half>(p, stream);
    case FDNN_BF16: return backward_t<__nv_bfloat16>(p, stream);
    default: return backward_t<float>(p, stream);
  }
}

}  // namespace fdnn
