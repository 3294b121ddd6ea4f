// What the group norm kernels for channels-last tensors share: vectors of neighbouring channels, and which width a tensor allows.
#pragma once
#include "sequence_internal.h"
#include "sequence_launch.h"
#include "sequence_math.cuh"

namespace fdnn {

// V neighbouring values, moved at once.
template <typename T, int V>
struct Pack {
  static constexpr int kBytes = V * int(sizeof(T));
  using Word = std::conditional_t<kBytes == 16, uint4, std::conditional_t<kBytes == 8, uint2, std::conditional_t<kBytes == 4, uint32_t, uint16_t>>>;
  Word q;
  __device__ __forceinline__ void clear() { q = Word{}; }
  __device__ __forceinline__ void load(const T* p) { q = __ldg(reinterpret_cast<const Word*>(p)); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Word*>(p) = q; }
  __device__ __forceinline__ float at(int j) const { return to_f32<T>(reinterpret_cast<const T*>(&q)[j]); }
  __device__ __forceinline__ void set(int j, float v) { reinterpret_cast<T*>(&q)[j] = from_f32<T>(v); }
};

// Whether the channels lie together and the pixels at one stride, in x and in what goes with it.
inline bool norm_rows(const NormParams& p, bool backward) {
  const long long* s[3] = {p.x_s, backward ? p.dy_s : p.y_s, p.dx_s};
  for (int i = 0; i < (backward ? 3 : 2); ++i)
    if ((s[i][1] != 1 && p.C > 1) || (p.H > 1 && p.W > 1 && s[i][2] != p.W * s[i][3])) return false;
  return true;
}

// The widest vector of channels (16 bytes, 4 bytes or one value) that `run` neighbouring channels are whole numbers of and
// every address is a multiple of; 0 where norm_rows() does not hold.
inline int norm_vector(int dtype, const NormParams& p, bool backward, int run) {
  const int es = dtype == FDNN_F32 ? 4 : 2;
  const void* q[3] = {p.x, backward ? p.dy : p.y, backward ? p.dx : nullptr};
  const long long* s[3] = {p.x_s, backward ? p.dy_s : p.y_s, p.dx_s};
  if (!norm_rows(p, backward)) return 0;
  for (int bytes = 16; bytes >= es; bytes = bytes == 16 ? (es == 4 ? 8 : 4) : bytes / 2) {
    const int v = bytes / es;
    bool ok = run % v == 0;
    for (int i = 0; i < 3; ++i)
      if (q[i] != nullptr)
        ok = ok && reinterpret_cast<uintptr_t>(q[i]) % bytes == 0 && s[i][0] % v == 0 && (p.H == 1 || s[i][2] % v == 0) &&
             (p.W == 1 || s[i][3] % v == 0);
    if (ok) return v;
  }
  return 0;
}

template <typename T>
struct TypeOf {
  using type = T;
};
// f(TypeOf<T>, integral_constant<int, V>) for a run-time type and vector width.
template <typename F>
cudaError_t norm_by_vector(int dtype, int v, F&& f) {
  auto go = [&](auto type, auto widest) -> cudaError_t {
    constexpr int kMost = decltype(widest)::value;
    if (v == kMost) return f(type, std::integral_constant<int, kMost>{});
    if (v == 2) return f(type, std::integral_constant<int, 2>{});
    return f(type, std::integral_constant<int, 1>{});
  };
  if (dtype == FDNN_F16) return go(TypeOf<__half>{}, std::integral_constant<int, 8>{});
  if (dtype == FDNN_BF16) return go(TypeOf<__nv_bfloat16>{}, std::integral_constant<int, 8>{});
  return go(TypeOf<float>{}, std::integral_constant<int, 4>{});
}

// dweight and dbias from `count` rows of [C] pairs, added in their order (group_norm.cu).
template <typename T>
cudaError_t launch_norm_dparams(const NormParams& p, const float2* rows, long long count, cudaStream_t stream);

// group_norm_tokens.cu: rows of tokens
bool norm_tokens_take(int dtype, const NormParams& p, bool backward);
long long norm_tokens_workspace(int dtype, const NormParams& p, bool backward);
cudaError_t launch_norm_tokens(int dtype, const NormParams& p, bool backward, cudaStream_t stream);

// group_norm_images.cu: images, and rows of tokens in wide groups
bool norm_images_take(int dtype, const NormParams& p, bool backward);
long long norm_images_workspace(int dtype, const NormParams& p, bool backward);
cudaError_t launch_norm_images(int dtype, const NormParams& p, bool backward, cudaStream_t stream);

}  // namespace fdnn
