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
  // Values 2 i and 2 i + 1 as fp32 (of a single value: it and zero).
  static constexpr int kPairs = (V + 1) / 2;
  __device__ __forceinline__ F2 pair(int i) const {
    if constexpr (V == 1) {
      return f2_pack(at(0), 0.0f);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const uint32_t w = reinterpret_cast<const uint32_t*>(&q)[i];
      return f2_make(w << 16, w & 0xffff0000u);
    } else {
      return f2_pack(at(2 * i), at(2 * i + 1));
    }
  }
  __device__ __forceinline__ void set_pair(int i, F2 v) {
    float lo, hi;
    f2_split(v, lo, hi);
    if constexpr (V == 1) {
      set(0, lo);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
      reinterpret_cast<uint32_t*>(&q)[i] = *reinterpret_cast<const uint32_t*>(&b);
    } else if constexpr (std::is_same<T, __half>::value) {
      const __half2 b = __floats2half2_rn(lo, hi);
      reinterpret_cast<uint32_t*>(&q)[i] = *reinterpret_cast<const uint32_t*>(&b);
    } else {
      set(2 * i, lo);
      set(2 * i + 1, hi);
    }
  }
};

// A vector on its way into shared memory while the thread works on: zeros where it is not `there` (`from` is then any valid
// address). What a thread has asked for it may read after async_wait(); nobody else may.
template <typename T, int V>
__device__ __forceinline__ void async_load(Pack<T, V>* to, const T* from, bool there) {
  const uint32_t at = uint32_t(__cvta_generic_to_shared(to));
  if constexpr (Pack<T, V>::kBytes == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(from), "r"(there ? 16 : 0) : "memory");
  } else if constexpr (Pack<T, V>::kBytes >= 4) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(at), "l"(from), "n"(Pack<T, V>::kBytes),
                 "r"(there ? Pack<T, V>::kBytes : 0)
                 : "memory");
  } else {   // (two bytes cannot be copied asynchronously)
    to->clear();
    if (there) to->load(from);
  }
}
__device__ __forceinline__ void async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the newest N groups of this thread have arrived.
template <int N>
__device__ __forceinline__ void async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A thread's parameters as pairs.
template <typename T, int V>
__device__ __forceinline__ void norm_params_of(const NormParams& p, int c, bool live, F2 (&w)[Pack<T, V>::kPairs], F2 (&b)[Pack<T, V>::kPairs]) {
#pragma unroll
  for (int i = 0; i < Pack<T, V>::kPairs; ++i) {
    float wv[2], bv[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const bool in = live && 2 * i + j < V;
      wv[j] = in && p.weight != nullptr ? param<T>(p.weight, p.param_f32, c + 2 * i + j) : 1.0f;
      bv[j] = in && p.bias != nullptr ? param<T>(p.bias, p.param_f32, c + 2 * i + j) : 0.0f;
    }
    w[i] = f2_pack(wv[0], wv[1]);
    b[i] = f2_pack(bv[0], bv[1]);
  }
}

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
