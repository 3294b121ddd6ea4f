// What the gated delta rule's kernels share: a token's decay and step size, and which loads its tensors allow.
#pragma once
#include "group_norm.cuh"

namespace fdnn {

constexpr float kKeyEps = 1e-6f;   // added to a key's sum of squares before its root is taken

// delta or beta of a token.
template <typename T>
__device__ __forceinline__ float gate_at(const DeltaParams& p, const void* gates, long long i) {
  return p.gate_f32 ? static_cast<const float*>(gates)[i] : to_f32<T>(static_cast<const T*>(gates)[i]);
}
// The logarithm of the decay.  Its softplus takes a power from the special function unit, of a rounded argument: below 4e-7 + 8e-8 |dt| of
// itself off (3.7e-7 measured at dt = -8 .. -6).  By expf in its place 2.5e-7, and the next tokens of 128 rows of 32 heads took 97 us in
// place of 90.5: registers, four blocks to an SM.  (Held to five: 94.5, and 57 for 43 with keys of 256 channels.)
__device__ __forceinline__ float log_decay(const DeltaParams& p, float delta, float bias, float A) {
  const float dt = delta + bias;
  return A * (p.softplus ? softplus(dt) : dt);
}
__device__ __forceinline__ float step_size(const DeltaParams& p, float beta) {
  return p.sigmoid ? 1.0f / (1.0f + expf(-beta)) : beta;
}

// Whether four neighbouring channels of a [n, l, head, channel] tensor can be loaded at once.
template <typename T>
bool fours(const void* q, const long long* s) {
  return reinterpret_cast<uintptr_t>(q) % (4 * sizeof(T)) == 0 && s[0] % 4 == 0 && s[1] % 4 == 0 && s[2] % 4 == 0 && s[3] == 1;
}

// Prompts token by token (delta_rule_step.cu).
cudaError_t launch_delta_rule_tokens(int dtype, const DeltaParams& p, cudaStream_t stream);

}  // namespace fdnn
