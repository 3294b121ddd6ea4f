// Internal declarations of the group norm and state space operators (group_norm*.cu, causal_conv.cu, selective_scan*.cu, delta_rule*.cu),
// shared with their C-ABI front end (sequence_api.cu).  Nothing here is exported.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/flagdnn_b200.h"

namespace fdnn {

// Records the text fdnn_last_error() answers on this thread and returns `status` (conv_api.cu).
int api_fail(int status, const char* text);
int api_fail_cuda(const char* what, cudaError_t e);

struct NormParams {
  int N, C, H, W, G;
  int act;               // FDNN_ACT_*
  int param_f32;         // 1: weight, bias and their gradients are float32, 0: of x's type
  float eps;
  long long x_s[4], y_s[4], dy_s[4], dx_s[4];   // element strides in (n, c, h, w) order
  const void *x, *dy, *weight, *bias;
  void *y, *dx, *dweight, *dbias;
  float *mean, *rstd;    // [N, G]; forward: written if not null, backward: read
  void* workspace;
  long long workspace_bytes;   // every launcher compares it with what it is about to write
};
long long group_norm_workspace(int dtype, const NormParams& p, bool backward);
cudaError_t launch_group_norm(int dtype, const NormParams& p, cudaStream_t stream);
cudaError_t launch_group_norm_backward(int dtype, const NormParams& p, cudaStream_t stream);

struct CausalConvParams {
  int N, L, C, width, act;
  long long x_s[3], y_s[3];         // element strides in (n, l, c) order
  const void *x, *weight, *bias;    // weight [C, width], bias [C] or null
  const void* initial;              // [N, width - 1, C] or null (zeros)
  const int* lengths;               // [N] or null
  void *y, *final_state;            // final_state [N, width - 1, C] or null
};
cudaError_t launch_causal_conv(int dtype, const CausalConvParams& p, cudaStream_t stream);
// One token a row: x [N, C] with strides x_s[0], x_s[2]; state [n_slots, width - 1, C] in place.
cudaError_t launch_causal_conv_step(int dtype, const CausalConvParams& p, void* state, int n_slots, const int* slots,
                                    cudaStream_t stream);

struct ScanParams {
  int N, L, C, S, G;
  int softplus;
  long long u_s[3], delta_s[3], z_s[3], y_s[3];   // element strides in (n, l, c) order
  long long b_s[4], c_s[4];                       // (n, l, group, state)
  const void *u, *delta, *B, *Cm, *z;             // z or null
  const float *A, *D, *delta_bias;                // A [C, S]; D, delta_bias [C] or null
  const float* initial;                           // [N, C, S] or null (zeros)
  const int* lengths;                             // [N] or null
  void* y;
  float* final_state;                             // [N, C, S] or null
  void* workspace;
};
long long selective_scan_workspace(int dtype, const ScanParams& p);
cudaError_t launch_selective_scan(int dtype, const ScanParams& p, cudaStream_t stream);
// One token a row (l strides unused): state [n_slots, C, S] in place.
cudaError_t launch_selective_scan_step(int dtype, const ScanParams& p, float* state, int n_slots, const int* slots,
                                       cudaStream_t stream);

struct DeltaParams {
  int N, L, G, H, K, V;                           // G key heads, H heads; K = dk, V = dv
  int gate_f32;                                   // 1: delta and beta are float32, 0: of q's type
  int softplus, sigmoid, norm;
  float scale;
  long long q_s[4], k_s[4], v_s[4], y_s[4];       // element strides in (n, l, head, channel) order
  long long delta_s[3], beta_s[3];                // (n, l, head)
  const void *q, *k, *v, *delta, *beta;
  const float *A, *delta_bias;                    // [H] or null
  const float* initial;                           // [N, H, V, K] or null (zeros)
  const int* lengths;                             // [N] or null
  void* y;
  float* final_state;                             // [N, H, V, K] or null
  void* workspace;
};
long long delta_rule_workspace(int dtype, const DeltaParams& p);
cudaError_t launch_delta_rule(int dtype, const DeltaParams& p, cudaStream_t stream);
// One token a row (l strides unused): state [n_slots, H, V, K] in place.
cudaError_t launch_delta_rule_step(int dtype, const DeltaParams& p, float* state, int n_slots, const int* slots,
                                   cudaStream_t stream);

}  // namespace fdnn
