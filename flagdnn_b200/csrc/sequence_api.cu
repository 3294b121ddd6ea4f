// C-ABI front end of the group norm, state space and delta rule operators and of products of few rows: validation and launches.  See include/flagdnn_b200.h.
#include "mm_rows.h"
#include "sequence_internal.h"

using namespace fdnn;

namespace {

constexpr int32_t kMaxTokens = 0x7fffffff - 1024;   // tiles past a row's end are counted in 32 bits
// Rows (images) past the last are counted in 32 bits: at most 1024 side by side in a block, or a stride of sixteen blocks an SM.
constexpr int32_t kMaxRows = 0x7fffffff - 65536;

bool float_type(int dtype) { return dtype == FDNN_F16 || dtype == FDNN_BF16 || dtype == FDNN_F32; }

int norm_params(const fdnn_norm_desc* d, NormParams* p) {
  if (d == nullptr) return api_fail(FDNN_BAD_PARAM, "descriptor is NULL");
  if (!float_type(d->dtype)) return api_fail(FDNN_NOT_SUPPORTED, "Unsupported dtype");
  if (d->param_dtype != d->dtype && d->param_dtype != FDNN_F32)
    return api_fail(FDNN_NOT_SUPPORTED, "weight and bias must be of the input's type or float32");
  if (d->n < 0 || d->c <= 0 || d->h < 0 || d->w < 0) return api_fail(FDNN_BAD_PARAM, "negative extent");
  if (d->n > kMaxRows) return api_fail(FDNN_NOT_SUPPORTED, "more rows than the kernels count");
  if (d->groups <= 0 || d->c % d->groups != 0) return api_fail(FDNN_BAD_PARAM, "channels must be divisible by groups");
  if (d->activation < FDNN_ACT_NONE || d->activation > FDNN_ACT_SILU) return api_fail(FDNN_BAD_PARAM, "unknown activation");
  if (!(d->eps >= 0.0f)) return api_fail(FDNN_BAD_PARAM, "eps must not be negative");
  p->N = d->n; p->C = d->c; p->H = d->h; p->W = d->w; p->G = d->groups;
  p->act = d->activation;
  p->param_f32 = d->param_dtype == FDNN_F32;
  p->eps = d->eps;
  for (int i = 0; i < 4; ++i) {
    p->x_s[i] = d->x_strides[i];
    p->y_s[i] = d->y_strides[i];
    p->dy_s[i] = d->dy_strides[i];
    p->dx_s[i] = d->dx_strides[i];
  }
  p->x = p->dy = p->weight = p->bias = nullptr;
  p->y = p->dx = p->dweight = p->dbias = nullptr;
  p->mean = p->rstd = nullptr;
  p->workspace = nullptr;
  p->workspace_bytes = 0;
  return FDNN_OK;
}

bool empty(const NormParams& p) { return p.N == 0 || p.H == 0 || p.W == 0; }

int check_workspace(const void* workspace, int64_t bytes, long long needed) {
  if (needed == 0) return FDNN_OK;
  if (workspace == nullptr || bytes < needed) return api_fail(FDNN_WORKSPACE_TOO_SMALL, "workspace smaller than the call needs");
  if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return api_fail(FDNN_BAD_PARAM, "workspace must be 16-byte aligned");
  return FDNN_OK;
}

int causal_params(const fdnn_causal_conv_desc* d, CausalConvParams* p) {
  if (d == nullptr) return api_fail(FDNN_BAD_PARAM, "descriptor is NULL");
  if (!float_type(d->dtype)) return api_fail(FDNN_NOT_SUPPORTED, "Unsupported dtype");
  if (d->n < 0 || d->l < 0 || d->c < 0) return api_fail(FDNN_BAD_PARAM, "negative extent");
  if (d->l > kMaxTokens) return api_fail(FDNN_NOT_SUPPORTED, "more tokens in a row than the kernels count");
  if (d->width < 1 || d->width > FDNN_CAUSAL_CONV_MAX_WIDTH) return api_fail(FDNN_NOT_SUPPORTED, "the filter must have 1 to 8 taps");
  if (d->activation < FDNN_ACT_NONE || d->activation > FDNN_ACT_SILU) return api_fail(FDNN_BAD_PARAM, "unknown activation");
  p->N = d->n; p->L = d->l; p->C = d->c; p->width = d->width; p->act = d->activation;
  for (int i = 0; i < 3; ++i) {
    p->x_s[i] = d->x_strides[i];
    p->y_s[i] = d->y_strides[i];
  }
  return FDNN_OK;
}

int scan_params(const fdnn_scan_desc* d, ScanParams* p) {
  if (d == nullptr) return api_fail(FDNN_BAD_PARAM, "descriptor is NULL");
  if (!float_type(d->dtype)) return api_fail(FDNN_NOT_SUPPORTED, "Unsupported dtype");
  if (d->n < 0 || d->l < 0 || d->c < 0) return api_fail(FDNN_BAD_PARAM, "negative extent");
  if (d->l > kMaxTokens) return api_fail(FDNN_NOT_SUPPORTED, "more tokens in a row than the kernels count");
  if (d->s < 1 || d->s > FDNN_SCAN_MAX_STATES) return api_fail(FDNN_NOT_SUPPORTED, "a channel must have 1 to 256 states");
  if (d->groups <= 0 || d->c % d->groups != 0) return api_fail(FDNN_BAD_PARAM, "channels must be divisible by groups");
  p->N = d->n; p->L = d->l; p->C = d->c; p->S = d->s; p->G = d->groups;
  p->softplus = d->delta_softplus != 0;
  for (int i = 0; i < 3; ++i) {
    p->u_s[i] = d->u_strides[i];
    p->delta_s[i] = d->delta_strides[i];
    p->z_s[i] = d->z_strides[i];
    p->y_s[i] = d->y_strides[i];
  }
  for (int i = 0; i < 4; ++i) {
    p->b_s[i] = d->b_strides[i];
    p->c_s[i] = d->c_strides[i];
  }
  p->initial = nullptr;
  p->lengths = nullptr;
  p->final_state = nullptr;
  p->workspace = nullptr;
  return FDNN_OK;
}

int delta_params(const fdnn_delta_rule_desc* d, DeltaParams* p) {
  if (d == nullptr) return api_fail(FDNN_BAD_PARAM, "descriptor is NULL");
  if (!float_type(d->dtype)) return api_fail(FDNN_NOT_SUPPORTED, "Unsupported dtype");
  if (d->gate_dtype != d->dtype && d->gate_dtype != FDNN_F32)
    return api_fail(FDNN_NOT_SUPPORTED, "delta and beta must be of the input's type or float32");
  if (d->n < 0 || d->l < 0 || d->heads < 0) return api_fail(FDNN_BAD_PARAM, "negative extent");
  if (d->l > kMaxTokens) return api_fail(FDNN_NOT_SUPPORTED, "more tokens in a row than the kernels count");
  if (d->n > kMaxRows) return api_fail(FDNN_NOT_SUPPORTED, "more rows than the kernels count");
  if (d->dk < 1 || d->dk > FDNN_DELTA_RULE_MAX_DK) return api_fail(FDNN_NOT_SUPPORTED, "a key must have 1 to 256 channels");
  if (d->dv < 1 || d->dv > FDNN_DELTA_RULE_MAX_DV) return api_fail(FDNN_NOT_SUPPORTED, "a value must have 1 to 1024 channels");
  if (d->heads > FDNN_DELTA_RULE_MAX_HEADS) return api_fail(FDNN_NOT_SUPPORTED, "more heads than the kernels count");
  if (d->key_heads <= 0 || d->heads % d->key_heads != 0) return api_fail(FDNN_BAD_PARAM, "heads must be divisible by key heads");
  p->N = d->n; p->L = d->l; p->G = d->key_heads; p->H = d->heads; p->K = d->dk; p->V = d->dv;
  p->gate_f32 = d->gate_dtype == FDNN_F32;
  p->softplus = d->delta_softplus != 0;
  p->sigmoid = d->beta_sigmoid != 0;
  p->norm = d->qk_norm != 0;
  p->scale = d->scale;
  for (int i = 0; i < 4; ++i) {
    p->q_s[i] = d->q_strides[i];
    p->k_s[i] = d->k_strides[i];
    p->v_s[i] = d->v_strides[i];
    p->y_s[i] = d->y_strides[i];
  }
  for (int i = 0; i < 3; ++i) {
    p->delta_s[i] = d->delta_strides[i];
    p->beta_s[i] = d->beta_strides[i];
  }
  p->initial = nullptr;
  p->lengths = nullptr;
  p->final_state = nullptr;
  p->workspace = nullptr;
  return FDNN_OK;
}

int mm_params(const fdnn_mm_desc* d, MmRowsParams* p) {
  if (d == nullptr) return api_fail(FDNN_BAD_PARAM, "descriptor is NULL");
  if (!float_type(d->dtype)) return api_fail(FDNN_NOT_SUPPORTED, "Unsupported dtype");
  if (d->m < 0 || d->n < 0 || d->k < 0) return api_fail(FDNN_BAD_PARAM, "negative extent");
  if (d->activation < FDNN_ACT_NONE || d->activation > FDNN_ACT_GELU_TANH) return api_fail(FDNN_BAD_PARAM, "unknown activation");
  if (d->m > 1 << 22 || d->n > kMaxTokens || d->k > kMaxTokens) return api_fail(FDNN_NOT_SUPPORTED, "an extent is more than the kernels count");
  p->M = d->m; p->N = d->n; p->K = d->k; p->act = d->activation;
  for (int i = 0; i < 2; ++i) {
    p->a_s[i] = d->a_strides[i];
    p->b_s[i] = d->b_strides[i];
    p->residual_s[i] = d->residual_strides[i];
    p->y_s[i] = d->y_strides[i];
  }
  return FDNN_OK;
}

}  // namespace

extern "C" {

int fdnn_group_norm_workspace_bytes(const fdnn_norm_desc* desc, int backward, int64_t* bytes) {
  if (bytes == nullptr) return api_fail(FDNN_BAD_PARAM, "bytes is NULL");
  NormParams p;
  const int st = norm_params(desc, &p);
  if (st != FDNN_OK) return st;
  *bytes = empty(p) ? 0 : group_norm_workspace(desc->dtype, p, backward != 0);
  return FDNN_OK;
}

int fdnn_group_norm_fwd(const fdnn_norm_desc* desc, const void* x, const void* weight, const void* bias, void* y, float* mean,
                        float* rstd, void* workspace, int64_t workspace_bytes, void* stream) {
  NormParams p;
  int st = norm_params(desc, &p);
  if (st != FDNN_OK) return st;
  if ((mean == nullptr) != (rstd == nullptr)) return api_fail(FDNN_BAD_PARAM, "mean and rstd come together");
  if (empty(p)) return FDNN_OK;
  if (x == nullptr || y == nullptr) return api_fail(FDNN_BAD_PARAM, "x and y must not be NULL");
  st = check_workspace(workspace, workspace_bytes, group_norm_workspace(desc->dtype, p, false));
  if (st != FDNN_OK) return st;
  p.x = x; p.weight = weight; p.bias = bias; p.y = y; p.mean = mean; p.rstd = rstd; p.workspace = workspace; p.workspace_bytes = workspace_bytes;
  const cudaError_t e = launch_group_norm(desc->dtype, p, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? FDNN_OK : api_fail_cuda("group_norm launch", e);
}

int fdnn_group_norm_bwd(const fdnn_norm_desc* desc, const void* dy, const void* x, const float* mean, const float* rstd,
                        const void* weight, const void* bias, void* dx, void* dweight, void* dbias, void* workspace,
                        int64_t workspace_bytes, void* stream) {
  NormParams p;
  int st = norm_params(desc, &p);
  if (st != FDNN_OK) return st;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (empty(p)) {   // sums over nothing
    const size_t es = p.param_f32 || desc->dtype == FDNN_F32 ? 4 : 2;
    for (void* d : {dweight, dbias})
      if (d != nullptr) {
        const cudaError_t e = cudaMemsetAsync(d, 0, es * size_t(p.C), s);
        if (e != cudaSuccess) return api_fail_cuda("group_norm gradient of nothing", e);
      }
    return FDNN_OK;
  }
  if (dy == nullptr || x == nullptr || mean == nullptr || rstd == nullptr)
    return api_fail(FDNN_BAD_PARAM, "dy, x, mean and rstd must not be NULL");
  st = check_workspace(workspace, workspace_bytes, group_norm_workspace(desc->dtype, p, true));
  if (st != FDNN_OK) return st;
  p.x = x; p.dy = dy; p.weight = weight; p.bias = bias; p.dx = dx; p.dweight = dweight; p.dbias = dbias;
  p.mean = const_cast<float*>(mean); p.rstd = const_cast<float*>(rstd); p.workspace = workspace; p.workspace_bytes = workspace_bytes;
  const cudaError_t e = launch_group_norm_backward(desc->dtype, p, s);
  return e == cudaSuccess ? FDNN_OK : api_fail_cuda("group_norm backward launch", e);
}

int fdnn_causal_conv1d_fwd(const fdnn_causal_conv_desc* desc, const void* x, const void* weight, const void* bias,
                           const void* initial_state, const int32_t* lengths, void* y, void* final_state, void* stream) {
  CausalConvParams p;
  const int st = causal_params(desc, &p);
  if (st != FDNN_OK) return st;
  if (p.N == 0 || p.C == 0) return FDNN_OK;
  if (weight == nullptr) return api_fail(FDNN_BAD_PARAM, "weight must not be NULL");
  if (p.L > 0 && (x == nullptr || y == nullptr)) return api_fail(FDNN_BAD_PARAM, "x and y must not be NULL");
  p.x = x; p.weight = weight; p.bias = bias; p.initial = initial_state; p.lengths = lengths; p.y = y; p.final_state = final_state;
  const cudaError_t e = launch_causal_conv(desc->dtype, p, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? FDNN_OK : api_fail_cuda("causal_conv1d launch", e);
}

int fdnn_causal_conv1d_step(const fdnn_causal_conv_desc* desc, const void* x, const void* weight, const void* bias, void* state,
                            int32_t n_slots, const int32_t* slots, void* y, void* stream) {
  CausalConvParams p;
  const int st = causal_params(desc, &p);
  if (st != FDNN_OK) return st;
  if (p.N == 0 || p.C == 0) return FDNN_OK;
  if (n_slots < 0 || (slots == nullptr && n_slots < p.N)) return api_fail(FDNN_BAD_PARAM, "fewer states than rows");
  if (x == nullptr || y == nullptr || weight == nullptr || (state == nullptr && p.width > 1 && n_slots > 0))
    return api_fail(FDNN_BAD_PARAM, "x, y, weight and state must not be NULL");
  p.x = x; p.weight = weight; p.bias = bias; p.initial = nullptr; p.lengths = nullptr; p.y = y; p.final_state = nullptr;
  const cudaError_t e = launch_causal_conv_step(desc->dtype, p, state, n_slots, slots, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? FDNN_OK : api_fail_cuda("causal_conv1d_step launch", e);
}

int fdnn_selective_scan_workspace_bytes(const fdnn_scan_desc* desc, int64_t* bytes) {
  if (bytes == nullptr) return api_fail(FDNN_BAD_PARAM, "bytes is NULL");
  ScanParams p;
  const int st = scan_params(desc, &p);
  if (st != FDNN_OK) return st;
  *bytes = p.N == 0 || p.C == 0 || p.L == 0 ? 0 : selective_scan_workspace(desc->dtype, p);
  return FDNN_OK;
}

int fdnn_selective_scan_fwd(const fdnn_scan_desc* desc, const void* u, const void* delta, const float* A, const void* B, const void* C,
                            const float* D, const void* z, const float* delta_bias, const float* initial_state,
                            const int32_t* lengths, void* y, float* final_state, void* workspace, int64_t workspace_bytes,
                            void* stream) {
  ScanParams p;
  int st = scan_params(desc, &p);
  if (st != FDNN_OK) return st;
  if (p.N == 0 || p.C == 0) return FDNN_OK;
  if (A == nullptr) return api_fail(FDNN_BAD_PARAM, "A must not be NULL");
  if (p.L > 0 && (u == nullptr || delta == nullptr || B == nullptr || C == nullptr || y == nullptr))
    return api_fail(FDNN_BAD_PARAM, "u, delta, B, C and y must not be NULL");
  if (p.L > 0) {
    st = check_workspace(workspace, workspace_bytes, selective_scan_workspace(desc->dtype, p));
    if (st != FDNN_OK) return st;
  }
  p.u = u; p.delta = delta; p.A = A; p.B = B; p.Cm = C; p.D = D; p.z = z; p.delta_bias = delta_bias;
  p.initial = initial_state; p.lengths = lengths; p.y = y; p.final_state = final_state; p.workspace = workspace;
  const cudaError_t e = launch_selective_scan(desc->dtype, p, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? FDNN_OK : api_fail_cuda("selective_scan launch", e);
}

int fdnn_selective_scan_step(const fdnn_scan_desc* desc, const void* u, const void* delta, const float* A, const void* B,
                             const void* C, const float* D, const void* z, const float* delta_bias, float* state, int32_t n_slots,
                             const int32_t* slots, void* y, void* stream) {
  ScanParams p;
  const int st = scan_params(desc, &p);
  if (st != FDNN_OK) return st;
  if (p.N == 0 || p.C == 0) return FDNN_OK;
  if (p.N > kMaxRows) return api_fail(FDNN_NOT_SUPPORTED, "more rows than the kernels count");
  if (n_slots < 0 || (slots == nullptr && n_slots < p.N)) return api_fail(FDNN_BAD_PARAM, "fewer states than rows");
  if (u == nullptr || delta == nullptr || A == nullptr || B == nullptr || C == nullptr || y == nullptr || (state == nullptr && n_slots > 0))
    return api_fail(FDNN_BAD_PARAM, "u, delta, A, B, C, state and y must not be NULL");
  p.u = u; p.delta = delta; p.A = A; p.B = B; p.Cm = C; p.D = D; p.z = z; p.delta_bias = delta_bias; p.y = y;
  const cudaError_t e = launch_selective_scan_step(desc->dtype, p, state, n_slots, slots, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? FDNN_OK : api_fail_cuda("selective_scan_step launch", e);
}

int fdnn_gated_delta_rule_workspace_bytes(const fdnn_delta_rule_desc* desc, int64_t* bytes) {
  if (bytes == nullptr) return api_fail(FDNN_BAD_PARAM, "bytes is NULL");
  DeltaParams p;
  const int st = delta_params(desc, &p);
  if (st != FDNN_OK) return st;
  *bytes = p.N == 0 || p.H == 0 || p.L == 0 ? 0 : delta_rule_workspace(desc->dtype, p);
  return FDNN_OK;
}

int fdnn_gated_delta_rule_fwd(const fdnn_delta_rule_desc* desc, const void* q, const void* k, const void* v, const void* delta,
                              const void* beta, const float* A, const float* delta_bias, const float* initial_state,
                              const int32_t* lengths, void* y, float* final_state, void* workspace, int64_t workspace_bytes,
                              void* stream) {
  DeltaParams p;
  int st = delta_params(desc, &p);
  if (st != FDNN_OK) return st;
  if (p.N == 0 || p.H == 0) return FDNN_OK;
  if (p.L > 0) {
    if (q == nullptr || k == nullptr || v == nullptr || delta == nullptr || beta == nullptr || y == nullptr)
      return api_fail(FDNN_BAD_PARAM, "q, k, v, delta, beta and y must not be NULL");
    st = check_workspace(workspace, workspace_bytes, delta_rule_workspace(desc->dtype, p));
    if (st != FDNN_OK) return st;
  }
  p.q = q; p.k = k; p.v = v; p.delta = delta; p.beta = beta; p.A = A; p.delta_bias = delta_bias;
  p.initial = initial_state; p.lengths = lengths; p.y = y; p.final_state = final_state; p.workspace = workspace;
  const cudaError_t e = launch_delta_rule(desc->dtype, p, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? FDNN_OK : api_fail_cuda("gated_delta_rule launch", e);
}

int fdnn_gated_delta_rule_step(const fdnn_delta_rule_desc* desc, const void* q, const void* k, const void* v, const void* delta,
                               const void* beta, const float* A, const float* delta_bias, float* state, int32_t n_slots,
                               const int32_t* slots, void* y, void* stream) {
  DeltaParams p;
  const int st = delta_params(desc, &p);
  if (st != FDNN_OK) return st;
  if (p.N == 0 || p.H == 0) return FDNN_OK;
  if (n_slots < 0 || (slots == nullptr && n_slots < p.N)) return api_fail(FDNN_BAD_PARAM, "fewer states than rows");
  if (q == nullptr || k == nullptr || v == nullptr || delta == nullptr || beta == nullptr || y == nullptr || (state == nullptr && n_slots > 0))
    return api_fail(FDNN_BAD_PARAM, "q, k, v, delta, beta, state and y must not be NULL");
  p.q = q; p.k = k; p.v = v; p.delta = delta; p.beta = beta; p.A = A; p.delta_bias = delta_bias; p.y = y;
  const cudaError_t e = launch_delta_rule_step(desc->dtype, p, state, n_slots, slots, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? FDNN_OK : api_fail_cuda("gated_delta_rule_step launch", e);
}

int fdnn_mm_rows_preferred(const fdnn_mm_desc* desc, int32_t* preferred) {
  if (preferred == nullptr) return api_fail(FDNN_BAD_PARAM, "preferred is NULL");
  MmRowsParams p;
  const int st = mm_params(desc, &p);
  if (st != FDNN_OK) return st;
  *preferred = mm_rows_preferred(desc->dtype, p);
  return FDNN_OK;
}

int fdnn_mm_rows_fwd(const fdnn_mm_desc* desc, const void* a, const void* b, const void* bias, const void* residual, void* y,
                     void* stream) {
  MmRowsParams p;
  const int st = mm_params(desc, &p);
  if (st != FDNN_OK) return st;
  if (p.M == 0 || p.N == 0) return FDNN_OK;
  if (y == nullptr || (p.K > 0 && (a == nullptr || b == nullptr))) return api_fail(FDNN_BAD_PARAM, "a, b and y must not be NULL");
  p.a = a; p.b = b; p.bias = bias; p.residual = residual; p.y = y;
  const cudaError_t e = launch_mm_rows(desc->dtype, p, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? FDNN_OK : api_fail_cuda("mm_rows launch", e);
}

}  // extern "C"
