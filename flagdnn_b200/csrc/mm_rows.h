// Products of few rows (mm_rows.cu), shared with their C-ABI front end (sequence_api.cu).
#pragma once
#include <cuda_runtime.h>

namespace fdnn {

struct MmRowsParams {
  int M, N, K, act;                                  // a [M, K], b [K, N]
  int a_bytes, b_bytes;                              // set by the launcher: 8, 4, or 0, that lie together and aligned along the reduction
  long long a_s[2], b_s[2], residual_s[2], y_s[2];   // element strides
  const void *a, *b, *bias, *residual;               // bias [N] or null; residual [M, N] or null
  void* y;
};
// Whether that is ahead of the 1x1 convolution.
bool mm_rows_preferred(int dtype, const MmRowsParams& p);
cudaError_t launch_mm_rows(int dtype, const MmRowsParams& p, cudaStream_t stream);

}  // namespace fdnn
