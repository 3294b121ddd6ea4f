// The gated delta rule over prompts.
#include "delta_rule.cuh"

namespace fdnn {

long long delta_rule_workspace(int, const DeltaParams&) { return 0; }

cudaError_t launch_delta_rule(int dtype, const DeltaParams& p, cudaStream_t stream) {
  return launch_delta_rule_tokens(dtype, p, stream);
}

}  // namespace fdnn
