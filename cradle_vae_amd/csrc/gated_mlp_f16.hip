// The gated feed-forward block's products for fp16 tensors.
#include "gated_mlp.h"

namespace cradle {
namespace gated {
int64_t forward_f16(const cradle_gated_mlp_desc* d, const Plan& p, void* workspace, hipStream_t s, bool run) {
  return forward<F16, 1>(d, p, workspace, s, run);
}
int64_t backward_f16(const cradle_gated_mlp_desc* d, const Plan& p, void* workspace, hipStream_t s, bool run) {
  return backward<F16, 1>(d, p, workspace, s, run);
}
}  // namespace gated
}  // namespace cradle
