// The gated feed-forward block's products for fp32 tensors, as three bf16 planes.
#include "gated_mlp.h"

namespace cradle {
namespace gated {
int64_t forward_f32(const cradle_gated_mlp_desc* d, const Plan& p, void* workspace, hipStream_t s, bool run) {
  return forward<BF16, 3, 3>(d, p, workspace, s, run);
}
int64_t backward_f32(const cradle_gated_mlp_desc* d, const Plan& p, void* workspace, hipStream_t s, bool run) {
  return backward<BF16, 3, 3>(d, p, workspace, s, run);
}
}  // namespace gated
}  // namespace cradle
