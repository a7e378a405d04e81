// The gated feed-forward block's products for bf16 tensors: h and [dg | du] as the tensors' numbers or in two planes.
#include "gated_mlp.h"

namespace cradle {
namespace gated {
int64_t forward_bf16(const cradle_gated_mlp_desc* d, const Plan& p, void* workspace, hipStream_t s, bool run) {
  return (p.nph == 2 ? forward<BF16, 1, 2> : forward<BF16, 1, 1>)(d, p, workspace, s, run);
}
int64_t backward_bf16(const cradle_gated_mlp_desc* d, const Plan& p, void* workspace, hipStream_t s, bool run) {
  return (p.nph == 2 ? backward<BF16, 1, 2> : backward<BF16, 1, 1>)(d, p, workspace, s, run);
}
}  // namespace gated
}  // namespace cradle
