// Scored attention of few query rows over many keys, head_dim 128 (compiled separately to build in parallel).
#include "prefill_scored_launch.hpp"

namespace sia {

int launch_prefill_scored_split_128(PrefillLaunch& L) {
  const bool bf = L.dtype == SIA_BF16;
  if (L.var == 3) return bf ? launch_scored_var<128, BF16, 3>(L) : launch_scored_var<128, F16, 3>(L);
  if (L.var == 4 && bf) return launch_scored_var<128, BF16, 4>(L);
  return fail(SIA_ERR_LAUNCH, "prefill variant %d is not built for head_dim %d", L.var, L.D);
}

}  // namespace sia
