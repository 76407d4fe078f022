// Scored attention of few query rows over many keys: the key blocks split over work-groups (variants 3 and 4), head_dim 64
// and 256.
#include "prefill_scored_launch.hpp"

namespace sia {

int launch_prefill_scored_split(PrefillLaunch& L) {
  const bool bf = L.dtype == SIA_BF16;
  if (L.D == 128) return launch_prefill_scored_split_128(L);
  if (L.D == 64 && bf && L.var == 3) return launch_scored_var<64, BF16, 3>(L);
  if (L.D == 64 && !bf && L.var == 4) return launch_scored_var<64, F16, 4>(L);
  if (L.D == 256 && L.var == 4) return bf ? launch_scored_var<256, BF16, 4>(L) : launch_scored_var<256, F16, 4>(L);
  return fail(SIA_ERR_LAUNCH, "prefill variant %d is not built for head_dim %d", L.var, L.D);
}

}  // namespace sia
