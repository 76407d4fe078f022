// Scored attention of prompts on the matrix cores: dispatch, and head_dim 64.
#include "prefill_scored_launch.hpp"

namespace sia {

int launch_prefill_scored(PrefillLaunch& L) {
  switch (L.D) {
    case 16: case 32: return launch_prefill_scored_small(L);
    case 64: return launch_scored_d<64>(L);
    case 128: return launch_prefill_scored_128(L);
    case 256: return launch_prefill_scored_256(L);
    default: return fail(SIA_ERR_UNSUPPORTED, "prefill head_dim %d not supported (16, 32, 64, 128, 256)", L.D);
  }
}

}  // namespace sia
