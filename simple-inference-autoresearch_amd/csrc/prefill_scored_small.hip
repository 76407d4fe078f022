// Scored attention of prompts on the matrix cores, head_dim 16 and 32 (compiled separately to build in parallel).
#include "prefill_scored_launch.hpp"

namespace sia {

int launch_prefill_scored_small(PrefillLaunch& L) { return L.D == 16 ? launch_scored_d<16>(L) : launch_scored_d<32>(L); }

}  // namespace sia
