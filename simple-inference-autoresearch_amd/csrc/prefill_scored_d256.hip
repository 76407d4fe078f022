// Scored attention of prompts on the matrix cores, head_dim 256 (compiled separately to build in parallel).
#include "prefill_scored_launch.hpp"

namespace sia {

int launch_prefill_scored_256(PrefillLaunch& L) { return launch_scored_d<256>(L); }

}  // namespace sia
