// Scored attention of prompts on the matrix cores, head_dim 128 (compiled separately to build in parallel).
#include "prefill_scored_launch.hpp"

namespace sia {

int launch_prefill_scored_128(PrefillLaunch& L) { return launch_scored_d<128>(L); }

}  // namespace sia
