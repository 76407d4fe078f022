// Float32 attention of decode calls with a score function (compiled separately to build in parallel).
#include "attn_f32_kernel.hpp"

namespace sia {

int launch_attn_f32_scored(F32Launch& L) { return launch_f32_types<true>(L); }

}  // namespace sia
