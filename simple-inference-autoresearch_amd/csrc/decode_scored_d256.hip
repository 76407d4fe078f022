// Decode kernel instantiations with a score function for head_dim 256 (all K/V types; as decode_d256.hip, with AGPRs).
#include "decode_launch.hpp"

namespace sia {

int launch_decode_scored_256(DecodeLaunch& L, int kv_dtype) {
  switch (kv_dtype) {
    case SIA_F16: return launch_decode_scored_q<256, F16, F32>(L);
    case SIA_BF16: return launch_decode_scored_q<256, BF16, F32>(L);
    default: return L.scale_dtype == SIA_F32 ? launch_decode_scored_q<256, I8, F32>(L) : launch_decode_scored_q<256, I8, F16>(L);
  }
}

}  // namespace sia
