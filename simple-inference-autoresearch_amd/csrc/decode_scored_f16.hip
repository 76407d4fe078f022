// Decode kernel instantiations with a score function for f16 K/V at head_dim 64 and 128.
#include "decode_launch.hpp"

namespace sia {

int launch_decode_scored_f16(DecodeLaunch& L) {
  return L.D == 64 ? launch_decode_scored_q<64, F16, F32>(L) : launch_decode_scored_q<128, F16, F32>(L);
}

}  // namespace sia
