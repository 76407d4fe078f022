// Decode kernel instantiations with a score function for int8 K/V at head_dim 64 and 128.
#include "decode_launch.hpp"

namespace sia {

int launch_decode_scored_i8(DecodeLaunch& L) {
  if (L.scale_dtype == SIA_F32)
    return L.D == 64 ? launch_decode_scored_q<64, I8, F32>(L) : launch_decode_scored_q<128, I8, F32>(L);
  return L.D == 64 ? launch_decode_scored_q<64, I8, F16>(L) : launch_decode_scored_q<128, I8, F16>(L);
}

}  // namespace sia
