// Decode kernel instantiations for int4 pools with pages of any size, head_dim 64 and 128.
#include "decode_launch.hpp"

namespace sia {

int launch_decode_i4_pages(DecodeLaunch& L) {
  if (L.D == 256) return launch_decode_i4_pages_256(L);
  if (L.D == 64)
    return L.lg_group == 5 ? launch_decode_i4_typed<64, 32, true>(L) : launch_decode_i4_typed<64, 64, true>(L);
  switch (L.lg_group) {
    case 5: return launch_decode_i4_typed<128, 32, true>(L);
    case 6: return launch_decode_i4_typed<128, 64, true>(L);
    default: return launch_decode_i4_typed<128, 128, true>(L);
  }
}

}  // namespace sia
