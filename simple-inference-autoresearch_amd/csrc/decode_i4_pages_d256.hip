// Decode kernel instantiations for int4 pools with pages of any size, head_dim 256.
#include "decode_launch.hpp"

namespace sia {

int launch_decode_i4_pages_256(DecodeLaunch& L) {
  switch (L.lg_group) {
    case 5: return launch_decode_i4_typed<256, 32, true>(L);
    case 6: return launch_decode_i4_typed<256, 64, true>(L);
    default: return launch_decode_i4_typed<256, 128, true>(L);
  }
}

}  // namespace sia
