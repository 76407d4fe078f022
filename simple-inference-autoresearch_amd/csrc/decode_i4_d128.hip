// Decode kernel instantiations for int4 K/V at head_dim 128.
#include "decode_launch.hpp"

namespace sia {

int launch_decode_i4_128(DecodeLaunch& L) {
  switch (L.lg_group) {
    case 5: return launch_decode_i4_typed<128, 32>(L);
    case 6: return launch_decode_i4_typed<128, 64>(L);
    default: return launch_decode_i4_typed<128, 128>(L);
  }
}

}  // namespace sia
