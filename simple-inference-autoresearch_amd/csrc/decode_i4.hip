// Decode kernel instantiations for int4 K/V at head_dim 64, and the choice by head_dim.
#include "decode_launch.hpp"

namespace sia {

int launch_decode_i4(DecodeLaunch& L) {
  if (L.q_dtype == SIA_F32) return launch_decode_i4_f32(L);
  if (L.a.page > 0) return launch_decode_i4_pages(L);
  switch (L.D) {
    case 64: return L.lg_group == 5 ? launch_decode_i4_typed<64, 32>(L) : launch_decode_i4_typed<64, 64>(L);
    case 128: return launch_decode_i4_128(L);
    case 256: return launch_decode_i4_256(L);
    default: return fail(SIA_ERR_UNSUPPORTED, "head_dim %d not supported by the int4 matrix kernels", L.D);
  }
}

}  // namespace sia
