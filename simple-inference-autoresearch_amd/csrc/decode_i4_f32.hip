// Decode kernel instantiations for int4 K/V and float32 queries.
#include "decode_launch.hpp"

namespace sia {

int launch_decode_i4_f32(DecodeLaunch& L) {
  const int g = L.lg_group;
  switch (L.D) {
    case 64:
      return g == 5 ? launch_decode_typed<64, I4G<32, false>, F32, F16>(L)
                    : launch_decode_typed<64, I4G<64, false>, F32, F16>(L);
    case 128:
      return g == 5   ? launch_decode_typed<128, I4G<32, false>, F32, F16>(L)
             : g == 6 ? launch_decode_typed<128, I4G<64, false>, F32, F16>(L)
                      : launch_decode_typed<128, I4G<128, false>, F32, F16>(L);
    case 256:
      return g == 5   ? launch_decode_typed<256, I4G<32, false>, F32, F16>(L)
             : g == 6 ? launch_decode_typed<256, I4G<64, false>, F32, F16>(L)
                      : launch_decode_typed<256, I4G<128, false>, F32, F16>(L);
    default: return fail(SIA_ERR_UNSUPPORTED, "head_dim %d not supported by the int4 matrix kernels", L.D);
  }
}

}  // namespace sia
