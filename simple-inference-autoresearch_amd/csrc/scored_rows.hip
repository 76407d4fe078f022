// Scored attention of 16-bit prompts one query row per wave (score.hpp): the calls whose cap, or whose scale beside
// slopes, is out of the matrix kernels' range.  K and V are read once per row, from the caches.
#include "host_util.hpp"
#include "scored.hpp"

namespace sia {

template <int D, class T>
__global__ __launch_bounds__(256) void scored_rows(const ScoredRowsArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * 4 + uniform(threadIdx.x >> 6);
  if (r >= a.rows) return;                                    // (whole waves)
  // rows of one sequence and position together, the heads of a position fastest, last positions first
  const int64_t bi = r / a.Hq;
  const int hq = (int)(r - bi * a.Hq);
  const int b = (int)(bi / a.Tq), i = a.Tq - 1 - (int)(bi - (int64_t)b * a.Tq);
  const int p = a.Tk - a.Tq + i;
  const SeqBounds sb = seq_bounds(a.s, b, a.Tk);
  const Documents d = documents(a.s, b, p, p, p, lane);
  const int lo = row_lo(a.s, sb, p, d.g_below), hi = row_hi(a.s, sb, p, d.g_above);
  const int hkv = hq / a.G;
  scored_row<D, T>(a.s, a.qk_scale, a.s.slopes != nullptr ? a.s.slopes[hq] * kLog2e : 0.f,
                   a.q + b * a.q_sb + (int64_t)hq * a.q_sh + (int64_t)i * a.q_sm, a.k + b * a.k_sb + (int64_t)hkv * a.k_sh,
                   a.k_sn, a.v + b * a.v_sb + (int64_t)hkv * a.v_sh, a.v_sn, p, lo, hi,
                   a.out + b * a.o_sb + (int64_t)hq * a.o_sh + (int64_t)i * a.o_sm, lane);
}

template <class T>
static int launch_rows_t(const ScoredRowsArgs& a, int D, dim3 grid, hipStream_t st) {
  switch (D) {
    case 16: hipLaunchKernelGGL((scored_rows<16, T>), grid, dim3(256), 0, st, a); break;
    case 32: hipLaunchKernelGGL((scored_rows<32, T>), grid, dim3(256), 0, st, a); break;
    case 64: hipLaunchKernelGGL((scored_rows<64, T>), grid, dim3(256), 0, st, a); break;
    case 128: hipLaunchKernelGGL((scored_rows<128, T>), grid, dim3(256), 0, st, a); break;
    case 256: hipLaunchKernelGGL((scored_rows<256, T>), grid, dim3(256), 0, st, a); break;
    default: return fail(SIA_ERR_UNSUPPORTED, "head_dim %d not supported (16, 32, 64, 128, 256)", D);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SIA_OK : fail(SIA_ERR_LAUNCH, "scored attention launch: %s", hipGetErrorString(e));
}

int launch_scored_rows(const ScoredRowsArgs& a, int D, int dtype, hipStream_t stream) {
  const int64_t groups = (a.rows + 3) / 4;
  if (groups > 0x7fffffff) return fail(SIA_ERR_UNSUPPORTED, "too many query rows");
  const dim3 grid((unsigned)groups);
  return dtype == SIA_F16 ? launch_rows_t<F16>(a, D, grid, stream) : launch_rows_t<BF16>(a, D, grid, stream);
}

}  // namespace sia
