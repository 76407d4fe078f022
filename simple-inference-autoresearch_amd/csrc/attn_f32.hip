// Float32 attention: calls without a score function, and the merge of split calls.
#include "attn_f32_kernel.hpp"

namespace sia {

// Combine the nsplit partials of each output row: D/4 lanes per row, PB
// pieces read together.  (One piece after the other, maxima first, a row of 4
// pieces took 3.8 us, and shorter pieces cost here what they gained before.)
template <int D, class OT>
__global__ __launch_bounds__(256) void attn_f32_merge(const F32Args a) {
  constexpr int LPT = D / 4, RPW = 64 / LPT;
  const int lane = threadIdx.x & 63;
  const int64_t row = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * RPW + lane / LPT;
  const int jj = lane % LPT;
  if (row >= (int64_t)a.B * a.Hq) return;
  const float* p = a.part + row * a.nsplit * (D + 4);
  constexpr int PB = 8;
  float M = -INFINITY, L = 0.f;
  f32x4 A = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < a.nsplit; s0 += PB) {
    float ms[PB], ls[PB];
    f32x4 x[PB];
#pragma unroll
    for (int i = 0; i < PB; ++i) {
      const float* ps = p + (int64_t)min(s0 + i, a.nsplit - 1) * (D + 4);
      ms[i] = ps[D];
      ls[i] = ps[D + 1];
      x[i] = *(const f32x4*)(ps + 4 * jj);
    }
    __builtin_amdgcn_sched_barrier(0);
    float mb = M;
#pragma unroll
    for (int i = 0; i < PB; ++i) {
      if (s0 + i >= a.nsplit) ms[i] = -INFINITY;         // (the last piece read again)
      mb = fmaxf(mb, ms[i]);
    }
    const float mu = mb == -INFINITY ? 0.f : mb;         // (a piece without a key weighs 2^-inf = 0)
    const float r = fast_exp2(M - mu);
    // (a batch adds up in pairs: one after the other, the roundings of 125
    // pieces made the error of 8000 keys 3.1e-7 of the result, now 2.0e-7)
#pragma unroll
    for (int i = 0; i < PB; ++i) {
      const float w = fast_exp2(ms[i] - mu);
      ls[i] *= w;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i][e] = w * keep_below(x[i][e], s0 + i, a.nsplit);
    }
#pragma unroll
    for (int o = 1; o < PB; o *= 2)
#pragma unroll
      for (int i = 0; i < PB; i += 2 * o) {
        ls[i] += ls[i + o];
        x[i] += x[i + o];
      }
    L = L * r + ls[0];
    A = A * r + x[0];
    M = mb;
  }
  const int b = (int)(row / a.Hq);
  const int hq = (int)(row - (int64_t)b * a.Hq);
  const float inv = L == 0.f ? 0.f : 1.0f / L;
  store4(OT{}, a.out + b * a.o_sb + (int64_t)hq * a.o_sh + jj * 4 * OT::bytes, A * inv);
}

template <int D>
static int launch_merge_d(const F32Args& a, int out_dtype, hipStream_t st) {
  constexpr int RPB = 4 * (64 / (D / 4));
  const int64_t rows = (int64_t)a.B * a.Hq;
  const int64_t blocks = (rows + RPB - 1) / RPB;
  if (blocks > 0x7fffffff) return fail(SIA_ERR_UNSUPPORTED, "split-K merge: too many rows");
  if (blocks == 0) return SIA_OK;
  if (out_dtype == SIA_F16) hipLaunchKernelGGL((attn_f32_merge<D, F16>), dim3((unsigned)blocks), dim3(256), 0, st, a);
  else if (out_dtype == SIA_BF16) hipLaunchKernelGGL((attn_f32_merge<D, BF16>), dim3((unsigned)blocks), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((attn_f32_merge<D, F32>), dim3((unsigned)blocks), dim3(256), 0, st, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SIA_OK : fail(SIA_ERR_LAUNCH, "split-K merge launch: %s", hipGetErrorString(e));
}

int launch_attn_merge(const F32Args& a, int D, int out_dtype, hipStream_t stream) {
  switch (D) {
    case 16: return launch_merge_d<16>(a, out_dtype, stream);
    case 32: return launch_merge_d<32>(a, out_dtype, stream);
    case 64: return launch_merge_d<64>(a, out_dtype, stream);
    case 128: return launch_merge_d<128>(a, out_dtype, stream);
    case 256: return launch_merge_d<256>(a, out_dtype, stream);
    default: return fail(SIA_ERR_UNSUPPORTED, "head_dim %d not supported (16, 32, 64, 128, 256)", D);
  }
}

int launch_attn_f32(F32Launch& L) { return launch_f32_types<false>(L); }

}  // namespace sia
