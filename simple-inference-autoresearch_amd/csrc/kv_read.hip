// KV read-back for gfx950: cached K/V tokens of a contiguous cache or a paged
// pool as plain (B, H, T, D) tensors, whatever the cache holds (16-bit, fp32,
// int8 with per-token-per-head scales, 4 bits with a step and a minimum per
// group).  Token t of sequence b is position start_host + start[b] + t; a
// position outside the source (past its capacity, page id outside the pool) reads
// as zeros.
//
// Bound: HBM.  16 x 5000 tokens, 4 heads of 256, 4 bits to bf16: 87.9 us, 415 MB
// at 4.7 TB/s, the rate of a large copy.
//
// A thread owns 8 consecutive elements of one row of K and of V: one word of
// codes and one of parameters for 4 bits.  Every value is rounded once, from
// the fp32 m + n s (int8: the fp32 product x s) to the output type.
#include "host_util.hpp"
#include "int4.hpp"
#include "kv_rows.hpp"
#include "kv_write.hpp"

namespace sia {

// Where row (b, h, t) lives: page (or sequence) and token in it.
struct RowAt {
  int64_t slot0, slot1;
  bool ok;
};
__device__ __forceinline__ RowAt row_at(const KvReadArgs& a, int b, int t) {
  const int64_t pos = (int64_t)t + a.start_host + (a.start ? a.start[a.start_per_seq ? b : 0] : 0);
  RowAt r;
  r.ok = pos >= 0 && pos < a.cap;
  const int p = r.ok ? (int)pos : 0;
  r.slot0 = b;
  r.slot1 = p;
  if (a.bt) {
    const int blk = fdiv(p, a.dpage);
    const int pg = r.ok ? a.bt[(int64_t)b * a.bt_sb + (int64_t)blk * a.bt_sl] : 0;
    r.ok = r.ok && pg >= 0 && pg < a.num_pages;
    r.slot0 = r.ok ? pg : 0;
    r.slot1 = p - blk * a.page;
  }
  return r;
}

// Elements [8 part, 8 part + 8) of the row at `src`, scales or parameters at `sc`.
template <class S>
__device__ __forceinline__ void read8(const KvReadArgs& a, const char* src, const char* sc, int part, float* x) {
  if constexpr (std::is_same<S, I4>::value) {
    const uint32_t w = *(const uint32_t*)(src + 4 * i4_place(part, a.D));
    const uint32_t sm = *(const uint32_t*)(sc + 4 * (part >> (a.lg_group - 3)));
    const float s = lo_f32(F16{}, sm), m = hi_f32(F16{}, sm);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i4_value(w, i, s, m);
  } else if constexpr (std::is_same<S, I8>::value) {
    const u32x2 w = *(const u32x2*)(src + 8 * part);
    const float s = a.scale_f32 ? *(const float*)sc : (float)*(const _Float16*)sc;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)(int8_t)(w[i >> 2] >> (8 * (i & 3))) * s;
  } else {
    load8<S>(src + part * 8 * S::bytes, x);
  }
}

template <class S, class DT>
__global__ __launch_bounds__(256) void kv_read_kernel(const KvReadArgs a) {
  const uint32_t gid = blockIdx.x * 256u + threadIdx.x;     // (the host keeps rows * width below 2^31)
  const uint32_t row = gid >> a.log2_width;
  const int part = (int)(gid & ((1u << a.log2_width) - 1u));
  if (row >= a.rows) return;
  const int bh = fdiv((int)row, a.dT), t = (int)row - bh * a.T;
  const int b = fdiv(bh, a.dH), h = bh - b * a.H;
  const RowAt r = row_at(a, b, t);
  const int64_t so = r.slot0 * a.s_s0 + (int64_t)h * a.s_sh + r.slot1 * a.s_sn;
  const int64_t co = r.slot0 * a.c_s0 + (int64_t)h * a.c_sh + r.slot1 * a.c_sn;
  const int64_t o = (int64_t)b * a.d_sb + (int64_t)h * a.d_sh + (int64_t)t * a.d_st + part * 8 * DT::bytes;
  float x[2][8] = {};
  if (r.ok) {
    read8<S>(a, a.src0 + so, a.sc0 + co, part, x[0]);
    read8<S>(a, a.src1 + so, a.sc1 + co, part, x[1]);       // (k again when there is no v)
  }
  store8<DT>(a.dst0 + o, x[0]);
  if (a.ntensors == 2) store8<DT>(a.dst1 + o, x[1]);
}

template <class S>
static int launch_read_dst(const KvReadArgs& a, int dst_dtype, hipStream_t stream) {
  const dim3 grid((unsigned)((((int64_t)a.rows << a.log2_width) + 255) / 256));
  switch (dst_dtype) {
    case SIA_F16: hipLaunchKernelGGL((kv_read_kernel<S, F16>), grid, dim3(256), 0, stream, a); break;
    case SIA_BF16: hipLaunchKernelGGL((kv_read_kernel<S, BF16>), grid, dim3(256), 0, stream, a); break;
    case SIA_F32: hipLaunchKernelGGL((kv_read_kernel<S, F32>), grid, dim3(256), 0, stream, a); break;
    default: return fail(SIA_ERR_UNSUPPORTED, "output dtype %s not supported", dtype_name(dst_dtype));
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(SIA_ERR_LAUNCH, "kv read launch: %s", hipGetErrorString(e));
  return SIA_OK;
}

int launch_kv_read(const KvReadArgs& a_in, int src_dtype, int dst_dtype, hipStream_t stream) {
  KvReadArgs a = a_in;
  if (a.src1 == nullptr) {
    a.src1 = a.src0;
    a.sc1 = a.sc0;
  }
  a.log2_width = __builtin_ctz((unsigned)(a.D / 8));
  switch (src_dtype) {
    case SIA_F16: return launch_read_dst<F16>(a, dst_dtype, stream);
    case SIA_BF16: return launch_read_dst<BF16>(a, dst_dtype, stream);
    case SIA_F32: return launch_read_dst<F32>(a, dst_dtype, stream);
    case SIA_I8: return launch_read_dst<I8>(a, dst_dtype, stream);
    case SIA_U8: return launch_read_dst<I4>(a, dst_dtype, stream);
    default: return fail(SIA_ERR_UNSUPPORTED, "source dtype %s not supported", dtype_name(src_dtype));
  }
}

}  // namespace sia
