// What the kernels that write K/V rows share: elements and rotary tables in
// fp32, the rotated query, a correctly rounded quotient.
#pragma once

#include "kv_write.hpp"
#include "sia_common.hpp"

namespace sia {

template <class T>
__device__ __forceinline__ void load8(const char* p, float* x);
template <>
__device__ __forceinline__ void load8<F16>(const char* p, float* x) {
  const u32x4 w = *(const u32x4*)p;
#pragma unroll
  for (int i = 0; i < 4; ++i) { x[2 * i] = lo_f32(F16{}, w[i]); x[2 * i + 1] = hi_f32(F16{}, w[i]); }
}
template <>
__device__ __forceinline__ void load8<BF16>(const char* p, float* x) {
  const u32x4 w = *(const u32x4*)p;
#pragma unroll
  for (int i = 0; i < 4; ++i) { x[2 * i] = lo_f32(BF16{}, w[i]); x[2 * i + 1] = hi_f32(BF16{}, w[i]); }
}
template <>
__device__ __forceinline__ void load8<F32>(const char* p, float* x) {
  const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 16);
#pragma unroll
  for (int i = 0; i < 4; ++i) { x[i] = a[i]; x[4 + i] = b[i]; }
}

template <class T>
__device__ __forceinline__ void store8(char* p, const float* x);
template <>
__device__ __forceinline__ void store8<F16>(char* p, const float* x) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack2(F16{}, x[2 * i], x[2 * i + 1]);
  *(u32x4*)p = w;
}
template <>
__device__ __forceinline__ void store8<BF16>(char* p, const float* x) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack2(BF16{}, x[2 * i], x[2 * i + 1]);
  *(u32x4*)p = w;
}
template <>
__device__ __forceinline__ void store8<F32>(char* p, const float* x) {
  *(f32x4*)p = f32x4{x[0], x[1], x[2], x[3]};
  *(f32x4*)(p + 16) = f32x4{x[4], x[5], x[6], x[7]};
}

// N (4 or 8) consecutive table values of dtype C from element j0 of `row`
// (a 16-byte aligned chunk: the host requires aligned tables).
template <class C, int N>
__device__ __forceinline__ void tab_n(const char* row, int j0, float* c) {
  if constexpr (std::is_same<C, F32>::value) {
    const f32x4 a = *(const f32x4*)(row + j0 * 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = a[i];
    if constexpr (N == 8) {
      const f32x4 b = *(const f32x4*)(row + j0 * 4 + 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) c[4 + i] = b[i];
    }
  } else {
    uint32_t w[N / 2];
    if constexpr (N == 8) {
      const u32x4 v = *(const u32x4*)(row + j0 * 2);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = v[i];
    } else {
      const u32x2 v = *(const u32x2*)(row + j0 * 2);
      w[0] = v[0]; w[1] = v[1];
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) { c[2 * i] = lo_f32(C{}, w[i]); c[2 * i + 1] = hi_f32(C{}, w[i]); }
  }
}

// Round a float to the source dtype (the rotated row is stored in that dtype
// before it is quantised or cast, as a separate RoPE pass would store it).
template <class S> __device__ __forceinline__ float to_src(float x) { return x; }
template <> __device__ __forceinline__ float to_src<F16>(float x) { return (float)(_Float16)x; }
template <> __device__ __forceinline__ float to_src<BF16>(float x) { return (float)(__bf16)x; }

// x / s correctly rounded, from inv = RN(1/s): q0 = RN(x inv) is within one
// ulp of x/s, r = x - q0 s is exact under an FMA, and RN(q0 + r inv) is the
// correctly rounded quotient (Markstein's correction step) while the scale
// stays a normal number, which the amax floor guarantees.  Three VALU
// operations per element instead of a full division; checked against the
// correctly rounded division for every bf16 and fp16 (x, amax) pair and for
// sampled fp32 pairs (tests/test_quant_division.py).
__device__ __forceinline__ float div_by_scale(float x, float s, float inv) {
#pragma clang fp contract(off)
  const float q0 = x * inv;
  const float r = __builtin_fmaf(-q0, s, x);
  return __builtin_fmaf(r, inv, q0);
}

// The q part of a RoPE write: one work-group per token (b, t); a work item is
// 8 pairs of one query head, read and written with 16-byte accesses (both
// halves of a split-half pair, or 16 consecutive elements of interleaved
// pairs, in the same thread).  A token whose position lies outside the table
// is written as zeros.  Loads are unconditional (a position outside the
// table reads row 0 and the result is then zeroed), so no branch sits
// between a load and its use.
template <class S, class C, int ROPE>
__device__ __forceinline__ void rope_q_token(const KvWriteArgs& a, uint32_t token) {
  constexpr int ES = S::bytes;
  const uint32_t b = token / (uint32_t)a.T, t = token - b * (uint32_t)a.T;
  const int pos = (int)t + a.start_host + (a.start ? a.start[a.start_per_seq ? b : 0] : 0);
  const bool tab_ok = pos >= 0 && pos < a.Tc;
  const int half = a.D >> 1;
  const int per_head = half >> 3;
  const int items = a.Hq * per_head;
  const char* qrow = a.q + (int64_t)b * a.q_sb + (int64_t)t * a.q_st;
  char* orow = a.qo + (int64_t)b * a.qo_sb + (int64_t)t * a.qo_st;
  const char* crow = a.cs + (int64_t)(tab_ok ? pos : 0) * a.tab_rs;
  const char* srow = a.sn + (int64_t)(tab_ok ? pos : 0) * a.tab_rs;
  for (int it = threadIdx.x; it < items; it += 256) {
    const int h = it / per_head;
    const int i0 = (it - h * per_head) * 8;
    const char* src = qrow + (int64_t)h * a.q_sh;
    char* dst = orow + (int64_t)h * a.qo_sh;
    float c[8], s[8], x0[8], x1[8];
    // split-half: x0 = elements [i0, i0+8), x1 = [i0+half, ...); interleaved: 16 consecutive
    const int o0 = ROPE == 1 ? i0 : 2 * i0;
    const int o1 = ROPE == 1 ? i0 + half : 2 * i0 + 8;
    load8<S>(src + o0 * ES, x0);
    load8<S>(src + o1 * ES, x1);
    tab_n<C, 8>(crow, i0, c);
    tab_n<C, 8>(srow, i0, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      c[i] = tab_ok ? c[i] : 0.f;
      s[i] = tab_ok ? s[i] : 0.f;
    }
    if constexpr (ROPE == 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) rope_rotate(x0[i], x1[i], c[i], s[i], x0[i], x1[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) rope_rotate(x0[2 * j], x0[2 * j + 1], c[j], s[j], x0[2 * j], x0[2 * j + 1]);
#pragma unroll
      for (int j = 0; j < 4; ++j) rope_rotate(x1[2 * j], x1[2 * j + 1], c[4 + j], s[4 + j], x1[2 * j], x1[2 * j + 1]);
    }
    store8<S>(dst + o0 * ES, x0);
    store8<S>(dst + o1 * ES, x1);
  }
}

}  // namespace sia
