// Eight consecutive elements of a K or V row, loaded to and stored from fp32.
#pragma once

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

}  // namespace sia
