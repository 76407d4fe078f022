// The 4-bit K/V format.
//
// A row is one (sequence, KV head, token) vector of D elements.  A group of g
// consecutive elements has two fp16 numbers, a minimum m and a step s, and each
// element a 4-bit code n that stands for m + n s:
//
//   lo, hi = min and max of the group, clamped to +-65504
//   m = fp16(lo), to nearest;  s = fp16(max(0, (hi - m) / 15)), towards zero
//   n = round((x - m) / s), 0 <= n <= 15 (half to even), 0 where s = 0
//
// with hi - m, its quotient, x - m and its quotient each rounded to fp32.  s
// is rounded down so that m + 15 s never exceeds hi: a value read back in fp16
// cannot overflow, and the attention kernels may form it in fp16.  (What it
// costs is 15 s 2^-10 at the group's maximum, a thirtieth of half a step.)  A
// group holding a NaN or an infinity gets NaN for s and m and codes 0, so
// that it reads back as NaN instead of as some finite value.
//
// Codes: element 8 p + i is in bits 4 i .. 4 i + 3 of 32-bit word p.  Word p
// of a block of min(D, 128) elements stands at place (p % 4) (block / 32) +
// p / 4, so that 16 consecutive bytes of a block of 128 hold words p, p + 4,
// p + 8 and p + 12.  That is the order in which the matrix kernels consume a row:
// the four lanes that share a token each load 16 consecutive bytes, and word
// j of all four covers elements [32 j, 32 j + 32), one k-step that lies inside
// one group.  (In element order a k-step would mix four groups of 32, whose
// scales cannot be applied after the product.)
//
// Parameters of a row, fp16: [s0, m0, s1, m1, ...]; one 32-bit load per group.
#pragma once

#include "sia_common.hpp"

namespace sia {

struct I4 { static constexpr int code = SIA_U8; };
// The same with groups of G elements known to the compiler (the matrix
// kernels); HALF: at most 8 query heads share a KV head, ANY: pages of any
// size, looked up per token (decode_i4.hpp).
template <int G, bool HALF, bool ANY = false>
struct I4G { static constexpr int group = G; static constexpr bool half = HALF, any = ANY; };
template <class KV> struct IsInt4 { static constexpr bool value = false; };
template <int G, bool HALF, bool ANY> struct IsInt4<I4G<G, HALF, ANY>> { static constexpr bool value = true; };
template <class KV>
constexpr bool i4_half() {
  if constexpr (IsInt4<KV>::value) return KV::half;
  else return false;
}

template <class KV>
constexpr bool i4_any() {
  if constexpr (IsInt4<KV>::value) return KV::any;
  else return false;
}

// Bytes of n consecutive elements.
template <class KV>
constexpr int kv_bytes(int n) {
  if constexpr (IsInt4<KV>::value) return n / 2;
  else return n * KV::bytes;
}

constexpr float kF16Max = 65504.0f;

// Place of word `p` (elements 8 p .. 8 p + 7) in a row of D elements.
__host__ __device__ __forceinline__ int i4_place(int p, int D) {
  if (D < 64) return p;                               // (one word or less per lane of a k-step: the same order)
  if (D == 64) return (p & 3) * 2 + (p >> 2);
  return (p & ~15) | ((p & 3) << 2) | ((p >> 2) & 3);
}
// The word at place `at`: i4_place's inverse.
__host__ __device__ __forceinline__ int i4_word(int at, int D) {
  if (D < 64) return at;
  if (D == 64) return (at & 1) * 4 + (at >> 1);
  return (at & ~15) | ((at & 3) << 2) | ((at >> 2) & 3);
}

// Bytes of a row's codes and of its parameters.
inline int64_t i4_code_bytes(int64_t D) { return D / 2; }

// The value of code bits [4 i, 4 i + 4) of `w` under the parameters `sm` (s
// low, m high): one rounding of m + n s to fp32.
__device__ __forceinline__ float i4_value(uint32_t w, int i, float s, float m) {
  return __builtin_fmaf((float)((w >> (4 * i)) & 15u), s, m);
}

}  // namespace sia
