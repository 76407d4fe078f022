// The score function of scored attention: what a query at position p makes of key j beside the scaled product, and which
// keys it sees.
//
//   x = sm_scale q . k;   x = c tanh(x / c);   x -= slope |p - j|
//
// and every mask it knows (causal with a bidirectional prefix, sliding window, documents, padding) leaves a row ONE
// interval of keys, whose two ends do not fall from one row to the next:
//
//   lo(p) = max(start, document's first position, p - W + 1)
//   hi(p) = min(len, next document's first position, p + W, causal ? max(p + 1, prefix) : len)
//
// So the kernels take a pair of bounds per row instead of a mask, walk the union of their rows' intervals and skip the rest.
#pragma once

#include "sia_common.hpp"

namespace sia {

struct ScoreArgs {
  float cap_in;                  // softcap: 2 log2(e) sm_scale / c, so that 2^(cap_in q.k) = e^(2 x / c)
  float cap_out;                 // c log2(e)
  float cap_inv;                 // sm_scale / c
  float cap_log2;                // 2 / c
  const float* slopes;           // (Hq) fp32, or nullptr
  const int32_t* start;          // first key of a row of the batch, (1) or (B), or nullptr (0)
  const int32_t* len;            // its keys, likewise, or nullptr (all)
  const int32_t* prefix;         // keys that a causal row sees whatever its position, likewise, or nullptr
  const int32_t* cuts;           // first positions of documents, any order, or nullptr
  int64_t cuts_sb;               // elements from one sequence's to the next's (0: shared)
  int32_t ncuts;
  int32_t start_per_seq, len_per_seq, prefix_per_seq;
  int32_t window;                // W, of prompts at most 2^30
  int32_t causal;
};

// Score kernels are compiled for: masks alone, capped scores, a bias by distance, or both (kModNone: none of this).
constexpr int kModNone = 0, kModMask = 4, kModCap = 5, kModBias = 6, kModCapBias = 7;
constexpr bool mod_cap(int m) { return (m & 1) != 0; }
constexpr bool mod_bias(int m) { return (m & 2) != 0; }
inline int score_mod(const ScoreArgs& s) { return kModMask | (s.cap_out > 0.f ? 1 : 0) | (s.slopes != nullptr ? 2 : 0); }

constexpr float kLog2e = 1.4426950408889634f;

// The largest cap of the matrix kernels: their `capped` is off by 2^-22 of it, at 512 as much as the weights' rounding to
// fp16 (2^-11 half a step; 512 2^-22 log2(e) = 2^-12.5).  Larger ones go to the vector kernels.
constexpr float kMaxFastCap = 512.0f;
// The prompts' matrix kernels take slopes in units of the cap or of the scale; below this the products could pass fp32's
// range, and the vector kernels take the call.
constexpr float kMinFastUnit = 1e-20f;

// c tanh(x / c) in log2 units from a score x in log2 units, as c (1 - 2 / (1 + e^(2 x / c))): two transcendentals and three
// instructions.  Off by at most about 3 ulp of c, 2^-22 c: below every rounding of 16-bit inputs and weights (c = 50: 2e-5
// of a weight).  The prompts' kernels take the same formula apart (`shape` in prefill_fwd); float32 calls use capped_f32.
__device__ __forceinline__ float capped_log2(const ScoreArgs& s, float x) {
  const float e = fast_exp2(x * s.cap_log2);
  return __builtin_fmaf(__builtin_amdgcn_rcpf(1.0f + e), -2.0f * s.cap_out, s.cap_out);
}
// The same off by a few ulp of itself: near 0 the series of tanh up to its 9th power (off by 1e-8 of it at 1/4), from
// there on (1 - e) / (1 + e) with e = e^(-2 |x| / c) <= 0.61.
__device__ __forceinline__ float capped_f32(const ScoreArgs& s, float raw) {
  const float z = raw * s.cap_inv, y = z * z;
  float t = __builtin_fmaf(y, 62.0f / 2835.0f, -17.0f / 315.0f);
  t = __builtin_fmaf(y, t, 2.0f / 15.0f);
  t = __builtin_fmaf(y, t, -1.0f / 3.0f);
  t = __builtin_fmaf(z * y, t, z);
  const float e = fast_exp2(fabsf(z) * (-2.0f * kLog2e));
  const float u = __builtin_copysignf((1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e), z);
  return s.cap_out * (y < 0.0625f ? t : u);
}

// What one sequence's bounds are made of, clamped to [0, Tk] (so that no sum of them passes 32 bits).
struct SeqBounds {
  int start, len, prefix;
};
__device__ __forceinline__ SeqBounds seq_bounds(const ScoreArgs& s, int b, int Tk) {
  SeqBounds r;
  r.start = s.start != nullptr ? min(Tk, max(0, s.start[s.start_per_seq ? b : 0])) : 0;
  r.len = s.len != nullptr ? min(Tk, max(0, s.len[s.len_per_seq ? b : 0])) : Tk;
  r.prefix = s.prefix != nullptr ? min(Tk, max(0, s.prefix[s.prefix_per_seq ? b : 0])) : 0;
  return r;
}
// Bounds of the row at position p inside the document [dlo, dhi).
__device__ __forceinline__ int row_lo(const ScoreArgs& s, const SeqBounds& r, int p, int dlo) {
  return max(max(r.start, dlo), p - s.window + 1);
}
__device__ __forceinline__ int row_hi(const ScoreArgs& s, const SeqBounds& r, int p, int dhi) {
  const int hi = min(min(r.len, dhi), p + s.window);
  return s.causal ? min(hi, max(p + 1, r.prefix)) : hi;
}

__device__ __forceinline__ int wave_max_i(int x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x = max(x, __shfl_xor(x, o));
  return x;
}
__device__ __forceinline__ int wave_min_i(int x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x = min(x, __shfl_xor(x, o));
  return x;
}
__device__ __forceinline__ uint32_t wave_or(uint32_t x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x |= __shfl_xor(x, o);
  return x;
}

// Documents around the 32 positions p0 .. p0 + 31 of a wave's rows and around a group's first and last position g0, g1:
// the cuts are read 64 at a time, each lane keeps what its own say, and five wave reductions join them, whatever their
// order or number.  Bit i of `in`: a document starts at p0 + i.  (Every lane active, every argument uniform.)
struct Documents {
  int below, above;      // first position of p0's document, and of the first one after p0 + 31
  int g_below, g_above;  // the same of g0 and g1
  uint32_t in;
  __device__ __forceinline__ int lo(int p0, int i) const {
    const uint32_t m = in & ((2u << i) - 1u);
    return m != 0u ? p0 + 31 - __builtin_clz(m) : below;
  }
  __device__ __forceinline__ int hi(int p0, int i) const {
    const uint32_t m = i < 31 ? in >> (i + 1) : 0u;
    return m != 0u ? p0 + i + 1 + __builtin_ctz(m) : above;
  }
};
__device__ __forceinline__ Documents documents(const ScoreArgs& s, int b, int p0, int g0, int g1, int lane) {
  Documents d;
  d.below = d.g_below = 0;
  d.above = d.g_above = 0x7fffffff;
  d.in = 0u;
  if (s.cuts == nullptr) return d;
  const int32_t* cuts = s.cuts + (int64_t)b * s.cuts_sb;
  for (int i = lane; i < s.ncuts; i += 64) {
    const int c = cuts[i];
    if (c <= p0) d.below = max(d.below, c);
    else if (c <= p0 + 31) d.in |= 1u << (c - p0);
    else d.above = min(d.above, c);
    if (c <= g0) d.g_below = max(d.g_below, c);
    if (c > g1) d.g_above = min(d.g_above, c);
  }
  d.below = uniform(wave_max_i(d.below));
  d.above = uniform(wave_min_i(d.above));
  d.g_below = uniform(wave_max_i(d.g_below));
  d.g_above = uniform(wave_min_i(d.g_above));
  d.in = (uint32_t)uniform((int)wave_or(d.in));
  return d;
}

// One row of attention by one wave, in fp32 on the vector ALUs: every lane takes the product of one key of 64, then the
// lanes share the dimensions and add up P V key by key.  Nothing of a key outside [lo, hi) is read, so whatever stands
// there stays out, and any value of a visible one is taken as it is.
template <class T>
__device__ __forceinline__ void row8(const char* p, float* x) {
  if constexpr (std::is_same<T, F32>::value) {
    const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[i] = a[i]; x[4 + i] = b[i]; }
  } else {
    const u32x4 w = *(const u32x4*)p;
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = lo_f32(T{}, w[i]); x[2 * i + 1] = hi_f32(T{}, w[i]); }
  }
}
template <class T>
__device__ __forceinline__ float elem_at(const char* p) {
  if constexpr (std::is_same<T, F32>::value) return *(const float*)p;
  else return to_f32(T{}, *(const uint16_t*)p);
}

// What fp16 makes of a bfloat16 V.  The prompts' kernels take V to fp16 for P V: exact from 2^-17 on, off by at most 2^-25 of
// a smaller value, so by as much of the result (the weights add up to 1).  Beside a value of 2^-13 or more that is under 2^-12
// of the largest one a row sees; a row that sees none, and some that are rounded, is computed again in fp32 (scored_row).
// Only rows whose results all lie below 2^-13 can be such, and only for those is V read again.
constexpr float kSmallV = 0x1p-13f;
// Keys of one KV head as a wave's rows see them, in rising order of their runs: scanned up to `done` as far as the rows need
// it, the last key found with a value that fp16 rounds, and the last one with a value of kSmallV or more.
// 4 x 2048 tokens, 32/8 heads of 128, capped: us 173, 395 over values that are all zero (V read once per wave), 17400 over
// values of 1e-6 (every row computed again).
struct SmallValues {
  int done = 0, rounded = -1, ample = -1;
  // Whether the row of keys [lo, hi) is to be computed again.  (Every lane active, every argument uniform; 16 bytes of a
  // key's row per lane.)
  template <int D>
  __device__ __forceinline__ bool lost(const char* v, int64_t v_sn, int lo, int hi, int lane) {
    constexpr int LPK = D / 8, KPL = 64 / LPK, U = 4;
    asm volatile("" : "+v"(lane));   // (its row and piece computed here: held through the block loop, they cost a wave per SIMD)
    done = max(lo, done);
#pragma unroll 1
    while (ample < lo && done < hi) {
      u32x4 w[U];
      int key[U], r = -1, m = -1;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        key[u] = min(done + u * KPL + lane / LPK, hi - 1);
        w[u] = *(const u32x4*)(v + (int64_t)key[u] * v_sn + 16 * (lane % LPK));
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t x = (w[u][i >> 1] >> (16 * (i & 1))) & 0x7fffu;   // |value|: 0x3700 is 2^-17, 0x3900 2^-13
          if (x - 1u < 0x3700u - 1u) r = key[u];
          if (x >= 0x3900u) m = key[u];
        }
      if (__any(r >= 0)) rounded = uniform(wave_max_i(r));
      if (__any(m >= 0)) ample = uniform(wave_max_i(m));
      done = min(hi, done + U * KPL);
    }
    return rounded >= lo && ample < lo;
  }
};

template <int D, class T>
__device__ __forceinline__ void scored_row(const ScoreArgs& s, float qk_scale, float slope2, const char* q, const char* k,
                                           int64_t k_sn, const char* v, int64_t v_sn, int p, int lo, int hi, char* out,
                                           int lane) {
  constexpr int DL = D < 64 ? 1 : D / 64;      // dimensions of a lane: DL lane + i (D < 64: lane % D, every KG-th key)
  constexpr int KG = D < 64 ? 64 / D : 1;
  const int grp = KG > 1 ? lane / D : 0;
  const int d0 = KG > 1 ? lane % D : DL * lane;
  float m = -INFINITY, l = 0.f, acc[DL];
#pragma unroll
  for (int i = 0; i < DL; ++i) acc[i] = 0.f;
  for (int base = lo; base < hi; base += 64) {
    const int n = min(64, hi - base), key = base + min(lane, n - 1);
    const char* kp = k + (int64_t)key * k_sn;
    float x = 0.f;
#pragma unroll 4
    for (int c = 0; c < D / 8; ++c) {
      float kk[8], qq[8];
      row8<T>(kp + c * 8 * T::bytes, kk);
      row8<T>(q + c * 8 * T::bytes, qq);
#pragma unroll
      for (int i = 0; i < 8; ++i) x = __builtin_fmaf(qq[i], kk[i], x);
    }
    x = s.cap_out > 0.f ? capped_f32(s, x) : x * qk_scale;
    x -= slope2 * fabsf((float)(p - key));
    if (lane >= n) x = -INFINITY;
    float top = x;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    const float mb = fmaxf(m, top);
    const float mu = mb == -INFINITY ? 0.f : mb;
    const float alpha = fast_exp2(m - mu);
    const float w = fast_exp2(x - mu);
    m = mb;
    l = l * alpha + w;
#pragma unroll
    for (int i = 0; i < DL; ++i) acc[i] *= alpha;
    const char* vp = v + (int64_t)base * v_sn + d0 * T::bytes;
    for (int j0 = 0; j0 < n; j0 += 8 * KG) {
      float x8[8][DL];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int j = min(j0 + u * KG + grp, n - 1);
#pragma unroll
        for (int i = 0; i < DL; ++i) x8[u][i] = elem_at<T>(vp + (int64_t)j * v_sn + i * T::bytes);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int j = j0 + u * KG + grp;
        const float wj = __shfl(w, j & 63);
#pragma unroll
        for (int i = 0; i < DL; ++i)
          if (j < n) acc[i] = __builtin_fmaf(wj, x8[u][i], acc[i]);
      }
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
#pragma unroll
  for (int i = 0; i < DL; ++i) {
#pragma unroll
    for (int o = D; o < 64; o <<= 1) acc[i] += __shfl_xor(acc[i], o);
    if (lane < (D < 64 ? D : 64))
      store_out(T{}, out + (d0 + i) * T::bytes, l == 0.f ? 0.f : acc[i] / l);     // (no visible key: zeros)
  }
}

}  // namespace sia
