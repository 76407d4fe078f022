// Rotary positions from frequencies, of a part of each head, for gfx950.
//
// Pair i of a token at position n is turned by the angle n f_i (frequency f_i per position) and stretched by a factor.
// A table of cosines costs its reads and a row per position that a long context reaches, and one built in fp32 is off by
// n 2^-24 radians, 0.06 at a million.  Here the angle is taken modulo one turn in 64-bit integers: F = frac(f / 2 pi) 2^64,
// and n F mod 2^64 is the fraction of a turn whatever n is; its top 32 bits give a quadrant and a rest of at most an eighth of
// a turn, where the Taylor series of sine and cosine to the 9th and 10th power are off by less than 2^-28.  F is rounded to a
// whole number, so a turn is off by |n| 2^-64 at most, that is 2^-24 at 2^40 positions.
//
// Memory-bound: q and k once in, once out.  A work-group takes a few tokens: it computes each token's R / 2 pairs of sine
// and cosine once, into LDS, while its first elements are in flight, and every head's items read them there.  An item is
// PP pairs of a head, in two runs of PP elements (half layout) or one of 2 PP (interleaved), 16 bytes each where the
// layout allows, or as many of the elements behind the rotated part: consecutive items take consecutive runs.
#include <string.h>

#include <algorithm>

#include "host_util.hpp"
#include "sia_common.hpp"

namespace sia {

struct RopeScaledArgs {
  const char* x[2]; int64_t sb[2], st[2], sh[2];       // q and k, byte strides
  char* o[2]; int64_t ob[2], ot[2], oh[2];
  const char* pos; int64_t p_sb, p_st;                 // element strides
  const char* freq;
  int32_t rows, T, Hq, H, D, R;                        // rows = B T, H = Hq + Hkv
  int32_t tokens, block;                               // per work-group; its threads
  int32_t pos64, freq64;
  float scale;
  FastDiv dT, dHead, dItems;                           // by T, items of a head, items of a token
  int32_t head_items;                                  // items of a head
  int32_t rot_items;                                   // of them in the rotated part
};

// f / 2 pi modulo 1 in units of 2^-64, for any finite f: 1 / 2 pi as a sum of two numbers, the product with the first as
// two (itself and what its rounding left), and whole turns taken out of each part.  (In fp64 alone f / 2 pi is off by
// 2^-53 of itself, 2^-13 of a radian after 2^40 positions.)
__device__ __forceinline__ uint64_t turn_per_position(double f) {
#pragma clang fp contract(off)
  constexpr double kHi = 0x1.45f306dc9c883p-3, kLo = -0x1.6b01ec5417056p-57;
  auto fixed = [](double x) {                       // |x| <= 1/2
    const double y = rint(x * 18446744073709551616.0);
    return y < 0.0 ? 0u - (uint64_t)-y : (uint64_t)y;
  };
  const double p = f * kHi, e = __builtin_fma(f, kLo, __builtin_fma(f, kHi, -p));
  return fixed(p - rint(p)) + fixed(e - rint(e));
}

// sine and cosine of `turn` / 2^64 of a turn
__device__ __forceinline__ float2 sincos_turn(uint64_t turn) {
  const uint32_t t = (uint32_t)(turn >> 32);
  const uint32_t quad = (t + 0x20000000u) >> 30;
  const float a = (float)(int32_t)(t - (quad << 30)) * 1.4629180792671596e-9f;   // 2 pi / 2^32
  const float b = a * a;
  float s = __builtin_fmaf(b, 2.7557319e-6f, -1.9841270e-4f);
  s = __builtin_fmaf(b, s, 8.3333333e-3f);
  s = __builtin_fmaf(b, s, -1.6666667e-1f);
  s = __builtin_fmaf(a * b, s, a);
  float c = __builtin_fmaf(b, -2.7557319e-7f, 2.4801587e-5f);
  c = __builtin_fmaf(b, c, -1.3888889e-3f);
  c = __builtin_fmaf(b, c, 4.1666667e-2f);
  c = __builtin_fmaf(b, c, -0.5f);
  c = __builtin_fmaf(b, c, 1.0f);
  const bool swap = (quad & 1u) != 0u;
  const float ys = swap ? c : s, yc = swap ? s : c;
  return float2{(quad & 2u) != 0u ? -ys : ys, ((quad + 1u) & 2u) != 0u ? -yc : yc};
}

template <int BYTES>
struct Words { uint32_t w[BYTES >= 4 ? BYTES / 4 : 1]; };
template <int BYTES>
__device__ __forceinline__ Words<BYTES> get(const char* p) {
  Words<BYTES> r;
  if constexpr (BYTES % 16 == 0) {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const u32x4 x = __builtin_nontemporal_load((const u32x4*)(p + 16 * i));
#pragma unroll
      for (int e = 0; e < 4; ++e) r.w[4 * i + e] = x[e];
    }
  } else if constexpr (BYTES == 8) {
    const u32x2 x = __builtin_nontemporal_load((const u32x2*)p);
    r.w[0] = x[0]; r.w[1] = x[1];
  } else if constexpr (BYTES == 4) {
    r.w[0] = __builtin_nontemporal_load((const uint32_t*)p);
  } else {
    r.w[0] = __builtin_nontemporal_load((const uint16_t*)p);
  }
  return r;
}
template <int BYTES>
__device__ __forceinline__ void put(char* p, const Words<BYTES>& r) {
  if constexpr (BYTES % 16 == 0) {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i)
      __builtin_nontemporal_store(u32x4{r.w[4 * i], r.w[4 * i + 1], r.w[4 * i + 2], r.w[4 * i + 3]}, (u32x4*)(p + 16 * i));
  } else if constexpr (BYTES == 8) {
    __builtin_nontemporal_store(u32x2{r.w[0], r.w[1]}, (u32x2*)p);
  } else if constexpr (BYTES == 4) {
    __builtin_nontemporal_store(r.w[0], (uint32_t*)p);
  } else {
    __builtin_nontemporal_store((uint16_t)r.w[0], (uint16_t*)p);
  }
}
// element i of the words of elements of type T, and all of them back
template <class T, int BYTES>
__device__ __forceinline__ float elem(const Words<BYTES>& r, int i) {
  if constexpr (std::is_same<T, F32>::value) return __builtin_bit_cast(float, r.w[i]);
  else return (i & 1) ? hi_f32(T{}, r.w[i >> 1]) : lo_f32(T{}, r.w[i >> 1]);
}
template <class T, int N>
__device__ __forceinline__ Words<N * T::bytes> words(const float* x) {
  Words<N * T::bytes> r;
  if constexpr (std::is_same<T, F32>::value) {
#pragma unroll
    for (int i = 0; i < N; ++i) r.w[i] = __builtin_bit_cast(uint32_t, x[i]);
  } else if constexpr (N == 1) {
    r.w[0] = pack2(T{}, x[0], 0.f) & 0xffffu;
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) r.w[i] = pack2(T{}, x[2 * i], x[2 * i + 1]);
  }
  return r;
}

// Two runs of BYTES as one item, and its run i.  (Runs of a single 16-bit element share a word.)
template <int BYTES>
__device__ __forceinline__ Words<2 * BYTES> join(const Words<BYTES>& a, const Words<BYTES>& b) {
  Words<2 * BYTES> r;
  if constexpr (BYTES == 2) {
    r.w[0] = a.w[0] | b.w[0] << 16;
  } else {
#pragma unroll
    for (int i = 0; i < BYTES / 4; ++i) { r.w[i] = a.w[i]; r.w[BYTES / 4 + i] = b.w[i]; }
  }
  return r;
}
template <int BYTES>
__device__ __forceinline__ Words<BYTES> part(const Words<2 * BYTES>& x, int i) {
  Words<BYTES> r;
  if constexpr (BYTES == 2) {
    r.w[0] = i ? x.w[0] >> 16 : x.w[0] & 0xffffu;
  } else {
#pragma unroll
    for (int k = 0; k < BYTES / 4; ++k) r.w[k] = x.w[i * (BYTES / 4) + k];
  }
  return r;
}

constexpr int kRopeThreads = 256;     // most threads of a work-group
constexpr int kRopeMaxSc = 2048;      // (sine, cosine) pairs that a work-group's LDS holds: 16 KB

template <class T, bool IL, int PP>
__global__ __launch_bounds__(kRopeThreads) void rope_scaled_kernel(const RopeScaledArgs a) {
  __shared__ float2 sc[kRopeMaxSc];
  constexpr int ES = T::bytes, N = PP * ES;
  constexpr bool kOneRun = IL && PP > 1;               // an item's 2 N bytes are one run (else two of N)
  const int row0 = blockIdx.x * a.tokens, nrow = min(a.tokens, a.rows - row0), half = a.R / 2;
  const int token_items = a.H * a.head_items;
  const int items = nrow * token_items;
  const int copy_items = a.head_items - a.rot_items;
  // item it -> its runs in and out, the distance of the second, and its first pair (-1: copied)
  struct Item { const char* src; char* dst; int gap, pair; };
  auto item = [&](int it) {
    Item r;
    const int t = fdiv(it, a.dItems), i = it - t * token_items;
    const int h = fdiv(i, a.dHead), c = i - h * a.head_items;
    const int row = row0 + t, b = fdiv(row, a.dT), tt = row - b * a.T;
    const int w = h < a.Hq ? 0 : 1, hh = h - (w ? a.Hq : 0);
    const bool rot = c < a.rot_items;
    const int at = rot ? c * (IL ? 2 * N : N) : a.R * ES + (c - a.rot_items) * (kOneRun ? 2 * N : N);
    r.src = a.x[w] + b * a.sb[w] + tt * a.st[w] + hh * a.sh[w] + at;
    r.dst = a.o[w] + b * a.ob[w] + tt * a.ot[w] + hh * a.oh[w] + at;
    r.gap = !rot ? copy_items * N : IL ? N : half * ES;
    r.pair = rot ? t * half + PP * c : -1;
    return r;
  };
  auto load = [&](const Item& r) {
    if constexpr (kOneRun) return get<2 * N>(r.src);
    else return join(get<N>(r.src), get<N>(r.src + r.gap));
  };
  // the first item's elements fly while the sines are computed
  int it = threadIdx.x;
  Item cur{};
  Words<2 * N> x{};
  if (it < items) {
    cur = item(it);
    x = load(cur);
  }
  for (int i = threadIdx.x; i < nrow * half; i += blockDim.x) {
    const int t = i / half, pair = i - t * half;
    const int row = row0 + t, b = fdiv(row, a.dT), tt = row - b * a.T;
    const int64_t pi = b * a.p_sb + tt * a.p_st;
    const int64_t n = a.pos64 ? ((const int64_t*)a.pos)[pi] : (int64_t)((const int32_t*)a.pos)[pi];
    const double f = a.freq64 ? ((const double*)a.freq)[pair] : (double)((const float*)a.freq)[pair];
    const bool finite = __builtin_isfinite(f);
    float2 y = sincos_turn((uint64_t)n * turn_per_position(finite ? f : 0.0));
    const float scale = finite ? a.scale : NAN;      // (a frequency that is not finite has no angle)
    y.x *= scale;
    y.y *= scale;
    sc[i] = y;
  }
  __syncthreads();
  while (it < items) {
    const int next = it + blockDim.x;
    Item nx{};
    Words<2 * N> y{};
    if (next < items) {
      nx = item(next);
      y = load(nx);
    }
    if (cur.pair >= 0) {
      float e[2 * PP];
#pragma unroll
      for (int i = 0; i < PP; ++i) {
        const float2 v = sc[cur.pair + i];
        const int p = IL ? 2 * i : i, q = IL ? 2 * i + 1 : PP + i;
        rope_rotate(elem<T>(x, p), elem<T>(x, q), v.y, v.x, e[p], e[q]);
      }
      x = words<T, 2 * PP>(e);
    }
    if constexpr (kOneRun) {
      put<2 * N>(cur.dst, x);
    } else {
      put<N>(cur.dst, part<N>(x, 0));
      put<N>(cur.dst + cur.gap, part<N>(x, 1));
    }
    it = next;
    cur = nx;
    x = y;
  }
}

namespace {

template <class T, bool IL>
int launch_rope_scaled_pp(const RopeScaledArgs& a, int pp, dim3 grid, hipStream_t st) {
  const dim3 block((unsigned)a.block);
  // (16 bytes a run: 8 or 4 pairs of 16-bit elements, 4 or 2 of 32-bit ones; half of that; single pairs)
  constexpr int kMost = 16 / (IL ? 2 * T::bytes : T::bytes);
  if (pp == kMost) hipLaunchKernelGGL((rope_scaled_kernel<T, IL, kMost>), grid, block, 0, st, a);
  else if (pp == kMost / 2 && kMost > 2) hipLaunchKernelGGL((rope_scaled_kernel<T, IL, kMost / 2>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((rope_scaled_kernel<T, IL, 1>), grid, block, 0, st, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SIA_OK : fail(SIA_ERR_LAUNCH, "rope launch: %s", hipGetErrorString(e));
}
template <class T>
int launch_rope_scaled_t(const RopeScaledArgs& a, bool il, int pp, dim3 grid, hipStream_t st) {
  return il ? launch_rope_scaled_pp<T, true>(a, pp, grid, st) : launch_rope_scaled_pp<T, false>(a, pp, grid, st);
}

bool empty(const sia_tensor* t) {
  for (int d = 0; d < t->ndim; ++d)
    if (t->shape[d] == 0) return true;
  return false;
}

}  // namespace
}  // namespace sia

using namespace sia;

extern "C" int sia_rope_scaled(const sia_tensor* q, const sia_tensor* k, const sia_tensor* positions,
                               const sia_tensor* inv_freq, int32_t rotary_dim, int32_t interleaved, float scale,
                               const sia_tensor* q_out, const sia_tensor* k_out, void* stream) {
  if (q == nullptr || positions == nullptr || inv_freq == nullptr || q_out == nullptr || (k != nullptr) != (k_out != nullptr))
    return fail(SIA_ERR_INVALID_ARGUMENT, "q, positions, inv_freq and q_out are required, and k_out exactly with k");
  const sia_tensor* in[2] = {q, k};
  const sia_tensor* out[2] = {q_out, k_out};
  if (q->ndim != 4) return fail(SIA_ERR_INVALID_ARGUMENT, "q must be (B, T, H, D)");
  const int64_t B = q->shape[0], T = q->shape[1], D = q->shape[3], R = rotary_dim;
  if (q->dtype != SIA_F16 && q->dtype != SIA_BF16 && q->dtype != SIA_F32)
    return fail(SIA_ERR_UNSUPPORTED, "q dtype %s: expected float16, bfloat16 or float32", dtype_name(q->dtype));
  const int es = elem_size(q->dtype);
  RopeScaledArgs a;
  memset(&a, 0, sizeof(a));
  int64_t H = 0;
  for (int w = 0; w < (k != nullptr ? 2 : 1); ++w) {
    const sia_tensor *x = in[w], *o = out[w];
    const char* name = w ? "k" : "q";
    if (x->ndim != 4 || o->ndim != 4) return fail(SIA_ERR_INVALID_ARGUMENT, "%s and its output must be (B, T, H, D)", name);
    if (x->dtype != q->dtype || o->dtype != q->dtype) return fail(SIA_ERR_INVALID_ARGUMENT, "q, k and the outputs must share one dtype");
    if (x->shape[0] != B || x->shape[1] != T || x->shape[3] != D)
      return fail(SIA_ERR_INVALID_ARGUMENT, "k must be (B, T, Hkv, D) with q's B, T and D");
    for (int d = 0; d < 4; ++d)
      if (o->shape[d] != x->shape[d]) return fail(SIA_ERR_INVALID_ARGUMENT, "output shape differs from its input");
    if ((x->stride[3] != 1 || o->stride[3] != 1) && D > 1)
      return fail(SIA_ERR_INVALID_ARGUMENT, "%s and its output must be contiguous along head_dim", name);
    if (!empty(x) && (x->data == nullptr || o->data == nullptr))
      return fail(SIA_ERR_INVALID_ARGUMENT, "a non-empty tensor has no data pointer");
    H += x->shape[2];
    a.x[w] = (const char*)x->data; a.sb[w] = bstride(x, 0); a.st[w] = bstride(x, 1); a.sh[w] = bstride(x, 2);
    a.o[w] = (char*)o->data; a.ob[w] = bstride(o, 0); a.ot[w] = bstride(o, 1); a.oh[w] = bstride(o, 2);
  }
  if (R < 2 || R % 2 || R > D) return fail(SIA_ERR_INVALID_ARGUMENT, "rotary_dim %d must be even, at least 2 and at most head_dim %lld", rotary_dim, (long long)D);
  if (R / 2 > kRopeMaxSc) return fail(SIA_ERR_UNSUPPORTED, "rotary_dim %d exceeds %d", rotary_dim, 2 * kRopeMaxSc);
  if (positions->dtype != SIA_I32 && positions->dtype != SIA_I64)
    return fail(SIA_ERR_INVALID_ARGUMENT, "positions must be int32 or int64");
  if (!((positions->ndim == 1 && positions->shape[0] == T) ||
        (positions->ndim == 2 && positions->shape[0] == B && positions->shape[1] == T)))
    return fail(SIA_ERR_INVALID_ARGUMENT, "positions must be (T,) or (B, T)");
  if ((inv_freq->dtype != SIA_F32 && inv_freq->dtype != SIA_F64) || inv_freq->ndim != 1 || inv_freq->shape[0] != R / 2 ||
      inv_freq->data == nullptr || (R > 2 && inv_freq->stride[0] != 1))
    return fail(SIA_ERR_INVALID_ARGUMENT, "inv_freq must be a contiguous float32 or float64 (rotary_dim / 2,) tensor");
  if (B * T == 0 || H == 0) return SIA_OK;
  if (positions->data == nullptr) return fail(SIA_ERR_INVALID_ARGUMENT, "positions has no data pointer");
  if (B * T > 0x7fffffff || H * D > 0x7fffff) return fail(SIA_ERR_UNSUPPORTED, "too many rows or heads");
  a.pos = (const char*)positions->data;
  a.p_sb = positions->ndim == 2 ? positions->stride[0] : 0;
  a.p_st = positions->stride[positions->ndim - 1];
  a.pos64 = positions->dtype == SIA_I64;
  a.freq = (const char*)inv_freq->data;
  a.freq64 = inv_freq->dtype == SIA_F64;
  a.rows = (int32_t)(B * T); a.T = (int32_t)T; a.Hq = (int32_t)q->shape[2]; a.H = (int32_t)H;
  a.D = (int32_t)D; a.R = (int32_t)R;
  a.scale = scale;
  // the widest items whose runs start at multiples of their size everywhere
  const int most = 16 / (interleaved ? 2 * es : es);
  int pp = 1;
  for (const int p : {most, most / 2}) {
    if (p < 2) break;
    const int64_t al = (interleaved ? 2 : 1) * p * es;
    bool ok = (R / 2) % p == 0 && (D - R) % (2 * p) == 0;
    for (int w = 0; w < (k != nullptr ? 2 : 1); ++w) {
      const int64_t at[] = {(int64_t)(uintptr_t)a.x[w], (int64_t)(uintptr_t)a.o[w], a.sb[w], a.st[w], a.sh[w], a.ob[w], a.ot[w], a.oh[w]};
      for (const int64_t x : at) ok = ok && x % al == 0;
    }
    if (ok) {
      pp = p;
      break;
    }
  }
  a.rot_items = (int32_t)(R / 2 / pp);
  // (single elements: what lies behind the rotated part is an even number of them, as D and R are, or D is refused)
  if ((D - R) % (2 * pp) != 0) return fail(SIA_ERR_UNSUPPORTED, "head_dim %lld must be even", (long long)D);
  a.head_items = a.rot_items + (int32_t)((D - R) / (2 * pp));
  a.dT = make_fastdiv((uint32_t)T);
  a.dHead = make_fastdiv((uint32_t)a.head_items);
  a.dItems = make_fastdiv((uint32_t)(H * a.head_items));
  int rc;
  if ((rc = device_ok())) return rc;
  // A token per work-group, or as many as give each thread an item (and whose sines fit).  8192 tokens, 32/8 heads of 128
  // (168 MB), half layout / interleaved, us: groups of 256 threads 30.3 / 32.0 (5.5 TB/s), with four tokens 32.3 / 34.2;
  // of 320 threads, an item each in the half layout, 34.0 / 37.3, of 128 32.3 / 36.5, of 64 35.5 / 46.5.
  int64_t tokens = std::max<int64_t>(1, kRopeThreads / (H * a.head_items));
  tokens = std::min(tokens, B * T);
  tokens = std::min<int64_t>(tokens, kRopeMaxSc / (R / 2));
  a.block = (int32_t)std::min<int64_t>(kRopeThreads, (tokens * H * a.head_items + 63) / 64 * 64);
  a.tokens = (int32_t)tokens;
  const dim3 grid((unsigned)((B * T + tokens - 1) / tokens));
  const hipStream_t st = (hipStream_t)stream;
  switch (q->dtype) {
    case SIA_F16: return launch_rope_scaled_t<F16>(a, interleaved != 0, pp, grid, st);
    case SIA_BF16: return launch_rope_scaled_t<BF16>(a, interleaved != 0, pp, grid, st);
    default: return launch_rope_scaled_t<F32>(a, interleaved != 0, pp, grid, st);
  }
}
